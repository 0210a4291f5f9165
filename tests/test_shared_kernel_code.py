"""The compiled gfx950 code of the attention over shared prefixes and 8-bit pages, kernel by kernel."""
import re
import shutil

import pytest

from test_kernel_code import BUILD, LLVM, kernels


def test_descriptors_stay_scalar_in_each_kernel(tmp_path):
    """A tile's descriptor that the compiler takes through vector registers costs four readfirstlanes a load, in a
    loop: the forms by themselves have 16 (wide) and 19 (narrow) of other kinds, those of both in one twice as many."""
    obj = BUILD / "k_attn_shared.o"
    if not obj.exists() or not shutil.which(LLVM / "llvm-objdump"):
        pytest.skip("no object of the build, or no disassembler")
    counts = {k: len(re.findall(r"\bv_readfirstlane_b32\b", v)) for k, v in kernels(obj, tmp_path).items()}
    for form, kinds, most in (("wide", 4, 20), ("narrow", 3, 22), ("both", 4, 40), ("merge", 2, 4)):
        some = {k: n for k, n in counts.items() if f"attn_shared_{form}_kernel" in k}
        assert len(some) == kinds and max(some.values()) <= most, some
