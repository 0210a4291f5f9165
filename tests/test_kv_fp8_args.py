"""Refusals of the entry points on the 8-bit page pool and on shared prefixes: every call below fails its host
checks before any GPU work (the context is never looked into).  CPU only."""
import pytest

from test_paged_serving_args import BATCH, BUF, CTX, IE_ERR_INVALID_ARG, ODD, WINDOW, ints


def append(lib, **k):
    a = dict(ctx=CTX, n=2, start=ints(0, 5), new=ints(3, 1), heads=32, qkv=BUF, stride=6144, wq=None, wk=None,
             cos=BUF, sin=BUF, rope=8192, q=BUF, pages=BUF, n_pages=4, tables=BUF, tstride=2, layer=0)
    a.update(k)
    return lib.ie_qk_norm_rope_paged_fp8(*a.values())


def attend(lib, **k):
    a = dict(ctx=CTX, n=2, start=ints(0, 5), new=ints(3, 1), window=64, sinks=4, heads=32, q=BUF, pages=BUF,
             n_pages=4, tables=BUF, tstride=2, layer=0, out=BUF, ws=BUF)
    a.update(k)
    return lib.ie_attn_window_paged_fp8(*a.values())


def shared(lib, **k):
    a = dict(ctx=CTX, fmt=1, groups=1, sizes=ints(2), lens=ints(64), n=2, start=ints(64, 69), new=ints(3, 1),
             window=64, sinks=4, heads=32, q=BUF, pages=BUF, n_pages=4, tables=BUF, tstride=2, layer=0, out=BUF,
             ws=BUF)
    a.update(k)
    return lib.ie_attn_shared_paged(*a.values())


def to_fp8(lib, **k):
    a = dict(ctx=CTX, n=2, src=BUF, dst=BUF, a=BUF, n_a=3, b=BUF, n_b=3)
    a.update(k)
    return lib.ie_kv_pages_to_fp8(*a.values())


def from_fp8(lib, **k):
    a = dict(ctx=CTX, n=2, src=BUF, dst=BUF, a=BUF, n_a=3, b=BUF, n_b=3)
    a.update(k)
    return lib.ie_kv_pages_from_fp8(*a.values())


OUT = [dict(out=None), dict(out=ODD), dict(ws=None), dict(ws=ODD)]
CONVERT = [dict(ctx=None), dict(n=-1), dict(n=65537), dict(src=None), dict(dst=None), dict(a=None), dict(a=ODD),
           dict(b=None), dict(b=ODD), dict(n_a=0), dict(n_b=0)]
CASES = (
    [(append, k) for k in BATCH + [dict(qkv=None), dict(qkv=ODD), dict(stride=6136), dict(stride=6148),
                                   dict(heads=64), dict(cos=None), dict(sin=None), dict(sin=ODD), dict(wq=ODD),
                                   dict(wk=ODD), dict(rope=5)]]
    + [(attend, k) for k in BATCH + WINDOW + OUT]
    + [(shared, k) for k in BATCH + WINDOW + OUT + [
        dict(fmt=-1), dict(fmt=2), dict(groups=0), dict(groups=-1), dict(groups=3), dict(sizes=None),
        dict(lens=None), dict(sizes=ints(1)), dict(sizes=ints(3)), dict(sizes=ints(0)), dict(sizes=ints(-2)),
        dict(sizes=ints(2**31 - 1)), dict(groups=2, sizes=ints(1, 2), lens=ints(0, 0)),
        dict(groups=2, sizes=ints(2, 0), lens=ints(0, 0)), dict(lens=ints(-64)), dict(lens=ints(32)),
        dict(lens=ints(128)), dict(groups=2, sizes=ints(1, 1), lens=ints(64, 128)),
        dict(lens=ints(2**31 - 64))]]
    + [(c, k) for c in (to_fp8, from_fp8) for k in CONVERT])


@pytest.mark.parametrize("call,change", CASES,
                         ids=[f"{c.__name__}-{i}" for i, (c, _) in enumerate(CASES)])
def test_refusals(hip, call, change):
    assert call(hip.lib, **change) == IE_ERR_INVALID_ARG
    assert hip.last_error()


def test_no_pages_is_no_work(hip):
    assert to_fp8(hip.lib, n=0) == 0 and from_fp8(hip.lib, n=0) == 0


def test_page_size(hip):
    assert hip.lib.ie_kv_page_size_fp8() == 32 * 2 * 8 * 64 * (128 + 1)
    assert (hip._lib.KV_BF16, hip._lib.KV_FP8) == (0, 1)


def test_workspaces_never_shrink(hip):
    """A workspace for a size serves every smaller one: 64 splits of up to 64 rows, and two partials of each row of
    sequences of up to 64 columns."""
    lib = hip.lib
    rows = sorted({r + d for r in (1, 2, 16, 63, 64, 65, 511, 512, 1023, 1024, 2048, 4096, 100000, 2**24)
                   for d in (0, 1)})
    for heads in (16, 32, 64):
        sizes = [lib.ie_attn_shared_workspace_size(r, heads) for r in rows]
        assert sizes == sorted(sizes) and sizes[0] > 0
        few = 64 * (64 // (heads // 8))
        assert all(s >= (64 * min(r, 64) + 2 * min(r, few)) * heads * 130 * 4 for r, s in zip(rows, sizes))
        assert sizes[-1] == sizes[-2]


def test_shared_attention_descriptors_stay_scalar(tmp_path):
    """The K and V tiles' descriptors are in scalar registers: one that the compiler took through a vector register
    would turn every load of a tile into a readfirstlane loop."""
    import re
    import shutil
    from test_kernel_code import BUILD, LLVM, kernels
    obj = BUILD / "k_attn_shared.o"
    if not obj.exists() or not shutil.which(LLVM / "llvm-objdump"):
        pytest.skip("no object of the build, or no disassembler")
    code = {k: v for k, v in kernels(obj, tmp_path).items() if "buffer_load" in v}
    assert len(code) >= 4
    # (a loop's exit test is an exec mask emptied lane by lane)
    loops = {k: len(re.findall(r"s_xor_b64 exec, exec", v)) for k, v in code.items()}
    counts = {k: len(re.findall(r"\bv_readfirstlane_b32\b", v)) for k, v in code.items()}
    assert max(counts.values()) <= 40, (counts, loops)
