"""Refusals of the paged-serving entry points: every call below fails its host checks before any GPU
work (the context is never looked into).  CPU only."""
import ctypes as C

import pytest

IE_ERR_INVALID_ARG = -1
CTX = C.c_void_p(0x1000)     # never dereferenced
BUF = C.c_void_p(0x1000)
ODD = C.c_void_p(0x1008)     # not 16-byte aligned
V = 128256


def ints(*v):
    return (C.c_int * len(v))(*v)


def append(lib, **k):
    a = dict(ctx=CTX, n=2, start=ints(0, 5), new=ints(3, 1), heads=32, qkv=BUF, stride=6144, wq=None,
             wk=None, cos=BUF, sin=BUF, rope=8192, q=BUF, pages=BUF, n_pages=4, tables=BUF, tstride=2,
             layer=0)
    a.update(k)
    return lib.ie_qk_norm_rope_paged(*a.values())


def attend(lib, **k):
    a = dict(ctx=CTX, n=2, start=ints(0, 5), new=ints(3, 1), window=64, sinks=4, heads=32, q=BUF,
             pages=BUF, n_pages=4, tables=BUF, tstride=2, layer=0, out=BUF, ws=BUF)
    a.update(k)
    return lib.ie_attn_window_paged(*a.values())


def fork(lib, **k):
    a = dict(ctx=CTX, n=2, src=ints(0, 0), dst=ints(1, 2), pos=ints(70, 70), fresh=ints(2, 3),
             pages=BUF, n_pages=4, tables=BUF, rows=3, tstride=2)
    a.update(k)
    return lib.ie_kv_fork_paged(*a.values())


def compact(lib, **k):
    a = dict(ctx=CTX, n=2, lens=ints(70, 0), window=64, sinks=4, pages=BUF, n_pages=4, tables=BUF,
             tstride=2, new=BUF, remap=BUF, counts=BUF, ws=BUF)
    a.update(k)
    return lib.ie_kv_compact_paged(*a.values())


def sample(lib, **k):
    a = dict(ctx=CTX, rows=2, vocab=V, logits=BUF, t=BUF, k=BUF, p=BUF, m=BUF, u=BUF, out=BUF, ws=BUF)
    a.update(k)
    return lib.ie_sample_filtered(*a.values())


BATCH = [dict(ctx=None), dict(n=0), dict(n=65), dict(n=-1), dict(start=None), dict(new=None),
         dict(start=ints(0, -1)), dict(new=ints(-1, 1)), dict(new=ints(129, 1)),
         dict(start=ints(0, 129), new=ints(1, 0)), dict(start=ints(0, 2**31 - 1)),
         dict(new=ints(2**31 - 1, 1)), dict(tstride=0), dict(tstride=2049), dict(heads=0),
         dict(heads=8), dict(heads=24), dict(heads=128), dict(n_pages=0), dict(layer=-1),
         dict(layer=32), dict(tables=None), dict(pages=None), dict(pages=ODD), dict(q=None),
         dict(q=ODD)]
WINDOW = [dict(window=0), dict(window=-5), dict(window=131073), dict(sinks=-1), dict(sinks=131073)]

CASES = (
    [(append, k) for k in BATCH + [dict(qkv=None), dict(qkv=ODD), dict(stride=6136),
                                   dict(stride=6148), dict(heads=64), dict(cos=None),
                                   dict(sin=None), dict(sin=ODD), dict(wq=ODD), dict(wk=ODD),
                                   dict(rope=5)]]
    + [(attend, k) for k in BATCH + WINDOW + [dict(out=None), dict(out=ODD), dict(ws=None),
                                              dict(ws=ODD)]]
    + [(fork, k) for k in [dict(ctx=None), dict(n=-1), dict(n=65), dict(src=None), dict(dst=None),
                           dict(pos=None), dict(fresh=None), dict(pages=None), dict(pages=ODD),
                           dict(tables=None), dict(n_pages=0), dict(rows=0), dict(rows=2),
                           dict(tstride=0), dict(tstride=1), dict(tstride=2049), dict(src=ints(0, -1)),
                           dict(dst=ints(1, 3)), dict(dst=ints(1, 1)), dict(dst=ints(1, 0)),
                           dict(src=ints(0, 1)), dict(pos=ints(70, 129)), dict(pos=ints(-1, 70)),
                           dict(fresh=ints(2, 4)), dict(fresh=ints(-1, 3)), dict(fresh=ints(3, 3))]]
    + [(compact, k) for k in WINDOW + [dict(ctx=None), dict(n=0), dict(n=65), dict(lens=None),
                                       dict(lens=ints(-1, 0)), dict(lens=ints(129, 0)),
                                       dict(pages=None), dict(pages=ODD), dict(n_pages=0),
                                       dict(n_pages=65537), dict(tables=None), dict(tstride=0),
                                       dict(tstride=2049), dict(new=None), dict(remap=None),
                                       dict(counts=None), dict(ws=None), dict(ws=ODD)]]
    + [(sample, k) for k in [dict(ctx=None), dict(rows=0), dict(rows=65536), dict(vocab=0),
                             dict(vocab=2**21 + 1), dict(logits=None), dict(u=None),
                             dict(out=None), dict(ws=None), dict(ws=ODD)]])


@pytest.mark.parametrize("call,change", CASES,
                         ids=[f"{c.__name__}-{i}" for i, (c, _) in enumerate(CASES)])
def test_refusals(hip, call, change):
    assert call(hip.lib, **change) == IE_ERR_INVALID_ARG
    assert hip.last_error()


def test_no_forks_is_no_work(hip):
    assert fork(hip.lib, n=0) == 0


def test_workspace_sizes(hip):
    lib = hip.lib
    assert hip._lib.MAX_SEQS == 64
    # partials of 4096 (row, split) pairs at most: 130 floats a head
    assert 0 < lib.ie_attn_window_workspace_size(1, 32) <= 4096 * 32 * 130 * 4
    assert lib.ie_attn_window_workspace_size(16, 64) == 2 * lib.ie_attn_window_workspace_size(16, 32)
    assert lib.ie_attn_window_workspace_size(100000, 32) > 0
    assert lib.ie_kv_compact_workspace_size(1000) >= 8000
    assert lib.ie_sample_filtered_workspace_size(64, V) >= lib.ie_sample_filtered_workspace_size(1, V) > 0


def test_workspaces_never_shrink(hip):
    """A workspace for a size serves every smaller one."""
    lib = hip.lib
    rows = sorted({r + d for r in (1, 2, 16, 63, 64, 65, 1000, 4095, 4096, 8192, 100000, 2**24) for d in (0, 1)})
    for heads in (16, 32, 64):
        sizes = [lib.ie_attn_window_workspace_size(r, heads) for r in rows]
        assert sizes == sorted(sizes) and sizes[0] > 0
        # every split of every row that a launch may make
        assert all(s >= min(64 * r, 4096) * heads * 130 * 4 for r, s in zip(rows, sizes))
    pages = [1, 2, 63, 64, 65, 1000, 65535, 65536]
    sizes = [lib.ie_kv_compact_workspace_size(n) for n in pages]
    assert sizes == sorted(sizes)
    for vocab in (1, 64, 65, 1000, V, V + 1, 2**21):
        sizes = [lib.ie_sample_filtered_workspace_size(r, vocab) for r in range(1, 65)]
        assert sizes == sorted(sizes) and sizes[0] > 0


def test_window_attention_descriptors_stay_scalar(tmp_path):
    """The window attention's K and V tile descriptors are in scalar registers: one that the compiler took
    through a vector register would turn every load of a tile into a readfirstlane loop."""
    import re
    import shutil
    from test_kernel_code import BUILD, LLVM, kernels
    obj = BUILD / "k_attn_window.o"
    if not obj.exists() or not shutil.which(LLVM / "llvm-objdump"):
        pytest.skip("no object of the build, or no disassembler")
    code = {k: v for k, v in kernels(obj, tmp_path).items() if "buffer_load" in v}
    assert len(code) == 2
    counts = {k: len(re.findall(r"\bv_readfirstlane_b32\b", v)) for k, v in code.items()}
    assert max(counts.values()) <= 16, counts
