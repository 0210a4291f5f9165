"""The 8-bit page pool (conversion of pages, quantising append, attention over it) and attention over shared
prefixes, against plain computations in 64 bits.

Tolerances, from the arithmetic:
  codes   a code is the nearest value: off by at most half a step, 2^-4 of the value (e4m3: eps / 2), or half of the
          least step, 2^-10, times the scale; values that no arithmetic went into (V, converted pages) have the
          nearest code itself; K's rotation in fp32 adds 2^-18 of the values that went into it, and may tip a
          scale whose row's maximum lies that near to its border
  attend  as the bf16 attention (test_gpu_paged_serving): codes times scales are exact in bf16
  shared  the same; the parts of a softmax are joined in fp32, 2^-22 of a few terms, inside 2^-12 A
"""
import pytest
import torch

from gpu_util import say
from test_gpu_paged_serving import (ALL, ATTEND, D, KVH, LAYER, LAYERS, PAGE, attend64, bf16, check_attend,
                                    gen, ints, make_pool, make_tables, ptr, rope, turned64)

pytestmark = pytest.mark.gpu
CODES = 2 * KVH * PAGE * D
LAYER_BYTES = CODES + 2 * KVH * PAGE
PAGE_BYTES = LAYERS * LAYER_BYTES
ROWS = torch.arange(PAGE)
AT = 4 * (ROWS % 16) + ROWS // 16          # where the scale of a page's row is


def pool8(n, fill=0):
    return torch.full((n, PAGE_BYTES), fill, dtype=torch.uint8, device="cuda")


def codes_of(pool):
    return pool.view(-1, LAYERS, LAYER_BYTES)[..., :CODES].unflatten(-1, (2, KVH, PAGE, D))


def scales_of(pool):
    """[pages][32][K|V][8][64], in the order in which they lie"""
    return pool.view(-1, LAYERS, LAYER_BYTES)[..., CODES:].unflatten(-1, (2, KVH, PAGE))


def pow2(e):
    """2^e in 64 bits, exactly (a library's power may be a bit off, which a border shows)."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def exponents(x):
    """The scales' bytes of rows [..., 128] of finite values in 64 bits: the least e >= -110 with max <= 448 2^e."""
    top = x.abs().amax(-1)
    e = torch.full_like(top, -110.0)
    for step in (128, 64, 32, 16, 8, 4, 2, 1):     # the largest multiple by which max is still too large
        e = torch.where(top > 448 * pow2(e + step - 1), e + step, e)
    return e + 127


def codes64(y):
    """The nearest codes of values in [-448, 448], by torch's own rounding from fp32."""
    return y.float().to(torch.float8_e4m3fn).view(torch.uint8)


def bf16_pool(pool, layer=LAYER):
    """A bf16 pool with the values of the one layer."""
    out = torch.zeros(pool.shape[0], LAYERS, 2, KVH, PAGE, D, dtype=torch.bfloat16, device="cuda")
    v = codes_of(pool)[:, layer].view(torch.float8_e4m3fn).double()
    e = scales_of(pool)[:, layer][..., AT.cuda()].double() - 127
    out[:, layer] = (v * pow2(e)[..., None]).bfloat16()
    return out


def put8(pool, layer, kv):
    """Rows kv [pages][K|V][8][64][128] (finite) into a layer of all pages."""
    e = exponents(kv.double())
    codes_of(pool)[:, layer] = codes64(kv.double() * pow2(127 - e)[..., None])
    scales = torch.empty_like(e)
    scales[..., AT.cuda()] = e
    scales_of(pool)[:, layer] = scales.to(torch.uint8)


def make_pool8(g, n, layer=LAYER):
    pool = pool8(n)
    put8(pool, layer, bf16(g, n, 2, KVH, PAGE, D))
    return pool


# ------------------------------------------------------------------------------- pages
def to_fp8(hip, ctx, src, dst, a, b):
    hip.check(hip.lib.ie_kv_pages_to_fp8(ctx.handle, src.numel(), ptr(src), ptr(dst), ptr(a), a.shape[0],
                                         ptr(b), b.shape[0]))


def from_fp8(hip, ctx, src, dst, b, a):
    hip.check(hip.lib.ie_kv_pages_from_fp8(ctx.handle, src.numel(), ptr(src), ptr(dst), ptr(b), b.shape[0],
                                           ptr(a), a.shape[0]))


def ids(*v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def check_page(src, pool, page):
    """The codes and scales of a page against those of bf16 rows [32][2][8][64][128] (finite)."""
    x = src.double()
    e = exponents(x)
    assert torch.equal(scales_of(pool)[page][..., AT.cuda()].double(), e)
    want = codes64(x * pow2(127 - e)[..., None])
    got = codes_of(pool)[page]
    assert torch.equal(got, want), int((got != want).sum())


def test_page_size(hip):
    assert hip.lib.ie_kv_page_size_fp8() == PAGE_BYTES


def test_pages_to_fp8_and_back(hip, ctx):
    say("pages: bf16 -> 8 bits -> bf16 -> 8 bits")
    g = gen(1)
    a = bf16(g, 5, LAYERS, 2, KVH, PAGE, D)
    a[1] *= torch.exp2(torch.randint(-60, 60, a.shape[1:-1], generator=g, device="cuda").float())[..., None].bfloat16()
    a[2] *= torch.exp2(torch.randint(-12, 12, a.shape[1:], generator=g, device="cuda").float()).bfloat16()
    b = pool8(7, 0x55)
    to_fp8(hip, ctx, ids(0, 1, 2, 1), ids(6, 0, 3, 5), a, b)
    torch.cuda.synchronize()
    for i, j in ((0, 6), (1, 0), (2, 3), (1, 5)):
        check_page(a[i], b, j)
    assert (b[[1, 2, 4]] == 0x55).all()
    back = torch.full_like(a, 7.0)
    from_fp8(hip, ctx, ids(6, 0, 3), ids(1, 2, 4), b, back)
    torch.cuda.synchronize()
    for i, j in ((6, 1), (0, 2), (3, 4)):
        v = codes_of(b)[i].view(torch.float8_e4m3fn).double()
        v = v * pow2(scales_of(b)[i][..., AT.cuda()].double() - 127)[..., None]
        assert torch.equal(back[j].double(), v)               # exact
    assert (back[[0, 3]] == 7.0).all()
    # values that codes and a scale hold come back to the same values
    c = pool8(2)
    to_fp8(hip, ctx, ids(1), ids(0), back, c)
    again = torch.empty_like(a)
    from_fp8(hip, ctx, ids(0), ids(0), c, again)
    torch.cuda.synchronize()
    assert torch.equal(again[0], back[1])


def test_pages_rows_at_the_borders(hip, ctx):
    """Maxima at and next to the borders of a scale, the smallest and the largest numbers, zeros, ties."""
    say("pages: rows at the borders")
    a = torch.zeros(1, LAYERS, 2, KVH, PAGE, D, dtype=torch.bfloat16, device="cuda")
    rows = a.view(-1, D)
    g = gen(2)
    rows.normal_(0, 0.3, generator=g)
    k = 0
    for e in list(range(-133, 128, 3)) + [127]:
        for m in (1.0, 1.4921875, 1.7421875, 1.75, 1.7578125, 1.9921875):
            top = m * 2.0 ** e
            rows[k] = (rows[k].float().clamp(-1, 1) * top).bfloat16()
            rows[k, k % D] = top if k % 2 else -top
            k += 1
    assert torch.isfinite(rows).all()
    rows[k] = 0.0
    rows[k + 1] = -0.0
    rows[k + 2], rows[k + 2, 5] = 0.0, 2.0 ** -133            # the least bf16
    # ties: halfway between two codes at scale 1 (maximum 448): 17 -> 16, 19 -> 20, 2^-10 -> 0, 3 x 2^-10 -> 2^-8
    rows[k + 3] = 0.0
    rows[k + 3, :8] = torch.tensor([448, 17, 19, -17, -19, 2.0 ** -10, 3 * 2.0 ** -10, 416])
    b = pool8(1)
    to_fp8(hip, ctx, ids(0), ids(0), a, b)
    torch.cuda.synchronize()
    check_page(a[0], b, 0)
    tie = codes_of(b).reshape(-1, D)[k + 3, :8].view(torch.float8_e4m3fn).float().tolist()
    assert tie == [448, 16, 20, -16, -20, 0, 2.0 ** -8, 416]


@pytest.mark.parametrize("value", [float("nan"), float("inf"), float("-inf")])
def test_pages_nonfinite_rows(hip, ctx, value):
    """A row with an infinity or a NaN becomes NaN, its neighbours as ever."""
    say(f"pages: rows with {value}")
    g = gen(3)
    a = bf16(g, 1, LAYERS, 2, KVH, PAGE, D)
    clean = a.clone()
    bad = torch.zeros(LAYERS, 2, KVH, PAGE, dtype=torch.bool, device="cuda")
    bad[3, 0, 2, 17] = bad[31, 1, 7, 63] = bad[0, 0, 0, 0] = True
    a[0, 3, 0, 2, 17, 5] = a[0, 31, 1, 7, 63, 127] = a[0, 0, 0, 0, 0, 0] = value
    b, back = pool8(1), torch.empty_like(a)
    to_fp8(hip, ctx, ids(0), ids(0), a, b)
    from_fp8(hip, ctx, ids(0), ids(0), b, back)
    want = pool8(1)
    to_fp8(hip, ctx, ids(0), ids(0), clean, want)
    torch.cuda.synchronize()
    assert torch.isnan(back[0][bad]).all() and torch.isfinite(back[0][~bad]).all()
    assert torch.equal(codes_of(b)[0][~bad], codes_of(want)[0][~bad])
    assert torch.equal(scales_of(b)[0][..., AT.cuda()][~bad], scales_of(want)[0][..., AT.cuda()][~bad])


def test_pages_every_code_and_scale(hip, ctx):
    """All 256 codes under all scales that rows can have."""
    say("pages: every code and scale")
    b = pool8(1)
    c = codes_of(b)
    c.unflatten(4, (PAGE // 2, 2))[:] = torch.arange(256, dtype=torch.uint8, device="cuda").view(2, D)
    e = (17 + torch.arange(LAYERS * 2 * KVH * PAGE, device="cuda") // 2 % 231).view(LAYERS, 2, KVH, PAGE)
    scales = torch.empty_like(e)
    scales[..., AT.cuda()] = e
    scales_of(b)[0] = scales.to(torch.uint8)
    assert int(e.min()) == 17 and int(e.max()) == 247
    back = torch.empty(1, LAYERS, 2, KVH, PAGE, D, dtype=torch.bfloat16, device="cuda")
    from_fp8(hip, ctx, ids(0), ids(0), b, back)
    torch.cuda.synchronize()
    v = c[0].view(torch.float8_e4m3fn).double() * pow2(e.double() - 127)[..., None]
    want = v.float().bfloat16()                               # (past the largest bf16: infinities)
    nan = torch.isnan(want)
    assert nan.sum() == nan.numel() // 128 and torch.isnan(back[0][nan]).all()
    assert torch.equal(back[0][~nan], want[~nan])
    assert torch.isinf(want).any() and (want[~nan].abs() > 0).any()


def test_pages_outside_the_pools_are_left_out(hip, ctx):
    say("pages outside the pools")
    g = gen(4)
    a, b = bf16(g, 2, LAYERS, 2, KVH, PAGE, D), pool8(3, 0x33)
    kept = a.clone()
    to_fp8(hip, ctx, ids(-1, 2, 0, 1, 2**31 - 1, -2**31, 1), ids(0, 0, 3, -1, 0, 1, 2), a, b)
    torch.cuda.synchronize()
    assert (b[:2] == 0x33).all()
    check_page(a[1], b, 2)
    from_fp8(hip, ctx, ids(3, -1, 2, 2, 2), ids(0, 0, 2, -1, 2**31 - 1), b, a)
    hip.check(hip.lib.ie_kv_pages_from_fp8(ctx.handle, 0, ptr(b), ptr(b), ptr(b), 3, ptr(a), 2))
    torch.cuda.synchronize()
    assert torch.equal(a, kept)


def test_pages_of_long_lists(hip, ctx):
    """The longest lists, nearly all of whose pairs are left out."""
    say("pages: lists of 65536")
    g = gen(5)
    a, b = bf16(g, 2, LAYERS, 2, KVH, PAGE, D), pool8(3, 0x33)
    src, dst = torch.full((65536,), -1, dtype=torch.int32, device="cuda"), torch.zeros(65536, dtype=torch.int32,
                                                                                      device="cuda")
    src[16383], src[16384], src[65535] = 0, 1, 0
    dst[16383], dst[16384], dst[65535] = 2, 1, 0
    to_fp8(hip, ctx, src, dst, a, b)
    torch.cuda.synchronize()
    for page, of in ((2, 0), (1, 1), (0, 0)):
        check_page(a[of], b, page)
    back, want = torch.full_like(a, 7.0), torch.full_like(a[:1], 7.0)
    from_fp8(hip, ctx, ids(1), ids(0), b, want)
    dst.fill_(-1)
    src.zero_()
    src[65535], dst[65535] = 1, 1
    from_fp8(hip, ctx, src, dst, b, back)
    torch.cuda.synchronize()
    assert torch.equal(back[1], want[0]) and (back[0] == 7.0).all()


# ------------------------------------------------------------------------------- append
def append8(hip, ctx, start, new, heads, qkv, wq, wk, cos, sin, q, pool, tables, layer=LAYER):
    hip.check(hip.lib.ie_qk_norm_rope_paged_fp8(
        ctx.handle, len(start), ints(start), ints(new), heads, ptr(qkv), qkv.stride(0), ptr(wq), ptr(wk),
        ptr(cos), ptr(sin), cos.shape[0], ptr(q), ptr(pool), pool.shape[0], ptr(tables), tables.shape[1],
        layer))


def rows_in(pool, tables, seq, pos, layer=LAYER):
    """(codes, scales' bytes) [rows][K|V][8] of the rows at these positions"""
    page, r = tables[seq, pos // PAGE].long(), pos % PAGE
    return codes_of(pool)[page, layer, :, :, r], scales_of(pool)[page, layer, :, :, 4 * (r % 16) + r // 16]


@pytest.mark.parametrize("start,new,heads,norm,pad", [
    ([0], [1], 32, True, 0),
    ([599], [1], 32, False, 0),
    ([0, 63, 64, 130, 7], [1, 2, 0, 65, 200], 32, True, 8),
    ([5] * 16, [1] * 16, 64, True, 0),
    ([100, 0], [0, 129], 16, False, 24),
    (list(range(64)), [1] * 64, 32, True, 0),
    ([130000], [1072], 32, True, 0),
])
def test_append(hip, ctx, start, new, heads, norm, pad):
    say(f"append, 8 bits: {start[:4]} {new[:4]} heads={heads} norm={norm}")
    g = gen(sum(new) + heads)
    n_pages, tables = make_tables(g, [a + n for a, n in zip(start, new)])
    for b, a in enumerate(start):            # pages before a sequence's first new row are not looked at
        tables[b, :a // PAGE] = -1
    used = tables[tables >= 0]
    remap = torch.full((n_pages,), -1, dtype=torch.int32, device="cuda")
    remap[used.long()] = torch.arange(used.numel(), dtype=torch.int32, device="cuda")
    tables = torch.where(tables >= 0, remap[tables.clamp(min=0).long()], -1)
    pool = pool8(used.numel() + 1, 0x55)
    rows, width = sum(new), (heads + 2 * KVH) * D
    qkv = bf16(g, rows + 2, width + pad)
    wq, wk = (bf16(g, D, mean=1.0, std=0.2) for _ in range(2)) if norm else (None, None)
    cos, sin = rope(max(a + n for a, n in zip(start, new)))
    q = torch.full((rows + 2, heads, D), 7.0, dtype=torch.bfloat16, device="cuda")
    append8(hip, ctx, start, new, heads, qkv, wq, wk, cos, sin, q, pool, tables)
    torch.cuda.synchronize()
    assert (q[rows:] == 7.0).all()
    x = qkv[:rows, :width].reshape(rows, heads + 2 * KVH, D)
    seq = torch.repeat_interleave(torch.arange(len(new)), torch.tensor(new)).cuda()
    pos = torch.cat([torch.arange(a, a + n) for a, n in zip(start, new)]).cuda()
    want, size = turned64(x[:, :heads], wq, cos[pos], sin[pos])
    assert ((q[:rows].double() - want).abs() <= want.abs() * 2**-8 + size * 2**-18).all()
    codes, scales = rows_in(pool, tables, seq, pos)
    # V: the nearest codes
    v = x[:, heads + KVH:].double()
    e = exponents(v)
    assert torch.equal(scales[:, 1].double(), e)
    assert torch.equal(codes[:, 1], codes64(v * pow2(127 - e)[..., None]))
    # K
    want, size = turned64(x[:, heads:heads + KVH], wk, cos[pos], sin[pos])
    slack = size * 2**-18
    e, top = scales[:, 0].double() - 127, want.abs().amax(-1)
    most = slack.amax(-1)
    assert (top - most <= 448 * pow2(e)).all() and (top + most > 448 * pow2(e - 1)).all()
    got = codes[:, 0].view(torch.float8_e4m3fn).double() * pow2(e)[..., None]
    err = (got - want).abs()
    assert (err <= torch.maximum(want.abs() * 2**-4, pow2(e - 10)[..., None]) + 2 * slack).all()
    # nothing else was written
    page, r = tables[seq, pos // PAGE].long(), pos % PAGE
    codes_of(pool)[page, LAYER, :, :, r] = 0x55
    scales_of(pool)[page, LAYER, :, :, 4 * (r % 16) + r // 16] = 0x55
    assert (pool == 0x55).all()


def test_append_nonfinite_and_bad_pages(hip, ctx):
    """A K or V row with an infinity or a NaN becomes NaN; ids outside the pool are not written."""
    say("append, 8 bits: NaN rows, bad pages")
    g = gen(6)
    pool = pool8(3, 0x55)
    tables = ids(2, 0, 3, -1, 2**31 - 1)[None]
    cos, sin = rope(320)
    qkv = bf16(g, 320, 48 * D)
    qkv[3, 33 * D + 7] = float("inf")                        # K head 1 of position 3
    qkv[70, 47 * D + 1] = float("nan")                       # V head 7 of position 70
    qkv[5, 32 * D:] = 0
    q = torch.empty(320, 32, D, dtype=torch.bfloat16, device="cuda")
    append8(hip, ctx, [0], [320], 32, qkv, None, None, cos, sin, q, pool, tables)
    torch.cuda.synchronize()
    pos = torch.arange(128, device="cuda")
    codes, scales = rows_in(pool, tables, torch.zeros_like(pos), pos)
    nan = torch.isnan(codes.view(torch.float8_e4m3fn).float())
    bad = torch.zeros(128, 2, KVH, dtype=torch.bool, device="cuda")
    bad[3, 0, 1] = bad[70, 1, 7] = True
    assert torch.equal(nan.all(-1), bad) and torch.equal(nan.any(-1), bad)
    assert (codes[5] & 0x7F == 0).all() and (scales[5] == 17).all()
    assert (pool[1] == 0x55).all()


def test_append_one_norm_and_layers(hip, ctx):
    """A weight for one of q and k alone; the first and the last layer."""
    say("append, 8 bits: one norm, layers 0 and 31")
    g = gen(7)
    cos, sin = rope(80)
    qkv, w = bf16(g, 80, 48 * D), bf16(g, D, mean=1.0, std=0.2)
    tables = ids(1, 0)[None]
    pos = torch.arange(80, device="cuda")
    x = qkv.view(80, 48, D)
    for layer, wq, wk in ((0, w, None), (31, None, w)):
        pool = pool8(2, 0x55)
        q = torch.empty(80, 32, D, dtype=torch.bfloat16, device="cuda")
        append8(hip, ctx, [0], [80], 32, qkv, wq, wk, cos, sin, q, pool, tables, layer)
        torch.cuda.synchronize()
        want, size = turned64(x[:, :32], wq, cos, sin)
        assert ((q.double() - want).abs() <= want.abs() * 2**-8 + size * 2**-18).all()
        want, size = turned64(x[:, 32:40], wk, cos, sin)
        codes, scales = rows_in(pool, tables, torch.zeros_like(pos), pos, layer)
        e = scales[:, 0].double() - 127
        got = codes[:, 0].view(torch.float8_e4m3fn).double() * pow2(e)[..., None]
        tol = torch.maximum(want.abs() * 2**-4, pow2(e - 10)[..., None]) + size * 2**-17
        assert ((got - want).abs() <= tol).all()
        v = pool.view(2, LAYERS, LAYER_BYTES)
        assert (v[:, [i for i in range(LAYERS) if i != layer]] == 0x55).all()


# ------------------------------------------------------------------------------- attend
def workspace(hip, rows, heads, fill=255):
    return torch.empty(hip.lib.ie_attn_shared_workspace_size(rows, heads), dtype=torch.uint8,
                       device="cuda").fill_(fill)


def attend8(hip, ctx, start, new, window, sinks, heads, q, pool, tables, out, ws=None, layer=LAYER):
    ws = workspace(hip, sum(new), heads) if ws is None else ws
    hip.check(hip.lib.ie_attn_window_paged_fp8(
        ctx.handle, len(start), ints(start), ints(new), window, sinks, heads, ptr(q), ptr(pool), pool.shape[0],
        ptr(tables), tables.shape[1], layer, ptr(out), ptr(ws)))
    return ws


MORE = [([700], [2500], 150, 5, 32), ([700], [1300], 4000, 70, 64), ([0], [2500], ALL, 0, 16),
        ([5000, 100], [4, 900], 1000, 0, 32), ([9000] * 24, [3] * 24, ALL, 0, 16),
        ([100, 5000], [2, 1], 64, 4, 64), ([3000], [12], ALL, 0, 32)]


@pytest.mark.parametrize("i", range(len(ATTEND + MORE)))
def test_attend(hip, ctx, i):
    start, new, window, sinks, heads = (ATTEND + MORE)[i]
    say(f"attend, 8 bits: {start[:4]} {new[:4]} window={window} sinks={sinks} heads={heads}")
    g = gen(i)
    n_pages, tables = make_tables(g, [a + n for a, n in zip(start, new)], extra=1)
    pool = make_pool8(g, n_pages)
    rows = sum(new)
    q = bf16(g, rows, heads, D)
    out = torch.full((rows + 3, heads, D), 7.0, dtype=torch.bfloat16, device="cuda")
    attend8(hip, ctx, start, new, window, sinks, heads, q, pool, tables, out)
    torch.cuda.synchronize()
    assert (out[rows:] == 7.0).all()
    want, tol = attend64(start, new, window, sinks, heads, q, bf16_pool(pool), tables)
    check_attend(out[:rows], want, tol)


@pytest.mark.parametrize("start,new", [([900, 300, 5000], [1, 1, 1]), ([900, 0], [100, 700]),
                                       ([900, 0], [1000, 2000])])
def test_attend_evicted_pages(hip, ctx, start, new):
    """Keys of missing pages are not seen; a row that sees nothing gets zeros."""
    say(f"attend, 8 bits: evicted pages {start} {new}")
    g = gen(11)
    n_pages, tables = make_tables(g, [a + n for a, n in zip(start, new)])
    pool = make_pool8(g, n_pages)
    tables[0] = -1
    tables[1, 1::2] = ids(-1, n_pages, 2**31 - 1, -2**31).repeat(tables.shape[1])[:tables[1, 1::2].numel()]
    q = bf16(g, sum(new), 32, D)
    plain = bf16_pool(pool)
    for window, sinks in ((ALL, 0), (200, 70), (40, 0)):
        out = torch.full((sum(new), 32, D), 7.0, dtype=torch.bfloat16, device="cuda")
        attend8(hip, ctx, start, new, window, sinks, 32, q, pool, tables, out)
        torch.cuda.synchronize()
        assert (out[:new[0]] == 0).all()
        want, tol = attend64(start, new, window, sinks, 32, q, plain, tables)
        check_attend(out, want, tol, f"window {window}")


@pytest.mark.parametrize("fill", [0xFF, 0x7F, 0x7E])
@pytest.mark.parametrize("start,new,heads", [([1000, 333], [1, 1], 32), ([1000, 70], [90, 500], 32),
                                             ([20000], [2], 32), ([700], [2500], 16)])
def test_attend_unseen_bytes_do_not_matter(hip, ctx, start, new, heads, fill):
    """NaN codes and scales (0xFF), NaN codes, or the largest ones, in every row that no new row sees: other layers,
    pages of no one, keys before the window, rows past the end."""
    say(f"attend, 8 bits: {fill:#x} in unseen places {start} {new}")
    window, sinks = 150, 5
    g = gen(12)
    lens = [a + n for a, n in zip(start, new)]
    n_pages, tables = make_tables(g, lens)
    pool = pool8(n_pages, fill)
    clean = make_pool8(g, n_pages)
    for b, (a, n) in enumerate(zip(start, new)):
        j = torch.cat([torch.arange(0, min(sinks, a + n)),
                       torch.arange(max(0, a - window + 1), a + n)]).unique().cuda()
        page, r = tables[b, j // PAGE].long(), j % PAGE
        codes_of(pool)[page, LAYER, :, :, r] = codes_of(clean)[page, LAYER, :, :, r]
        at = 4 * (r % 16) + r // 16
        scales_of(pool)[page, LAYER, :, :, at] = scales_of(clean)[page, LAYER, :, :, at]
    q = bf16(g, sum(new), heads, D)
    out = torch.empty(sum(new), heads, D, dtype=torch.bfloat16, device="cuda")
    attend8(hip, ctx, start, new, window, sinks, heads, q, pool, tables, out)
    torch.cuda.synchronize()
    want, tol = attend64(start, new, window, sinks, heads, q, bf16_pool(clean), tables)
    check_attend(out, want, tol)


@pytest.mark.parametrize("rows", [120, 2500])
@pytest.mark.parametrize("at,part", [(130, 0), (130, 1), (1, 1), (175, 1)])
def test_attend_nan_row_reaches_only_rows_that_see_it(hip, ctx, rows, at, part):
    say(f"attend, 8 bits: a NaN row at key {at}, part {part}, {rows} rows")
    g = gen(13)
    start, new, window, sinks = [100], [rows], 60, 2
    n_pages, tables = make_tables(g, [100 + rows])
    pool = make_pool8(g, n_pages)
    q = bf16(g, rows, 32, D)
    clean, out = torch.empty_like(q), torch.empty_like(q)
    attend8(hip, ctx, start, new, window, sinks, 32, q, pool, tables, clean)
    codes_of(pool)[tables[0, at // PAGE].long(), LAYER, part, 2, at % PAGE] = 0x7F
    attend8(hip, ctx, start, new, window, sinks, 32, q, pool, tables, out)
    torch.cuda.synchronize()
    p = torch.arange(100, 100 + rows, device="cuda")
    sees = (at <= p) & ((at > p - window) | (at < sinks))
    assert sees.any() and torch.equal(out[~sees], clean[~sees])
    other = [h for h in range(32) if h // 4 != 2]
    assert torch.equal(out[:, other], clean[:, other])
    assert torch.isnan(out[sees][:, 8:12]).all()


@pytest.mark.parametrize("start,new", [([900], [8]), ([900], [100]), ([900], [2500]), ([3000] * 5, [1] * 5)])
def test_attend_rows_do_not_depend_on_their_neighbours(hip, ctx, start, new):
    """Other queries in one row, whose scores outgrow their first tiles' by far, leave the others' bits."""
    say(f"attend, 8 bits: a row among others {start} {new}")
    g = gen(23)
    n_pages, tables = make_tables(g, [a + n for a, n in zip(start, new)])
    pool = make_pool8(g, n_pages)
    q = bf16(g, sum(new), 32, D)
    outs = [torch.empty_like(q) for _ in range(2)]
    for out, factor in zip(outs, (1, 30)):
        q[1] *= factor
        attend8(hip, ctx, start, new, ALL, 0, 32, q, pool, tables, out)
    torch.cuda.synchronize()
    others = [r for r in range(sum(new)) if r != 1]
    assert torch.equal(outs[0][others], outs[1][others]) and not torch.equal(outs[0][1], outs[1][1])


@pytest.mark.parametrize("start,new,heads", [([6000, 20, 3], [1, 1, 1], 32), ([0, 900], [333, 65], 32),
                                             ([30000], [200], 16), ([40000], [2], 64)])
def test_attend_in_place(hip, ctx, start, new, heads):
    say(f"attend, 8 bits, in place: {start} {new}")
    g = gen(17)
    n_pages, tables = make_tables(g, [a + n for a, n in zip(start, new)])
    pool = make_pool8(g, n_pages)
    q = bf16(g, sum(new), heads, D)
    out = torch.empty_like(q)
    ws = attend8(hip, ctx, start, new, 20000, 4, heads, q, pool, tables, out)
    attend8(hip, ctx, start, new, 20000, 4, heads, q, pool, tables, q, ws)
    torch.cuda.synchronize()
    assert torch.equal(q, out)


def test_attend_large_scores(hip, ctx):
    """Equal scores: the plain mean; rows whose weight is all on one key."""
    say("attend, 8 bits: equal and large scores")
    g = gen(14)
    n_pages, tables = make_tables(g, [700])
    pool = make_pool8(g, n_pages)
    plain = bf16_pool(pool)
    for start, new in (([650], [50]), ([699], [1])):
        q = torch.zeros(new[0], 32, D, dtype=torch.bfloat16, device="cuda")
        out = torch.empty_like(q)
        attend8(hip, ctx, start, new, 300, 4, 32, q, pool, tables, out)
        torch.cuda.synchronize()
        want, tol = attend64(start, new, 300, 4, 32, q, plain, tables)
        check_attend(out, want, tol, "equal scores")
        q = bf16(g, new[0], 32, D, std=200.0)
        attend8(hip, ctx, start, new, 300, 4, 32, q, pool, tables, out)
        torch.cuda.synchronize()
        want, tol = attend64(start, new, 300, 4, 32, q, plain, tables)
        # scores reach 200 x 1.28 x 128^0.5 x 5: their fp32 sums are off by up to 128 x 2^-24 x
        # sum |q k| / 128^0.5, below 0.5 x 2^-4, which moves the weights of keys that nearly tie by that share
        kv = plain[tables[0].long(), LAYER, 1].float().abs().max()
        assert ((out.double() - want).abs() <= tol + 2**-4 * kv).all()


def test_attend_workspace_of_a_larger_batch(hip, ctx):
    """One workspace for calls of several sizes, nothing behind it touched; its contents are of no account."""
    say("attend, 8 bits: one workspace for several batches")
    g = gen(21)
    start, new = [3000, 100, 70000], [1, 4200, 2]
    n_pages, tables = make_tables(g, [a + b for a, b in zip(start, new)])
    pool = make_pool8(g, n_pages)
    plain = bf16_pool(pool)
    size = hip.lib.ie_attn_shared_workspace_size(sum(new), 32)
    ws = torch.empty(size // 4 + 1024, device="cuda").normal_(generator=g)
    ws[size // 4:] = 7.0
    for some in ((0, 1, 2), (0,), (2,), (0, 2), (2,)):
        st, n, t = [start[i] for i in some], [new[i] for i in some], tables[list(some)].contiguous()
        q = bf16(g, sum(n), 32, D)
        out = torch.empty_like(q)
        attend8(hip, ctx, st, n, 40000, 4, 32, q, pool, t, out, ws)
        torch.cuda.synchronize()
        assert (ws[size // 4:] == 7.0).all()
        want, tol = attend64(st, n, 40000, 4, 32, q, plain, t)
        check_attend(out, want, tol)


@pytest.mark.parametrize("window,evicted", [(ALL, False), (16500, True)])
def test_attend_long_runs_of_many_sequences(hip, ctx, window, evicted):
    """More tiles a wave than it looks up at a time (64): 64 sequences of one table, uncut."""
    say(f"attend, 8 bits: 64 sequences over 20000 keys, window {window}")
    g = gen(22)
    start, new = [20000 + 7 * i for i in range(64)], [1 + i % 2 for i in range(64)]
    n_pages, row = make_tables(g, [max(start) + 2])
    pool = make_pool8(g, n_pages)
    if evicted:
        row[0, 100:330:5] = -1
    tables = row.repeat(64, 1)
    q = bf16(g, sum(new), 16, D)
    out = torch.empty_like(q)
    attend8(hip, ctx, start, new, window, 70, 16, q, pool, tables, out)
    torch.cuda.synchronize()
    want, tol = attend64(start, new, window, 70, 16, q, bf16_pool(pool), tables)
    check_attend(out, want, tol)


@pytest.mark.parametrize("layer", [0, 31])
def test_layers_and_pages_far_into_the_pool(hip, ctx, layer):
    """Pages past 2^32 bytes from the pool's start, the first and the last layer; other bytes NaN."""
    say(f"append and attend, 8 bits: layer {layer}, far pages")
    n_pages, near, far = 1100, [1, 3], [1099, 1030]
    assert min(far) * PAGE_BYTES > 2**32
    g = gen(layer)
    pool = torch.empty(n_pages, PAGE_BYTES, dtype=torch.uint8, device="cuda")
    pool[near + far] = 0xFF
    tables = torch.tensor([near, far], dtype=torch.int32, device="cuda")
    cos, sin = rope(128)
    qkv = bf16(g, 100, 48 * D).repeat(2, 1)
    q, out = (torch.empty(200, 32, D, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    append8(hip, ctx, [0, 0], [100, 100], 32, qkv, None, None, cos, sin, q, pool, tables, layer)
    attend8(hip, ctx, [0, 0], [100, 100], 70, 3, 32, q, pool, tables, out, layer=layer)
    back = torch.zeros(4, LAYERS, 2, KVH, PAGE, D, dtype=torch.bfloat16, device="cuda")
    from_fp8(hip, ctx, ids(*near, *far), ids(0, 1, 2, 3), pool, back)
    torch.cuda.synchronize()
    # (rows past the end read as NaN: no row sees them)
    back[1, layer, :, :, 36:] = back[3, layer, :, :, 36:] = 0
    assert torch.equal(back[0, layer], back[2, layer]) and torch.equal(back[1, layer], back[3, layer])
    want, tol = attend64([0], [100], 70, 3, 32, q[:100], back, ids(0, 1)[None], layer=layer)
    check_attend(out[:100], want, tol)
    assert torch.equal(out[100:], out[:100])
    tail = torch.empty(2, LAYERS, 2, KVH, PAGE, D, dtype=torch.bfloat16, device="cuda")
    to_fp8(hip, ctx, ids(0), ids(1098), back[:1], pool)
    from_fp8(hip, ctx, ids(1098), ids(1), pool, tail)
    torch.cuda.synchronize()
    assert torch.equal(tail[1, layer], back[0, layer])


# ------------------------------------------------------------------------------- shared prefixes
def shared(hip, ctx, fmt, sizes, lens, start, new, window, sinks, heads, q, pool, tables, out, ws=None,
           layer=LAYER):
    ws = workspace(hip, sum(new), heads) if ws is None else ws
    hip.check(hip.lib.ie_attn_shared_paged(
        ctx.handle, fmt, len(sizes), ints(sizes), ints(lens), len(start), ints(start), ints(new), window, sinks,
        heads, ptr(q), ptr(pool), pool.shape[0], ptr(tables), tables.shape[1], layer, ptr(out), ptr(ws)))
    return ws


def shared_tables(g, sizes, lens, start, new, spare=2):
    """Tables as forks leave them: (pool pages, tables)."""
    stride = max(1, max(-(-(a + n) // PAGE) for a, n in zip(start, new)))
    own = [-(-(a + n) // PAGE) for a, n in zip(start, new)]
    group = [i for i, s in enumerate(sizes) for _ in range(s)]
    need = sum(x // PAGE for x in lens) + sum(max(0, o - lens[group[b]] // PAGE) for b, o in enumerate(own))
    order = torch.randperm(need + spare, device="cuda", generator=g).to(torch.int32)
    table = torch.full((len(start), stride), -1, dtype=torch.int32, device="cuda")
    at, first = 0, 0
    for size, x in zip(sizes, lens):
        n = min(x // PAGE, stride)
        table[first:first + size, :n] = order[at:at + n]
        at += x // PAGE
        first += size
    for b, o in enumerate(own):
        n = max(0, o - lens[group[b]] // PAGE)
        table[b, o - n:o] = order[at:at + n]
        at += n
    return need + spare, table


def pools(g, fmt, n):
    """(the pool, its values)"""
    pool = make_pool8(g, n) if fmt else make_pool(g, n)
    return pool, bf16_pool(pool) if fmt else pool


SHARED = [
    # (sizes, shared positions, start, new, window, sinks, heads)
    ([2], [64], [64, 64], [1, 1], ALL, 0, 32),                        # the first tokens of two answers
    ([2], [64], [64, 70], [1, 0], ALL, 0, 32),                        # one of them has none
    ([3], [640], [640, 700, 1000], [1, 1, 1], ALL, 0, 32),            # 12 columns: the narrow form for the prefix
    ([16], [4992], [4992 + 17 * i for i in range(16)], [1] * 16, ALL, 0, 32),
    ([16], [4992], [4992 + 17 * i for i in range(16)], [1] * 16, 3000, 100, 16),
    ([5, 1, 3], [1024, 512, 0], [1024, 1100, 2000, 1024, 1500, 600, 5, 0, 64], [1] * 9, ALL, 0, 64),
    ([4, 4], [320, 2048], [320, 400, 333, 1000, 2048, 2050, 2111, 2500], [5, 1, 16, 3, 1, 2, 0, 7], 500, 70, 32),
    ([3], [2048], [2048, 2100, 2050], [1, 900, 4], ALL, 0, 32),       # one is a chunk that attends by itself
    ([3], [2048], [2048, 2100, 2050], [300, 900, 4], 1500, 4, 32),    # only one of few rows: nothing is shared
    ([64], [1984], [1984 + i for i in range(64)], [1] * 64, ALL, 0, 32),
    ([64], [1984], [1984 + 3 * i for i in range(64)], [8] * 64, ALL, 0, 64),
    ([64], [640], [640 + 3 * i for i in range(64)], [16 if i % 2 else 5 for i in range(64)], 600, 64, 32),
    ([6], [6400], [6400, 6500, 7000, 9000, 6400, 6401], [1, 2, 1, 1, 1, 1], 80, 0, 32),   # behind most windows
    ([6], [6400], [6464, 6500, 7000, 9000, 6470, 6465], [1] * 6, 64, 0, 32),              # behind all of them
    ([6], [6400], [6464, 6500, 7000, 9000, 6470, 6465], [1] * 6, 64, 6400, 32),           # all of it sinks
    ([6], [6400], [6464, 6500, 7000, 9000, 6470, 6465], [1] * 6, 64, 7000, 32),           # and some own keys too
    ([20], [30016], [30016 + i for i in range(20)], [2] * 20, ALL, 0, 32),
    ([2, 2], [131008, 64], [131008, 131071, 64, 64], [1, 1, 40, 2], 3000, 10, 32),        # the last positions
    ([1] * 5, [64, 0, 128, 64, 0], [64, 0, 200, 100, 77], [1, 2, 3, 70, 1], ALL, 0, 32),
    ([3], [640], [640, 700, 1000], [0, 0, 1], ALL, 0, 32),            # the only one with rows is not the first
    ([1, 1], [64, 128], [3000, 1500], [10, 13], ALL, 0, 32),          # few columns, nothing shared
]


@pytest.mark.parametrize("fmt", [0, 1])
@pytest.mark.parametrize("i", range(len(SHARED)))
def test_shared(hip, ctx, i, fmt):
    sizes, lens, start, new, window, sinks, heads = SHARED[i]
    say(f"shared, {8 if fmt else 16} bits: {sizes[:4]} {lens[:4]} {start[:4]} {new[:4]} window={window} "
        f"sinks={sinks} heads={heads}")
    g = gen(100 + i)
    n_pages, tables = shared_tables(g, sizes, lens, start, new)
    pool, plain = pools(g, fmt, n_pages)
    rows = sum(new)
    q = bf16(g, rows, heads, D)
    out = torch.full((rows + 3, heads, D), 7.0, dtype=torch.bfloat16, device="cuda")
    shared(hip, ctx, fmt, sizes, lens, start, new, window, sinks, heads, q, pool, tables, out)
    torch.cuda.synchronize()
    assert (out[rows:] == 7.0).all()
    want, tol = attend64(start, new, window, sinks, heads, q, plain, tables)
    check_attend(out[:rows], want, tol)
    # in place, with the workspace as the call before left it, and again: the same bits
    ws = shared(hip, ctx, fmt, sizes, lens, start, new, window, sinks, heads, q, pool, tables, out)
    again = q.clone()
    shared(hip, ctx, fmt, sizes, lens, start, new, window, sinks, heads, again, pool, tables, again, ws)
    torch.cuda.synchronize()
    assert torch.equal(again, out[:rows])


@pytest.mark.parametrize("fmt", [0, 1])
def test_shared_agrees_with_the_windowed_attention(hip, ctx, fmt):
    """Groups of one, and groups that share nothing, are the attention without groups, bit for bit in 8 bits;
    the bf16 pool's against ie_attn_window_paged within both tolerances."""
    say(f"shared vs windowed, format {fmt}")
    g = gen(60)
    start, new = [500, 3000, 64, 0], [1, 3, 150, 20]
    n_pages, tables = make_tables(g, [a + n for a, n in zip(start, new)])
    pool, plain = pools(g, fmt, n_pages)
    q = bf16(g, sum(new), 32, D)
    outs = [torch.empty_like(q) for _ in range(3)]
    shared(hip, ctx, fmt, [1] * 4, [448, 3008 - 64, 64, 0], start, new, 1000, 3, 32, q, pool, tables, outs[0])
    shared(hip, ctx, fmt, [4], [0], start, new, 1000, 3, 32, q, pool, tables, outs[1])
    if fmt:
        attend8(hip, ctx, start, new, 1000, 3, 32, q, pool, tables, outs[2])
    else:
        from test_gpu_paged_serving import attend
        attend(hip, ctx, start, new, 1000, 3, 32, q, pool, tables, outs[2])
    torch.cuda.synchronize()
    assert torch.equal(outs[0], outs[1])
    _, tol = attend64(start, new, 1000, 3, 32, q, plain, tables)
    if fmt:
        assert torch.equal(outs[0], outs[2])
    else:
        assert ((outs[0].double() - outs[2].double()).abs() <= 2 * tol).all()


@pytest.mark.parametrize("fmt", [0, 1])
def test_shared_evicted_pages(hip, ctx, fmt):
    """Pages of a prefix that are gone are not seen by any of its sequences; rows that see nothing get zeros."""
    say(f"shared: evicted pages, format {fmt}")
    g = gen(61)
    sizes, lens = [4, 3], [1280, 640]
    start, new = [1280, 1300, 1281, 1400, 640, 641, 650], [1, 2, 1, 9, 1, 1, 1]
    n_pages, tables = shared_tables(g, sizes, lens, start, new)
    pool, plain = pools(g, fmt, n_pages)
    tables[:4, 2:20:3] = -1
    tables[:4, 3] = n_pages
    tables[4:] = -1
    q = bf16(g, sum(new), 32, D)
    for window, sinks in ((ALL, 0), (300, 130)):
        out = torch.full_like(q, 7.0)
        shared(hip, ctx, fmt, sizes, lens, start, new, window, sinks, 32, q, pool, tables, out)
        torch.cuda.synchronize()
        assert (out[-3:] == 0).all()
        want, tol = attend64(start, new, window, sinks, 32, q, plain, tables)
        check_attend(out, want, tol, f"window {window}")


@pytest.mark.parametrize("fmt,fill", [(0, float("nan")), (0, float("inf")), (1, 0xFF), (1, 0x7E)])
@pytest.mark.parametrize("sizes,lens,start,new", [
    ([6], [1024], [1024, 1100, 1180, 1250, 1330, 1390], [1, 3, 1, 16, 1, 1]),
    ([2], [64], [560, 700], [90, 2500]),                              # chunks, each by itself
])
def test_shared_unseen_values_do_not_matter(hip, ctx, fmt, fill, sizes, lens, start, new):
    """Windows of different positions cut a prefix at different keys: what a row does not see never reaches it, and
    what lies in no row's sight may be anything."""
    say(f"shared: unseen values {fill}, format {fmt}, rows {new}")
    g = gen(62)
    window, sinks = 400, 5
    n_pages, tables = shared_tables(g, sizes, lens, start, new)
    clean, plain = pools(g, fmt, n_pages)
    pool = pool8(n_pages, fill) if fmt else torch.full_like(clean, fill)
    last = [a + n for a, n in zip(start, new)]
    keep = torch.zeros(len(start), tables.shape[1] * PAGE, dtype=torch.bool, device="cuda")
    for b, (a, n) in enumerate(zip(start, new)):
        keep[b, :sinks] = keep[b, max(0, a - window + 1):last[b]] = True
    for b in range(len(start)):
        j = keep[b].nonzero()[:, 0]
        page, r = tables[b, j // PAGE].long(), j % PAGE
        if fmt:
            at = 4 * (r % 16) + r // 16
            codes_of(pool)[page, LAYER, :, :, r] = codes_of(clean)[page, LAYER, :, :, r]
            scales_of(pool)[page, LAYER, :, :, at] = scales_of(clean)[page, LAYER, :, :, at]
        else:
            pool[page, LAYER, :, :, r] = clean[page, LAYER, :, :, r]
    q = bf16(g, sum(new), 32, D)
    out, want_bits = torch.empty_like(q), torch.empty_like(q)
    shared(hip, ctx, fmt, sizes, lens, start, new, window, sinks, 32, q, clean, tables, want_bits)
    shared(hip, ctx, fmt, sizes, lens, start, new, window, sinks, 32, q, pool, tables, out)
    torch.cuda.synchronize()
    want, tol = attend64(start, new, window, sinks, 32, q, plain, tables)
    check_attend(out, want, tol)
    assert torch.equal(out, want_bits)
    # a NaN value at key 700, which some rows' windows have passed
    at = 700
    for b in range(len(start)):
        page = tables[b, at // PAGE].long()
        if fmt:
            codes_of(pool)[page, LAYER, 1, 2, at % PAGE] = 0x7F
        else:
            pool[page, LAYER, 1, 2, at % PAGE] = float("nan")
    shared(hip, ctx, fmt, sizes, lens, start, new, window, sinks, 32, q, pool, tables, out)
    torch.cuda.synchronize()
    pos = torch.cat([torch.arange(a, a + n) for a, n in zip(start, new)]).cuda()
    sees = (at <= pos) & (at > pos - window)
    assert sees.any() and not sees.all()
    assert torch.equal(out[~sees], want_bits[~sees])
    assert torch.isnan(out[sees][:, 8:12]).all()
    other = [h for h in range(32) if h // 4 != 2]
    assert torch.equal(out[:, other], want_bits[:, other])


@pytest.mark.parametrize("fmt", [0, 1])
def test_shared_sequences_that_are_over(hip, ctx, fmt):
    """Sequences of a group without new rows may have no pages at all."""
    say(f"shared: sequences that are over, format {fmt}")
    g = gen(63)
    sizes, lens, start, new = [5], [1280], [1300, 1290, 1280, 1400, 1281], [0, 2, 0, 1, 1]
    n_pages, tables = shared_tables(g, sizes, lens, start, new)
    pool, plain = pools(g, fmt, n_pages)
    tables[0] = tables[2] = -1
    q = bf16(g, sum(new), 32, D)
    out = torch.empty_like(q)
    shared(hip, ctx, fmt, sizes, lens, start, new, ALL, 0, 32, q, pool, tables, out)
    torch.cuda.synchronize()
    want, tol = attend64(start, new, ALL, 0, 32, q, plain, tables)
    check_attend(out, want, tol)


def test_shared_after_very_many_rows(hip, ctx):
    """Two sequences that share a prefix, behind 2^21 rows: more than one launch of the join."""
    start, new, heads = [0] * 16 + [200, 300], [131072] * 16 + [1, 1], 64
    say(f"shared, {sum(new)} rows of {heads} heads")
    g = gen(330)
    pool = make_pool8(g, 40)
    plain = bf16_pool(pool)
    tables = torch.randint(0, 40, (18, 2048), dtype=torch.int32, device="cuda", generator=g)
    tables[17, :2] = tables[16, :2]
    rows = sum(new)
    q = torch.empty(rows, heads, D, dtype=torch.bfloat16, device="cuda").normal_(generator=g)
    out = torch.full_like(q, 7.0)
    shared(hip, ctx, 1, [16, 2], [0, 128], start, new, 64, 0, heads, q, pool, tables, out)
    torch.cuda.synchronize()
    for first, n, seqs, at in ((rows - 2, 2, slice(16, 18), [200, 300]), (rows - 9, 7, slice(15, 16), [131065]),
                               (131072 * 7 + 1000, 5, slice(7, 8), [1000]), (0, 3, slice(0, 1), [0])):
        count = [1, 1] if len(at) == 2 else [n]
        want, tol = attend64(at, count, 64, 0, heads, q[first:first + n], plain, tables[seqs])
        check_attend(out[first:first + n], want, tol, first)


def test_no_new_rows_is_no_work(hip, ctx):
    say("8 bits and shared: batches without new rows")
    g = gen(9)
    n_pages, tables = make_tables(g, [100, 70])
    pool = make_pool8(g, n_pages)
    before = pool.clone()
    q = torch.full((2, 32, D), 7.0, dtype=torch.bfloat16, device="cuda")
    out = q.clone()
    cos, sin = rope(128)
    append8(hip, ctx, [100, 70], [0, 0], 32, bf16(g, 1, 48 * D), None, None, cos, sin, q, pool, tables)
    attend8(hip, ctx, [100, 70], [0, 0], 10, 0, 32, q, pool, tables, out, workspace(hip, 1, 32))
    shared(hip, ctx, 1, [2], [64], [100, 70], [0, 0], 10, 0, 32, q, pool, tables, out, workspace(hip, 1, 32))
    torch.cuda.synchronize()
    assert (q == 7.0).all() and (out == 7.0).all() and torch.equal(pool, before)


# ------------------------------------------------------------------------------- together
class Serving8:
    """A prompt in bf16 pages becomes 8-bit pages, is forked at a full page, and its continuations take a step:
    append, attention over the shared prompt, sampling."""

    def __init__(self, hip, ctx, seed, forks=7, prompt=448):
        self.hip, self.ctx, self.n, self.prompt = hip, ctx, forks, prompt
        self.g = g = gen(seed)
        self.blocks = prompt // PAGE
        self.bf16 = make_pool(g, self.blocks + 1)
        self.src = torch.randperm(self.blocks + 1, generator=g, device="cuda")[:self.blocks].to(torch.int32)
        self.pages = self.blocks + 2 * forks + 1
        self.pool = pool8(self.pages, 0xFF)
        order = torch.randperm(self.pages, device="cuda", generator=g).to(torch.int32)
        self.stride = self.blocks + 2
        self.tables = torch.full((forks + 1, self.stride), -1, dtype=torch.int32, device="cuda")
        self.tables[0, :self.blocks] = order[:self.blocks]
        self.fresh = order[self.blocks:self.blocks + 2 * forks].view(forks, 2)
        self.new = [1 + i % 3 for i in range(forks)]
        rows = sum(self.new)
        self.cos, self.sin = rope(4096)
        self.qkv = bf16(g, rows, 48 * D)
        self.w = bf16(g, D, mean=1.0, std=0.1)
        self.q, self.out = (torch.zeros(rows, 32, D, dtype=torch.bfloat16, device="cuda") for _ in range(2))
        self.alone = torch.zeros_like(self.out)
        self.ws = workspace(hip, rows, 32)

    def begin(self):
        to_fp8(self.hip, self.ctx, self.src, self.tables[0, :self.blocks], self.bf16, self.pool)
        n = self.n
        # (a fork at a full page copies ids only: it serves any pool)
        self.hip.check(self.hip.lib.ie_kv_fork_paged(
            self.ctx.handle, n, ints([0] * n), ints(range(1, n + 1)), ints([self.prompt] * n), ints([-1] * n),
            ptr(self.pool), self.pages, ptr(self.tables), n + 1, self.stride))
        self.tables[1:, self.blocks:] = self.fresh

    def step(self):
        start = [self.prompt + 5 * i for i in range(self.n)]
        t = self.tables[1:]
        append8(self.hip, self.ctx, start, self.new, 32, self.qkv, self.w, self.w, self.cos, self.sin, self.q,
                self.pool, t)
        shared(self.hip, self.ctx, 1, [self.n], [self.prompt], start, self.new, ALL, 0, 32, self.q, self.pool, t,
               self.out, self.ws)
        attend8(self.hip, self.ctx, start, self.new, ALL, 0, 32, self.q, self.pool, t, self.alone, self.ws)

    def check(self):
        start = [self.prompt + 5 * i for i in range(self.n)]
        seq = torch.repeat_interleave(torch.arange(self.n), torch.tensor(self.new)).cuda()
        pos = torch.cat([torch.arange(a, a + n) for a, n in zip(start, self.new)]).cuda()
        x = self.qkv.view(-1, 48, D)
        want, size = turned64(x[:, :32], self.w, self.cos[pos], self.sin[pos])
        assert ((self.q.double() - want).abs() <= want.abs() * 2**-8 + size * 2**-18).all()
        v = x[:, 40:].double()
        codes, scales = rows_in(self.pool, self.tables[1:], seq, pos)
        assert torch.equal(codes[:, 1], codes64(v * pow2(127 - exponents(v))[..., None]))
        # positions between the prompt's end and a continuation's first row were never written: zeros here
        plain = bf16_pool(self.pool)
        want, tol = attend64(start, self.new, ALL, 0, 32, self.q, plain, self.tables[1:])
        check_attend(self.out, want, tol, "shared")
        check_attend(self.alone, want, tol, "each by itself")


def fill_gaps(s):
    """Zero rows where a continuation's earlier tokens would be."""
    for b in range(s.n):
        page = s.tables[1 + b, s.blocks:].long()
        s.pool[page] = 0


def test_step(hip, ctx):
    say("8 bits: convert, fork, append, attend")
    s = Serving8(hip, ctx, 30)
    s.begin()
    fill_gaps(s)
    s.step()
    torch.cuda.synchronize()
    for i in range(s.blocks):
        check_page(s.bf16[int(s.src[i])], s.pool, int(s.tables[0, i]))
    assert (s.tables[1:, :s.blocks] == s.tables[0, :s.blocks]).all()
    s.check()


def test_step_captured(hip, ctx):
    """The step recorded into graphs and replayed with new inputs, eager work and other calls between; two graphs
    of one workspace replay in turn."""
    say("8 bits: captured step")
    a, b = Serving8(hip, ctx, 31), Serving8(hip, ctx, 32, forks=5, prompt=1984)
    b.ws = a.ws = workspace(hip, 64, 32)
    for s in (a, b):
        s.begin()
        fill_gaps(s)
    graphs = []
    for s in (a, b):
        s.step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=ctx.stream):
            s.step()
        graphs.append(graph)
    for i in range(4):
        for s, graph in zip((a, b), graphs):
            s.qkv.normal_(0, 1.28, generator=gen(100 + i))
            s.out.fill_(9.0)
            s.alone.fill_(9.0)
            graph.replay()
            torch.cuda.synchronize()
            got = s.out.clone(), s.alone.clone(), s.pool.clone()
            s.check()
            s.step()                               # eager, same bits
            torch.cuda.synchronize()
            for x, y in zip(got, (s.out, s.alone, s.pool)):
                assert torch.equal(x, y)


def test_convert_captured(hip, ctx):
    say("pages: captured")
    g = gen(70)
    a, b = bf16(g, 3, LAYERS, 2, KVH, PAGE, D), pool8(3)
    back = torch.empty_like(a)
    src, dst = ids(0, 1, 2), ids(2, 0, 1)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=ctx.stream):
        to_fp8(hip, ctx, src, dst, a, b)
        from_fp8(hip, ctx, dst, src, b, back)
    for i in range(3):
        a.normal_(0, 2.0 ** i, generator=g)
        dst.copy_(dst.roll(1))                     # (the lists are read at the replay)
        graph.replay()
        torch.cuda.synchronize()
        for s, d in zip(src.tolist(), dst.tolist()):
            check_page(a[s], b, d)
            assert torch.equal(back[s].double(), bf16_page(b, d))


def bf16_page(pool, page):
    v = codes_of(pool)[page].view(torch.float8_e4m3fn).double()
    return v * pow2(scales_of(pool)[page][..., AT.cuda()].double() - 127)[..., None]


def test_two_streams_at_once(hip, ctx):
    """Two contexts on streams of their own, each with its workspace, at the same time."""
    from infengine_amd.engine import Context
    say("8 bits: two streams")
    g = gen(40)
    start, new = [9000, 5000, 4992], [1, 1, 2]
    n_pages, tables = shared_tables(g, [1, 2], [0, 4992], start, new)
    pool = make_pool8(g, n_pages)
    q = bf16(g, 4, 32, D)
    torch.cuda.synchronize()
    main = torch.cuda.current_stream()
    other = Context(0, graph=False)
    torch.cuda.set_stream(main)
    try:
        outs = [[torch.empty_like(q) for _ in range(2)] for _ in range(2)]
        wss = [workspace(hip, 4, 32) for _ in range(2)]
        torch.cuda.synchronize()
        for _ in range(10):
            for i, c in enumerate((ctx, other)):
                attend8(hip, c, start, new, 8000, 4, 32, q, pool, tables, outs[i][0], wss[i])
                shared(hip, c, 1, [1, 2], [0, 4992], start, new, 8000, 4, 32, q, pool, tables, outs[i][1], wss[i])
        torch.cuda.synchronize()
        want, tol = attend64(start, new, 8000, 4, 32, q, bf16_pool(pool), tables)
        for k in range(2):
            assert torch.equal(outs[0][k], outs[1][k])
            check_attend(outs[0][k], want, tol)
    finally:
        torch.cuda.synchronize()
        other.close()
