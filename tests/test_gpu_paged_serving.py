"""The paged-serving operators (ragged append with norms and rotation, windowed attention with sinks,
fork, compaction, filtered sampling) against plain computations in 64 bits.

Tolerances, from the arithmetic (a rounding to bf16 is off by at most 2^-8 of the value):
  append  one rounding at the end: 2^-8 |y|, and what fp32 does before it: a sum of 128 squares and a
          few products, 2^-18 of |x| in all (a x c - b x s cancels, so relative to the inputs)
  attend  the weights are rounded to bf16 and divided by the sum of the rounded ones: an output moves
          by at most 2^-8 sum_j w_j |v_j - o| <= 2^-8 (A + |o|), A = sum_j w_j |v_j|; the output's own
          rounding 2^-8 |o|; the scores are fp32 sums of 128 products: 128 x 2^-24 x sum |q k|, below
          2^-13 for the values here, moves a weight by that share, an output by 2^-12 A
  the rest is copied, or counted in integers: equal
"""
import ctypes as C

import numpy as np
import pytest
import torch

from gpu_util import say

pytestmark = pytest.mark.gpu
KVH, D, PAGE, LAYERS, V = 8, 128, 64, 32, 128256
LAYER = 7
ALL = 131072


def ptr(t):
    return None if t is None else C.c_void_p(t.data_ptr())


def ints(v):
    return (C.c_int * len(v))(*v)


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def bf16(g, *shape, std=1.28, mean=0.0):
    return torch.empty(*shape, dtype=torch.bfloat16, device="cuda").normal_(mean, std, generator=g)


def make_pool(g, n):
    pool = torch.zeros(n, LAYERS, 2, KVH, PAGE, D, dtype=torch.bfloat16, device="cuda")
    pool[:, LAYER] = bf16(g, n, 2, KVH, PAGE, D)
    return pool


def make_tables(g, lens, spare=3, extra=0):
    """Shuffled pages for sequences of these lengths: (pool pages, tables)."""
    need = [-(-n // PAGE) for n in lens]
    order = torch.randperm(sum(need) + spare, device="cuda", generator=g).to(torch.int32)
    stride = min(max(max(need), 1) + extra, ALL // PAGE)      # (a table row holds 2048 pages at most)
    table = torch.full((len(lens), stride), -1, dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    return sum(need) + spare, table


# ------------------------------------------------------------------------------- append
def append(hip, ctx, start, new, heads, qkv, wq, wk, cos, sin, q, pool, tables, layer=LAYER):
    hip.check(hip.lib.ie_qk_norm_rope_paged(
        ctx.handle, len(start), ints(start), ints(new), heads, ptr(qkv), qkv.stride(0), ptr(wq),
        ptr(wk), ptr(cos), ptr(sin), cos.shape[0], ptr(q), ptr(pool), pool.shape[0], ptr(tables),
        tables.shape[1], layer))


def rope(n):
    freq = 500000.0 ** (-torch.arange(64, device="cuda", dtype=torch.float64) / 64)
    a = torch.arange(n, device="cuda", dtype=torch.float64)[:, None] * freq
    return a.cos().float(), a.sin().float()


def turned64(x, w, cos, sin):
    """(the normed and rotated heads, the size of the values that went into each output)"""
    x = x.double()
    if w is not None:
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-5) * w.double()
    a, b, c, s = x[..., :64], x[..., 64:], cos.double()[:, None], sin.double()[:, None]
    y = torch.cat([a * c - b * s, a * s + b * c], -1)
    return y, torch.cat([a.abs() + b.abs()] * 2, -1)


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
    say(f"append {start[:4]} {new[:4]} heads={heads} norm={norm}")
    g = gen(sum(new) + heads)
    n_pages, tables = make_tables(g, [a + n for a, n in zip(start, new)])
    # pages before a sequence's first new row are not looked at
    for b, a in enumerate(start):
        tables[b, :a // PAGE] = -1
    used = tables[tables >= 0]
    remap = torch.full((n_pages,), -1, dtype=torch.int32, device="cuda")
    remap[used.long()] = torch.arange(used.numel(), dtype=torch.int32, device="cuda")
    tables = torch.where(tables >= 0, remap[tables.clamp(min=0).long()], -1)
    pool = make_pool(g, used.numel() + 1)
    rows, width = sum(new), (heads + 2 * KVH) * D
    qkv = bf16(g, rows + 2, width + pad)
    wq, wk = (bf16(g, D, mean=1.0, std=0.2) for _ in range(2)) if norm else (None, None)
    cos, sin = rope(max(a + n for a, n in zip(start, new)))
    q = torch.full((rows + 2, heads, D), 7.0, dtype=torch.bfloat16, device="cuda")
    before = pool.clone()
    append(hip, ctx, start, new, heads, qkv, wq, wk, cos, sin, q, pool, tables)
    torch.cuda.synchronize()
    assert (q[rows:] == 7.0).all()
    x = qkv[:rows, :width].reshape(rows, heads + 2 * KVH, D)
    seq = torch.repeat_interleave(torch.arange(len(new)), torch.tensor(new)).cuda()
    pos = torch.cat([torch.arange(a, a + n) for a, n in zip(start, new)]).cuda()
    page = tables[seq, pos // PAGE].long()
    got = pool[page, LAYER, :, :, pos % PAGE]            # [rows][K|V][8][128]
    for what, y, xs, w in (("q", q[:rows], x[:, :heads], wq),
                           ("k", got[:, 0], x[:, heads:heads + KVH], wk)):
        want, size = turned64(xs, w, cos[pos], sin[pos])
        bad = (y.double() - want).abs() > want.abs() * 2**-8 + size * 2**-18
        assert not bad.any(), (what, int(bad.sum()))
    assert torch.equal(got[:, 1], x[:, heads + KVH:])
    pool[page, LAYER, :, :, pos % PAGE] = before[page, LAYER, :, :, pos % PAGE]
    assert torch.equal(pool.view(torch.int16), before.view(torch.int16))   # nothing else written


def test_append_without_norm_is_apply_rope(hip, ctx):
    """The rotation alone gives ie_apply_rope's bits."""
    say("append vs ie_apply_rope")
    g = gen(3)
    n, start = 70, 50
    n_pages, tables = make_tables(g, [start + n])
    pool = make_pool(g, n_pages)
    qkv = bf16(g, n, 48 * D)
    cos, sin = rope(256)
    q = torch.empty(n, 32, D, dtype=torch.bfloat16, device="cuda")
    append(hip, ctx, [start], [n], 32, qkv, None, None, cos, sin, q, pool, tables)
    heads_first = qkv.view(n, 48, D)[:, :32].transpose(0, 1).contiguous()
    out = torch.empty_like(heads_first)
    hip.check(hip.lib.ie_apply_rope(start, 32, n, ptr(cos), ptr(sin), ptr(heads_first), ptr(out), 0,
                                    ctx.stream_ptr))
    torch.cuda.synchronize()
    assert torch.equal(out.transpose(0, 1), q)


@pytest.mark.parametrize("which", ["q", "k"])
def test_append_one_norm_alone(hip, ctx, which):
    say(f"append with a norm of the {which} heads alone")
    g = gen(4)
    n_pages, tables = make_tables(g, [150])
    pool = make_pool(g, n_pages)
    qkv = bf16(g, 70, 48 * D)
    w = bf16(g, D, mean=1.0, std=0.2)
    wq, wk = (w, None) if which == "q" else (None, w)
    cos, sin = rope(150)
    q = torch.empty(70, 32, D, dtype=torch.bfloat16, device="cuda")
    append(hip, ctx, [80], [70], 32, qkv, wq, wk, cos, sin, q, pool, tables)
    torch.cuda.synchronize()
    x = qkv.view(70, 48, D)
    pos = torch.arange(80, 150, device="cuda")
    k = pool[tables[0, pos // PAGE].long(), LAYER, 0, :, pos % PAGE]
    for got, heads, wt in ((q, x[:, :32], wq), (k, x[:, 32:40], wk)):
        want, size = turned64(heads, wt, cos[pos], sin[pos])
        assert ((got.double() - want).abs() <= want.abs() * 2**-8 + size * 2**-18).all()


def test_append_bad_pages_are_not_written(hip, ctx):
    say("append with page ids outside the pool")
    g = gen(4)
    pool = make_pool(g, 2)
    before = pool.clone()
    tables = torch.tensor([[-1, 2, 2**31 - 1, -2**31]], dtype=torch.int32, device="cuda")
    cos, sin = rope(256)
    qkv = bf16(g, 256, 48 * D)
    q = torch.empty(256, 32, D, dtype=torch.bfloat16, device="cuda")
    append(hip, ctx, [0], [256], 32, qkv, None, None, cos, sin, q, pool, tables)
    torch.cuda.synchronize()
    assert torch.equal(pool, before)
    want, size = turned64(qkv.view(256, 48, D)[:, :32], None, cos, sin)
    assert ((q.double() - want).abs() <= want.abs() * 2**-8 + size * 2**-18).all()


# ------------------------------------------------------------------------------- attend
def attend(hip, ctx, start, new, window, sinks, heads, q, pool, tables, out, ws=None, layer=LAYER):
    if ws is None:
        ws = torch.empty(hip.lib.ie_attn_window_workspace_size(sum(new), heads), dtype=torch.uint8,
                         device="cuda").fill_(255)
    hip.check(hip.lib.ie_attn_window_paged(
        ctx.handle, len(start), ints(start), ints(new), window, sinks, heads, ptr(q), ptr(pool),
        pool.shape[0], ptr(tables), tables.shape[1], layer, ptr(out), ptr(ws)))
    return ws


def attend64(start, new, window, sinks, heads, q, pool, tables, layer=LAYER):
    """(outputs, tolerances) [rows][heads][128]: dense over every position whose page is there."""
    out, tol = [], []
    row, group = 0, heads // KVH
    for b, (a, n) in enumerate(zip(start, new)):
        o = torch.zeros(n, heads, D, dtype=torch.float64, device="cuda")
        t = torch.zeros_like(o)
        table = tables[b].long()
        held = ((table >= 0) & (table < pool.shape[0])).nonzero()[:, 0]
        j = (held[:, None] * PAGE + torch.arange(PAGE, device="cuda")).reshape(-1)
        kv = pool[table[held], layer].permute(1, 2, 0, 3, 4).reshape(2, KVH, -1, D)
        kv, j = kv[:, :, j < a + n].double(), j[j < a + n]
        for r0 in range(0, n if j.numel() else 0, 512):
            r1 = min(n, r0 + 512)
            p = torch.arange(a + r0, a + r1, device="cuda")[:, None]
            seen = (j <= p) & ((j > p - window) | (j < sinks))
            any_seen = seen.any(1, keepdim=True)
            some = seen.any(0)                      # keys that no row sees are left out (NaN there)
            for h in range(heads):
                k, v = kv[0, h // group][some], kv[1, h // group][some]
                s = (q[row + r0:row + r1, h].double() @ k.t()) / D ** 0.5
                w = torch.softmax(s.masked_fill(~seen[:, some], -1e300), -1) * any_seen
                w = w.masked_fill(~seen[:, some], 0.0)
                o[r0:r1, h] = w @ v
                t[r0:r1, h] = (2**-8 + 2**-12) * (w @ v.abs()) + 2**-7 * o[r0:r1, h].abs()
        out.append(o)
        tol.append(t)
        row += n
    return torch.cat(out), torch.cat(tol)


def check_attend(out, want, tol, what=""):
    err = (out.double() - want).abs()
    share = float((err / (tol + 1e-30)).max()) if out.numel() else 0.0
    say(f"  {what} worst {share:.2f} of its tolerance")
    assert not torch.isnan(out).any()
    assert (err <= tol + 1e-30).all(), (what, int((err > tol).sum()), share)


ATTEND = [
    # (start, new, window, sinks, heads)
    ([0], [1], ALL, 0, 32),                                   # the very first token
    ([600], [1], ALL, 0, 32),
    ([0], [1], 1, 0, 32),
    ([100], [3], 1, 0, 32),                                   # each row sees itself alone
    ([1000], [5], 64, 0, 32), ([1000], [64], 63, 1, 32), ([999], [130], 65, 64, 32),
    ([63, 64, 65, 127, 128, 0], [1, 1, 1, 1, 1, 1], 64, 4, 32),
    ([0, 10, 0, 500], [17, 0, 300, 33], 100, 5, 32),          # a sequence without new rows
    ([0] * 3, [0, 0, 2], 10, 0, 32),
    ([6000, 20, 3000, 777], [1, 1, 1, 1], 4096, 4, 32),       # decode batch, mixed lengths
    ([6000, 20, 3000, 777], [1, 200, 4, 16], 1000, 100, 64),
    ([6000, 20, 3000, 777], [1, 200, 4, 16], 1000, 3, 16),
    ([40000], [1], 4096, 4, 32), ([40000], [1], ALL, 0, 32),  # many splits
    ([30000], [200], ALL, 0, 32),
    ([0], [2100], 512, 16, 32), ([0], [1500], ALL, 0, 64),
    ([131071], [1], 200, 130000, 16),                         # nearly everything a sink
    ([131000], [72], 500, 64, 32),                            # the last positions
    (list(range(0, 64 * 37, 37)), [1] * 64, 300, 2, 32),
    ([3] * 20, [9] * 20, 5, 1, 32),
    ([2000], [1], 70, 2000, 32),                              # the sinks meet the window
]


@pytest.mark.parametrize("i", range(len(ATTEND)))
def test_attend(hip, ctx, i):
    start, new, window, sinks, heads = ATTEND[i]
    say(f"attend {start[:4]} {new[:4]} window={window} sinks={sinks} heads={heads}")
    g = gen(i)
    n_pages, tables = make_tables(g, [a + n for a, n in zip(start, new)], extra=1)
    pool = make_pool(g, n_pages)
    rows = sum(new)
    q = bf16(g, rows, heads, D)
    out = torch.full((rows + 3, heads, D), 7.0, dtype=torch.bfloat16, device="cuda")
    attend(hip, ctx, start, new, window, sinks, heads, q, pool, tables, out)
    torch.cuda.synchronize()
    assert (out[rows:] == 7.0).all()
    want, tol = attend64(start, new, window, sinks, heads, q, pool, tables)
    check_attend(out[:rows], want, tol)


def test_attend_workspace_of_a_larger_batch(hip, ctx):
    """A workspace made for more rows holds the partials of fewer; a single token beside a chunk of more
    than 4096 rows is split like one alone."""
    say("attend: one workspace for a large and a small batch")
    g = gen(21)
    start, new = [3000, 100], [1, 4200]
    n_pages, tables = make_tables(g, [a + b for a, b in zip(start, new)])
    pool = make_pool(g, n_pages)
    size = hip.lib.ie_attn_window_workspace_size(sum(new), 32)
    ws = torch.full((size // 4 + 1024,), 7.0, device="cuda")
    for st, n in ((start, new), (start[:1], [1])):
        rows = sum(n)
        q = bf16(g, rows, 32, D)
        out = torch.empty_like(q)
        hip.check(hip.lib.ie_attn_window_paged(
            ctx.handle, len(n), ints(st), ints(n), 2500, 4, 32, ptr(q), ptr(pool), n_pages, ptr(tables),
            tables.shape[1], LAYER, ptr(out), ptr(ws)))
        torch.cuda.synchronize()
        assert (ws[size // 4:] == 7.0).all()
        want, tol = attend64(st, n, 2500, 4, 32, q, pool, tables)
        check_attend(out, want, tol)


@pytest.mark.parametrize("start,new,heads", [([6000, 20, 3], [1, 1, 1], 32), ([0, 900], [333, 65], 32),
                                             ([0], [2100], 16), ([3000], [40], 64)])
def test_attend_in_place(hip, ctx, start, new, heads):
    say(f"attend into the queries' own buffer {start} {new} heads={heads}")
    g = gen(heads)
    n_pages, tables = make_tables(g, [a + b for a, b in zip(start, new)])
    pool = make_pool(g, n_pages)
    q = bf16(g, sum(new), heads, D)
    out = torch.empty_like(q)
    attend(hip, ctx, start, new, 700, 4, heads, q, pool, tables, out)
    attend(hip, ctx, start, new, 700, 4, heads, q, pool, tables, q)
    torch.cuda.synchronize()
    assert torch.equal(q, out)


def test_no_new_rows_is_no_work(hip, ctx):
    say("batches without new rows")
    g = gen(9)
    n_pages, tables = make_tables(g, [100, 5])
    pool = make_pool(g, n_pages)
    before = pool.clone()
    q = torch.full((2, 32, D), 7.0, dtype=torch.bfloat16, device="cuda")
    out = q.clone()
    cos, sin = rope(128)
    append(hip, ctx, [100, 5], [0, 0], 32, bf16(g, 1, 48 * D), None, None, cos, sin, q, pool, tables)
    attend(hip, ctx, [100, 5], [0, 0], 10, 0, 32, q, pool, tables, out)
    torch.cuda.synchronize()
    assert (q == 7.0).all() and (out == 7.0).all() and torch.equal(pool, before)


@pytest.mark.parametrize("layer", [0, 31])
def test_layers(hip, ctx, layer):
    """The first and the last layer's planes of the pages, in pages far apart."""
    say(f"append and attend, layer {layer}")
    g = gen(layer)
    pool = torch.full((300, LAYERS, 2, KVH, PAGE, D), float("nan"), dtype=torch.bfloat16, device="cuda")
    tables = torch.tensor([[299, 0], [1, 298]], dtype=torch.int32, device="cuda")
    cos, sin = rope(128)
    qkv = bf16(g, 170, 48 * D)
    q, out = (torch.empty(170, 32, D, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    append(hip, ctx, [0, 0], [70, 100], 32, qkv, None, None, cos, sin, q, pool, tables, layer)
    attend(hip, ctx, [0, 0], [70, 100], 30, 2, 32, q, pool, tables, out, layer=layer)
    torch.cuda.synchronize()
    want, tol = attend64([0, 0], [70, 100], 30, 2, 32, q, pool, tables, layer)
    check_attend(out, want, tol)
    pool[:, layer] = float("nan")
    assert torch.isnan(pool).all()               # no other layer was written


@pytest.mark.parametrize("start,new", [([900, 300, 5000], [1, 1, 1]), ([900, 0], [100, 700])])
def test_attend_evicted_pages(hip, ctx, start, new):
    """Keys of missing pages are not seen; a row that sees nothing gets zeros."""
    say(f"attend with evicted pages {start} {new}")
    g = gen(11)
    n_pages, tables = make_tables(g, [a + n for a, n in zip(start, new)])
    pool = make_pool(g, n_pages)
    tables[0] = -1                                            # a sequence without any page
    tables[1, 1::2] = torch.tensor([-1, n_pages, 2**31 - 1, -2**31], device="cuda",
                                   dtype=torch.int32).repeat(tables.shape[1])[:tables[1, 1::2].numel()]
    q = bf16(g, sum(new), 32, D)
    for window, sinks in ((ALL, 0), (200, 70), (40, 0)):
        out = torch.full((sum(new), 32, D), 7.0, dtype=torch.bfloat16, device="cuda")
        attend(hip, ctx, start, new, window, sinks, 32, q, pool, tables, out)
        torch.cuda.synchronize()
        assert (out[:new[0]] == 0).all()
        want, tol = attend64(start, new, window, sinks, 32, q, pool, tables)
        check_attend(out, want, tol, f"window {window}")


@pytest.mark.parametrize("start,new", [([1000, 333], [1, 1]), ([1000, 70], [90, 500]),
                                       ([20000], [2])])
def test_attend_unseen_values_do_not_matter(hip, ctx, start, new):
    """NaN and infinities in every row that no new row sees: other layers, pages of no one, keys
    before the window, rows past the end."""
    say(f"attend with NaN in unseen places {start} {new}")
    window, sinks = 150, 5
    g = gen(12)
    lens = [a + n for a, n in zip(start, new)]
    n_pages, tables = make_tables(g, lens)
    pool = torch.full((n_pages, LAYERS, 2, KVH, PAGE, D), float("nan"), dtype=torch.bfloat16,
                      device="cuda")
    pool[:, :, :, 1::2] = float("inf")
    for b, (a, n) in enumerate(zip(start, new)):
        j = torch.cat([torch.arange(0, min(sinks, a + n)),
                       torch.arange(max(0, a - window + 1), a + n)]).unique().cuda()
        page = tables[b, j // PAGE].long()
        pool[page, LAYER, :, :, j % PAGE] = bf16(g, j.numel(), 2, KVH, D)
    q = bf16(g, sum(new), 32, D)
    out = torch.empty(sum(new), 32, D, dtype=torch.bfloat16, device="cuda")
    attend(hip, ctx, start, new, window, sinks, 32, q, pool, tables, out)
    torch.cuda.synchronize()
    want, tol = attend64(start, new, window, sinks, 32, q, pool, tables)
    check_attend(out, want, tol)


@pytest.mark.parametrize("value", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("at,part", [(130, 0), (130, 1), (40, 1), (175, 1)])
def test_attend_nonfinite_key_reaches_only_rows_that_see_it(hip, ctx, value, at, part):
    """One key's K (part 0) or V (part 1) is NaN or infinite in dim 3 of kv head 2: rows that do not
    see it keep their bits; in V, the rows that see it get that value in that dim alone."""
    say(f"attend: {value} at key {at}, part {part}")
    g = gen(13)
    start, new, window, sinks = [100], [120], 60, 2
    n_pages, tables = make_tables(g, [220])
    pool = make_pool(g, n_pages)
    q = bf16(g, 120, 32, D)
    clean, out = (torch.empty(120, 32, D, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    attend(hip, ctx, start, new, window, sinks, 32, q, pool, tables, clean)
    pool[tables[0, at // PAGE].long(), LAYER, part, 2, at % PAGE, 3] = value
    attend(hip, ctx, start, new, window, sinks, 32, q, pool, tables, out)
    torch.cuda.synchronize()
    p = torch.arange(100, 220, device="cuda")
    sees = (at <= p) & (at > p - window)
    assert torch.equal(out[~sees], clean[~sees])
    other = [h for h in range(32) if h // 4 != 2]
    assert torch.equal(out[:, other], clean[:, other])
    if part == 1:
        hit = out[sees][:, 8:12]
        dims = [d for d in range(D) if d != 3]
        assert torch.equal(hit[..., dims], clean[sees][:, 8:12][..., dims])
        if value != value:
            assert torch.isnan(hit[..., 3]).all()
        else:
            assert (hit[..., 3] == value).all()
    elif value != value:
        assert torch.isnan(out[sees][:, 8:12]).all()


def test_attend_extreme_scores(hip, ctx):
    """Scores far apart: a row's weight is all on its largest key; huge equal scores stay even."""
    say("attend with large scores")
    g = gen(14)
    n_pages, tables = make_tables(g, [700])
    pool = make_pool(g, n_pages)
    q = bf16(g, 50, 32, D, std=200.0)
    out = torch.empty(50, 32, D, dtype=torch.bfloat16, device="cuda")
    attend(hip, ctx, [650], [50], 300, 4, 32, q, pool, tables, out)
    torch.cuda.synchronize()
    want, tol = attend64([650], [50], 300, 4, 32, q, pool, tables)
    # scores reach 200 x 1.28 x 128^0.5 x 5: their fp32 sums are off by up to 128 x 2^-24 x
    # sum |q k| / 128^0.5, below 0.5 x 2^-4, which moves the weights of keys that nearly tie by that share
    kv = pool[tables[0].long(), LAYER, 1].float().abs().max()
    assert ((out.double() - want).abs() <= tol + 2**-4 * kv).all()
    q.zero_()                                   # equal scores: the plain mean
    attend(hip, ctx, [650], [50], 300, 4, 32, q, pool, tables, out)
    torch.cuda.synchronize()
    want, tol = attend64([650], [50], 300, 4, 32, q, pool, tables)
    check_attend(out, want, tol, "equal scores")


def test_attend_agrees_with_prefill_core_paged(hip, ctx):
    say("attend vs ie_attn_prefill_core_paged")
    g = gen(15)
    start, n = 500, 200
    n_pages, tables = make_tables(g, [start + n])
    pool = make_pool(g, n_pages)
    q = bf16(g, n, 32, D)
    out, other = (torch.empty(n, 32, D, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    attend(hip, ctx, [start], [n], ALL, 0, 32, q, pool, tables, out)
    hip.check(hip.lib.ie_attn_prefill_core_paged(ctx.handle, n, start, ptr(q), ptr(pool), n_pages,
                                                 ptr(tables), LAYER, ptr(other)))
    torch.cuda.synchronize()
    _, tol = attend64([start], [n], ALL, 0, 32, q, pool, tables)
    assert ((out.double() - other.double()).abs() <= 2 * tol).all()


# ------------------------------------------------------------------------------- fork
def test_fork(hip, ctx):
    """Several forks of two rows, full and partial last pages, all layers; table rows whole."""
    say("fork")
    g = gen(20)
    n_pages = 14
    pool = torch.randint(-2**15, 2**15, (n_pages, LAYERS, 2, KVH, PAGE, D), dtype=torch.int16,
                         device="cuda", generator=g)
    tables = torch.full((9, 5), 99, dtype=torch.int32, device="cuda")
    tables[0] = torch.tensor([3, 1, 4, 5, -1])
    tables[4] = torch.tensor([2, 0, -7, 55, 3])
    forks = [(0, 1, 200, 6), (0, 2, 192, -1), (0, 3, 1, 7), (4, 5, 127, 8), (4, 6, 0, 0),
             (0, 7, 255, 9), (4, 8, 150, 10)]      # the last one's source page is outside the pool
    before, t = pool.clone(), tables.clone()
    src, dst, pos, fresh = (ints(x) for x in zip(*forks))
    hip.check(hip.lib.ie_kv_fork_paged(ctx.handle, len(forks), src, dst, pos, fresh, ptr(pool), n_pages,
                                       ptr(tables), 9, 5))
    torch.cuda.synchronize()
    for a, b, n, page in forks:
        t[b] = -1
        t[b, :n // PAGE] = t[a, :n // PAGE]
        if n % PAGE:
            t[b, n // PAGE] = page
            old = int(t[a, n // PAGE])
            if 0 <= old < n_pages:
                before[page, :, :, :, :n % PAGE] = before[old, :, :, :, :n % PAGE]
    assert torch.equal(tables, t)
    assert torch.equal(pool, before)


# ------------------------------------------------------------------------------- compaction
def compact_plan(tables, lens, window, sinks, n_pages):
    """The host's plan: (new tables, remap, [live, moved])."""
    def kept(i, n):
        return n > 0 and (i * PAGE < sinks or (i + 1) * PAGE > n - window + 1 or i >= -(-n // PAGE))
    keep = [[0 <= p < n_pages and kept(i, n) for i, p in enumerate(row)]
            for row, n in zip(tables, lens)]
    live = {p for row, k in zip(tables, keep) for p, yes in zip(row, k) if yes}
    count = len(live)
    holes = [p for p in range(count) if p not in live]
    movers = sorted(p for p in live if p >= count)
    remap = {p: p for p in live} | dict(zip(movers, holes))
    new = [[remap[p] if yes else -1 for p, yes in zip(row, k)] for row, k in zip(tables, keep)]
    return new, [remap.get(p, -1) for p in range(n_pages)], [count, len(movers)]


@pytest.mark.parametrize("n_pages,stride,lens,window,sinks,in_place", [
    (1, 1, [64], ALL, 0, True),
    (1, 1, [0], ALL, 0, False),
    (40, 6, [384, 0, 65, 1, 320], ALL, 0, False),
    (40, 6, [384, 0, 65, 1, 320], 64, 0, True),
    (40, 6, [384, 100, 65, 1, 320], 100, 70, False),
    (70, 3, [130] * 20, 1, 1, True),
    (64, 6, [384, 383, 300, 257], 65, 4, False),
])
def test_compact(hip, ctx, n_pages, stride, lens, window, sinks, in_place):
    say(f"compact {n_pages} pages, lens {lens[:5]}, window {window}, sinks {sinks}")
    rng = np.random.default_rng(n_pages + window)
    tables = rng.permutation(max(n_pages, len(lens) * stride))[:len(lens) * stride]
    tables = np.where(tables < n_pages, tables, -1).reshape(len(lens), stride)
    if len(lens) > 3:
        tables[2] = tables[0]                       # shared pages
        tables[3, -1] = 2**31 - 1                   # set aside, outside the pool
    pool = torch.randint(-2**15, 2**15, (n_pages, LAYERS, 2, KVH, PAGE, D), dtype=torch.int16,
                         device="cuda")
    before = pool.clone()
    t = torch.from_numpy(tables.astype(np.int32)).cuda()
    new = t if in_place else torch.empty_like(t)
    remap = torch.full((n_pages,), 77, dtype=torch.int32, device="cuda")
    counts = torch.full((2,), 77, dtype=torch.int32, device="cuda")
    ws = torch.empty(hip.lib.ie_kv_compact_workspace_size(n_pages), dtype=torch.uint8,
                     device="cuda").fill_(255)
    hip.check(hip.lib.ie_kv_compact_paged(ctx.handle, len(lens), ints(lens), window, sinks, ptr(pool),
                                          n_pages, ptr(t), stride, ptr(new), ptr(remap), ptr(counts),
                                          ptr(ws)))
    torch.cuda.synchronize()
    want, want_remap, want_counts = compact_plan(tables.tolist(), lens, window, sinks, n_pages)
    assert counts.tolist() == want_counts
    assert remap.tolist() == want_remap
    assert new.tolist() == want
    for old, to in enumerate(want_remap):
        if to >= 0:
            before[to] = before[old] if to == old else pool.new_tensor(0)
    moved = [(o, n) for o, n in enumerate(want_remap) if n >= 0 and n != o]
    ref = pool.clone()
    for old, to in moved:
        assert torch.equal(pool[to], pool[old])     # sources keep their values
    keep = [p for p in range(n_pages) if p not in {n for _, n in moved}]
    assert torch.equal(ref[keep], before[keep])


def test_compact_large_pool_of_ids(hip, ctx):
    """More ids than pages held: the planning alone, over the largest tables (the live pages already
    lie at the front, so that nothing moves)."""
    say("compact: 64 x 2048 tables")
    n_pages = 16
    t = torch.full((64, 2048), -1, dtype=torch.int32, device="cuda")
    t[63, :8] = torch.arange(8, dtype=torch.int32)
    t[0, 2040:] = torch.arange(8, dtype=torch.int32)
    lens = [131072] * 64
    pool = torch.zeros(n_pages, LAYERS, 2, KVH, PAGE, D, dtype=torch.bfloat16, device="cuda")
    new, remap = torch.empty_like(t), torch.empty(n_pages, dtype=torch.int32, device="cuda")
    counts = torch.empty(2, dtype=torch.int32, device="cuda")
    ws = torch.empty(hip.lib.ie_kv_compact_workspace_size(n_pages), dtype=torch.uint8, device="cuda")
    hip.check(hip.lib.ie_kv_compact_paged(ctx.handle, 64, ints(lens), ALL, 0, ptr(pool), n_pages, ptr(t),
                                          2048, ptr(new), ptr(remap), ptr(counts), ptr(ws)))
    torch.cuda.synchronize()
    assert counts.tolist() == [8, 0]
    assert torch.equal(new, t)
    assert remap.tolist() == list(range(8)) + [-1] * 8


# ------------------------------------------------------------------------------- sampling
def sample64(l, t, k, p, m, u):
    """One row on the host, in 64 bits: (token, distance of the draw to the nearest border)."""
    l = np.where(np.isnan(l), -np.inf, l).astype(np.float64)
    order = np.lexsort((np.arange(l.size), -l))
    top = l[order[0]]
    if top == -np.inf:
        return -1
    if not t > 0 or m > 1:
        return int(order[0])
    with np.errstate(invalid="ignore"):
        w = np.where(l == top, 1.0, np.exp(np.where(l == -np.inf, -np.inf, (l - top) / t)))
    kept = min(k, l.size) if k > 0 else l.size
    s = w[order][:kept]
    if p < 1:
        kept = min(kept, int(np.searchsorted(np.cumsum(s), max(p, 0.0) * s.sum())) + 1)
    if m > 0:
        kept = min(kept, int((s >= m).sum()))
    ids = np.sort(order[:max(kept, 1)])
    cum = np.cumsum(w[ids])
    u = u if u > 0 else 0.0
    at = min(int(np.searchsorted(cum, u * cum[-1], side="right")), ids.size - 1)
    while w[ids[at]] == 0:
        at -= 1
    return int(ids[at])


def sample(hip, ctx, logits, t, k, p, m, u):
    rows, vocab = logits.shape
    f = [None if x is None else torch.tensor(x, dtype=d, device="cuda")
         for x, d in ((t, torch.float32), (k, torch.int32), (p, torch.float32), (m, torch.float32))]
    uu = torch.tensor(u, dtype=torch.float32, device="cuda")
    out = torch.full((rows + 1,), -7, dtype=torch.int32, device="cuda")
    ws = torch.empty(hip.lib.ie_sample_filtered_workspace_size(rows, vocab), dtype=torch.uint8,
                     device="cuda").fill_(255)
    hip.check(hip.lib.ie_sample_filtered(ctx.handle, rows, vocab, ptr(logits), *map(ptr, f), ptr(uu),
                                         ptr(out), ptr(ws)))
    torch.cuda.synchronize()
    assert int(out[rows]) == -7
    return out[:rows].tolist()


def f32(x):
    return [float(np.float32(v)) for v in x]


def check_sample(hip, ctx, logits, t, k, p, m, u):
    rows = logits.shape[0]
    got = sample(hip, ctx, logits, t, k, p, m, u)
    host = logits.cpu().numpy()
    tt, kk, pp, mm = ([d] * rows if x is None else x for x, d in ((t, 1.0), (k, 0), (p, 1.0), (m, 0.0)))
    want = [sample64(host[r], *(float(np.float32(x[r])) if x is not kk else x[r]
                                for x in (tt, kk, pp, mm, u))) for r in range(rows)]
    assert got == want, [(r, g, w) for r, (g, w) in enumerate(zip(got, want)) if g != w][:8]


SETTINGS = [(1.0, 0, 1.0, 0.0), (0.7, 50, 0.9, 0.0), (0.7, 1, 1.0, 0.0), (1.3, 0, 0.3, 0.0),
            (0.8, 40, 1.0, 0.05), (1.0, 0, 1.0, 0.2), (0.5, 300, 0.95, 0.001), (0.0, 5, 0.5, 0.1),
            (2.0, 5000, 0.99, 0.0), (1.0, 0, 0.0, 0.0), (1.0, 0, 1.0, 1.0), (1.0, 0, 1.0, 1.5),
            (1.0, 0, 0.999999, 0.0), (0.05, 0, 0.9, 0.0), (30.0, 0, 0.5, 0.0), (-1.0, 0, 1.0, 0.0)]


@pytest.mark.parametrize("vocab", [1, 2, 7, 255, 1023, 1025, 8193, 50001, V, 200000])
@pytest.mark.parametrize("std,ties", [(2.0, False), (2.0, True), (0.1, True), (8.0, False)])
def test_sample(hip, ctx, vocab, std, ties):
    say(f"sample vocab={vocab} std={std} ties={ties}")
    g = gen(vocab)
    rows = len(SETTINGS)
    logits = torch.empty(rows, vocab, device="cuda").normal_(0.0, std, generator=g)
    if ties:
        logits = logits.bfloat16().float()
    t, k, p, m = map(list, zip(*SETTINGS))
    check_sample(hip, ctx, logits, t, k, p, m, torch.rand(rows, generator=g, device="cuda").tolist())


def test_sample_odd_rows(hip, ctx):
    """Flat rows, rows of few tokens above -inf, infinities, NaN, none at all; uniforms at the ends."""
    say("sample: odd rows")
    n = 5000
    rows = []
    flat = np.zeros(n, np.float32)
    rows += [(flat, s, u) for s in SETTINGS[:7] for u in (0.0, 0.37, 1 - 2**-24)]
    rows += [(flat + 3e38, SETTINGS[0], 0.5), (flat - 3e38, SETTINGS[1], 0.5)]
    few = np.full(n, -np.inf, np.float32)
    few[[17, 4000, 4999]] = [1.0, 1.0, 0.5]
    rows += [(few, s, u) for s in SETTINGS for u in (0.0, 0.2, 0.6, 0.99)]
    one = np.full(n, -np.inf, np.float32)
    one[4321] = -1e30
    rows += [(one, s, 0.9) for s in SETTINGS]
    none = np.full(n, -np.inf, np.float32)
    rows += [(none, s, 0.5) for s in SETTINGS]
    nans = np.full(n, np.nan, np.float32)
    rows += [(nans, SETTINGS[0], 0.5)]
    some = np.random.default_rng(0).standard_normal(n).astype(np.float32)
    some[::3] = np.nan
    some[1::3] = -np.inf
    rows += [(some, s, 0.4) for s in SETTINGS]
    inf = some.copy()
    inf[[100, 2000]] = np.inf
    rows += [(inf, s, u) for s in SETTINGS[:9] for u in (0.1, 0.9)]
    zeros = np.where(np.arange(n) % 2, np.float32(0.0), np.float32(-0.0)).astype(np.float32)
    rows += [(zeros, (1.0, 3, 1.0, 0.0), u) for u in (0.0, 0.5, 0.9)]
    rows += [(some, (1.0, 0, float("nan"), float("nan")), 0.4),
             (some, (float("nan"), 0, 1.0, 0.0), 0.4), (some, SETTINGS[0], float("nan")),
             (some, SETTINGS[0], -1.0), (some, SETTINGS[0], 2.0), (some, SETTINGS[1], 1.0),
             (some, (float("inf"), 0, 1.0, 0.0), 0.7), (some, (1.0, 2**31 - 1, 1.0, 0.0), 0.7),
             (some, (1.0, -2**31, -1.0, -1.0), 0.7)]
    logits = torch.from_numpy(np.stack([r[0] for r in rows])).cuda()
    t, k, p, m = map(list, zip(*[r[1] for r in rows]))
    # (the host's rule: NaN top-p and min-p are off, a uniform past 1 the last token)
    p = [1.0 if x != x else x for x in p]
    m = [0.0 if x != x else x for x in m]
    check_sample(hip, ctx, logits, t, k, p, m, [r[2] for r in rows])
    nan_off = sample(hip, ctx, logits[-9:-8].clone(), [1.0], [0], [float("nan")], [float("nan")], [0.4])
    off = sample(hip, ctx, logits[-9:-8].clone(), None, None, None, None, [0.4])
    assert nan_off == off


@pytest.mark.parametrize("base,t", [(30.0, 1e-6), (100.0, 2e-7), (-30.0, 1e-6), (1e7, 0.7), (-3e5, 0.01),
                                    (1e6, 0.3), (1e10, 900.0)])
def test_sample_logits_far_from_zero(hip, ctx, base, t):
    """Logits of neighbouring fp32 values, some nats apart at their temperature: 8 l / T is far past the
    24 bits of an fp32 product there."""
    say(f"sample: logits next to {base} at temperature {t}")
    rng = np.random.default_rng(3)
    steps = rng.integers(0, 12, 4000)
    ulp = float(np.spacing(np.float32(abs(base))))
    row = (base - steps * ulp).astype(np.float32)
    row[rng.permutation(4000)[:3900]] = np.float32(base - 3000 * ulp - 4000 * t)   # nothing of those
    rows = []
    for share in np.exp(-np.arange(0.3, 8.0, 0.7) * ulp / t):
        rows += [(row, (t, 0, 1.0, float(share)), u) for u in (0.05, 0.5, 0.95, 0.9999)]
    for top_p in (0.2, 0.5, 0.9, 0.99, 0.99999):
        rows += [(row, (t, k, top_p, 0.0), u) for u in (0.05, 0.5, 0.95, 0.9999) for k in (0, 30, 70, 90)]
    logits = torch.from_numpy(np.stack([r[0] for r in rows])).cuda()
    tt, k, p, m = map(list, zip(*[r[1] for r in rows]))
    check_sample(hip, ctx, logits, tt, k, p, m, [r[2] for r in rows])


def test_sample_chunk_that_weighs_next_to_nothing(hip, ctx):
    """A first chunk about 32 nats below the largest logit, and a draw of zero: a token all the same."""
    say("sample: a first chunk of next to no weight")
    depths = np.arange(29.0, 34.0, 0.05, dtype=np.float32)
    logits = np.full((depths.size, 1000), -100.0, np.float32)
    logits[:, :60] = -depths[:, None]
    logits[:, 500] = 0.0
    for rows in (31, depths.size):
        for top_p in (1.0, 0.999999):
            got = sample(hip, ctx, torch.from_numpy(logits[:rows].copy()).cuda(), [1.0] * rows, [0] * rows,
                         [top_p] * rows, [0.0] * rows, [0.0] * rows)
            assert set(got) <= {0, 500}, got


@pytest.mark.parametrize("low", [15.0, 26.0, 28.0])
def test_sample_uniform_of_one_draws_the_last(hip, ctx, low):
    say(f"sample: a uniform of one, last tokens {low} nats down")
    g = gen(1)
    for rows in (30, 60):
        logits = torch.empty(rows, 20000, device="cuda").normal_(0.0, 0.1, generator=g)
        logits[:, -300:] = logits.max(1, keepdim=True).values - low
        for p in (1.0, 0.9999999):
            got = sample(hip, ctx, logits, None, None, [p] * rows, None, [1.0, 2.0, float("inf")] * (rows // 3))
            assert set(got) == {19999} if p == 1 else min(got) > 19000, (rows, p, [
                (i, x) for i, x in enumerate(got) if x != 19999][:6])


def test_sample_infinite_logits_and_temperature(hip, ctx):
    say("sample: infinite logits at an infinite temperature")
    logits = torch.zeros(2, 3000, device="cuda")
    logits[:, [700, 2100]] = float("inf")
    logits[:, 5] = -float("inf")
    for k, p, m in ((0, 1.0, 0.0), (2, 1.0, 0.0), (5, 0.9, 0.0), (0, 0.9, 0.0), (0, 1.0, 0.5), (1000, 0.9, 0.5)):
        got = sample(hip, ctx, logits, [float("inf")] * 2, [k] * 2, [p] * 2, [m] * 2, [0.1, 0.7])
        assert got == [700, 2100], (k, p, m, got)


def test_sample_settings_off(hip, ctx):
    """NULL settings are off; a vocabulary of equal logits gives floor(u x vocab)."""
    say("sample: settings off")
    logits = torch.full((4, V), 2.5, device="cuda")
    u = [0.0, 0.25, 0.5, 1 - 2**-24]
    assert sample(hip, ctx, logits, None, None, None, None, u) == [int(x * V) for x in u]
    check_sample(hip, ctx, logits, None, [1000] * 4, None, None, u)
    check_sample(hip, ctx, logits, None, None, [0.5] * 4, None, u)


def test_sample_many_draws_follow_the_distribution(hip, ctx):
    """Many uniforms on one row: counts against the kept probabilities (exact borders, so that each
    count is off by at most one from the grid's)."""
    say("sample: draws of one row")
    l = torch.tensor([0.0, 1.0, -1.0, 2.0, 0.5], device="cuda")
    n = 4096
    u = [(i + 0.5) / n for i in range(n)]
    got = np.bincount(sample(hip, ctx, l.repeat(n, 1), None, [3] * n, None, None, u), minlength=5)
    w = np.exp(l.double().cpu().numpy())
    w[[0, 2]] = 0
    assert (np.abs(got - n * w / w.sum()) <= 1).all()


@pytest.mark.parametrize("rows,vocab", [(40, V), (33, 100003), (2, 2**21), (35, 2**18)])
def test_sample_many_rows_and_large_vocabularies(hip, ctx, rows, vocab):
    """Past 32 rows each is cut into fewer chunks; chunks of several rounds; the largest vocabulary."""
    say(f"sample {rows} rows of {vocab}")
    g = gen(rows)
    logits = torch.empty(rows, vocab, device="cuda").normal_(0.0, 2.0, generator=g)
    if rows % 2:
        logits = logits.bfloat16().float()
    settings = [SETTINGS[r % len(SETTINGS)] for r in range(rows)]
    t, k, p, m = map(list, zip(*settings))
    check_sample(hip, ctx, logits, t, k, p, m, torch.rand(rows, generator=g, device="cuda").tolist())


def test_sample_rounds_of_small_and_large_cuts(hip, ctx):
    """Rows at the border between the forms of the last step: 63, 64 and 65 tokens to choose from, ties
    across it, and with each filter the one that decides."""
    say("sample: borders of the listed tokens")
    n, rows = 3000, []
    for top in (62, 63, 64, 65, 66, 300):
        l = np.full(n, -8.0, np.float32)
        l[np.random.default_rng(top).permutation(n)[:top]] = np.linspace(0, 3, top, dtype=np.float32)
        tie = l.copy()
        tie[tie > -8] = 1.0
        for row in (l, tie):
            for k in (1, 40, 63, 64, 65, 200):
                for p, m in ((1.0, 0.0), (0.6, 0.0), (1.0, 0.3), (0.9, 0.01)):
                    rows.append((row, (0.9, k, p, m), 0.77))
    logits = torch.from_numpy(np.stack([r[0] for r in rows])).cuda()
    t, k, p, m = map(list, zip(*[r[1] for r in rows]))
    check_sample(hip, ctx, logits, t, k, p, m, [r[2] for r in rows])


# ------------------------------------------------------------------------------- together
class Serving:
    """Several continuations of one prompt over one layer: fork, then append, attend, sample."""

    def __init__(self, hip, ctx, seed, forks=3, prompt=333, window=100, sinks=4):
        self.hip, self.ctx, self.n = hip, ctx, forks
        g = gen(seed)
        self.prompt, self.window, self.sinks = prompt, window, sinks
        self.pages = -(-prompt // PAGE) + forks + 3
        self.pool = make_pool(g, self.pages)
        order = torch.randperm(self.pages, device="cuda", generator=g).to(torch.int32)
        n = -(-prompt // PAGE)
        self.stride = n + 2
        self.tables = torch.full((forks + 1, self.stride), -1, dtype=torch.int32, device="cuda")
        self.tables[0, :n] = order[:n]
        self.fresh = order[n:n + forks].tolist()
        self.cos, self.sin = rope(4096)
        self.qkv = bf16(g, forks, 48 * D)
        self.w = bf16(g, D, mean=1.0, std=0.1)
        self.q, self.out = (torch.zeros(forks, 32, D, dtype=torch.bfloat16, device="cuda")
                            for _ in range(2))
        self.head = torch.empty(32 * D, 1000, device="cuda").normal_(0, 0.05, generator=g)
        self.logits = torch.empty(forks, 1000, device="cuda")
        self.u = torch.rand(forks, device="cuda", generator=g)
        self.k = torch.full((forks,), 40, dtype=torch.int32, device="cuda")
        self.p = torch.full((forks,), 0.9, device="cuda")
        self.token = torch.zeros(forks, dtype=torch.int32, device="cuda")
        self.ws = torch.empty(hip.lib.ie_attn_window_workspace_size(forks, 32), dtype=torch.uint8,
                              device="cuda")
        self.ws2 = torch.empty(hip.lib.ie_sample_filtered_workspace_size(forks, 1000),
                               dtype=torch.uint8, device="cuda")

    def fork(self):
        n = self.n
        self.hip.check(self.hip.lib.ie_kv_fork_paged(
            self.ctx.handle, n, ints([0] * n), ints(range(1, n + 1)), ints([self.prompt] * n),
            ints(self.fresh), ptr(self.pool), self.pages, ptr(self.tables), n + 1, self.stride))

    def step(self):
        start, new = [self.prompt] * self.n, [1] * self.n
        append(self.hip, self.ctx, start, new, 32, self.qkv, self.w, self.w, self.cos, self.sin, self.q,
               self.pool, self.tables[1:])
        attend(self.hip, self.ctx, start, new, self.window, self.sinks, 32, self.q, self.pool,
               self.tables[1:], self.out, self.ws)
        torch.mm(self.out.view(self.n, -1).float(), self.head, out=self.logits)
        self.hip.check(self.hip.lib.ie_sample_filtered(
            self.ctx.handle, self.n, 1000, ptr(self.logits), None, ptr(self.k), ptr(self.p), None,
            ptr(self.u), ptr(self.token), ptr(self.ws2)))

    def check(self):
        """The step against the formulas, from what went into each operator."""
        start, new = [self.prompt] * self.n, [1] * self.n
        pos = torch.full((self.n,), self.prompt, device="cuda")
        x = self.qkv.view(self.n, 48, D)
        want, size = turned64(x[:, :32], self.w, self.cos[pos], self.sin[pos])
        assert ((self.q.double() - want).abs() <= want.abs() * 2**-8 + size * 2**-18).all()
        want, tol = attend64(start, new, self.window, self.sinks, 32, self.q, self.pool, self.tables[1:])
        check_attend(self.out, want, tol, "step")
        host = self.logits.cpu().numpy()
        assert self.token.tolist() == [sample64(host[r], 1.0, 40, float(np.float32(0.9)), 0.0,
                                                float(self.u[r])) for r in range(self.n)]


def test_serving_step(hip, ctx):
    say("fork, append, attend, sample, compact")
    s = Serving(hip, ctx, 30)
    prompt_pages = s.pool[s.tables[0, :6].long()].clone()
    s.fork()
    s.step()
    torch.cuda.synchronize()
    s.check()
    assert torch.equal(s.pool[s.tables[0, :6].long()], prompt_pages)   # the prompt's pages stand
    # the prompt is over, the continuations outgrow their windows: what is left attends as before
    lens = [0] + [s.prompt + 1] * s.n
    remap = torch.empty(s.pages, dtype=torch.int32, device="cuda")
    counts = torch.empty(2, dtype=torch.int32, device="cuda")
    ws = torch.empty(hip.lib.ie_kv_compact_workspace_size(s.pages), dtype=torch.uint8, device="cuda")
    kept = s.out.clone()
    hip.check(hip.lib.ie_kv_compact_paged(ctx.handle, 1 + s.n, ints(lens), s.window, s.sinks, ptr(s.pool),
                                          s.pages, ptr(s.tables), s.stride, ptr(s.tables), ptr(remap),
                                          ptr(counts), ptr(ws)))
    attend(hip, ctx, [s.prompt] * s.n, [1] * s.n, s.window, s.sinks, 32, s.q, s.pool, s.tables[1:],
           s.out, s.ws)
    torch.cuda.synchronize()
    # block 0 (sinks), block 4 (positions 256 on; the window of the next token starts at 235, in block
    # 3) shared, the three last blocks of their own
    assert counts.tolist()[0] == 3 + s.n
    assert int(s.tables.max()) == counts.tolist()[0] - 1
    assert torch.equal(s.out, kept)


def test_serving_step_captured(hip, ctx):
    """The step recorded into a graph and replayed, with new inputs, eager work and other calls between;
    two graphs with workspaces of their own replay in turn."""
    say("captured step")
    a, b = Serving(hip, ctx, 31), Serving(hip, ctx, 32, forks=5, prompt=2000, window=1900)
    a.fork()
    b.fork()
    graphs = []
    for s in (a, b):
        s.step()                                   # (the library product's own set-up)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=ctx.stream):
            s.step()
        graphs.append(graph)
    for i in range(4):
        for s, graph in zip((a, b), graphs):
            s.qkv.normal_(0, 1.28, generator=gen(100 + i))
            s.u.uniform_(0, 1, generator=gen(200 + i))
            s.out.fill_(9.0)
            graph.replay()
            torch.cuda.synchronize()
            got = s.token.tolist(), s.out.clone()
            s.check()
            s.step()                               # eager, same bits
            torch.cuda.synchronize()
            assert got[0] == s.token.tolist() and torch.equal(got[1], s.out)


def test_two_streams_at_once(hip, ctx):
    """Two contexts on streams of their own, each with its workspace, at the same time."""
    from infengine_amd.engine import Context
    say("two streams")
    g = gen(40)
    start, new = [9000, 5000, 100], [1, 1, 1]
    n_pages, tables = make_tables(g, [a + n for a, n in zip(start, new)])
    pool = make_pool(g, n_pages)
    q = bf16(g, 3, 32, D)
    logits = torch.empty(8, V, device="cuda").normal_(0, 2, generator=g)
    u = torch.rand(8, device="cuda", generator=g)
    k = torch.full((8,), 50, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    main = torch.cuda.current_stream()
    other = Context(0, graph=False)
    torch.cuda.set_stream(main)
    try:
        outs, tokens = [], []
        for c in (ctx, other):
            outs.append(torch.empty(3, 32, D, dtype=torch.bfloat16, device="cuda"))
            tokens.append(torch.empty(8, dtype=torch.int32, device="cuda"))
        wss = [torch.empty(hip.lib.ie_attn_window_workspace_size(3, 32), dtype=torch.uint8,
                           device="cuda") for _ in range(2)]
        wst = [torch.empty(hip.lib.ie_sample_filtered_workspace_size(8, V), dtype=torch.uint8,
                           device="cuda") for _ in range(2)]
        torch.cuda.synchronize()
        for _ in range(10):
            for i, c in enumerate((ctx, other)):
                attend(hip, c, start, new, 8000, 4, 32, q, pool, tables, outs[i], wss[i])
                hip.check(hip.lib.ie_sample_filtered(c.handle, 8, V, ptr(logits), None, ptr(k), None,
                                                     None, ptr(u), ptr(tokens[i]), ptr(wst[i])))
        torch.cuda.synchronize()
        assert torch.equal(outs[0], outs[1])
        assert torch.equal(tokens[0], tokens[1])
        want, tol = attend64(start, new, 8000, 4, 32, q, pool, tables)
        check_attend(outs[0], want, tol)
        host = logits.cpu().numpy()
        assert tokens[0].tolist() == [sample64(host[r], 1.0, 50, 1.0, 0.0, float(u[r]))
                                      for r in range(8)]
    finally:
        torch.cuda.synchronize()
        other.close()
