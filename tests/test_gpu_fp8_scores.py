"""Scores of 8-bit keys whose products differ much in size: channels in which keys and queries are large throughout,
queries of a wide range.  The sums of the products are fp32 sums.

Tolerance: a score, a sum of 128 exact products in fp32 whose steps may cut, is off by at most
  E = 128 x 2^-23 x sum |q k| / 128^0.5,
so a weight by a factor within exp(+-2 E): exp(2 E) - 1 of the sum of w |v|, on top of what the attention's own
roundings take (test_gpu_paged_serving)."""
import pytest
import torch

from gpu_util import say
from test_gpu_kv_fp8 import attend8, bf16_pool, pool8, put8, shared, shared_tables
from test_gpu_paged_serving import ALL, D, KVH, LAYER, LAYERS, PAGE, attend64, bf16, check_attend, gen, make_tables

pytestmark = pytest.mark.gpu


def wide_queries(g, rows, heads, scale):
    """Values spread over 2^-30 .. 1 of a row's largest."""
    q = bf16(g, rows, heads, D)
    q *= torch.exp2(torch.randint(-28, 1, q.shape, generator=g, device="cuda").float()).bfloat16()
    q[..., 0] = 7.0
    return q * scale


def check(out, start, new, heads, q, plain, tables, window=ALL, sinks=0):
    want, tol = attend64(start, new, window, sinks, heads, q, plain, tables)
    size = plain.clone()                                          # for sum w |v|
    size[:, LAYER, 1] = size[:, LAYER, 1].abs()
    mass, _ = attend64(start, new, window, sinks, heads, q, size, tables)
    of, k = q.double().abs(), plain[:, LAYER, 0].double().abs().transpose(0, 1).reshape(KVH, -1, D)
    e = torch.stack([2**-16 * (of[:, h] @ k[h // (heads // KVH)].t()).amax(-1) for h in range(heads)], 1)
    check_attend(out, want, tol + torch.expm1(2 * e / D**0.5)[..., None] * mass)


@pytest.mark.parametrize("fmt", [0, 1])
@pytest.mark.parametrize("sizes,lens,start,new,heads", [
    ([1], [0], [2000], [4], 32),                          # the narrow form
    ([1], [0], [1500], [600], 32),                        # the wide form
    ([1], [0], [300], [2500], 16),
    ([1, 1], [0, 0], [40000, 30], [1, 90], 64),
    ([5], [1280], [1280, 1290, 1400, 1281, 1300], [1, 2, 1, 9, 1], 32),
])
@pytest.mark.parametrize("key,query", [(30.0, 0.0), (30.0, 20.0), (8.0, 60.0)])
def test_channels_that_are_large_throughout(hip, ctx, sizes, lens, start, new, heads, fmt, key, query):
    """Four channels of the keys, and of the queries, lie about a large value: their products outweigh the others
    in every score, but for the softmax it is the others that count."""
    say(f"shared, {8 if fmt else 16} bits: {start[:2]} {new[:2]} heads={heads} large channels {key} {query}")
    g = gen(sum(new) + int(key + query))
    n_pages, tables = shared_tables(g, sizes, lens, start, new)
    kv = bf16(g, n_pages, 2, KVH, PAGE, D)
    q = bf16(g, sum(new), heads, D)
    at = torch.randperm(D, generator=g, device="cuda")[:4]
    kv[:, 0, ..., at] += key * torch.tensor([1.0, -1.0, 1.0, 0.5], device="cuda").bfloat16()
    q[..., at] += query * torch.tensor([1.0, -1.0, -0.75, 0.5], device="cuda").bfloat16()
    if fmt:
        pool = pool8(n_pages)
        put8(pool, LAYER, kv)
        plain = bf16_pool(pool)
    else:
        plain = pool = torch.zeros(n_pages, LAYERS, 2, KVH, PAGE, D, dtype=torch.bfloat16, device="cuda")
        pool[:, LAYER] = kv
    out = torch.empty_like(q)
    shared(hip, ctx, fmt, sizes, lens, start, new, ALL, 0, heads, q, pool, tables, out)
    torch.cuda.synchronize()
    check(out, start, new, heads, q, plain, tables)
    if fmt:
        attend8(hip, ctx, start, new, ALL, 0, heads, q, pool, tables, out)
        torch.cuda.synchronize()
        check(out, start, new, heads, q, plain, tables)


@pytest.mark.parametrize("start,new", [([700], [1]), ([700, 300], [3, 70]), ([500], [900])])
@pytest.mark.parametrize("keys", [1.0, 64.0])
def test_small_values_of_a_query_count(hip, ctx, start, new, keys):
    """Keys that are zero where the query is largest: what the scores come from are the query's small values."""
    say(f"attend, 8 bits: queries of a wide range {start} {new} keys {keys}")
    g = gen(int(keys) + sum(new))
    n_pages, tables = make_tables(g, [a + n for a, n in zip(start, new)])
    kv = bf16(g, n_pages, 2, KVH, PAGE, D)
    kv[:, 0] *= keys
    kv[:, 0, ..., 0] = 0
    pool = pool8(n_pages)
    put8(pool, LAYER, kv)
    plain = bf16_pool(pool)
    q = wide_queries(g, sum(new), 32, 1.0)
    out = torch.empty_like(q)
    attend8(hip, ctx, start, new, ALL, 0, 32, q, pool, tables, out)
    torch.cuda.synchronize()
    check(out, start, new, 32, q, plain, tables)


@pytest.mark.parametrize("power", [-100, -60, 60, 100])
def test_queries_of_any_magnitude(hip, ctx, power):
    """Queries times 2^n against keys times 2^-n: the same bits."""
    say(f"attend and shared, 8 bits: queries times 2^{power}")
    g = gen(77)
    start, new, sizes, lens = [640, 700, 900], [1, 4, 1], [3], [640]
    n_pages, tables = shared_tables(g, sizes, lens, start, new)
    kv = bf16(g, n_pages, 2, KVH, PAGE, D)
    q = wide_queries(g, sum(new), 32, 1.0)
    q = torch.where(q.abs() < 2.0**-13, 0.0, q.float()).bfloat16()       # (normal numbers all)
    outs = []
    for f in (0, power):
        pool = pool8(n_pages)
        some = kv.clone()
        some[:, 0] = (kv[:, 0].double() * 2.0**-f).bfloat16()
        put8(pool, LAYER, some)
        p = (q.double() * 2.0**f).bfloat16()
        a, b = torch.empty_like(q), torch.empty_like(q)
        attend8(hip, ctx, start, new, ALL, 0, 32, p, pool, tables, a)
        shared(hip, ctx, 1, sizes, lens, start, new, ALL, 0, 32, p, pool, tables, b)
        torch.cuda.synchronize()
        outs.append((a, b))
    assert torch.equal(outs[0][0], outs[1][0]) and torch.equal(outs[0][1], outs[1][1])


@pytest.mark.parametrize("fmt", [0, 1])
@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("sizes,lens,start,new", [
    ([1], [0], [300], [2]), ([1], [0], [20000], [1]), ([1], [0], [300], [200]), ([3], [256], [300, 256, 310], [1, 2, 1]),
])
def test_scores_of_the_largest_size(hip, ctx, sizes, lens, start, new, sign, fmt):
    """Sums q . k of nearly 2^33, all of one sign: a row's weight is all on the key of its largest, whose value it gets."""
    say(f"shared, {8 if fmt else 16} bits: scores of 2^33, sign {sign}, {start} {new}")
    g = gen(5 + sum(new))
    n_pages, tables = shared_tables(g, sizes, lens, start, new)
    kv = bf16(g, n_pages, 2, KVH, PAGE, D)
    steps = torch.randint(1, 7, (n_pages, KVH, PAGE, 1), generator=g, device="cuda")
    kv[:, 0] = (2.0**11 * (1 + steps / 8)).bfloat16()
    # position 37 of every sequence has the largest score: 1.875 x 2^11 or, of negative scores, 2^11
    kv[tables[:, 0].long(), 0, :, 37] = 2.0**11 * (1.875 if sign > 0 else 1.0)
    kv[:, 1] = torch.randint(-15, 16, kv[:, 1].shape, generator=g, device="cuda").bfloat16() * 28    # (codes of scale 1)
    pool = pool8(n_pages) if fmt else torch.zeros(n_pages, LAYERS, 2, KVH, PAGE, D, dtype=torch.bfloat16, device="cuda")
    if fmt:
        put8(pool, LAYER, kv)
        assert torch.equal(bf16_pool(pool)[:, LAYER, 0], kv[:, 0])
        kv = bf16_pool(pool)[:, LAYER]
    else:
        pool[:, LAYER] = kv
    q = torch.full((sum(new), 32, D), sign * 2.0**14, dtype=torch.bfloat16, device="cuda")
    out = torch.empty_like(q)
    shared(hip, ctx, fmt, sizes, lens, start, new, ALL, 0, 32, q, pool, tables, out)
    torch.cuda.synchronize()
    seq = torch.repeat_interleave(torch.arange(len(new)), torch.tensor(new)).cuda()
    want = kv[tables[seq, 0].long(), 1, :, 37].repeat_interleave(4, 1)
    assert torch.equal(out, want)
