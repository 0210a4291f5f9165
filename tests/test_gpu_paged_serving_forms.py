"""Forms of the paged-serving kernels that only large batches and pools reach: attention by 32 columns a
wave around infinities and NaN, pages gigabytes into a pool, compaction of pools of more than 4096 pages,
and page operators in a graph."""
import numpy as np
import pytest
import torch

from gpu_util import say
from test_gpu_paged_serving import (ALL, D, KVH, LAYER, LAYERS, PAGE, append, attend, attend64, bf16,
                                    check_attend, compact_plan, gen, ints, make_pool, make_tables, ptr,
                                    rope)

pytestmark = pytest.mark.gpu


# thousands of rows take the 32-column form, whose masked tiles hold values of two column sets back
@pytest.mark.parametrize("heads,rows", [(32, 2500), (16, 2500), (64, 1300)])
def test_attend_unseen_values_do_not_matter_to_chunks(hip, ctx, heads, rows):
    say(f"attend: NaN in unseen places, {rows} rows of {heads} heads")
    start, new, window, sinks = [700], [rows], 150, 5
    g = gen(heads)
    n_pages, tables = make_tables(g, [700 + rows])
    pool = torch.full((n_pages, LAYERS, 2, KVH, PAGE, D), float("nan"), dtype=torch.bfloat16, device="cuda")
    pool[:, :, :, 1::2] = float("inf")
    j = torch.cat([torch.arange(sinks), torch.arange(700 - window + 1, 700 + rows)]).cuda()
    page = tables[0, j // PAGE].long()
    pool[page, LAYER, :, :, j % PAGE] = bf16(g, j.numel(), 2, KVH, D)
    q = bf16(g, rows, heads, D)
    out = torch.empty_like(q)
    attend(hip, ctx, start, new, window, sinks, heads, q, pool, tables, out)
    torch.cuda.synchronize()
    want, tol = attend64(start, new, window, sinks, heads, q, pool, tables)
    check_attend(out, want, tol)


@pytest.mark.parametrize("value", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("at,part", [(1500, 0), (1500, 1), (701, 1), (2239, 1), (3, 1)])
def test_attend_nonfinite_key_reaches_only_rows_of_a_chunk_that_see_it(hip, ctx, value, at, part):
    """One key's K (part 0) or V (part 1) is NaN or infinite in dim 3 of kv head 2: rows that do not see it
    keep their bits; in V, the rows that see it get that value in that dim alone."""
    say(f"attend: {value} at key {at}, part {part}, 2500 rows")
    g = gen(13)
    start, new, window, sinks = [700], [2500], 150, 5
    n_pages, tables = make_tables(g, [3200])
    pool = make_pool(g, n_pages)
    q = bf16(g, 2500, 32, D)
    clean, out = torch.empty_like(q), torch.empty_like(q)
    attend(hip, ctx, start, new, window, sinks, 32, q, pool, tables, clean)
    pool[tables[0, at // PAGE].long(), LAYER, part, 2, at % PAGE, 3] = value
    attend(hip, ctx, start, new, window, sinks, 32, q, pool, tables, out)
    torch.cuda.synchronize()
    p = torch.arange(700, 3200, device="cuda")
    sees = (at <= p) & ((at > p - window) | (at < sinks))
    assert sees.any()
    assert torch.equal(out[~sees], clean[~sees])
    other = [h for h in range(32) if h // 4 != 2]
    assert torch.equal(out[:, other], clean[:, other])
    if part == 1:
        hit = out[sees][:, 8:12]
        dims = [d for d in range(D) if d != 3]
        assert torch.equal(hit[..., dims], clean[sees][:, 8:12][..., dims])
        # (every weight here is far above the smallest number: scores lie within 60 nats)
        assert torch.isnan(hit[..., 3]).all() if value != value else (hit[..., 3] == value).all()
    elif value != value:
        assert torch.isnan(out[sees][:, 8:12]).all()


@pytest.mark.parametrize("window,sinks", [(200, 70), (40, 0)])
def test_attend_evicted_pages_of_chunks(hip, ctx, window, sinks):
    say(f"attend: evicted pages, chunks, window {window}")
    start, new = [900, 0], [1000, 2000]
    g = gen(11)
    n_pages, tables = make_tables(g, [a + n for a, n in zip(start, new)])
    pool = make_pool(g, n_pages)
    tables[0] = -1
    tables[1, 1::2] = torch.tensor([-1, n_pages, 2**31 - 1, -2**31], device="cuda",
                                   dtype=torch.int32).repeat(tables.shape[1])[:tables[1, 1::2].numel()]
    q = bf16(g, 3000, 32, D)
    out = torch.full_like(q, 7.0)
    attend(hip, ctx, start, new, window, sinks, 32, q, pool, tables, out)
    torch.cuda.synchronize()
    assert (out[:1000] == 0).all()
    want, tol = attend64(start, new, window, sinks, 32, q, pool, tables)
    check_attend(out, want, tol)


@pytest.mark.parametrize("rows", [1, 70, 2500])
def test_attend_scores_of_minus_infinity_weigh_nothing(hip, ctx, rows):
    """Rows that see only their own key: zeros where its score is -inf, its value elsewhere."""
    say(f"attend: scores of -inf, {rows} rows")
    g = gen(rows)
    n_pages, tables = make_tables(g, [rows])
    pool = make_pool(g, n_pages)
    j = torch.arange(0, rows, 3, device="cuda")
    pool[tables[0, j // PAGE].long(), LAYER, 0, :, j % PAGE, 3] = -float("inf")
    q = torch.zeros(rows, 32, D, dtype=torch.bfloat16, device="cuda")
    q[..., 3] = 1.0
    out = torch.full_like(q, 7.0)
    attend(hip, ctx, [0], [rows], 1, 0, 32, q, pool, tables, out)
    torch.cuda.synchronize()
    p = torch.arange(rows, device="cuda")
    own = pool[tables[0, p // PAGE].long(), LAYER, 1, :, p % PAGE].repeat_interleave(4, dim=1)
    own[::3] = 0
    assert torch.equal(out, own)


@pytest.mark.parametrize("n_pages,held,pick,window", [(4700, 4400, "any", ALL), (4700, 300, "last", 900),
                                                      (4500, 4500, "any", 900)])
def test_compact_pool_of_thousands_of_pages(hip, ctx, n_pages, held, pick, window):
    """Pools of more than 4096 pages: ranks over several waves of the plan, pages moved across them."""
    say(f"compact {held} of {n_pages} pages")
    rng = np.random.default_rng(held)
    ids = rng.permutation(n_pages)[:held] if pick == "any" else n_pages - 1 - rng.permutation(held)
    rows, stride = 60, 80
    tables = np.full(rows * stride, -1)
    tables[:held] = ids
    tables = rng.permutation(tables).reshape(rows, stride)
    lens = rng.integers(0, stride * PAGE, rows).tolist()
    lens[0], lens[1] = 0, stride * PAGE
    want, want_remap, want_counts = compact_plan(tables.tolist(), lens, window, 70, n_pages)
    assert want_counts[1] > 100 and (window != ALL or want_counts[0] > 4096)
    pool = torch.empty(n_pages, LAYERS * 2 * KVH * PAGE * D // 2, dtype=torch.int32, device="cuda")
    inside = torch.arange(pool.shape[1], dtype=torch.int32, device="cuda") * 8192
    torch.add(torch.arange(n_pages, dtype=torch.int32, device="cuda")[:, None], inside, out=pool)
    t = torch.from_numpy(tables.astype(np.int32)).cuda()
    new = torch.empty_like(t)
    remap = torch.empty(n_pages, dtype=torch.int32, device="cuda")
    counts = torch.empty(2, dtype=torch.int32, device="cuda")
    ws = torch.empty(hip.lib.ie_kv_compact_workspace_size(n_pages), dtype=torch.uint8, device="cuda")
    hip.check(hip.lib.ie_kv_compact_paged(ctx.handle, rows, ints(lens), window, 70, ptr(pool), n_pages, ptr(t),
                                          stride, ptr(new), ptr(remap), ptr(counts), ptr(ws)))
    torch.cuda.synchronize()
    assert counts.tolist() == want_counts
    assert remap.tolist() == want_remap
    assert new.tolist() == want
    holds = np.arange(n_pages)
    for old, to in enumerate(want_remap):
        if to >= 0:
            holds[to] = old
    holds = torch.from_numpy(holds.astype(np.int32)).cuda()
    for a in range(0, n_pages, 500):
        assert torch.equal(pool[a:a + 500], holds[a:a + 500, None] + inside)


def test_pages_far_into_the_pool(hip, ctx):
    """Append, attend and fork in pages past 2^32 elements (8 GiB) from the pool's start: as in pages near it."""
    say("pages far into the pool")
    n_pages, near = 1100, [1, 3, 5]
    far = [1099, 1030, 1025]
    assert min(far) * LAYERS * 2 * KVH * PAGE * D > 2**32
    g = gen(50)
    pool = torch.empty(n_pages, LAYERS, 2, KVH, PAGE, D, dtype=torch.bfloat16, device="cuda")
    tables = torch.tensor([near[:2] + [-1], far[:2] + [-1], [-1] * 3, [-1] * 3], dtype=torch.int32, device="cuda")
    cos, sin = rope(128)
    qkv = bf16(g, 100, 48 * D).repeat(2, 1)
    q, out = (torch.empty(200, 32, D, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    pool[near + far] = 0
    append(hip, ctx, [0, 0], [100, 100], 32, qkv, None, None, cos, sin, q, pool, tables, layer=31)
    attend(hip, ctx, [0, 0], [100, 100], 70, 3, 32, q, pool, tables, out, layer=31)
    hip.check(hip.lib.ie_kv_fork_paged(ctx.handle, 2, ints([0, 1]), ints([2, 3]), ints([90, 90]),
                                       ints([near[2], far[2]]), ptr(pool), n_pages, ptr(tables), 4, 3))
    torch.cuda.synchronize()
    want, tol = attend64([0], [100], 70, 3, 32, q[:100], pool, tables, layer=31)
    check_attend(out[:100], want, tol)
    assert torch.equal(out[100:], out[:100])
    for a, b in zip(near, far):
        assert torch.equal(pool[a], pool[b])
    assert pool[near[2], 31, :, :, :26].ne(0).any() and not pool[near[2], :, :, :, 26:].any()
    assert tables[2:].tolist() == [[near[0], near[2], -1], [far[0], far[2], -1]]


def test_fork_and_compact_captured(hip, ctx):
    """A fork and a compaction recorded into one graph and replayed over new pages and tables."""
    say("captured fork and compaction")
    g = gen(51)
    n_pages, stride, lens = 24, 4, [0, 150, 150, 70]
    pool = torch.empty(n_pages, LAYERS, 2, KVH, PAGE, D, dtype=torch.bfloat16, device="cuda")
    tables = torch.empty(4, stride, dtype=torch.int32, device="cuda")
    new, remap = torch.empty_like(tables), torch.empty(n_pages, dtype=torch.int32, device="cuda")
    counts = torch.empty(2, dtype=torch.int32, device="cuda")
    ws = torch.empty(hip.lib.ie_kv_compact_workspace_size(n_pages), dtype=torch.uint8, device="cuda")

    def fill():
        pool.normal_(0.0, 1.0, generator=g)
        ids = torch.randperm(20, device="cuda", generator=g).int()
        tables.fill_(-1)
        tables[0, :3] = ids[:3]
        tables[3, :2] = ids[3:5]
        torch.cuda.synchronize()

    def step():
        hip.check(hip.lib.ie_kv_fork_paged(ctx.handle, 2, ints([0, 0]), ints([1, 2]), ints([150, 150]),
                                           ints([21, 23]), ptr(pool), n_pages, ptr(tables), 4, stride))
        hip.check(hip.lib.ie_kv_compact_paged(ctx.handle, 4, ints(lens), ALL, 0, ptr(pool), n_pages, ptr(tables),
                                              stride, ptr(new), ptr(remap), ptr(counts), ptr(ws)))

    fill()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=ctx.stream):
        step()
    for _ in range(4):
        fill()
        kept = pool.clone(), tables.clone()
        graph.replay()
        torch.cuda.synchronize()
        got = [x.clone() for x in (pool, tables, new, remap, counts)]
        pool.copy_(kept[0])
        tables.copy_(kept[1])
        step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, (pool, tables, new, remap, counts)))
        plan = compact_plan(tables.tolist(), lens, ALL, 0, n_pages)
        assert (new.tolist(), remap.tolist(), counts.tolist()) == tuple(plan)
        assert counts.tolist()[0] == 6                    # two shared pages, two of the forks, two of the last
        old = tables[0, 2].long()
        assert torch.equal(pool[new[1, 2].long(), :, :, :, :22], kept[0][old, :, :, :, :22])
