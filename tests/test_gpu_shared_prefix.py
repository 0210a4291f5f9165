"""Attention over shared prefixes whose sequences are at different positions behind a sliding window, against plain
computations in 64 bits: the tables as compaction leaves them.

Tolerances as in test_gpu_kv_fp8."""
import pytest
import torch

from gpu_util import say
from test_gpu_kv_fp8 import pools, shared, shared_tables
from test_gpu_paged_serving import D, PAGE, attend64, bf16, check_attend, gen, ints, ptr

pytestmark = pytest.mark.gpu

AHEAD = [
    # (sizes, shared positions, start, new, window, sinks, heads): the first of a group is not the last in position
    ([3], [1280], [3000, 1400, 1290], [1, 1, 1], 400, 0, 32),
    ([3], [1280], [3000, 1400, 1290], [2, 0, 3], 400, 70, 16),
    ([4], [2048], [2500, 2048, 4000, 2100], [1, 4, 1, 2], 300, 4, 64),
    ([2, 3], [640, 1280], [1000, 700, 2600, 1300, 1290], [1, 2, 1, 1, 5], 500, 0, 32),
    ([4], [1280], [5000, 4000, 1300, 1500], [1, 0, 900, 1], 600, 10, 32),    # the last in position attends by itself
    ([3], [1984], [1984, 9000, 1984], [1, 1, 2], 1000, 64, 32),
]


def evict(tables, lens, window, sinks):
    """Each row's entries that its next token does not need, away (as ie_kv_compact_paged does)."""
    for b, n in enumerate(lens):
        for i in range(-(-n // PAGE)):
            if not (i * PAGE < sinks or (i + 1) * PAGE > n - window + 1):
                tables[b, i] = -1


@pytest.mark.parametrize("fmt", [0, 1])
@pytest.mark.parametrize("i", range(len(AHEAD)))
def test_shared_rows_evicted_by_their_own_lengths(hip, ctx, i, fmt):
    """A sequence that is further on no longer names pages that others of its group still see."""
    sizes, lens, start, new, window, sinks, heads = AHEAD[i]
    say(f"shared, {8 if fmt else 16} bits, evicted by length: {start} {new} window={window} sinks={sinks} heads={heads}")
    g = gen(200 + i)
    n_pages, tables = shared_tables(g, sizes, lens, start, new)
    whole = tables.clone()
    evict(tables, start, window, sinks)
    assert (tables != whole).any()
    pool, plain = pools(g, fmt, n_pages)
    q = bf16(g, sum(new), heads, D)
    out = torch.full_like(q, 7.0)
    shared(hip, ctx, fmt, sizes, lens, start, new, window, sinks, heads, q, pool, tables, out)
    torch.cuda.synchronize()
    want, tol = attend64(start, new, window, sinks, heads, q, plain, tables)
    full, _ = attend64(start, new, window, sinks, heads, q, plain, whole)
    assert torch.equal(want, full)                 # (what went, no new row sees)
    check_attend(out, want, tol)


def test_shared_after_compaction(hip, ctx):
    """Forks of one prompt at different lengths, compacted, attend on: each row as by itself."""
    say("shared, 16 bits: behind a compaction")
    g = gen(220)
    prompt, start, new, window, sinks = 1280, [2900, 1500, 1290, 1281], [1, 1, 2, 3], 500, 20
    n_pages, tables = shared_tables(g, [4], [prompt], start, new, spare=5)
    pool, _ = pools(g, 0, n_pages)
    remap = torch.empty(n_pages, dtype=torch.int32, device="cuda")
    counts = torch.empty(2, dtype=torch.int32, device="cuda")
    ws = torch.empty(hip.lib.ie_kv_compact_workspace_size(n_pages), dtype=torch.uint8, device="cuda")
    hip.check(hip.lib.ie_kv_compact_paged(ctx.handle, 4, ints(start), window, sinks, ptr(pool), n_pages, ptr(tables),
                                          tables.shape[1], ptr(tables), ptr(remap), ptr(counts), ptr(ws)))
    torch.cuda.synchronize()
    assert (tables[0, 1:20] == -1).all() and (tables[3, 13:20] >= 0).all()
    q = bf16(g, sum(new), 32, D)
    out = torch.full_like(q, 7.0)
    shared(hip, ctx, 0, [4], [prompt], start, new, window, sinks, 32, q, pool, tables, out)
    torch.cuda.synchronize()
    want, tol = attend64(start, new, window, sinks, 32, q, pool, tables)
    check_attend(out, want, tol)


def test_fork_without_a_pool(hip, ctx):
    """Forks at full pages copy ids only: the pool, which may have any format, need not be given."""
    say("fork without a pool")
    tables = torch.arange(40, dtype=torch.int32, device="cuda").view(4, 10)
    want = tables.clone()
    want[1, 3:], want[3, :] = -1, -1
    want[1, :3] = tables[0, :3]
    hip.check(hip.lib.ie_kv_fork_paged(ctx.handle, 2, ints([0, 2]), ints([1, 3]), ints([192, 0]), ints([-1, -1]), None,
                                       5, ptr(tables), 4, 10))
    torch.cuda.synchronize()
    assert torch.equal(tables, want)
