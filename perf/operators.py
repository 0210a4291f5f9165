"""Cases of the operators that serve many conversations, and several continuations of one prompt,
over the paged K/V cache:

  append    ie_qk_norm_rope_paged: norms and rotation of a ragged batch's queries and keys, K/V into
            the pages
  attend    ie_attn_window_paged: attention of ragged chunks of new tokens over the pages, with a
            sliding window and sinks
  fork      ie_kv_fork_paged: continuations that share a sequence's full pages
  compact   ie_kv_compact_paged: pages behind the windows freed, the live ones moved to the front
  sample    ie_sample_filtered: temperature, top-k, top-p and min-p from given uniforms

listed() fixes twelve; draw() gives others of the same ranges.  With `own` false a pass is the
operator's plain form in elementary torch operations, with `own` true the library's call.
"""
import functools
import random

import torch

own = False

KVH, D, PAGE, LAYERS, V = 8, 128, 64, 32, 128256
MAX_LONG = 131072
LAYER = 5         # the layer whose pages the attention reads and the append writes
EPS = 1e-5
KV_STD = 1.28     # keys and values of a random-init model: sqrt(4096) * 0.02
EVERYTHING = MAX_LONG   # a window that nothing falls out of


# ------------------------------------------------------------------------------- cases
def listed():
    return [
        # the new tokens of a full decode batch, without norms (the served model's own form)
        {"name": "append_16x1", "kind": "append", "seqs": 16, "rows": 1, "ctx": 6000, "heads": 32,
         "norm": False},
        # a step that prefills five prompts at once, queries and keys normed
        {"name": "append_5x1500", "kind": "append", "seqs": 5, "rows": 1500, "ctx": 900,
         "heads": 32, "norm": True},
        # one user's next token, everything visible: the latency of a single chat
        {"name": "attend_1_at_600", "kind": "attend", "seqs": 1, "rows": 1, "ctx": 600,
         "heads": 32, "window": EVERYTHING, "sinks": 0},
        # a full batch of long sessions, one token each, over windows of 4096
        {"name": "attend_16_at_60000", "kind": "attend", "seqs": 16, "rows": 1, "ctx": 60000,
         "heads": 32, "window": 4096, "sinks": 4},
        # a mixed step: the next turns of six sessions, 1 to 333 tokens, odd window and sinks
        {"name": "attend_6x333_at_9000", "kind": "attend", "seqs": 6, "rows": 333, "ctx": 9000,
         "heads": 32, "window": 1500, "sinks": 5},
        # a long document's chunk, one prefill call's worth of tokens
        {"name": "attend_8192_at_8192", "kind": "attend", "seqs": 1, "rows": 8192, "ctx": 8192,
         "heads": 32, "window": 4096, "sinks": 64},
        # four answers to one short question
        {"name": "fork_4_at_600", "kind": "fork", "forks": 4, "ctx": 600},
        # a full batch of continuations of one long prompt
        {"name": "fork_16_at_5050", "kind": "fork", "forks": 16, "ctx": 5050},
        # a few chats, one of them over: its pages are closed up
        {"name": "compact_4_at_1000", "kind": "compact", "seqs": 4, "ctx": 1000,
         "window": EVERYTHING, "sinks": 0},
        # a batch of sessions that have outgrown their windows
        {"name": "compact_8_at_4000", "kind": "compact", "seqs": 8, "ctx": 4000, "window": 1000,
         "sinks": 4},
        # one user's token
        {"name": "sample_1", "kind": "sample", "rows": 1, "ties": False},
        # a large batch whose requests ask for different filters; bf16 logits, so many are equal
        {"name": "sample_64", "kind": "sample", "rows": 64, "ties": True},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(lo * (hi / lo) ** rng.random())))


def draw(rng):
    kind = rng.choice(["append", "attend", "attend", "attend", "fork", "compact", "sample"])
    heads = rng.choice([32, 32, 32, 16, 64])
    if kind == "append":
        seqs = rng.randint(1, 16)
        return {"kind": kind, "seqs": seqs, "rows": _log(rng, 1, 6000 // seqs),
                "ctx": _log(rng, 8, 6000), "heads": heads, "norm": rng.random() < 0.5}
    if kind == "attend":
        seqs = _log(rng, 1, 32)
        rows = 1 if rng.random() < 0.4 else _log(rng, 2, 6000 // seqs)
        case = {"kind": kind, "seqs": seqs, "rows": rows, "ctx": _log(rng, 8, 60000),
                "heads": heads, "sinks": rng.choice([0, 1, 4, 16, 64, 100]),
                "window": 16384 if seqs <= 4 and rng.random() < 0.5 else _log(rng, 64, 4096)}
        while work(case)["flops"] > 5e11:     # the largest listed case's
            case["rows"] //= 2
        return case
    if kind == "fork":
        return {"kind": kind, "forks": rng.randint(1, 16), "ctx": _log(rng, 3, 5100)}
    if kind == "compact":
        return {"kind": kind, "seqs": rng.randint(2, 8), "ctx": _log(rng, 130, 4000),
                "window": rng.choice([_log(rng, 64, 2048), EVERYTHING]),
                "sinks": rng.choice([0, 4, 64])}
    return {"kind": kind, "rows": _log(rng, 1, 64), "ties": rng.random() < 0.5}


def _batch(case):
    """(positions before the new tokens, new tokens) of each sequence: the first has the case's
    ctx and rows, the others between an eighth of the one and all of it, and 1 to the other."""
    r = random.Random(case["seqs"] * 1000003 + case["ctx"] * 17 + case["rows"])
    start = [r.randint(case["ctx"] // 8, case["ctx"]) for _ in range(case["seqs"])]
    new = [r.randint(1, case["rows"]) for _ in range(case["seqs"])]
    start[0], new[0] = case["ctx"], case["rows"]
    return start, new


def _compact_lens(case):
    """The rows' lengths; every fourth row's sequence is over."""
    r = random.Random(case["seqs"] * 1000003 + case["ctx"])
    lens = [r.randint(case["ctx"] // 8, case["ctx"]) for _ in range(case["seqs"])]
    lens[0] = case["ctx"]
    return [0 if b % 4 == 1 else n for b, n in enumerate(lens)]


def _blocks_kept(n, window, sinks):
    """The position blocks that a sequence of n positions still needs for its next token."""
    return [i for i in range(-(-n // PAGE)) if i * PAGE < sinks or (i + 1) * PAGE > n - window + 1]


def _filters(rows):
    """Requests' settings by row: (temperature, top_k, top_p, min_p)."""
    kinds = [(0.7, 50, 0.9, 0.0), (1.0, 0, 0.95, 0.0), (0.8, 40, 1.0, 0.05), (1.2, 0, 1.0, 0.02),
             (0.6, 200, 0.8, 0.01), (0.0, 0, 1.0, 0.0), (1.0, 0, 1.0, 0.0), (0.9, 1000, 0.5, 0.0)]
    return [kinds[r % len(kinds)] for r in range(rows)]


def _visible(p, window, sinks):
    """Keys that the row at position p sees."""
    first = max(0, p - window + 1)
    return p + 1 - first + min(first, sinks)


def work(case):
    k = case["kind"]
    if k == "append":
        rows, heads = sum(_batch(case)[1]), case["heads"]
        return {"bytes": rows * (2 * (heads + 2 * KVH) * D * 2 + 2 * 4 * D // 2),
                "flops": rows * (heads + KVH) * D * (7 if case["norm"] else 3)}
    if k == "attend":
        w, s, heads = case["window"], case["sinks"], case["heads"]
        keys = flops = rows = 0
        for start, new in zip(*_batch(case)):
            first = max(0, start - w + 1)     # the oldest key that the first new row sees
            keys += start + new - first + min(first, s)
            flops += 4 * heads * D * sum(_visible(p, w, s) for p in range(start, start + new))
            rows += new
        return {"bytes": keys * 2 * KVH * D * 2 + 2 * rows * heads * D * 2, "flops": flops}
    if k == "fork":
        part, pages = case["ctx"] % PAGE, -(-case["ctx"] // PAGE)
        return {"bytes": (case["forks"] + 1) * (part * LAYERS * 2 * KVH * D * 2 + 4 * pages),
                "flops": case["forks"] * pages}
    if k == "compact":
        lens, table = _compact_lens(case), _compact_table(case)
        live, moved = _plan(case, lens, table)[:2]
        entries = len(table) * len(table[0])
        return {"bytes": moved * 2 * LAYERS * 2 * KVH * PAGE * D * 2 + 8 * entries,
                "flops": entries}
    # the logits are read once; a few operations each
    return {"bytes": case["rows"] * V * 4, "flops": case["rows"] * V * 10}


# ------------------------------------------------------------------------------- inputs
def _compact_table(case):
    """Block tables (host) over a pool half as large again as the sequences need."""
    r = random.Random(case["seqs"] * 7919 + case["ctx"])
    lens = _compact_lens(case)
    # a sequence that is over still holds its pages
    need = [-(-(n or case["ctx"] // 2) // PAGE) for n in lens]
    ids = r.sample(range(_compact_pages(case)), sum(need))
    stride, at, table = max(need), 0, []
    for n in need:
        table.append(ids[at:at + n] + [-1] * (stride - n))
        at += n
    return table


def _compact_pages(case):
    need = sum(-(-(n or case["ctx"] // 2) // PAGE) for n in _compact_lens(case))
    return need + need // 2 + 1


def _plan(case, lens, table):
    """(live pages, moved pages, old page -> new page) of a compaction, on the host."""
    live = set()
    for row, n in zip(table, lens):
        kept = set(_blocks_kept(n, case["window"], case["sinks"]))
        past = -(-n // PAGE)
        live |= {p for i, p in enumerate(row) if p >= 0 and n > 0 and (i in kept or i >= past)}
    n = len(live)
    holes = iter(i for i in range(n) if i not in live)
    move = {p: next(holes) for p in sorted(live) if p >= n}
    return n, len(move), {p: move.get(p, p) for p in live}


class _Gen:
    """Seeded tensors on the GPU."""

    def __init__(self, seed):
        self.g = torch.Generator(device="cuda").manual_seed(seed)

    def bf16(self, *shape, mean=0.0, std=1.0):
        return torch.empty(*shape, dtype=torch.bfloat16, device="cuda").normal_(
            mean, std, generator=self.g)


@functools.cache
def _rope():
    """fp32 tables [131072][64] of the angles pos * 500000^(-j/64)."""
    freq = 500000.0 ** (-torch.arange(64, device="cuda", dtype=torch.float64) / 64)
    angle = torch.arange(MAX_LONG, device="cuda", dtype=torch.float64)[:, None] * freq
    return angle.cos().float(), angle.sin().float()


def _pool(n_pages):
    return torch.zeros(n_pages, LAYERS, 2, KVH, PAGE, D, dtype=torch.bfloat16, device="cuda")


def _tables(g, blocks, stride):
    """A shuffled pool for sequences that hold the given position blocks: (pages, tables)."""
    n = sum(len(b) for b in blocks)
    order = torch.randperm(n, device="cuda", generator=g.g).to(torch.int32)
    table = torch.full((len(blocks), stride), -1, dtype=torch.int32, device="cuda")
    at = 0
    for b, kept in enumerate(blocks):
        table[b, torch.tensor(kept, device="cuda", dtype=torch.long)] = order[at:at + len(kept)]
        at += len(kept)
    return n, table


def _ints(values):
    """The lengths as the call takes them."""
    if not own:
        return list(values)
    import ctypes
    return (ctypes.c_int * len(values))(*values)


@functools.cache
def _stream():
    return torch.cuda.Stream(0)


def _context():
    from infengine_amd.engine import Context
    return Context(0, stream=_stream())


def prepare(case, seed):
    k = case["kind"]
    ctx = _context() if own else None   # (makes its stream torch's current one)
    g = _Gen(seed)
    s = {"kind": k, "ctx": ctx, "case": case}
    ws = 0
    if k in ("append", "attend"):
        start, new = _batch(case)
        s["start"], s["new"], s["seqs"] = _ints(start), _ints(new), len(start)
        rows, heads = sum(new), case["heads"]
        stride = max(-(-(a + n) // PAGE) for a, n in zip(start, new))
    if k == "append":
        # the blocks that the new rows fall into (the older ones are not touched)
        n, s["tables"] = _tables(g, [range(a // PAGE, -(-(a + n) // PAGE))
                                     for a, n in zip(start, new)], stride)
        s["pool"] = _pool(n)
        s["pool"][:, LAYER] = g.bf16(n, 2, KVH, PAGE, D, std=KV_STD)
        s["qkv"] = g.bf16(rows, (heads + 2 * KVH) * D, std=KV_STD)
        s["wq"] = g.bf16(D, mean=1.0, std=0.1) if case["norm"] else None
        s["wk"] = g.bf16(D, mean=1.0, std=0.1) if case["norm"] else None
        s["cos"], s["sin"] = _rope()
        s["q"] = torch.empty(rows, heads, D, dtype=torch.bfloat16, device="cuda")
    elif k == "attend":
        # pages behind the window of a sequence's first new row are gone
        blocks = []
        for a, n in zip(start, new):
            kept = set(_blocks_kept(a, case["window"], case["sinks"]))
            blocks.append([i for i in range(-(-(a + n) // PAGE)) if i in kept or i >= a // PAGE])
        n, s["tables"] = _tables(g, blocks, stride)
        s["pool"] = _pool(n)
        s["pool"][:, LAYER] = g.bf16(n, 2, KVH, PAGE, D, std=KV_STD)
        s["q"] = g.bf16(rows, heads, D, std=KV_STD)
        s["out"] = torch.empty(rows, heads, D, dtype=torch.bfloat16, device="cuda")
        if own:
            from infengine_amd import lib
            ws = lib.ie_attn_window_workspace_size(rows, heads)
    elif k == "fork":
        n, forks = case["ctx"], case["forks"]
        pages = -(-n // PAGE)
        order = torch.randperm(pages + forks, generator=g.g, device="cuda").to(torch.int32)
        s["pool"] = _pool(pages + forks)
        s["pool"].normal_(0.0, KV_STD, generator=g.g)
        s["tables"] = torch.full((forks + 1, pages + 2), -1, dtype=torch.int32, device="cuda")
        s["tables"][0, :pages] = order[:pages]
        s["src"], s["dst"] = _ints([0] * forks), _ints(range(1, forks + 1))
        s["n_pos"], s["fresh"] = _ints([n] * forks), _ints(order[pages:].tolist())
    elif k == "compact":
        s["lens"], n = _ints(_compact_lens(case)), _compact_pages(case)
        s["tables"] = torch.tensor(_compact_table(case), dtype=torch.int32, device="cuda")
        s["pool"] = _pool(n).normal_(0.0, KV_STD, generator=g.g)
        s["new_tables"] = torch.empty_like(s["tables"])
        s["remap"] = torch.empty(n, dtype=torch.int32, device="cuda")
        s["counts"] = torch.empty(2, dtype=torch.int32, device="cuda")
        if own:
            from infengine_amd import lib
            ws = lib.ie_kv_compact_workspace_size(n)
    else:
        r = case["rows"]
        # a bulk of unlikely tokens and a few hundred that stand out
        logits = torch.empty(r, V, device="cuda").normal_(0.0, 2.0, generator=g.g)
        head = torch.randint(0, V, (r, 300), device="cuda", generator=g.g)
        logits.scatter_add_(1, head, torch.empty(r, 300, device="cuda").exponential_(
            0.4, generator=g.g))
        s["logits"] = logits.bfloat16().float() if case["ties"] else logits
        t, kk, p, m = zip(*_filters(r))
        s["t"], s["p"], s["m"] = (torch.tensor(x, dtype=torch.float32, device="cuda")
                                  for x in (t, p, m))
        s["k"] = torch.tensor(kk, dtype=torch.int32, device="cuda")
        s["u"] = torch.rand(r, device="cuda", generator=g.g)
        s["token"] = torch.empty(r, dtype=torch.int32, device="cuda")
        if own:
            from infengine_amd import lib
            ws = lib.ie_sample_filtered_workspace_size(r, V)
    s["ws"] = torch.empty(max(ws, 16), dtype=torch.uint8, device="cuda") if own else None
    return s


# ------------------------------------------------------------------------------- one pass
def run(s):
    return (_run_own if own else _run_plain)(s)


def _run_own(s):
    from infengine_amd import check, lib
    from infengine_amd.engine import ptr
    k, c, h = s["kind"], s["case"], s["ctx"].handle
    if k == "append":
        check(lib.ie_qk_norm_rope_paged(
            h, s["seqs"], s["start"], s["new"], c["heads"], ptr(s["qkv"]), s["qkv"].shape[1],
            ptr(s["wq"]), ptr(s["wk"]), ptr(s["cos"]), ptr(s["sin"]), MAX_LONG, ptr(s["q"]),
            ptr(s["pool"]), s["pool"].shape[0], ptr(s["tables"]), s["tables"].shape[1], LAYER))
        return {"q": s["q"], "pool": s["pool"]}
    if k == "attend":
        check(lib.ie_attn_window_paged(
            h, s["seqs"], s["start"], s["new"], c["window"], c["sinks"], c["heads"], ptr(s["q"]),
            ptr(s["pool"]), s["pool"].shape[0], ptr(s["tables"]), s["tables"].shape[1], LAYER,
            ptr(s["out"]), ptr(s["ws"])))
        return s["out"]
    if k == "fork":
        check(lib.ie_kv_fork_paged(
            h, c["forks"], s["src"], s["dst"], s["n_pos"], s["fresh"], ptr(s["pool"]),
            s["pool"].shape[0], ptr(s["tables"]), s["tables"].shape[0], s["tables"].shape[1]))
        return {"pool": s["pool"], "tables": s["tables"]}
    if k == "compact":
        check(lib.ie_kv_compact_paged(
            h, len(s["lens"]), s["lens"], c["window"], c["sinks"], ptr(s["pool"]),
            s["pool"].shape[0], ptr(s["tables"]), s["tables"].shape[1], ptr(s["new_tables"]),
            ptr(s["remap"]), ptr(s["counts"]), ptr(s["ws"])))
        return {"pool": s["pool"], "tables": s["new_tables"], "remap": s["remap"],
                "counts": s["counts"]}
    check(lib.ie_sample_filtered(h, c["rows"], V, ptr(s["logits"]), ptr(s["t"]), ptr(s["k"]),
                                 ptr(s["p"]), ptr(s["m"]), ptr(s["u"]), ptr(s["token"]),
                                 ptr(s["ws"])))
    return s["token"]


def _rows_of(s):
    """(sequence, position) of every new row, in the rows' order."""
    seq = torch.cat([torch.full((n,), b, device="cuda") for b, n in enumerate(s["new"])])
    pos = torch.cat([torch.arange(a, a + n, device="cuda") for a, n in zip(s["start"], s["new"])])
    return seq, pos


def _run_plain(s):
    return {"append": _append, "attend": _attend, "fork": _fork, "compact": _compact,
            "sample": _sample}[s["kind"]](s)


def _append(s):
    heads = s["case"]["heads"]
    seq, pos = _rows_of(s)
    x = s["qkv"].view(-1, heads + 2 * KVH, D)
    cos, sin = s["cos"][pos][:, None], s["sin"][pos][:, None]

    def turn(v, w):
        v = v.float()
        if w is not None:
            v = v * torch.rsqrt(v.square().mean(-1, keepdim=True) + EPS) * w.float()
        a, b = v[..., :64], v[..., 64:]
        return torch.cat([a * cos - b * sin, a * sin + b * cos], dim=-1).bfloat16()

    s["q"].copy_(turn(x[:, :heads], s["wq"]))
    page = s["tables"][seq, pos // PAGE].long()
    s["pool"][page, LAYER, 0, :, pos % PAGE] = turn(x[:, heads:heads + KVH], s["wk"])
    s["pool"][page, LAYER, 1, :, pos % PAGE] = x[:, heads + KVH:]
    return {"q": s["q"], "pool": s["pool"]}


def _attend(s):
    c = s["case"]
    group, w, sinks = c["heads"] // KVH, c["window"], c["sinks"]
    row = 0
    for b, (a, n) in enumerate(zip(s["start"], s["new"])):
        for p0 in range(a, a + n, 512):          # 512 rows at a time
            p1 = min(p0 + 512, a + n)
            first = max(0, p0 - w + 1)
            j = torch.cat([torch.arange(0, min(first, sinks), device="cuda"),
                           torch.arange(first, p1, device="cuda")])
            page = s["tables"][b, j // PAGE].long()
            kv = s["pool"][page, LAYER, :, :, j % PAGE].float()     # [keys][K|V][8][128]
            p = torch.arange(p0, p1, device="cuda")[:, None]
            hidden = (j > p) | ((j <= p - w) & (j >= sinks))
            q = s["q"][row:row + p1 - p0].float().view(-1, KVH, group, D)
            for g in range(KVH):
                key, value = kv[:, 0, g].t().contiguous(), kv[:, 1, g].contiguous()
                for h in range(group):
                    sc = (q[:, g, h] @ key) * D ** -0.5
                    sc.masked_fill_(hidden, float("-inf"))
                    e = (sc - sc.amax(-1, keepdim=True)).exp()
                    s["out"][row:row + p1 - p0, g * group + h] = (
                        (e @ value) / e.sum(-1, keepdim=True)).bfloat16()
            row += p1 - p0
    return s["out"]


def _fork(s):
    t = s["tables"]
    for a, b, n, page in zip(s["src"], s["dst"], s["n_pos"], s["fresh"]):
        full, part = n // PAGE, n % PAGE
        t[b] = -1
        t[b, :full] = t[a, :full]
        if part:
            s["pool"][page, :, :, :, :part] = s["pool"][t[a, full].long(), :, :, :, :part]
            t[b, full] = page
    return {"pool": s["pool"], "tables": t}


def _compact(s):
    c, t, n = s["case"], s["tables"], s["pool"].shape[0]
    lens = torch.tensor(s["lens"], device="cuda")[:, None]
    i = torch.arange(t.shape[1], device="cuda")[None]
    past = (lens + PAGE - 1) // PAGE
    keep = (i * PAGE < c["sinks"]) | ((i + 1) * PAGE > lens - c["window"] + 1) | (i >= past)
    keep &= (lens > 0) & (t >= 0) & (t < n)
    live = torch.zeros(n, dtype=torch.bool, device="cuda")
    live[t[keep].long()] = True
    count = int(live.sum())
    page = torch.arange(n, device="cuda")
    moved, holes = page[live & (page >= count)], page[~live & (page < count)]
    remap = torch.where(live, page, -1)
    remap[moved] = holes
    s["pool"][holes] = s["pool"][moved]
    s["remap"].copy_(remap)
    s["new_tables"].copy_(torch.where(keep, remap[t.clamp(0, n - 1).long()], -1))
    s["counts"].copy_(torch.stack([live.sum(), (live & (page >= count)).sum()]))
    return {"pool": s["pool"], "tables": s["new_tables"], "remap": s["remap"],
            "counts": s["counts"]}


def _sample(s):
    """In 64 bits: a draw may fall next to a border of the cumulative distribution."""
    l = s["logits"].double()
    r, n = l.shape
    greedy = (s["t"] <= 0)[:, None]
    t = torch.where(greedy, 1.0, s["t"][:, None].double())
    order = torch.sort(l, dim=1, descending=True, stable=True).indices
    w = ((l.gather(1, order) - l.amax(1, keepdim=True)) / t).exp()
    rank = torch.arange(n, device="cuda")[None]
    k = torch.where(s["k"] > 0, s["k"], n)[:, None]
    k = torch.where(greedy, 1, k)
    w = torch.where(rank < k, w, 0.0)
    cum = w.cumsum(1)
    # a token is in the shortest prefix with the mass as long as the prefix before it lacks it
    p = s["p"][:, None].double()
    keep = (rank < k) & ((p >= 1) | (cum - w < p * cum[:, -1:])) & (w >= s["m"][:, None].double())
    keep |= rank == 0
    mass = torch.zeros_like(l).scatter_(1, order, torch.where(keep, w, 0.0)).cumsum(1)
    target = mass[:, -1:] * s["u"][:, None].double()
    s["token"].copy_((mass > target).int().argmax(1))
    return s["token"]


# ------------------------------------------------------------------------------- 64 bits
def exact(case, seed):
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    k = s["kind"]
    if k == "append":
        return _append64(s, case)
    if k == "attend":
        return _attend64(s, case)
    if k == "fork":
        return _fork64(s)
    if k == "compact":
        return _compact64(s, case)
    return _sample64(s)


def _append64(s, case):
    """Row by row of the batch as complex numbers: the pair (x_j, x_{j+64}) turned by the angle."""
    heads, pool = case["heads"], s["pool"].clone()
    x, out, row = s["qkv"].view(-1, heads + 2 * KVH, D), [], 0
    table = s["tables"].tolist()
    for b, (a, n) in enumerate(zip(s["start"], s["new"])):
        v = x[row:row + n].double()
        turn = torch.complex(s["cos"][a:a + n].double(), s["sin"][a:a + n].double())[:, None]
        parts = []
        for y, w in ((v[:, :heads], s["wq"]), (v[:, heads:heads + KVH], s["wk"])):
            if w is not None:
                y = w.double() * y / torch.sqrt((y * y).sum(-1, keepdim=True) / D + EPS)
            z = torch.complex(y[..., :64].contiguous(), y[..., 64:].contiguous()) * turn
            parts.append(torch.cat([z.real, z.imag], dim=-1))
        out.append(parts[0])
        if not row:
            pool = pool.double()
        for first in range(a // PAGE * PAGE, a + n, PAGE):
            lo, hi = max(first, a), min(first + PAGE, a + n)
            page = pool[table[b][first // PAGE], LAYER, :, :, lo - first:hi - first]
            page[0] = parts[1][lo - a:hi - a].transpose(0, 1)
            page[1] = v[lo - a:hi - a, heads + KVH:].transpose(0, 1)
        row += n
    return {"q": torch.cat(out), "pool": pool}


def _attend64(s, case):
    """Over the dense keys of each sequence that are in a page, by the definition's mask."""
    group, out, row = case["heads"] // KVH, torch.empty_like(s["q"], dtype=torch.float64), 0
    for b, (a, n) in enumerate(zip(s["start"], s["new"])):
        page = s["tables"][b].long()
        held = (page >= 0).nonzero()[:, 0]
        j = (held[:, None] * PAGE + torch.arange(PAGE, device="cuda")).reshape(-1)
        kv = s["pool"][page[held], LAYER].permute(1, 2, 0, 3, 4).reshape(2, KVH, -1, D)
        kv = kv[:, :, j < a + n].double()
        j = j[j < a + n]
        for r0 in range(0, n, 1024):
            r1 = min(n, r0 + 1024)
            p = torch.arange(a + r0, a + r1, device="cuda")[:, None]
            seen = (j <= p) & ((p - j < case["window"]) | (j < case["sinks"]))
            for h in range(case["heads"]):
                q = s["q"][row + r0:row + r1, h].double()
                sc = torch.where(seen, (q @ kv[0, h // group].t()) / D ** 0.5, float("-inf"))
                out[row + r0:row + r1, h] = torch.softmax(sc, dim=-1) @ kv[1, h // group]
        row += n
    return out


def _fork64(s):
    """The pool and tables written on the host's list of copies (the values as they stand)."""
    pool, table = s["pool"].clone(), s["tables"].tolist()
    for a, b, n, page in zip(s["src"], s["dst"], s["n_pos"], s["fresh"]):
        row = [table[a][i] if (i + 1) * PAGE <= n else -1 for i in range(len(table[b]))]
        if n % PAGE:
            for pos in range(n % PAGE):
                pool[page, :, :, :, pos] = pool[table[a][n // PAGE], :, :, :, pos]
            row[n // PAGE] = page
        table[b] = row
    return {"pool": pool, "tables": torch.tensor(table, dtype=torch.int32, device="cuda")}


def _compact64(s, case):
    """By the host's plan."""
    table, lens, pool = s["tables"].tolist(), list(s["lens"]), s["pool"].clone()
    live, moved, remap = _plan(case, lens, table)
    for old, new in remap.items():
        if old != new:
            pool[new] = s["pool"][old]
    rows = []
    for row, n in zip(table, lens):
        kept, past = set(_blocks_kept(n, case["window"], case["sinks"])), -(-n // PAGE)
        rows.append([remap[p] if n and p >= 0 and (i in kept or i >= past) else -1
                     for i, p in enumerate(row)])
    as_ints = functools.partial(torch.tensor, dtype=torch.int32, device="cuda")
    return {"pool": pool, "tables": as_ints(rows),
            "remap": as_ints([remap.get(p, -1) for p in range(pool.shape[0])]),
            "counts": as_ints([live, moved])}


def _sample64(s):
    """Row by row on the host: the sorted order walked to the cut, the ids walked to the draw."""
    import numpy as np
    tokens = []
    rows = zip(s["logits"].cpu().numpy().astype(np.float64), s["t"].tolist(), s["k"].tolist(),
               s["p"].tolist(), s["m"].tolist(), s["u"].tolist())
    for l, t, k, p, m, u in rows:
        order = np.lexsort((np.arange(l.size), -l))
        if t <= 0:
            tokens.append(int(order[0]))
            continue
        w = np.exp((l[order] - l[order[0]]) / t)
        kept = order.size if k <= 0 else min(k, order.size)
        w = w[:kept]
        if p < 1:
            kept = min(kept, int(np.searchsorted(np.cumsum(w), p * w.sum())) + 1)
        kept = max(1, min(kept, int((w >= m).sum())))
        ids = np.sort(order[:kept])
        cum = np.cumsum(np.exp((l[ids] - l[order[0]]) / t))
        tokens.append(int(ids[min(np.searchsorted(cum, u * cum[-1], side="right"), kept - 1)]))
    return torch.tensor(tokens, dtype=torch.int32, device="cuda")
