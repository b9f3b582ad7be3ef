"""The operators of a step that serves many requests at once, each with an adapter and a way of sampling of its own.

"group": the step's rows by the adapter of their request, the order the products below go by.  "adapters": low-rank
adapters beside a shared projection, out = base + scale_a B_a (A_a x) with a row's own adapter a, for single tokens
(a row a request) and for prompts (the rows of several requests, each in one piece).  "sample": a token a request
from the logits, with its own temperature, top-k, top-p, min-p and given random number.

Projections have the sizes of Qwen3-8B, width 4,096: the stacked q | k | v (4,096 + 1,024 + 1,024 columns, an
adapter each), gate and up (2 x 12,288, woven column by column), down (12,288 to 4,096); the vocabulary is 151,936.
"""

import math

import torch

own = False
DEVICE = "cuda:0"
WIDTHS = (64, 999, 1000, 1024, 2048, 2560, 4096, 5120, 8192, 12288)
KINDS = {"qkv": 3, "gate_up": 2, "one": 1}


def listed():
    def group(name, rows, adapters, seqs):
        return dict(name=name, op="group", rows=rows, adapters=adapters, seqs=seqs)

    def adapters(name, rows, seqs, kind, width, cols, rank, count, bare, dtype="bf16", out="bf16", mixed=False):
        return dict(name=name, op="adapters", rows=rows, seqs=seqs, kind=kind, width=width, cols=cols, rank=rank,
                    adapters=count, bare=bare, dtype=dtype, out=out, mixed=mixed)

    def sample(name, rows, vocab, cuts, spread, masked=0.0):
        return dict(name=name, op="sample", rows=rows, vocab=vocab, cuts=cuts, spread=spread, masked=masked)

    return [
        # the rows of a decode step of 64 requests over 32 resident adapters: the smallest call
        group("group_step_b64", 64, 32, 64),
        # prompts of many requests packed together, hundreds of adapters resident
        group("group_prompts", 16384, 500, 48),
        # one request decoding through the stacked q | k | v: latency
        adapters("qkv_step_b1", 1, 1, "qkv", 4096, 4096, 16, 4, 0.0, out="f32"),
        # a full batch, half of the requests on adapters of their own, ranks 8 to 64
        adapters("qkv_step_b64", 64, 64, "qkv", 4096, 4096, 64, 32, 0.15, out="f32", mixed=True),
        # eight requests through the woven gate and up: the widest projection
        adapters("gate_up_step_b8", 8, 8, "gate_up", 4096, 12288, 16, 8, 0.0),
        # prompts of five requests through the down projection
        adapters("down_prompts", 2047, 5, "one", 12288, 4096, 32, 4, 0.1),
        # long prompts through q | k | v, large ranks: the most work
        adapters("qkv_prompts", 8192, 9, "qkv", 4096, 4096, 64, 8, 0.1),
        # the true 32-bit path on a few unequal prompts
        adapters("one_prompts_f32", 701, 3, "one", 1024, 2048, 16, 3, 0.0, dtype="f32", out="f32"),
        # one request, a nucleus of a peaked distribution
        sample("sample_b1", 1, 151936, "top_p", 3.0),
        # a full batch in which every request has its own cuts, some are greedy and a grammar masks some logits
        sample("sample_mixed_b64", 64, 151936, "mixed", 2.5, masked=0.3),
        # no cut at all: every probability of the row counts
        sample("sample_plain_b8", 8, 151936, "none", 1.5),
        # many short rows of an odd vocabulary, flat: cuts deep in the row
        sample("sample_flat_b256", 256, 32003, "all", 1.0),
    ]


def draw(rng):
    def spread(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(("group", "adapters", "adapters", "adapters", "sample", "sample"))
    if op == "group":
        rows = spread(1, 16384)
        return dict(op=op, rows=rows, adapters=spread(1, 500), seqs=rng.choice((rows, max(1, min(rows, spread(1, 64))))))
    if op == "sample":
        rows = spread(1, 256)
        return dict(op=op, rows=rows, vocab=spread(1, min(262144, 9700000 // rows)),
                    cuts=rng.choice(("none", "top_k", "top_p", "min_p", "all", "mixed")),
                    spread=rng.choice((0.5, 1.0, 2.0, 3.0, 5.0)), masked=rng.choice((0.0, 0.0, 0.5, 0.99)))
    kind = rng.choice(("qkv", "gate_up", "one"))
    steps = rng.random() < 0.5
    f32 = rng.random() < 0.25
    rows = spread(1, 256) if steps else spread(17, 1024 if f32 else 8192)
    width = rng.choice(WIDTHS[:6] if f32 else WIDTHS if rows <= 2048 else WIDTHS[:7])
    rank, count = spread(1, 16 if f32 else 64), spread(1, 16)
    cols = spread(1, min(24576, 40000000 // rows) // KINDS[kind])
    if rng.random() < 0.7:
        cols = (cols + 63) // 64 * 64
    return dict(op=op, rows=rows, seqs=rows if steps else min(rows // 8, rng.choice((1, 2, 3, 5, 9))), kind=kind,
                width=width, cols=cols, rank=rank, adapters=count, bare=rng.choice((0.0, 0.1, 0.5)),
                dtype="f32" if f32 else "bf16", out="f32" if f32 or (steps and rows <= 64) else "bf16",
                mixed=rng.random() < 0.5)


def _parts(case):
    """The columns of the projection's parts, an adapter's A each: q | k | v, gate and up (woven), or one."""
    c = case["cols"]
    return {"qkv": (c, max(1, c // 4), max(1, c // 4)), "gate_up": (c, c), "one": (c,)}[case["kind"]]


def _dtype(name):
    return torch.float32 if name == "f32" else torch.bfloat16


def _ids(case, gen):
    """Each row's adapter, int32, -1 for none: `seqs` requests in pieces of unequal length."""
    rows, seqs, n = case["rows"], case["seqs"], case["adapters"]
    of_seq = torch.randint(0, n, (seqs,), generator=gen, device=DEVICE)
    bare = torch.rand((seqs,), generator=gen, device=DEVICE) < case.get("bare", 0.1)
    of_seq = torch.where(bare, -1, of_seq)
    starts = torch.rand((rows,), generator=gen, device=DEVICE).argsort()[:seqs].sort().values
    marks = torch.zeros((rows,), dtype=torch.int64, device=DEVICE)
    marks[starts] = 1
    return of_seq[(marks.cumsum(0) - 1).clamp_min(0)].to(torch.int32)


def _tile(rows):
    """Rows of one adapter that a product takes together."""
    return 16 if rows <= 256 else 128


def _grouped(ids, n, tile):
    """(order, first, tiles): the rows by adapter, in order within one, those without an adapter last (as adapter
    `n`); where each adapter's begin; and the groups cut into tiles of at most `tile` rows: (adapter, place, rows),
    -1, 0, 0 behind the last."""
    rows = ids.numel()
    key = torch.where((ids < 0) | (ids >= n), n, ids).long()
    order = key.sort(stable=True).indices
    counts = (key[None, :] == torch.arange(n + 1, device=ids.device)[:, None]).sum(1)
    first = torch.cat([counts.new_zeros(1), counts.cumsum(0)])
    per = (counts + tile - 1) // tile
    ends = per.cumsum(0)
    t = torch.arange(min(rows, n + 1) + rows // tile, device=ids.device)
    a = torch.searchsorted(ends, t, right=True)
    have, a = a <= n, a.clamp_max(n)
    place = first[a] + (t - (ends - per)[a]) * tile
    count = (first[a + 1] - place).clamp_max(tile)
    tiles = torch.stack([torch.where(have, a, -1), torch.where(have, place, 0), torch.where(have, count, 0)], 1)
    return order.to(torch.int32), first.to(torch.int32), tiles.to(torch.int32)


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE)
    gen.manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, generator=gen, device=DEVICE)

    def uniform(*shape):
        return torch.rand(shape, generator=gen, device=DEVICE)

    if case["op"] == "group":
        return dict(case=case, ids=_ids(case, gen))
    if case["op"] == "sample":
        rows, vocab = case["rows"], case["vocab"]
        logits = normal(rows, vocab) * case["spread"]
        # a few likely tokens above the rest, as a trained head gives
        if vocab >= 64:
            likely = ((torch.arange(12, device=DEVICE) + uniform(rows, 12)) / 12 * vocab).long().clamp_max(vocab - 1)
            logits.scatter_add_(1, likely, uniform(rows, 12) * 4 * case["spread"])
        if case["masked"]:
            logits = torch.where(uniform(rows, vocab) < case["masked"], -math.inf, logits)
        cuts = case["cuts"]
        some = uniform(4, rows) if cuts == "mixed" else None

        def on(i, value, off):
            return value if some is None else torch.where(some[i] < 0.5, value, off)

        temperature = 0.3 + uniform(rows)
        if cuts == "mixed":
            temperature = torch.where(some[3] < 0.1, 0.0, temperature)
        state = dict(case=case, logits=logits, temperature=temperature, uniform=torch.floor(uniform(rows) * 2 ** 24) / 2 ** 24,
                     top_k=None, top_p=None, min_p=None)
        if cuts in ("top_k", "all", "mixed"):
            state["top_k"] = on(0, (torch.exp(uniform(rows) * math.log(500)) + 0.5).to(torch.int32), 0).to(torch.int32)
        if cuts in ("top_p", "all", "mixed"):
            state["top_p"] = on(1, 0.5 + 0.5 * uniform(rows), 1.0)
        if cuts in ("min_p", "all", "mixed"):
            state["min_p"] = on(2, 0.2 * uniform(rows) ** 2, 0.0)
        return state
    rows, width, rank, n = (case[k] for k in ("rows", "width", "rank", "adapters"))
    parts, dtype = _parts(case), _dtype(case["dtype"])
    ids = _ids(case, gen)
    ranks = torch.full((n,), rank, dtype=torch.int32, device=DEVICE)
    if case["mixed"]:
        ranks = (rank / 2 ** torch.randint(0, 4, (n,), generator=gen, device=DEVICE)).ceil().to(torch.int32)
    used = (torch.arange(rank, device=DEVICE) < ranks[:, None]).float()
    a = normal(n, len(parts), rank, width) * width ** -0.5 * used[:, None, :, None]
    b = normal(n, sum(parts), rank) * rank ** -0.5 * used[:, None, :]
    state = dict(case=case, ids=ids, x=normal(rows, width).to(dtype), base=normal(rows, sum(parts)).to(_dtype(case["out"])),
                 a=a.to(dtype), b=b.to(dtype), scale=0.5 + uniform(n), ranks=ranks)
    tile = _tile(rows)
    state["grouped"] = _grouped(ids, n, tile)
    if own:  # the handles that a program keeps: the adapters as they were loaded, the step's rows as they were grouped
        from reflex_b200 import ops

        state["bank"] = ops.AdapterBank(state["a"], state["b"], state["scale"], parts, woven=case["kind"] == "gate_up",
                                        ranks=ranks)
        state["grouped"] = ops.AdapterRows(*state["grouped"], tile)
    return state


def run(state):
    return {"group": _run_group, "adapters": _run_adapters, "sample": _run_sample}[state["case"]["op"]](state)


def _run_group(state):
    case = state["case"]
    if own:
        from reflex_b200 import ops

        g = ops.adapter_rows(state["ids"], case["adapters"], _tile(case["rows"]))
        return g.order, g.first, g.tiles
    return _grouped(state["ids"], case["adapters"], _tile(case["rows"]))


def _run_adapters(state):
    if own:
        from reflex_b200 import ops

        return ops.adapter_add(state["base"], state["x"], state["bank"], state["grouped"])
    case, parts = state["case"], _parts(state["case"])
    n, rank = case["adapters"], case["rank"]
    ids = state["ids"]
    # every row against every adapter, and only its own adapter's numbers kept
    mine = (ids[:, None] == torch.arange(n, device=ids.device)) * state["scale"]
    low = state["x"].float() @ state["a"].float().reshape(n * len(parts) * rank, -1).T
    low = low.view(-1, n, len(parts), rank) * mine[:, :, None, None]
    b = state["b"].float()
    edges = [sum(parts[:i]) for i in range(len(parts) + 1)]
    if case["kind"] == "gate_up":  # column 2 j is gate j, column 2 j + 1 up j
        b = torch.cat([b[:, 0::2], b[:, 1::2]], 1)
    delta = [low[:, :, i].reshape(-1, n * rank) @ b[:, edges[i]:edges[i + 1]].transpose(1, 2).reshape(n * rank, -1)
             for i in range(len(parts))]
    delta = torch.stack(delta, 2).flatten(1) if case["kind"] == "gate_up" else torch.cat(delta, 1)
    return (state["base"].float() + delta).to(state["base"].dtype)


def _run_sample(state):
    if own:
        from reflex_b200 import ops

        return ops.sample_rows(state["logits"], state["temperature"], state["uniform"], state["top_k"], state["top_p"],
                               state["min_p"])
    # in 64 bits: a token's place in the running sum decides, and the sums are long
    logits, t = state["logits"].double(), state["temperature"].double()[:, None]
    top = logits.max(1, keepdim=True).values
    e = torch.exp((logits - top) / torch.where(t > 0, t, 1.0))
    e = torch.where(logits == -math.inf, 0.0, e)
    down, order = logits.sort(dim=1, descending=True, stable=True)
    e_down = e.gather(1, order)
    before = e_down.cumsum(1) - e_down
    keep = e_down > 0
    if state["top_k"] is not None:
        k = state["top_k"][:, None]
        keep &= (k <= 0) | (torch.arange(e.shape[1], device=e.device) < k)
    if state["top_p"] is not None:
        p = state["top_p"].double()[:, None]
        keep &= (p >= 1) | (before < p * e.sum(1, keepdim=True))
    if state["min_p"] is not None:
        keep &= e_down >= state["min_p"].double()[:, None]
    keep[:, 0] = True
    kept = torch.zeros_like(e).scatter_(1, order, e_down * keep)
    sums = kept.cumsum(1)
    reached = (sums >= state["uniform"].double()[:, None] * sums[:, -1:]) & (kept > 0)
    tokens = reached.to(torch.int8).argmax(1)
    return torch.where(t[:, 0] > 0, tokens, logits.argmax(1)).to(torch.int32)


def work(case):
    if case["op"] == "group":
        rows, n = case["rows"], case["adapters"]
        return {"bytes": 4 * (2 * rows + n + 2) + 12 * (min(rows, n + 1) + rows // _tile(rows)), "flops": rows}
    if case["op"] == "sample":
        rows = case["rows"]
        cuts = {"none": 0, "top_k": 1, "top_p": 1, "min_p": 1}.get(case["cuts"], 3)
        return {"bytes": 4 * rows * (case["vocab"] + 3 + cuts), "flops": 4 * rows * case["vocab"]}
    rows, width, parts = case["rows"], case["width"], _parts(case)
    size, out = (4 if case["dtype"] == "f32" else 2), (4 if case["out"] == "f32" else 2)
    # the adapters that are met, at the rank that a request of the case has on average
    rank = case["rank"] * (15 / 32 if case["mixed"] else 1.0)
    n, with_one = case["adapters"], case["seqs"] * (1 - case["bare"])
    met = n * (1 - (1 - 1 / n) ** with_one)
    per = rank * (len(parts) * width + sum(parts))
    adapted = rows * (1 - case["bare"])
    return {"bytes": int(adapted * width * size + 2 * rows * sum(parts) * out + met * per * size),
            "flops": int(2 * adapted * per)}


def exact(case, seed):
    if case["op"] != "adapters":
        return None
    state = prepare(case, seed)
    parts = _parts(case)
    out = state["base"].double()
    # the part that a column belongs to
    if case["kind"] == "gate_up":
        part = torch.arange(sum(parts), device=DEVICE) % 2
    else:
        part = torch.repeat_interleave(torch.arange(len(parts), device=DEVICE), torch.tensor(parts, device=DEVICE))
    for i in range(case["adapters"]):
        rows = (state["ids"] == i).nonzero()[:, 0]
        for s in range(len(parts)):
            cols = (part == s).nonzero()[:, 0]
            low = state["x"][rows].double() @ state["a"][i, s].double().T
            delta = low @ state["b"][i][cols].double().T
            out[rows[:, None], cols[None, :]] += state["scale"][i].double() * delta
    return out
