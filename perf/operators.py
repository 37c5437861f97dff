"""The operators of a paged KV cache, as a serving program calls them, and their plain forms.

Such a program keeps the keys and values of its requests in pages of a few rows, [pages][kv heads][page rows][head_dim]
for K and for V, and a table of page numbers per request.  A step of it is three calls:

  "map"     from each request's length and the rows it gains or loses: pages taken from and given back to the free
            ones, the table's new entries, and for every new row its slot (page * page rows + row in the page), its
            position and its request (`PagedKVCache.map_rows`);
  "append"  bias, QK-norm and rotation of the new rows of q, k and v, keys and values into their slots
            (`AttnContext.append_paged`);
  "attend"  attention of one new row per request over its pages (`AttnContext.attend_paged`).

Activations are float32, as everywhere in this framework; pages hold float32, bfloat16 or float16.  Head geometries and
batches are those of the repository's decode and prefill workloads, and generic ones (heads of 80 and 96, seven or sixteen query heads to a kv head).
"""
import math
import random

import numpy as np
import torch

own = False

# query heads, kv heads, head_dim, rope theta, QK-norm, biases
HEADS = {
    "llama1b": (32, 8, 64, 5e5, False, False),
    "qwen3_8b": (32, 8, 128, 1e6, True, False),
    "qwen3_30b": (32, 4, 128, 1e6, True, False),
    "gemma": (16, 8, 256, 1e4, False, False),
    "mha80": (20, 20, 80, 1e4, False, False),
    "gqa7": (28, 4, 96, 1e6, False, True),
    "mqa": (16, 1, 128, 1e4, False, False),
}
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
EPS = 1e-6


def listed():
    return [
        # a decode step of a small batch gains a row per request; the rows are dropped again, as after a refused draft
        {"name": "map_step_b16", "op": "map", "requests": 16, "low": 2048, "high": 8192, "page_rows": 16, "change": "step"},
        # a batch of prompts is admitted and, answered, dropped
        {"name": "map_prompts_b300", "op": "map", "requests": 300, "low": 1, "high": 4000, "page_rows": 32, "change": "admit"},
        # a busy server: some requests end, others begin or go on by a row
        {"name": "map_mixed_b1000", "op": "map", "requests": 1000, "low": 30, "high": 2000, "page_rows": 16, "change": "mixed"},
        # the new rows of a decode step, with QK-norm, into float32 pages
        {"name": "append_b16_f32", "op": "append", "heads": "qwen3_8b", "rows": 16, "far": 8192, "page_rows": 16, "dtype": "f32"},
        # a prompt into bfloat16 pages
        {"name": "append_t2048_bf16", "op": "append", "heads": "llama1b", "rows": 2048, "far": 2048, "page_rows": 16, "dtype": "bf16"},
        # the new rows of an odd batch, far into long contexts, with biases
        {"name": "append_b333_f16", "op": "append", "heads": "gqa7", "rows": 333, "far": 32768, "page_rows": 32, "dtype": "f16"},
        # one user, short context: the smallest call, nothing but latency
        {"name": "attend_b1_ctx1024_f32", "op": "attend", "heads": "llama1b", "requests": 1, "low": 1024, "high": 1024,
         "page_rows": 16, "dtype": "f32"},
        # the same of a wider batch in bfloat16, contexts of a short chat
        {"name": "attend_b24_ctx20-700_bf16", "op": "attend", "heads": "llama1b", "requests": 24, "low": 20, "high": 700,
         "page_rows": 16, "dtype": "bf16"},
        # the serving batch of this repository's headline workload, float32 pages
        {"name": "attend_b16_ctx2048-8192_f32", "op": "attend", "heads": "qwen3_8b", "requests": 16, "low": 2048, "high": 8192,
         "page_rows": 16, "dtype": "f32"},
        # one long document in bfloat16 pages: work only over the keys
        {"name": "attend_b1_ctx131072_bf16", "op": "attend", "heads": "qwen3_30b", "requests": 1, "low": 131072, "high": 131072,
         "page_rows": 64, "dtype": "bf16"},
        # the largest: 64 requests with long contexts in bfloat16 pages
        {"name": "attend_b64_ctx8192-32768_bf16", "op": "attend", "heads": "qwen3_8b", "requests": 64, "low": 8192, "high": 32768,
         "page_rows": 32, "dtype": "bf16"},
        # odd heads, small pages that end inside tiles, float16, requests without a row yet
        {"name": "attend_b77_ctx0-5000_f16", "op": "attend", "heads": "gqa7", "requests": 77, "low": 0, "high": 5000,
         "page_rows": 8, "dtype": "f16"},
    ]


def _spread(rng, low, high):
    """A whole number from low to high, even in its logarithm."""
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def _cost(case):
    w = work(case)
    return max(w["bytes"], w["flops"] / 50)


def draw(rng):
    most = {op: max(_cost(c) for c in listed() if c["op"] == op) for op in ("map", "append", "attend")}
    while True:
        op = rng.choice(["map", "append", "attend", "attend"])
        case = {"op": op}
        if op == "map":
            change = rng.choice(["step", "admit", "mixed"])
            low = _spread(rng, 1, 4096)
            case.update(requests=_spread(rng, 1, 1000), low=low, high=min(8192, low * rng.choice([1, 2, 8])),
                        page_rows=rng.choice([8, 16, 32, 64, 128]), change=change)
        elif op == "append":
            case.update(heads=rng.choice(sorted(HEADS)), rows=_spread(rng, 1, 2048), far=_spread(rng, 16, 32768),
                        page_rows=rng.choice([8, 16, 32, 64, 128]), dtype=rng.choice(sorted(DTYPES)))
        else:
            low = _spread(rng, 1, 131072) - 1
            case.update(heads=rng.choice(sorted(HEADS)), requests=_spread(rng, 1, 128), low=low,
                        high=min(131072, low * rng.choice([1, 2, 4]) + rng.choice([1, 100])),
                        page_rows=rng.choice([8, 16, 32, 64, 128]), dtype=rng.choice(sorted(DTYPES)))
        if _cost(case) <= most[op]:
            return case


# ---- what a pass cannot do without -------------------------------------------------------------

def _lengths(case):
    """Rows of each request: before the step, or those that it is admitted with, or that it attends over."""
    r = random.Random(case["requests"] * 1000003 + case["low"] * 31 + case["high"])
    return [r.randint(case["low"], case["high"]) for _ in range(case["requests"])]


def _changes(case):
    """(length, change) of each request."""
    r, lengths = random.Random(case["requests"] + case["low"]), _lengths(case)
    if case["change"] == "step":
        return [(n, 1) for n in lengths]
    if case["change"] == "admit":
        return [(0, n) for n in lengths]
    kinds = [r.choices(["on", "end", "begin", "idle"], [6, 1, 1, 2])[0] for _ in lengths]
    return [{"on": (n, 1), "end": (n, -n), "begin": (0, n), "idle": (n, 0)}[kind] for n, kind in zip(lengths, kinds)]


def _pages(n, page_rows):
    return (n + page_rows - 1) // page_rows


def work(case):
    if case["op"] == "map":
        # both halves: lengths and changes in, lengths out, moved pages read and written, three numbers out per new row
        total = 0
        for n, d in _changes(case):
            moved = abs(_pages(n + d, case["page_rows"]) - _pages(n, case["page_rows"]))
            total += 4 * (2 * 4 + 2 * 2 * moved + 3 * abs(d))
        return {"bytes": total, "flops": 0}
    H, KV, hd = HEADS[case["heads"]][:3]
    size = 4 if case["dtype"] == "f32" else 2
    if case["op"] == "append":
        rows = case["rows"]
        return {"bytes": rows * (4 * hd * (2 * H + 2 * KV) + 2 * KV * hd * size + 8), "flops": 6 * rows * hd * (H + KV)}
    visible = sum(_lengths(case))
    return {"bytes": 2 * KV * hd * size * visible + 2 * 4 * H * hd * case["requests"], "flops": 4 * H * hd * visible}


# ---- inputs --------------------------------------------------------------------------------------

def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _context(case, weights):
    import shainet_amd as sa

    H, KV, hd, theta, _, _ = HEADS[case["heads"]]
    qn, kn, biases = weights
    host = lambda t: None if t is None else t.cpu().numpy()  # noqa: E731
    ctx = sa.AttnContext(H, KV, hd, rope_theta=theta, q_norm=host(qn), k_norm=host(kn), eps=EPS)
    if biases is not None:
        ctx.set_bias(*(host(b) for b in biases))
    ctx.set_stream(torch.cuda.current_stream().cuda_stream)
    return ctx


def _map_inputs(case, seed):
    rng, P = np.random.default_rng(seed), case["page_rows"]
    changes = _changes(case)
    wide = max(_pages(max(n, n + d), P) for n, d in changes)
    most = sum(_pages(max(n, n + d), P) for n, d in changes)
    n_pages = most + 7
    pages = torch.from_numpy(rng.permutation(n_pages).astype(np.int32)).cuda()
    lens = _ints([n for n, _ in changes])
    counts = _pages(lens, P)
    grid = torch.arange(wide, device="cuda")[None]
    held = grid < counts[:, None]
    starts = torch.cumsum(counts, 0) - counts
    table = torch.where(held, pages[torch.where(held, starts[:, None] + grid, 0).long()], -1).to(torch.int32)
    used = int(counts.sum())
    free = torch.full((n_pages,), -1, dtype=torch.int32, device="cuda")
    free[:n_pages - used] = pages[used:]
    order = torch.from_numpy(rng.permutation(len(changes)).astype(np.int32)).cuda()  # requests in the scheduler's order
    delta = _ints([d for _, d in changes])[order.long()].contiguous()
    rows = [sum(max(0, s * d) for _, d in changes) for s in (1, -1)]
    s = {"page_rows": P, "n_pages": n_pages, "table": table, "lens": lens, "free": free,
         "n_free": _ints([n_pages - used]), "seq_ids": order, "delta": delta, "back": -delta,
         # a program has the arrays of its largest step; 13 rows more than this one has
         "rows": [[torch.full((n + 13,), -1, dtype=torch.int32, device="cuda") for _ in range(3)] for n in rows]}
    return s


def _weights(case, gen):
    H, KV, hd, _, norm, bias = HEADS[case["heads"]]
    qn, kn = (1 + 0.02 * torch.randn(hd, generator=gen, device="cuda") for _ in range(2)) if norm else (None, None)
    biases = [0.1 * torch.randn(n * hd, generator=gen, device="cuda") for n in (H, KV, KV)] if bias else None
    return qn, kn, biases


def _append_inputs(case, seed):
    H, KV, hd, theta, _, _ = HEADS[case["heads"]]
    gen, P, rows = torch.Generator(device="cuda").manual_seed(seed), case["page_rows"], case["rows"]
    n_pages = _pages(rows, P) + 5
    q, k, v = (torch.randn((rows, n * hd), generator=gen, device="cuda") for n in (H, KV, KV))
    pool = [torch.randn((n_pages, KV, P, hd), generator=gen, device="cuda").to(DTYPES[case["dtype"]]) for _ in range(2)]
    slots = torch.randperm(n_pages * P, generator=gen, device="cuda")[:rows].to(torch.int32)
    if rows >= case["far"]:
        positions = torch.arange(rows, dtype=torch.int32, device="cuda") % case["far"]
    else:
        positions = torch.randint(0, case["far"], (rows,), generator=gen, device="cuda", dtype=torch.int32)
    # (the frequencies as the framework holds them: 64 bits, rounded once)
    freq = torch.tensor([theta ** (-2.0 * i / hd) for i in range(hd // 2)], dtype=torch.float64).float().cuda()
    return {"q": q, "k": k, "v": v, "K": pool[0], "V": pool[1], "slots": slots, "positions": positions,
            "weights": _weights(case, gen), "freq": freq}


def _attend_inputs(case, seed):
    H, KV, hd = HEADS[case["heads"]][:3]
    gen, P = torch.Generator(device="cuda").manual_seed(seed), case["page_rows"]
    lengths = _lengths(case)
    wide = max(1, _pages(max(lengths), P))
    n_pages = sum(_pages(n, P) for n in lengths) + 3
    lens = _ints(lengths)
    counts = _pages(lens, P)
    grid = torch.arange(wide, device="cuda")[None]
    pages = torch.randperm(n_pages, generator=gen, device="cuda").to(torch.int32)
    held = grid < counts[:, None]
    starts = torch.cumsum(counts, 0) - counts
    table = torch.where(held, pages[torch.where(held, starts[:, None] + grid, 0).long()], -1).to(torch.int32)
    dtype = DTYPES[case["dtype"]]
    K, V = (torch.randn((n_pages, KV, P, hd), generator=gen, device="cuda", dtype=torch.bfloat16 if dtype is torch.bfloat16 else
                        torch.float32).to(dtype) for _ in range(2))
    # queries of several sizes: from nearly even weights to a few keys that count
    q = torch.randn((len(lengths), H * hd), generator=gen, device="cuda")
    q = q * torch.linspace(0.3, 2.0, H, device="cuda").repeat_interleave(hd)
    return {"q": q, "K": K, "V": V, "table": table, "row_seqs": torch.arange(len(lengths), dtype=torch.int32, device="cuda"),
            "positions": lens - 1}


def prepare(case, seed):
    if case["op"] == "map":
        s = _map_inputs(case, seed)
        if own:
            import shainet_amd as sa

            s["ctx"] = sa.AttnContext(1, 1, 8, max_positions=1)
            s["ctx"].set_stream(torch.cuda.current_stream().cuda_stream)
            cache = s["cache"] = sa.PagedKVCache(s["ctx"], s["n_pages"], s["page_rows"], *s["table"].shape, dtype="bf16")
            for have, want in ((cache.table, s["table"]), (cache.lens, s["lens"]), (cache.free_pages, s["free"]),
                               (cache.n_free, s["n_free"])):
                have.copy_(want)
    else:
        s = (_append_inputs if case["op"] == "append" else _attend_inputs)(case, seed)
        H, KV, hd = HEADS[case["heads"]][:3]
        s["heads"] = (H, KV, hd)
        if own:
            import shainet_amd as sa

            ctx = s["ctx"] = _context(case, s.get("weights", (None, None, None)))
            wide = _pages(case["far"], case["page_rows"]) if case["op"] == "append" else s["table"].shape[1]
            cache = s["cache"] = sa.PagedKVCache(ctx, len(s["K"]), case["page_rows"], case.get("requests", 1), wide,
                                                 dtype=case["dtype"])
            cache.k.copy_(s.pop("K"))
            cache.v.copy_(s.pop("V"))
            if case["op"] == "attend":
                cache.table.copy_(s["table"])
            s["out"] = torch.empty_like(s["q"])
    s["op"] = case["op"]
    torch.cuda.synchronize()
    return s


# ---- a pass ---------------------------------------------------------------------------------------

def _map_once(s, delta, out):
    """Plain form: lengths change by delta; pages move; the new rows' slots, positions and requests into `out`."""
    P, table, lens, free, ids = s["page_rows"], s["table"], s["lens"], s["free"], s["seq_ids"].long()
    delta, old, top = delta.long(), s["lens"][ids].long(), s["n_free"].long()
    new = old + delta
    had, has = _pages(old, P), _pages(new, P)
    gone, taken = (had - has).clamp(min=0), (has - had).clamp(min=0)
    n_gone, n_taken, n_rows = gone.sum(), taken.sum(), delta.clamp(min=0).sum()
    ok = (new.min() >= 0) & (has.max() <= table.shape[1]) & (n_taken <= top + n_gone) & (n_rows <= len(out[0]))
    # released pages on top of the free ones: the last request's last page first
    grid = torch.arange(table.shape[1], device=table.device)[None]
    behind = gone.flip(0).cumsum(0).flip(0) - gone
    mine = table[ids]
    at = top + behind[:, None] + had[:, None] - 1 - grid
    leaves = ok & (grid >= has[:, None]) & (grid < had[:, None])
    spare = len(free)
    stack = torch.cat([free, free[:1]])  # (the last place is nobody's)
    stack = stack.scatter(0, torch.where(leaves, at, spare).flatten(), mine.flatten())
    # taken from the top
    before = taken.cumsum(0) - taken
    at = top + n_gone - 1 - (before[:, None] + grid - had[:, None])
    comes = ok & (grid >= had[:, None]) & (grid < has[:, None])
    mine = torch.where(comes, stack[torch.where(comes, at, spare)], mine)
    table[ids] = mine
    free.copy_(stack[:spare])
    s["n_free"].copy_(torch.where(ok, top + n_gone - n_taken, top))
    lens[ids] = torch.where(ok, new, old).to(torch.int32)
    # the new rows
    ends = delta.clamp(min=0).cumsum(0)
    r = torch.arange(len(out[0]), device=table.device)
    i = torch.searchsorted(ends, r, right=True).clamp(max=len(ids) - 1)
    real = ok & (r < n_rows)
    pos = torch.where(real, old[i] + r - (ends[i] - delta[i].clamp(min=0)), 0)
    slot = mine[i, pos // P].long() * P + pos % P
    for have, value in zip(out, (slot, pos, ids[i])):
        have.copy_(torch.where(real, value, -1))


def _rotated(x, norm, bias, cos, sin, hd):
    """Plain form: rows [n, heads * hd] with bias, QK-norm and half-split rotation."""
    if bias is not None:
        x = x + bias
    x = x.view(len(x), -1, hd)
    if norm is not None:
        x = x * (1 / torch.sqrt((x * x).sum(-1, keepdim=True) / hd + EPS)) * norm
    a, b = x[..., :hd // 2], x[..., hd // 2:]
    return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)


def _append_plain(s):
    H, KV, hd = s["heads"]
    qn, kn, biases = s["weights"]
    bq, bk, bv = biases or (None, None, None)
    # the framework's rotation turns by the float32 product of position and frequency; its cosine and sine in 64 bits
    angle = (s["positions"].float()[:, None] * s["freq"]).double()[:, None]
    cos, sin = torch.cos(angle).float(), torch.sin(angle).float()
    P, slots = s["K"].shape[2], s["slots"].long()
    q = _rotated(s["q"], qn, bq, cos, sin, hd).flatten(1)
    s["K"][slots // P, :, slots % P] = _rotated(s["k"], kn, bk, cos, sin, hd).to(s["K"].dtype)
    v = s["v"] if bv is None else s["v"] + bv
    s["V"][slots // P, :, slots % P] = v.view(len(v), KV, hd).to(s["V"].dtype)
    return q, s["K"], s["V"]


def _attend_plain(s):
    H, KV, hd = s["heads"]
    n, P = s["positions"] + 1, s["K"].shape[2]
    pages = s["table"][s["row_seqs"].long()].clamp(min=0).long()

    def rows(pool):  # [requests * kv heads, longest, hd]
        return pool[pages].transpose(1, 2).reshape(-1, pages.shape[1] * P, hd).float()

    seen = torch.arange(pages.shape[1] * P, device=n.device) < n[:, None]
    seen = seen[:, None, None].expand(-1, KV, -1, -1).flatten(0, 1)
    q = s["q"].view(-1, H // KV, hd)
    scores = torch.bmm(q, rows(s["K"]).transpose(1, 2).contiguous()) / math.sqrt(hd)
    scores = torch.where(seen, scores, -math.inf)
    best = scores.amax(-1, keepdim=True)
    weights = torch.exp(scores - torch.where(best == -math.inf, 0.0, best))
    total = weights.sum(-1, keepdim=True)
    out = torch.bmm(weights, rows(s["V"])) / torch.where(total == 0, 1.0, total)
    return out.view(len(n), H * hd)


def run(state):
    s = state
    if s["op"] == "map":
        there, back = s["rows"]
        if own:
            s["cache"].map_rows(s["delta"], *there, seq_ids=s["seq_ids"])
            s["cache"].map_rows(s["back"], *back, seq_ids=s["seq_ids"])
            c = s["cache"]
            return there, back, c.table, c.lens, c.free_pages, c.n_free
        _map_once(s, s["delta"], there)
        _map_once(s, s["back"], back)
        return there, back, s["table"], s["lens"], s["free"], s["n_free"]
    if s["op"] == "append":
        if own:
            s["ctx"].append_paged(s["cache"], s["slots"], s["positions"], s["q"], s["k"], s["v"], q_rot=s["out"])
            return s["out"], s["cache"].k, s["cache"].v
        return _append_plain(s)
    if own:
        return s["ctx"].attend_paged(s["cache"], s["row_seqs"], s["positions"], s["q"], out=s["out"])
    return _attend_plain(s)


# ---- the definition in 64 bits --------------------------------------------------------------------

def _turn_exactly(x, weight, bias, positions, freq, hd):
    x = x.double() + (0 if bias is None else bias.double())
    x = x.unflatten(1, (-1, hd))
    if weight is not None:
        x = x / (x.square().mean(-1, keepdim=True) + EPS).sqrt() * weight.double()
    # position and frequency are float32 numbers and so is, by the rotation's definition here, their product
    z = torch.view_as_complex(torch.stack(x.chunk(2, -1), -1).contiguous())
    angle = torch.mul(positions.float().unsqueeze(1), freq.unsqueeze(0)).double().unsqueeze(1)
    z = z * torch.polar(torch.ones_like(angle), angle)
    return torch.cat([z.real, z.imag], -1)


def exact(case, seed):
    if case["op"] == "map":
        return None
    H, KV, hd = HEADS[case["heads"]][:3]
    if case["op"] == "append":
        s = _append_inputs(case, seed)
        qn, kn, biases = s["weights"]
        bq, bk, bv = biases or (None, None, None)
        K, V = s["K"].double().transpose(1, 2).flatten(0, 1), s["V"].double().transpose(1, 2).flatten(0, 1)  # [slots, KV, hd]
        at = s["slots"].long()
        K[at] = _turn_exactly(s["k"], kn, bk, s["positions"], s["freq"], hd)
        V[at] = (s["v"].double() + (0 if bv is None else bv.double())).unflatten(1, (KV, hd))
        P = case["page_rows"]
        whole = lambda t: t.unflatten(0, (-1, P)).transpose(1, 2).contiguous()  # noqa: E731
        return _turn_exactly(s["q"], qn, bq, s["positions"], s["freq"], hd).flatten(1), whole(K), whole(V)
    s = _attend_inputs(case, seed)
    q = s["q"].double().unflatten(1, (KV, H // KV, hd))
    out = torch.zeros_like(q)
    for i, n in enumerate((s["positions"] + 1).tolist()):
        if n == 0:
            continue  # nothing to attend over: zeros
        k, v = (s[name][s["table"][i, :_pages(n, case["page_rows"])].long()].transpose(0, 1).flatten(1, 2)[:, :n].double()
                for name in "KV")
        share = torch.softmax((q[i] / hd ** 0.5) @ k.mT.contiguous(), -1)
        out[i] = share @ v
    return out.flatten(1)
