"""Attention over bounded caches, as calls that can be timed and compared.

Every case is one pass through one operator, in a plain form (``own`` false: elementary torch operations in
fp32) or as a user calls the package (``own`` true). Kinds of case:

* ``window``  -- a decode step's attention over pages, each row seeing its last ``window`` tokens and its first ``sinks``;
* ``prompt``  -- a packed group's causal attention with the same mask (query i sees key j <= i where i - j < window or j < sinks);
* ``weigh``   -- a decode step's attention that also adds each token's weights (summed over the query heads of a
  KV head) to an account per row, KV head and token;
* ``observe`` -- the same account of a prompt: the weights that its last ``observe`` queries (0: all) give each key;
* ``evict``   -- rows longer than ``budget`` cut to it per KV head: their first ``sinks`` and last ``recent`` tokens and the
  heaviest of the rest (the lowest index where weights are equal) are kept in their order, K, V and
  account, in blocks of their own.
"""

import math
import os
import sys

import torch

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}

own = False

# 8 prompts, lognormal(median 512, sigma 0.6) clipped to [64, 2048]: a packed group of 4311 tokens
PROMPTS = "1742,110,658,364,390,450,152,445"


def _package():
    folder = os.path.join(os.getcwd(), "llm-serving_amd")
    if folder not in sys.path:
        sys.path.insert(0, folder)
    import miattn

    return miattn


def listed():
    qwen3 = {"H": 16, "H_kv": 8, "D": 128}
    wide = {"H": 8, "H_kv": 2, "D": 256}
    return [
        # one user's long chat under a window: a single row, launched call by call; latency is all there is
        {"name": "window_one_row", "kind": "window", "B": 1, "lo": 6000, "hi": 6000, "window": 1024, "sinks": 4,
         "block": 16, "layers": 28, "dtype": "bf16", "graph": False, **qwen3},
        # the ordinary serving batch: 32 rows, some shorter than the window, some far longer
        {"name": "window_ragged_batch", "kind": "window", "B": 32, "lo": 128, "hi": 16384, "window": 2048, "sinks": 4,
         "block": 16, "layers": 8, "dtype": "bf16", "graph": True, **qwen3},
        # four query heads per KV head at head_dim 256, fp16, pages of 32, long contexts
        {"name": "window_wide_heads", "kind": "window", "B": 16, "lo": 1000, "hi": 40000, "window": 4096, "sinks": 64,
         "block": 32, "layers": 8, "dtype": "fp16", "graph": True, **wide},
        # an admitted group of prompts under a short window
        {"name": "prompt_group", "kind": "prompt", "lengths": PROMPTS, "window": 256, "sinks": 4, "layers": 4,
         "dtype": "bf16", **qwen3},
        # one long document
        {"name": "prompt_long", "kind": "prompt", "lengths": "16384", "window": 2048, "sinks": 4, "layers": 1,
         "dtype": "bf16", **qwen3},
        # a group that fills the server's prefill budget, head_dim 256 in fp16, a window that is no multiple of a tile
        {"name": "prompt_wide_heads", "kind": "prompt", "lengths": "3001,1700,2048,903,540", "window": 500, "sinks": 17,
         "layers": 2, "dtype": "fp16", **wide},
        # one user's chat while its cache is being weighed: a short row, launched call by call
        {"name": "weigh_one_row", "kind": "weigh", "B": 1, "lo": 300, "hi": 300, "block": 16, "layers": 28,
         "dtype": "bf16", "graph": False, **qwen3},
        # the ordinary serving batch, weighed
        {"name": "weigh_ragged_batch", "kind": "weigh", "B": 32, "lo": 128, "hi": 2048, "block": 16, "layers": 28,
         "dtype": "bf16", "graph": True, **qwen3},
        # an admitted group, judged by the last 32 queries of each prompt
        {"name": "observe_group", "kind": "observe", "lengths": PROMPTS, "observe": 32, "layers": 4, "dtype": "bf16",
         **qwen3},
        # long prompts judged by all of their queries
        {"name": "observe_all", "kind": "observe", "lengths": "4096,2048,1742,306", "observe": 0, "layers": 1,
         "dtype": "bf16", **qwen3},
        # one row, 64 tokens over its budget: what a decode loop calls every 64 steps
        {"name": "evict_one_row", "kind": "evict", "B": 1, "lo": 1088, "hi": 1088, "budget": 1024, "recent": 256,
         "sinks": 4, "block": 16, "layers": 28, "dtype": "bf16", **qwen3},
        # a batch of prompts cut to their budget after their prefill, some of them shorter than it
        {"name": "evict_batch", "kind": "evict", "B": 32, "lo": 64, "hi": 4096, "budget": 512, "recent": 128,
         "sinks": 4, "block": 16, "layers": 4, "dtype": "bf16", **qwen3},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _some_lengths(rng, most_prompts, hi, most_tokens):
    got = []
    for _ in range(rng.randint(1, most_prompts)):
        k = _log_int(rng, 1 if rng.random() < 0.15 else 24, hi)
        if sum(got) + k > most_tokens:
            break
        got.append(k)
    return ",".join(str(k) for k in got or [hi])


def draw(rng):
    kind = rng.choice(["window", "prompt", "weigh", "observe", "evict"])
    heads = rng.choice([{"H": 16, "H_kv": 8, "D": 128}, {"H": 16, "H_kv": 8, "D": 128}, {"H": 8, "H_kv": 2, "D": 256},
                        {"H": 32, "H_kv": 4, "D": 128}, {"H": 16, "H_kv": 16, "D": 64}, {"H": 24, "H_kv": 2, "D": 128}])
    if kind in ("prompt", "observe"):
        case = {"kind": kind, "dtype": rng.choice(["bf16", "bf16", "fp16"]), **heads,
                "lengths": _some_lengths(rng, 12, rng.choice([60, 2048, 6000]), 8192), "layers": rng.randint(1, 2)}
        if kind == "prompt":
            return {**case, "window": _log_int(rng, 1, 3000), "sinks": rng.choice([0, 1, 4, _log_int(rng, 1, 300)])}
        longest = max(int(n) for n in case["lengths"].split(","))
        return {**case, "observe": rng.choice([1, 16, 32, 64, _log_int(rng, 1, 400), 0 if longest <= 4096 else 32])}
    case = {"kind": kind, "dtype": rng.choice(["bf16", "bf16", "bf16", "fp16", "fp16", "fp32"]),
            "block": rng.choice([16, 16, 32, 64]), **heads}
    B, hi = _log_int(rng, 1, 64), _log_int(rng, 20, 20000 if rng.random() < 0.2 else 6000)
    lo = rng.choice([0, max(1, int(hi * 0.06)), max(1, hi // 2), hi])
    most = 32 * 2048 if kind == "weigh" else 32 * 4096
    while B > 1 and B * hi * heads["H_kv"] * heads["D"] > most * 1024:
        B = max(1, B // 2)
    room = (1 << 30) // (B * (hi + 64) * heads["H_kv"] * heads["D"])
    case.update(B=B, lo=lo, hi=hi, layers=max(1, min(rng.choice([1, 4, 16]) if kind != "evict" else rng.choice([1, 4]), room)))
    if kind == "window":
        return {**case, "window": _log_int(rng, 1, 5000), "sinks": rng.choice([0, 1, 4, _log_int(rng, 1, 300)]),
                "graph": rng.random() < 0.6}
    if kind == "weigh":
        return {**case, "graph": rng.random() < 0.6}
    budget = _log_int(rng, 4, max(8, min(hi, 2048)))
    sinks = rng.choice([0, min(4, budget // 4)])
    return {**case, "budget": budget, "recent": rng.randint(0, budget - sinks), "sinks": sinks}


# ------------------------------------------------------------------------------- inputs
def _gen(seed, device="cpu"):
    return torch.Generator(device=device).manual_seed(int(seed))


def _normal(g, *shape, dtype=torch.float32):
    """N(0, 1) on the card, drawn in fp32 and cast, in slabs that need no second large copy."""
    out = torch.empty(shape, dtype=dtype, device=DEV)
    flat = out.view(-1)
    for at in range(0, flat.numel(), 1 << 26):
        n = min(1 << 26, flat.numel() - at)
        flat[at: at + n] = torch.randn(n, generator=g, device=DEV)
    return out


def _pages(n, block):
    return max(1, -(-n // block))


def _table(lengths, most, block, perm):
    """Block table of rows that take their pages from ``perm`` in turn (0 past a row's own), wide enough for ``most``."""
    need = [_pages(n, block) for n in lengths]
    table = torch.zeros(len(lengths), _pages(most, block), dtype=torch.int32)
    at = 0
    for r, n in enumerate(need):
        table[r, :n] = perm[at: at + n]
        at += n
    return table.to(DEV), perm[at:]


def _captured(step):
    """The step recorded in a graph that the program keeps, and the tensors that a replay fills."""
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    torch.cuda.synchronize()
    return graph, outs


def _account(g, L, lengths, H_kv, width):
    """What some hundred steps leave in the accounts: a few heavy tokens, many light ones, some of exactly 0."""
    w = torch.exp(1.5 * _normal(g, L, len(lengths), H_kv, width) - 3)
    w = torch.where(torch.rand(w.shape, generator=g, device=DEV) < 0.05, torch.zeros_like(w), w)
    end = torch.tensor(lengths, device=DEV).view(1, -1, 1, 1)
    return torch.where(torch.arange(width, device=DEV) < end, w, torch.zeros_like(w))


def prepare(case, seed):
    g, dg = _gen(seed), _gen(seed + 1, DEV)
    dt, H, H_kv, D, L = DTYPES[case["dtype"]], case["H"], case["H_kv"], case["D"], case["layers"]
    s = {"case": case, "graph": None}
    if case["kind"] in ("prompt", "observe"):
        lengths = [int(n) for n in case["lengths"].split(",")]
        T = sum(lengths)
        s["cu"] = [sum(lengths[:i]) for i in range(len(lengths) + 1)]
        s["longest"] = max(lengths)
        s["q"] = [_normal(dg, T, H, D, dtype=dt) for _ in range(L)]
        s["k"] = [_normal(dg, T, H_kv, D, dtype=dt) for _ in range(L)]
        s["v"] = [_normal(dg, T, H_kv, D, dtype=dt) for _ in range(L)] if case["kind"] == "prompt" else []
        if own:
            backend = _package().HipVarlen()
            qs, ks, vs, cu, longest = s["q"], s["k"], s["v"], s["cu"], s["longest"]
            if case["kind"] == "prompt":
                s["step"] = lambda: [backend.prefill_varlen(qs[i], ks[i], vs[i], cu_seqlens=cu, max_seqlen=longest,
                                                            window=case["window"], sinks=case["sinks"]) for i in range(L)]
            else:
                s["step"] = lambda: [backend.prompt_weights(qs[i], ks[i], cu_seqlens=cu, max_seqlen=longest,
                                                            observe=case["observe"] or None) for i in range(L)]
        return s
    B, block = case["B"], case["block"]
    lengths = torch.randint(case["lo"], case["hi"] + 1, (B,), generator=g).tolist()
    most = case["hi"]  # a table and a pool hold the longest row that may come, whatever the lengths of today
    n_pages = B * (_pages(most, block) + (_pages(min(most, case["budget"]), block) if case["kind"] == "evict" else 0)) + 1
    s["table"], perm = _table(lengths, most, block, torch.randperm(n_pages, generator=g).int())
    s["seqlen"] = torch.tensor(lengths, dtype=torch.int32, device=DEV)
    capacity = s["table"].shape[1] * block
    s["k"] = [_normal(dg, n_pages, block, H_kv, D, dtype=dt) for _ in range(L)]
    s["v"] = [_normal(dg, n_pages, block, H_kv, D, dtype=dt) for _ in range(L)]
    if case["kind"] != "window":
        s["before"] = _account(dg, L, lengths, H_kv, capacity)
        s["weights"] = s["before"].clone()
    if case["kind"] == "evict":
        kept = min(most, case["budget"])
        s["to"], _ = _table([min(n, kept) for n in lengths], kept, block, perm)
        s["lengths"] = s["seqlen"].clone()
        if own:
            pool = _package().PagedPool(L, n_pages, block, H_kv, D, dtype=dt, device=DEV, n_head=H)
            pool.keys, pool.values = s["k"], s["v"]
            s["pool"] = pool
        return s
    s["q"] = [_normal(dg, B, H, D, dtype=dt) for _ in range(L)]
    if own:
        qs = s["q"]  # no call below holds the state itself: a cycle would keep its graph until some later capture
        if case["kind"] == "window":
            plan = _package().paged_decode_plan(qs[0], s["k"], s["v"], s["table"], s["seqlen"], window=case["window"],
                                                sinks=case["sinks"])
            s["step"] = lambda: [plan.run(i, qs[i]) for i in range(L)]
        else:
            plan = _package().paged_decode_plan(qs[0], s["k"], s["v"], s["table"], s["seqlen"])
            weights, before = s["weights"], s["before"]

            def step():
                torch.mul(before, 1.0, out=weights)  # each pass starts from the same account
                return [*(plan.run_weighed(i, qs[i], weights[i]) for i in range(L)), weights]
            s["step"] = step
        if case["graph"]:
            s["graph"], s["outs"] = _captured(s["step"])
    return s


# ------------------------------------------------------------------------------- the plain forms
def _softmax(scores, visible):
    """exp(scores - max) / sum over the visible entries of the last axis; rows of none give zeros."""
    scores = torch.where(visible, scores, torch.full_like(scores, -math.inf))
    most = scores.amax(-1, True)
    p = torch.exp(scores - torch.where(most == -math.inf, torch.zeros_like(most), most))
    total = p.sum(-1, True)
    return p / torch.where(total == 0, torch.ones_like(total), total)


def _rows_of(pages, table, at):
    """fp32 rows ``(B, H_kv, n, D)`` of the tokens ``at`` ``(B, n)`` of each row."""
    block = pages.shape[1]
    page = torch.gather(table.long(), 1, (at // block).clamp(0, table.shape[1] - 1))
    return pages[page, at % block].float().transpose(1, 2).contiguous()


def _attend(q, kp, vp, table, at, visible):
    """softmax(q K^T / sqrt(D)) V over the tokens ``at`` that are visible, and the weights ``(B, H, n)``."""
    B, H, D = q.shape
    k, v = _rows_of(kp, table, at), _rows_of(vp, table, at)
    H_kv = k.shape[1]
    v = torch.where(visible[:, None, :, None], v, torch.zeros_like(v))
    scores = torch.matmul(q.float().view(B, H_kv, H // H_kv, D), k.transpose(-1, -2).contiguous()) * (1.0 / math.sqrt(D))
    p = _softmax(scores, visible[:, None, None, :])
    return torch.matmul(p, v).reshape(B, H, D).to(q.dtype), p


def _windowed(s, i):
    case = s["case"]
    n = min(case["sinks"] + case["window"], s["table"].shape[1] * case["block"])
    t = torch.arange(n, device=DEV)
    length = s["seqlen"].long().view(-1, 1)
    seen = length.clamp(max=case["sinks"] + case["window"])
    at = torch.where(t < case["sinks"], t, t + (length - seen))
    return _attend(s["q"][i], s["k"][i], s["v"][i], s["table"], at, t < seen)[0]


def _weighed(s, i):
    n = s["weights"].shape[-1]
    t = torch.arange(n, device=DEV)
    visible = t < s["seqlen"].view(-1, 1)
    out, p = _attend(s["q"][i], s["k"][i], s["v"][i], s["table"], t.expand(len(visible), n), visible)
    s["weights"][i] += p.sum(2)
    return out


def _prompt(s, i, a, b, out):
    """One prompt's attention under the window, 512 queries at a time over the keys that any of them sees."""
    case = s["case"]
    H, H_kv, D, window, sinks = case["H"], case["H_kv"], case["D"], case["window"], case["sinks"]
    k, v = (s[name][i][a:b].float().transpose(0, 1).contiguous() for name in ("k", "v"))
    for lo in range(0, b - a, 512):
        hi = min(lo + 512, b - a)
        first = max(0, lo - window + 1)
        at = torch.cat([torch.arange(min(sinks, first), device=DEV), torch.arange(first, hi, device=DEV)])
        back = torch.arange(lo, hi, device=DEV).view(-1, 1) - at
        visible = (back >= 0) & ((back < window) | (at < sinks))
        q = s["q"][i][a + lo: a + hi].float().view(hi - lo, H_kv, H // H_kv, D).permute(1, 2, 0, 3).contiguous()
        scores = torch.matmul(q.flatten(1, 2), k[:, at].transpose(-1, -2).contiguous()) * (1.0 / math.sqrt(D))
        p = _softmax(scores.unflatten(1, (H // H_kv, hi - lo)), visible)
        y = torch.matmul(p.flatten(1, 2), v[:, at]).unflatten(1, (H // H_kv, hi - lo))
        out[a + lo: a + hi] = y.permute(2, 0, 1, 3).reshape(hi - lo, H, D).to(out.dtype)


def _observed(s, i):
    """Weights ``(prompts, H_kv, longest)`` that each prompt's last queries give its keys."""
    case, cu = s["case"], s["cu"]
    H, H_kv, D = case["H"], case["H_kv"], case["D"]
    out = torch.zeros(len(cu) - 1, H_kv, s["longest"], device=DEV)
    for r, (a, b) in enumerate(zip(cu, cu[1:])):
        k = s["k"][i][a:b].float().transpose(0, 1).contiguous()
        begin = max(a, b - case["observe"]) if case["observe"] else a
        for lo in range(begin, b, 512):
            hi = min(lo + 512, b)
            q = s["q"][i][lo:hi].float().view(hi - lo, H_kv, H // H_kv, D).permute(1, 2, 0, 3).contiguous()
            scores = torch.matmul(q.flatten(1, 2), k.transpose(-1, -2).contiguous()) * (1.0 / math.sqrt(D))
            visible = torch.arange(b - a, device=DEV) <= torch.arange(lo - a, hi - a, device=DEV).view(-1, 1)
            out[r, :, : b - a] += _softmax(scores.unflatten(1, (H // H_kv, hi - lo)), visible).sum((1, 2))
    return out


def _evicted(s):
    """Keep the protected and the heaviest tokens of the rows past the budget, in ``to``'s blocks."""
    case = s["case"]
    B, H_kv, block = case["B"], case["H_kv"], case["block"]
    budget, recent, sinks = case["budget"], case["recent"], case["sinks"]
    n_all, n_to = s["table"].shape[1] * block, s["to"].shape[1] * block
    t = torch.arange(n_all, device=DEV)
    length = s["seqlen"].long().view(B, 1, 1)
    keep = length.clamp(max=budget)
    held = torch.arange(n_to, device=DEV) < keep.view(B, 1)
    row, slot = held.nonzero(as_tuple=True)
    to_page, to_at = s["to"].long()[row, slot // block], slot % block
    heads = torch.arange(H_kv, device=DEV)
    for i in range(case["layers"]):
        w = s["weights"][i]
        # protected tokens first, tokens past the row last, the heaviest between; equal ones in their order
        rank = torch.where((t < sinks) | (t >= length - recent), torch.full_like(w, math.inf), w)
        rank = torch.where(t < length, rank, torch.full_like(rank, -math.inf))
        order = torch.sort(rank, dim=-1, descending=True, stable=True)[1]
        chosen = torch.zeros(w.shape, dtype=torch.bool, device=DEV).scatter_(-1, order, t < keep.expand_as(order[..., :1]))
        source = torch.sort(chosen.to(torch.uint8), dim=-1, descending=True, stable=True)[1]  # the kept ones, in their order
        at = source[row, :, slot]  # (kept tokens, H_kv)
        page = s["table"].long()[row.view(-1, 1), at // block]
        for pool in (s["k"][i], s["v"][i]):
            pool[to_page, to_at] = pool[page, at % block, heads]
        s["weights"][i] = torch.where(t < keep, torch.gather(w, -1, source), torch.zeros_like(w))
    s["seqlen"].clamp_(max=budget)


def run(s):
    case, L = s["case"], s["case"]["layers"]
    if case["kind"] == "evict":
        s["seqlen"].copy_(s["lengths"])  # each pass starts from the same rows and account
        torch.mul(s["before"], 1.0, out=s["weights"])
        if own:
            s["pool"].evict(s["table"], s["seqlen"], s["weights"], budget=case["budget"], recent=case["recent"],
                            sinks=case["sinks"], to=s["to"])
        else:
            _evicted(s)
        return s["k"], s["v"], s["weights"], s["seqlen"]
    if own:
        if s["graph"] is None:
            return s["step"]()
        s["graph"].replay()
        return s["outs"]
    if case["kind"] == "window":
        return [_windowed(s, i) for i in range(L)]
    if case["kind"] == "weigh":
        torch.mul(s["before"], 1.0, out=s["weights"])
        return [*(_weighed(s, i) for i in range(L)), s["weights"]]
    if case["kind"] == "observe":
        return [_observed(s, i) for i in range(L)]
    outs = [torch.empty_like(q) for q in s["q"]]
    for i in range(L):
        for a, b in zip(s["cu"], s["cu"][1:]):
            _prompt(s, i, a, b, outs[i])
    return outs


def _mean(f, case):
    """The mean of ``f`` over the lengths that a case's rows are drawn from."""
    lo, hi = case["lo"], case["hi"]
    points = range(lo, hi + 1, max(1, (hi - lo) // 256))
    return sum(f(n) for n in points) / len(points)


def work(case):
    H, H_kv, D, L = case["H"], case["H_kv"], case["D"], case["layers"]
    size = 4 if case["dtype"] == "fp32" else 2
    if case["kind"] in ("window", "weigh"):
        most = case["window"] + case["sinks"] if case["kind"] == "window" else math.inf
        tokens = case["B"] * _mean(lambda n: min(n, most), case)
        moved = 2 * tokens * H_kv * D * size + 2 * case["B"] * H * D * size + 4 * tokens / case["block"]
        if case["kind"] == "weigh":
            moved += 2 * 4 * tokens * H_kv
        return {"bytes": L * moved, "flops": L * 4 * tokens * H * D}
    if case["kind"] == "evict":
        tokens = case["B"] * _mean(lambda n: n, case)
        kept = case["B"] * _mean(lambda n: min(n, case["budget"]), case)
        return {"bytes": L * H_kv * (2 * 2 * kept * D * size + 2 * 4 * tokens), "flops": 0}
    lengths = [int(n) for n in case["lengths"].split(",")]
    T = sum(lengths)
    if case["kind"] == "observe":
        seen = [(n, min(n, case["observe"] or n)) for n in lengths]
        pairs = sum(m * (n - m) + m * (m + 1) // 2 for n, m in seen)
        moved = T * H_kv * (D * size + 4) + sum(m for _, m in seen) * H * D * size
        return {"bytes": L * moved, "flops": L * 2 * pairs * H * D}
    full = case["window"] + case["sinks"]
    pairs = sum(n * (n + 1) // 2 if n <= full else full * (full + 1) // 2 + (n - full) * full for n in lengths)
    return {"bytes": L * T * 2 * (H + H_kv) * D * size, "flops": L * 4 * pairs * H * D}


# ------------------------------------------------------------------------------- in 64 bits
def _gathered(pages, row, n):
    """float64 rows ``(H_kv, n, D)`` of one row's first ``n`` tokens."""
    block = pages.shape[1]
    return pages[row[: -(-n // block)].long()].double().flatten(0, 1)[:n].permute(1, 0, 2).contiguous()


def _exact_row(q, k, v, mask):
    """One query ``(H, D)`` over ``k``, ``v`` ``(H_kv, n, D)``: output and weights ``(H_kv, n)``."""
    H, D = q.shape
    x = torch.bmm(q.double().reshape(len(k), -1, D), k.transpose(1, 2).contiguous()) / math.sqrt(D)
    w = torch.softmax(x.masked_fill(~mask, -math.inf), -1)
    return torch.bmm(w, v).reshape(H, D), w.sum(1)


def _exact_rows(s, i):
    case = s["case"]
    outs = torch.zeros(s["q"][i].shape, dtype=torch.float64, device=DEV)
    account = s["before"][i].double() if case["kind"] == "weigh" else None
    for b, n in enumerate(s["seqlen"].tolist()):
        if n == 0:
            continue
        j = torch.arange(n, device=DEV)
        mask = (j >= n - case["window"]) | (j < case["sinks"]) if case["kind"] == "window" else j >= 0
        outs[b], w = _exact_row(s["q"][i][b], _gathered(s["k"][i], s["table"][b], n),
                                _gathered(s["v"][i], s["table"][b], n), mask)
        if account is not None:
            account[b, :, :n] += w
    return outs, account


def _exact_prompt(s, i):
    case, cu = s["case"], s["cu"]
    H, H_kv, D = case["H"], case["H_kv"], case["D"]
    prompt = case["kind"] == "prompt"
    outs = torch.zeros(s["q"][i].shape if prompt else (len(cu) - 1, H_kv, s["longest"]), dtype=torch.float64, device=DEV)
    for r in range(len(cu) - 1):
        a, n = cu[r], cu[r + 1] - cu[r]
        start = 0 if prompt or not case["observe"] else max(0, n - case["observe"])
        for h in range(H):
            k = s["k"][i][a: a + n, h // (H // H_kv)].double()
            for lo in range(start, n, 2048):
                hi = min(lo + 2048, n)
                x = torch.mm(s["q"][i][a + lo: a + hi, h].double(), k[:hi].t().contiguous()) / math.sqrt(D)
                back = torch.arange(lo, hi, device=DEV)[:, None] - torch.arange(hi, device=DEV)[None, :]
                hidden = back < 0
                if prompt:
                    hidden |= (back >= case["window"]) & (torch.arange(hi, device=DEV) >= case["sinks"])
                w = torch.softmax(x.masked_fill(hidden, -math.inf), -1)
                if prompt:
                    outs[a + lo: a + hi, h] = torch.mm(w, s["v"][i][a: a + hi, h // (H // H_kv)].double())
                else:
                    outs[r, h // (H // H_kv), :hi] += w.sum(0)
    return outs


def _exact_evicted(s):
    case, block = s["case"], s["case"]["block"]
    keys, values = ([x.double() for x in s[name]] for name in ("k", "v"))
    account = s["before"].double()
    lengths = s["lengths"].tolist()
    for i in range(case["layers"]):
        for b, n in enumerate(lengths):
            keep = min(n, case["budget"])
            w = account[i, b, :, :n].clone()
            w[:, : case["sinks"]] = math.inf
            w[:, max(0, n - case["recent"]):] = math.inf
            # of two equal weights the lower index is the heavier one
            best = torch.argsort(w, dim=-1, descending=True, stable=True)[:, :keep].sort(-1)[0]
            held = account[i, b, :, :n].gather(1, best)
            account[i, b, :, :n] = 0
            account[i, b, :, :keep] = held
            slot = torch.arange(keep, device=DEV)
            page, at = s["to"][b].long()[slot // block], slot % block
            for source, target in ((s["k"][i], keys[i]), (s["v"][i], values[i])):
                rows = _gathered(source, s["table"][b], n) if n else None
                for h in range(case["H_kv"] if n else 0):
                    target[page, at, h] = rows[h][best[h]]
    return keys, values, account, torch.tensor([min(n, case["budget"]) for n in lengths], device=DEV)


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "evict":
        return _exact_evicted(s)
    if case["kind"] in ("prompt", "observe"):
        return [_exact_prompt(s, i) for i in range(case["layers"])]
    rows = [_exact_rows(s, i) for i in range(case["layers"])]
    outs = [out for out, _ in rows]
    return outs if case["kind"] == "window" else [*outs, torch.stack([account for _, account in rows])]
