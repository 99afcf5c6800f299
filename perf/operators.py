"""The 4-bit paged KV cache and the moving of cache pages, as calls that can be timed and compared.

Every case is one pass through one operator, in a plain form (``own`` false: elementary torch
operations in fp32) or as a user calls the package (``own`` true). Kinds of case:

* ``decode``   -- a decode step's attention over pages held in 4 bits, every layer of it;
* ``write``    -- a packed group's (or a step's) K and V written into the 4-bit pool and read back;
* ``epilogue`` -- q/k norm, position rotation and the 4-bit K/V write in one, with what the pool then holds;
* ``copy``     -- pages of a pool copied to other pages, all layers (a fork, a compaction).

The 4-bit format, per (token, KV head) row of ``D`` elements: groups of 32 elements share one
scale 2^e, each element is a 4-bit float (sign, then one of 0, 0.5, 1, 1.5, 2, 3, 4, 6) times it.
e is the smallest integer with max|x| <= 7 * 2^e over the group, held to [-120, 125]; x * 2^-e is
rounded to the nearest level, ties to the even code, past 6 to 6. A group with a value that is not
finite reads back as NaN. A page of one KV head is ``bs * D / 2`` bytes of codes, token by token (element
2i in the low half of byte i), then ``D / 32`` rows of ``bs`` scale bytes, e + 127 (255: NaN).
"""

import math
import os
import sys

import torch

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
EPS = 1e-6
GROUP = 32
LEVELS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)

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
        # one user's chat: a single short row, launched call by call; latency is all there is
        {"name": "decode_one_row", "kind": "decode", "B": 1, "lo": 300, "hi": 300, "block": 16, "layers": 28,
         "dtype": "bf16", "graph": False, **qwen3},
        # a few users at an even length, the step replayed from a graph
        {"name": "decode_small_batch", "kind": "decode", "B": 8, "lo": 512, "hi": 512, "block": 16, "layers": 28,
         "dtype": "bf16", "graph": True, **qwen3},
        # the ordinary serving batch: 32 ragged rows
        {"name": "decode_ragged_batch", "kind": "decode", "B": 32, "lo": 128, "hi": 2048, "block": 16, "layers": 28,
         "dtype": "bf16", "graph": True, **qwen3},
        # long documents: 32 rows of 8192 tokens, the most bytes a step here reads
        {"name": "decode_long_rows", "kind": "decode", "B": 32, "lo": 8192, "hi": 8192, "block": 16, "layers": 4,
         "dtype": "bf16", "graph": False, **qwen3},
        # one very long context, of an odd length: a single row has to fill the chip
        {"name": "decode_one_long_row", "kind": "decode", "B": 1, "lo": 100003, "hi": 100003, "block": 16, "layers": 4,
         "dtype": "bf16", "graph": True, **qwen3},
        # four query heads per KV head at head_dim 256, fp16, pages of 32
        {"name": "decode_wide_heads", "kind": "decode", "B": 16, "lo": 128, "hi": 2048, "block": 32, "layers": 28,
         "dtype": "fp16", "graph": True, **wide},
        # an admitted group's K and V into the pool
        {"name": "write_group", "kind": "write", "lengths": PROMPTS, "layers": 4, "dtype": "bf16", "block": 16,
         "graph": False, **qwen3},
        # one decode step's K and V (32 rows of one token) into the pool, from a graph
        {"name": "write_step", "kind": "write", "lengths": ",".join(["1"] * 32), "layers": 28, "dtype": "bf16",
         "block": 16, "graph": True, **qwen3},
        # the attention epilogue of a group that fills the server's prefill budget (8192 tokens)
        {"name": "epilogue_full_group", "kind": "epilogue", "lengths": "3001,1700,2048,903,540", "layers": 1,
         "dtype": "bf16", "block": 16, "packed": True, "graph": False, **qwen3},
        # the attention epilogue of one decode step of 32 rows, from a graph
        {"name": "epilogue_step", "kind": "epilogue", "lengths": ",".join(["1"] * 32), "layers": 14, "dtype": "bf16",
         "block": 16, "packed": False, "graph": True, **qwen3},
        # forking four conversations: the partly filled last page of each, in every layer
        {"name": "copy_fork", "kind": "copy", "pages": 40, "moves": 4, "layers": 28, "dtype": "bf16", "block": 16,
         **qwen3},
        # compacting a fragmented pool: 1000 pages move
        {"name": "copy_compact", "kind": "copy", "pages": 2100, "moves": 1000, "layers": 8, "dtype": "bf16",
         "block": 16, **qwen3},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _some_lengths(rng, most_prompts, hi, most_tokens):
    n = rng.randint(1, most_prompts)
    got = []
    for _ in range(n):
        k = _log_int(rng, 1 if rng.random() < 0.15 else 24, hi)
        if sum(got) + k > most_tokens:
            break
        got.append(k)
    return ",".join(str(k) for k in got or [hi])


def draw(rng):
    kind = rng.choice(["decode", "decode", "decode", "write", "epilogue", "copy"])
    heads = rng.choice([{"H": 16, "H_kv": 8, "D": 128}, {"H": 16, "H_kv": 8, "D": 128}, {"H": 8, "H_kv": 2, "D": 256},
                        {"H": 32, "H_kv": 4, "D": 128}, {"H": 16, "H_kv": 16, "D": 64}, {"H": 24, "H_kv": 2, "D": 128}])
    dtype = rng.choice(["bf16", "bf16", "bf16", "fp16", "fp16", "fp32"])
    block = rng.choice([16, 16, 32, 64])
    common = {"dtype": dtype, "block": block, **heads}
    if kind == "decode":
        B, hi = _log_int(rng, 1, 64), _log_int(rng, 20, 60000 if rng.random() < 0.2 else 8192)
        lo = rng.choice([0, max(1, int(hi * 0.06)), max(1, hi // 2), hi])
        while B > 1 and B * hi * heads["H_kv"] * heads["D"] > 32 * 8192 * 8 * 128:
            B = max(1, B // 2)
        most = (1 << 31) // (B * (hi + 64) * heads["H_kv"] * heads["D"])
        return {"kind": kind, "B": B, "lo": lo, "hi": hi, "layers": max(1, min(rng.choice([1, 4, 28]), most)),
                "graph": rng.random() < 0.6, **common}
    if kind == "write":
        return {"kind": kind, "lengths": _some_lengths(rng, 40, rng.choice([1, 60, 2048]), 8192),
                "layers": rng.randint(1, 4), "graph": rng.random() < 0.3, **common}
    if kind == "epilogue":
        return {"kind": kind, "lengths": _some_lengths(rng, 40, rng.choice([1, 60, 2048]), 8192), "layers": 1,
                "packed": rng.random() < 0.5, "graph": rng.random() < 0.3, **common}
    pages = _log_int(rng, 8, 1500)
    return {"kind": kind, "pages": pages, "moves": rng.randint(1, max(1, pages // 2 - 1)), "layers": rng.randint(1, 8),
            **common}


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


def _tables(lengths, block, n_pages, g):
    """Disjoint pages for each row from one permutation of the pool."""
    perm = torch.randperm(n_pages, generator=g).tolist()
    got, at = [], 0
    for n in lengths:
        need = max(1, -(-n // block))
        got.append(perm[at: at + need])
        at += need
    return got


def _pages(lengths, block):
    return sum(max(1, -(-n // block)) for n in lengths)


def _page_bytes(block, D):
    return block * (D // 2 + D // GROUP)


def _random_pages(g, n_pages, case):
    """Pages whose rows are N(0, 1) in 4 bits: what a pool holds after prompts were written to it."""
    block, H_kv, D = case["block"], case["H_kv"], case["D"]
    out = torch.empty(n_pages, H_kv, _page_bytes(block, D), dtype=torch.uint8, device=DEV)
    slab = max(1, (1 << 25) // (H_kv * block * D))
    for at in range(0, n_pages, slab):
        n = min(slab, n_pages - at)
        out[at: at + n] = _pack(*_quantise(_normal(g, n, H_kv, block, D)))
    return out


def _captured(step):
    """The step recorded in a graph that the program keeps, and the tensors that a replay fills."""
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    torch.cuda.synchronize()
    return graph, outs


def _prompt_slots(case, g):
    """Slots of every token of the prompts, pages in a random order, and the pool's page count."""
    lengths = [int(n) for n in case["lengths"].split(",")]
    block = case["block"]
    n_pages = _pages(lengths, block) * 5 // 4 + 1
    slots = []
    for n, table in zip(lengths, _tables(lengths, block, n_pages, g)):
        at = torch.arange(n)
        slots.append(torch.tensor(table)[at // block] * block + at % block)
    return lengths, torch.cat(slots).to(DEV), n_pages


def _new_pool(case, n_pages):
    """The package's 4-bit pool (own) or bare page tensors (plain form), one K and one V per layer."""
    if own:
        return _package().Fp4PagedPool(case["layers"], n_pages, case["block"], case["H_kv"], case["D"],
                                       dtype=DTYPES[case["dtype"]], device=DEV, n_head=case["H"])
    shape = (n_pages, case["H_kv"], _page_bytes(case["block"], case["D"]))
    return [[torch.zeros(shape, dtype=torch.uint8, device=DEV) for _ in range(case["layers"])] for _ in range(2)]


def prepare(case, seed):
    g, dg = _gen(seed), _gen(seed + 1, DEV)
    dt, H, H_kv, D, L = DTYPES[case["dtype"]], case["H"], case["H_kv"], case["D"], case["layers"]
    s = {"case": case, "graph": None}
    if case["kind"] == "decode":
        lengths = torch.randint(case["lo"], case["hi"] + 1, (case["B"],), generator=g).tolist()
        n_pages = _pages(lengths, case["block"]) * 5 // 4 + 1
        tables = _tables(lengths, case["block"], n_pages, g)
        table = torch.zeros(case["B"], max(len(t) for t in tables), dtype=torch.int32)
        for r, t in enumerate(tables):
            table[r, : len(t)] = torch.tensor(t, dtype=torch.int32)
        s["table"], s["seqlen"] = table.to(DEV), torch.tensor(lengths, dtype=torch.int32, device=DEV)
        s["k"] = [_random_pages(dg, n_pages, case) for _ in range(L)]
        s["v"] = [_random_pages(dg, n_pages, case) for _ in range(L)]
        s["q"] = [_normal(dg, case["B"], H, D, dtype=dt) for _ in range(L)]
        if own:
            plan = _package().paged_decode_fp4_plan(s["q"][0], s["k"], s["v"], s["table"], s["seqlen"])
            qs = s["q"]  # no call below holds the state itself: a cycle would keep its graph until some later capture
            s["step"] = lambda: [plan.run(i, qs[i]) for i in range(L)]
    elif case["kind"] == "write":
        lengths, s["slots"], n_pages = _prompt_slots(case, g)
        s["k"] = [_normal(dg, sum(lengths), H_kv, D, dtype=dt) for _ in range(L)]
        s["v"] = [_normal(dg, sum(lengths), H_kv, D, dtype=dt) for _ in range(L)]
        s["pool"] = pool = _new_pool(case, n_pages)
        if own:
            slots, ks, vs = s["slots"], s["k"], s["v"]
            s["step"] = lambda: [(pool.write_slots(i, slots, ks[i], vs[i]), pool.read_slots(i, slots))[1]
                                 for i in range(L)]
    elif case["kind"] == "epilogue":
        lengths, s["slots"], n_pages = _prompt_slots(case, g)
        T = sum(lengths)
        # a prompt's tokens start at position 0, a step's single tokens lie anywhere in the context
        where = [torch.arange(n) if n > 1 else torch.randint(0, 2048, (1,), generator=g) for n in lengths]
        s["pos"] = torch.cat(where).to(DEV)
        n_pos = max(2048, max(lengths))
        angle = torch.outer(torch.arange(n_pos, dtype=torch.float64),
                            1e6 ** -(torch.arange(0, D, 2, dtype=torch.float64) / D))
        s["cos"], s["sin"] = angle.cos().to(dt).to(DEV), angle.sin().to(dt).to(DEV)
        s["qkv"] = [_normal(dg, T, (H + 2 * H_kv) * D, dtype=dt) for _ in range(L)]
        s["qw"] = (1 + 0.1 * _normal(dg, D)).to(dt)
        s["kw"] = (1 + 0.1 * _normal(dg, D)).to(dt)
        s["pool"] = pool = _new_pool(case, n_pages)
        if own:
            slots, qkv, args, packed = s["slots"], s["qkv"], [s[n] for n in ("qw", "kw", "cos", "sin", "pos")], case["packed"]

            def one(i):
                k = torch.empty(T, H_kv, D, dtype=dt, device=DEV) if packed else None
                v = torch.empty(T, H_kv, D, dtype=dt, device=DEV) if packed else None
                q = pool.write_qk_norm_rope(i, slots, qkv[i], *args, EPS, k_out=k, v_out=v)
                return [q, *([k, v] if packed else []), *pool.read_slots(i, slots)]
            s["step"] = lambda: [one(i) for i in range(L)]
    else:
        order = torch.randperm(case["pages"], generator=g)
        s["dst"] = order[: case["moves"]].tolist()
        # a page may be forked more than once; no page is both source and destination
        rest = order[case["moves"]:]
        s["src"] = rest[torch.randint(0, len(rest), (case["moves"],), generator=g)].tolist()
        shape = (case["pages"], case["block"], H_kv, D)
        s["keys"] = [_normal(dg, *shape, dtype=dt) for _ in range(L)]
        s["values"] = [_normal(dg, *shape, dtype=dt) for _ in range(L)]
        if own:
            pool = _package().PagedPool(L, case["pages"], case["block"], H_kv, D, dtype=dt, device=DEV)
            pool.keys, pool.values = s["keys"], s["values"]
            src, dst = s["src"], s["dst"]
            s["step"] = lambda: (pool.copy_blocks(src, dst), pool.keys, pool.values)[1:]
    if own and case.get("graph"):
        s["graph"], s["outs"] = _captured(s["step"])
    return s


# ------------------------------------------------------------------------------- the plain forms
def _quantise(x):
    """(codes, scale bytes) of fp32 rows ``(.., D)``: uint8 ``(.., D)`` and ``(.., D / 32)``."""
    g = x.unflatten(-1, (-1, GROUP))
    most = g.abs().amax(-1)
    mantissa, power = torch.frexp(most)  # most = mantissa * 2^power, mantissa in [0.5, 1): 7 * 2^e = 0.875 * 2^(e + 3)
    e = torch.where(mantissa <= 0.875, power - 3, power - 2).clamp(-120, 125)
    e = torch.where(most == 0, torch.full_like(e, -120), e)
    a = torch.ldexp(g.abs(), -e.unsqueeze(-1))
    code = ((a > 0.25).to(torch.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0))
    code = code + 8 * torch.signbit(g).to(torch.uint8)
    bad = ~torch.isfinite(most)
    code = torch.where(bad.unsqueeze(-1), torch.zeros_like(code), code)
    return code.flatten(-2), torch.where(bad, torch.full_like(e, 255), e + 127).to(torch.uint8)


def _pack(code, scale):
    """Pages ``(.., page_bytes)`` of ``(.., bs, D)`` codes and ``(.., bs, D / 32)`` scale bytes."""
    pairs = code.unflatten(-1, (-1, 2))
    return torch.cat([(pairs[..., 0] | (pairs[..., 1] << 4)).flatten(-2), scale.transpose(-1, -2).flatten(-2)], -1)


def _values(code, scale):
    """fp32 values of codes ``(.., D)`` under scale bytes ``(.., D / 32)``."""
    levels = torch.tensor(LEVELS + tuple(-x for x in LEVELS), device=code.device)
    by = torch.ldexp(torch.ones(1, device=code.device), scale.int() - 127)
    by = torch.where(scale == 255, torch.full_like(by, math.nan), by)
    return (levels[code.int()].unflatten(-1, (-1, GROUP)) * by.unsqueeze(-1)).flatten(-2)


def _unpack(pages, D):
    """fp32 values ``(.., bs, D)`` of pages ``(.., page_bytes)``."""
    block = pages.shape[-1] * GROUP // (D * 17)
    byte = pages[..., : block * D // 2].unflatten(-1, (block, D // 2))
    scale = pages[..., block * D // 2:].unflatten(-1, (D // GROUP, block)).transpose(-1, -2)
    return _values(torch.stack([byte & 15, byte >> 4], -1).flatten(-2), scale)


def _attend(q, kp, vp, table, seqlen):
    """softmax(q K^T / sqrt(D)) V over each row's first seqlen tokens; a row of none gives zeros."""
    B, H, D = q.shape
    H_kv = kp.shape[1]
    k = _unpack(kp[table.long()], D).transpose(1, 2).flatten(2, 3)  # (B, H_kv, tokens, D)
    v = _unpack(vp[table.long()], D).transpose(1, 2).flatten(2, 3)
    out_of = torch.arange(k.shape[2], device=q.device) >= seqlen.view(-1, 1, 1, 1)
    v = torch.where(out_of.transpose(-1, -2), torch.zeros_like(v), v)
    scores = torch.matmul(q.float().view(B, H_kv, H // H_kv, D), k.transpose(-1, -2)) * (1.0 / math.sqrt(D))
    scores = torch.where(out_of, torch.full_like(scores, -math.inf), scores)
    most = scores.amax(-1, True)
    p = torch.exp(scores - torch.where(most == -math.inf, torch.zeros_like(most), most))
    total = p.sum(-1, True)
    out = torch.matmul(p, v) / torch.where(total == 0, torch.ones_like(total), total)
    return out.reshape(B, H, D).to(q.dtype)


def _store(pages, slots, x, block):
    """Rows ``(n, H_kv, D)`` into pages at their slots."""
    D = x.shape[-1]
    code, scale = _quantise(x.float())
    page, at = slots // block, slots % block
    pairs = code.unflatten(-1, (-1, 2))
    pages[..., : block * D // 2].unflatten(-1, (block, D // 2))[page, :, at] = pairs[..., 0] | (pairs[..., 1] << 4)
    pages[..., block * D // 2:].unflatten(-1, (D // GROUP, block))[page, :, :, at] = scale


def _load(pages, slots, block, D, dtype):
    """Rows ``(n, H_kv, D)`` of pages at their slots."""
    page, at = slots // block, slots % block
    byte = pages[..., : block * D // 2].unflatten(-1, (block, D // 2))[page, :, at]
    scale = pages[..., block * D // 2:].unflatten(-1, (D // GROUP, block))[page, :, :, at]
    return _values(torch.stack([byte & 15, byte >> 4], -1).flatten(-2), scale).to(dtype)


def _write_read(pools, i, slots, k, v, block):
    _store(pools[0][i], slots, k, block)
    _store(pools[1][i], slots, v, block)
    return tuple(_load(p[i], slots, block, k.shape[-1], k.dtype) for p in pools)


def _rotated(x, w, cos, sin):
    """RMSNorm times w over the last axis, then the rotation of the halves; rounded once."""
    y = x.float() * torch.rsqrt(x.float().pow(2).mean(-1, True) + EPS) * w.float()
    a, b = y.chunk(2, -1)
    return torch.cat([a * cos - b * sin, a * sin + b * cos], -1).to(x.dtype)


def _epilogue(s, i):
    case = s["case"]
    H, H_kv, D = case["H"], case["H_kv"], case["D"]
    q, k, v = s["qkv"][i].view(-1, H + 2 * H_kv, D).split([H, H_kv, H_kv], 1)
    cos, sin = s["cos"][s["pos"]].float().unsqueeze(1), s["sin"][s["pos"]].float().unsqueeze(1)
    q, k = _rotated(q, s["qw"], cos, sin), _rotated(k, s["kw"], cos, sin)
    held = _write_read(s["pool"], i, s["slots"], k, v, case["block"])
    return [q, *([k, v.contiguous()] if case["packed"] else []), *held]


def _copied(pages, src, dst):
    pages[dst] = pages[src]
    return pages


def run(s):
    case, L = s["case"], s["case"]["layers"]
    if own:
        if s["graph"] is None:
            return s["step"]()
        s["graph"].replay()
        return s["outs"]
    if case["kind"] == "decode":
        return [_attend(s["q"][i], s["k"][i], s["v"][i], s["table"], s["seqlen"]) for i in range(L)]
    if case["kind"] == "write":
        return [_write_read(s["pool"], i, s["slots"], s["k"][i], s["v"][i], case["block"]) for i in range(L)]
    if case["kind"] == "epilogue":
        return [_epilogue(s, i) for i in range(L)]
    src, dst = (torch.tensor(s[name], device=DEV) for name in ("src", "dst"))
    return tuple([_copied(p, src, dst) for p in s[name]] for name in ("keys", "values"))


def work(case):
    H, H_kv, D, L = case["H"], case["H_kv"], case["D"], case["layers"]
    size = 4 if case["dtype"] == "fp32" else 2
    if case["kind"] == "decode":
        tokens = case["B"] * (case["lo"] + case["hi"]) / 2
        per = 2 * tokens * H_kv * D * 17 / 32 + 2 * case["B"] * H * D * size + 4 * tokens / case["block"]
        return {"bytes": L * per, "flops": L * 4 * tokens * H * D}
    if case["kind"] == "copy":
        return {"bytes": 2 * 2 * L * case["moves"] * case["block"] * H_kv * D * size, "flops": 0}
    n = sum(int(x) for x in case["lengths"].split(","))
    rows = 2 * n * H_kv * D
    if case["kind"] == "write":  # read, written in 4 bits, read in 4 bits, written
        return {"bytes": L * rows * (2 * size + 2 * 17 / 32), "flops": 0}
    move = n * (H + 2 * H_kv) * D * size + n * H * D * size + rows * (17 / 32) + (rows * size if case["packed"] else 0)
    return {"bytes": L * (move + rows * (17 / 32 + size)), "flops": L * 10 * n * (H + H_kv) * D}


# ------------------------------------------------------------------------------- in 64 bits
def _exact_row(byte, scale):
    """float64 values of code bytes ``(.., D / 2)`` under scale bytes ``(.., D / 32)``."""
    table = torch.tensor([[s * x for s in (1, -1) for x in LEVELS]], dtype=torch.float64, device=byte.device)[0]
    code = torch.empty(*byte.shape[:-1], byte.shape[-1] * 2, dtype=torch.long, device=byte.device)
    code[..., 0::2], code[..., 1::2] = byte.long() % 16, byte.long() // 16
    return table[code] * (2.0 ** (scale.double() - 127)).repeat_interleave(GROUP, -1)


def _exact_held(x):
    """What the format holds of float64 rows ``(.., D)``: the nearest level, the even code on a tie."""
    g = x.reshape(*x.shape[:-1], -1, GROUP)
    most = g.abs().amax(-1, keepdim=True)
    e = torch.ceil(torch.log2(torch.clamp(most, min=1e-300) / 7)).clamp(-120, 125)
    u = g / 2.0 ** e
    best = torch.zeros_like(u)
    off = torch.full_like(u, math.inf)
    for code in (0, 2, 4, 6, 1, 3, 5, 7):  # even codes first: an odd one has to be strictly nearer
        d = (u.abs() - LEVELS[code]).abs()
        best = torch.where(d < off, torch.full_like(u, LEVELS[code]), best)
        off = torch.minimum(d, off)
    return (torch.sign(u) * best * 2.0 ** e).reshape(x.shape)


def exact(case, seed):
    s = prepare(case, seed)
    H, H_kv, D, L = case["H"], case["H_kv"], case["D"], case["layers"]
    if case["kind"] == "decode":
        outs = []
        block = case["block"]
        for i in range(L):
            out = torch.zeros(case["B"], H, D, dtype=torch.float64, device=DEV)
            for b, n in enumerate(s["seqlen"].tolist()):
                if n == 0:
                    continue
                rows = []
                for cache in (s["k"][i], s["v"][i]):
                    page = cache[s["table"][b, : -(-n // block)].long()]
                    byte = page[:, :, : block * D // 2].reshape(-1, H_kv, block, D // 2)
                    scale = page[:, :, block * D // 2:].reshape(-1, H_kv, D // GROUP, block).permute(0, 1, 3, 2)
                    rows.append(_exact_row(byte, scale).permute(1, 0, 2, 3).reshape(H_kv, -1, D)[:, :n].contiguous())
                q = s["q"][i][b].double().reshape(H_kv, H // H_kv, D)
                w = torch.softmax(torch.bmm(q, rows[0].transpose(1, 2).contiguous()) / math.sqrt(D), -1)
                out[b] = torch.bmm(w, rows[1]).reshape(H, D)
            outs.append(out)
        return outs
    if case["kind"] == "write":
        return [tuple(_exact_held(x.double()) for x in (s["k"][i], s["v"][i])) for i in range(L)]
    if case["kind"] == "epilogue":
        outs = []
        for i in range(L):
            x = s["qkv"][i].double().reshape(-1, H + 2 * H_kv, D)
            angle = [s[name][s["pos"]].double()[:, None, :] for name in ("cos", "sin")]
            made = []
            for part, w in ((x[:, :H], s["qw"]), (x[:, H: H + H_kv], s["kw"])):
                y = part / torch.sqrt((part * part).sum(-1, keepdim=True) / D + EPS) * w.double()
                a, b = y[..., : D // 2], y[..., D // 2:]
                made.append(torch.cat([a * angle[0] - b * angle[1], b * angle[0] + a * angle[1]], -1))
            v = x[:, H + H_kv:]
            # the cache holds what the 16-bit row would have held, so the row is rounded to its type first
            k_row = made[1].to(DTYPES[case["dtype"]]).double()
            outs.append([made[0], *([made[1], v] if case["packed"] else []), _exact_held(k_row), _exact_held(v)])
        return outs
    outs = []
    for name in ("keys", "values"):
        after = [x.clone() for x in s[name]]
        for x, y in zip(s[name], after):
            for a, b in zip(s["src"], s["dst"]):
                y[b] = x[a]
        outs.append([y.double() for y in after])
    return tuple(outs)
