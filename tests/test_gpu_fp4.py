"""The 4-bit paged cache on the GPU: writes, reads and the fused epilogue bit by bit against the 64-bit
oracle's rounding, the attention against the oracle's within bounds derived below, refusals and reports,
captured and replayed calls, other streams, and the operators together as a server uses them.

Attention bound, per output element: the output's own rounding, ``finfo.eps / 2 * |ref|``, and a relative error of
each term p_t v_t times ``sum_t p_t |v_t|``. That error: p_t from a score that is off by its fp32 sum's
rounding, (D + 16) * 2^-24 times ``scale * sum_d |q_d k_td|`` (the sum itself, and the product with
the scale and the subtraction of the maximum, each 2^-24 of at most that); twice, for the term and for the total; the
exponential's own 2^-22; p_t cut to bf16 parts, the last one truncated, 2^-14 with two parts (fp16, bf16) and 2^-22
with three (fp32); fp32 sums over n tokens, n * 2^-24 each for the terms and the total.
"""

from __future__ import annotations

import math

import pytest
import torch

from miattn import Fp4PagedPool, PackedPrefill, PagedKV, PagedPool, _lib, paged_decode_fp4, paged_decode_fp4_plan
from miattn.fp4 import page_bytes
from miattn.qwen3 import GraphDecoder, Qwen3, Qwen3Config, random_weights
from miattn.rows import Parts
from miattn.serve import BlockFreeList, ContinuousServer, poisson_trace
from oracle import fp4 as oracle

pytestmark = pytest.mark.gpu
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _half_step(size, dtype):
    """What rounding values of this size to ``dtype`` is off by at most: ``eps / 2`` of the size, and below the
    smallest normal number, where the type's steps no longer shrink (fp16: 2^-24 apart under 2^-14), half
    of that step, ``smallest_normal * eps / 2``."""
    info = torch.finfo(dtype)
    return info.eps / 2 * size.clamp(min=info.smallest_normal)


def _assert_within(got, want, bound):
    got = got.cpu().double()
    share = ((got - want).abs() / bound).nan_to_num(nan=math.inf)
    at = share.flatten().argmax()
    assert share.max() <= 1, (f"{int((share > 1).sum())} of {share.numel()} off; element {at.item()} is {got.flatten()[at]:.9g}, "
                              f"want {want.flatten()[at]:.9g} +- {bound.flatten()[at]:.3g}")


# ------------------------------------------------------------------ writes and reads
def _hard_rows(n, H_kv, D, dtype, seed):
    """N(0, 1) rows with what is hard among them: ties and scale borders, zeros of both signs, values
    that are not finite, the type's largest and smallest, one outlier in a group."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(n, H_kv, D, generator=g)
    ties = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 7.0, -0.25, -0.75, -5.0, 0.0, -0.0, 6.5, 1.0])
    x[0, 0, :16], x[0, 0, 16:32] = ties, -ties
    x[0, -1] = 0.0
    x[1 % n, 0, :32] = ties.repeat(2) * 2.0 ** -9
    x = x.to(dtype)
    info = torch.finfo(dtype)
    if n > 3:
        x[2, 0, 3], x[2, -1, -1] = float("nan"), float("inf")
        x[3, 0, 0], x[3, 0, 1], x[3, -1, 40 % D] = info.max, info.max / 3, -info.max
        x[3, 0, 32:] = info.smallest_normal * x[3, 0, 32:].float().abs().clamp(max=4).to(dtype)
    if n > 4:
        x[4, 0, 7] = 300.0
    return x


def _want_pages(pool, before, slots, rows):
    """The pages ``before`` with ``rows`` at ``slots``, byte by byte from the oracle."""
    bs, D = pool.block_size, pool.head_dim
    codes, scales = oracle.encode(rows)
    want = before.clone().cpu()
    for i, s in enumerate(slots):
        page, at = divmod(int(s), bs)
        want[page, :, at * D // 2: (at + 1) * D // 2] = codes[i, :, 0::2] | (codes[i, :, 1::2] << 4)
        for grp in range(D // 32):
            want[page, :, bs * D // 2 + grp * bs + at] = scales[i, :, grp]
    return want


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("H_kv,D,bs", [(8, 128, 16), (1, 64, 32), (3, 256, 16), (2, 64, 128)])
@pytest.mark.parametrize("layout", ["contiguous", "permuted", "strided", "misaligned"])
def test_write_slots_stores_the_oracles_bytes_and_read_slots_returns_them(dtype, H_kv, D, bs, layout, cuda):
    dt, n = DTYPES[dtype], 13
    k, v = _hard_rows(n, H_kv, D, dt, 1), _hard_rows(n, H_kv, D, dt, 2)
    pool = Fp4PagedPool(2, 5, bs, H_kv, D, dtype=dt, device=cuda)
    for store in pool.keys + pool.values:
        store.random_(0, 256)
    before = [s.clone() for s in pool.keys + pool.values]
    slots = torch.randperm(pool.n_slots, generator=torch.Generator().manual_seed(3))[:n]

    def placed(x):
        if layout == "permuted":
            return x.permute(1, 0, 2).contiguous().cuda().permute(1, 0, 2)
        if layout == "strided":
            wide = torch.zeros(*x.shape[:2], 2 * D, dtype=dt, device=cuda)
            wide[..., ::2] = x.cuda()
            return wide[..., ::2]
        if layout == "misaligned":
            flat = torch.zeros(x.numel() + 1, dtype=dt, device=cuda)
            flat[1:] = x.reshape(-1).cuda()
            return flat[1:].view(x.shape)
        return x.cuda()

    slot_dtype = torch.int32 if layout in ("strided", "permuted") else torch.int64
    pool.write_slots(1, slots.to(slot_dtype).cuda(), placed(k), placed(v))
    pool.check_writes()
    for got, old, rows in ((pool.keys, before[1], k), (pool.values, before[3], v)):
        assert torch.equal(got[1].cpu(), _want_pages(pool, old, slots, rows))
    assert torch.equal(pool.keys[0], before[0]) and torch.equal(pool.values[0], before[2])
    again = torch.cat([slots, slots[:3]])  # repeats may be read
    for got, rows in zip(pool.read_slots(1, again.to(slot_dtype).cuda()), (k, v)):
        want = oracle.held(rows)[torch.cat([torch.arange(n), torch.arange(3)])]
        if dt == torch.float16:
            want = torch.where(want.isnan(), want, want.clamp(-65504, 65504))
        assert torch.equal(got.cpu().isnan(), want.isnan())
        assert torch.equal(got.cpu().double().nan_to_num(), want.to(dt).double().nan_to_num())
    pool.check_writes()


@pytest.mark.parametrize("n", [0, 1, 2, 65, 8191, 8197])
def test_write_of_no_few_and_many_tokens(n, cuda):
    pool = Fp4PagedPool(1, max(8, n // 8), 16, 2, 128, dtype=torch.bfloat16, device=cuda)
    k, v = torch.randn(n, 2, 128).bfloat16(), torch.randn(n, 2, 128).bfloat16()
    slots = torch.randperm(pool.n_slots)[:n]
    pool.write_slots(0, slots.cuda(), k.cuda(), v.cuda())
    got_k, got_v = pool.read_slots(0, slots.cuda())
    assert got_k.shape == k.shape
    pool.check_writes()
    if 0 < n < 100:
        assert torch.equal(got_k.cpu().double(), oracle.held(k)) and torch.equal(got_v.cpu().double(), oracle.held(v))


def test_many_tokens_are_stored_as_the_same_tokens_one_call_at_a_time(cuda):
    """Large calls work on two rows per lane: the same bytes as small ones, a bad slot among them skipped."""
    n, H_kv, D = 9001, 3, 128
    k, v = torch.randn(n, H_kv, D).half().cuda(), torch.randn(n, H_kv, D).half().cuda()
    pools = [Fp4PagedPool(1, 600, 16, H_kv, D, dtype=torch.float16, device=cuda) for _ in range(2)]
    slots = torch.randperm(9600, generator=torch.Generator().manual_seed(0))[:n].cuda()
    slots[4321] = 9600
    pools[0].write_slots(0, slots, k, v)
    with pytest.raises(IndexError, match="token 4321 of"):
        pools[0].check_writes()
    for a in range(0, n, 500):
        pools[1].write_slots(0, slots[a: a + 500], k[a: a + 500], v[a: a + 500])
    assert torch.equal(pools[0].keys[0], pools[1].keys[0]) and torch.equal(pools[0].values[0], pools[1].values[0])
    whole = pools[0].read_slots(0, slots)
    for a in range(0, n, 500):
        part = pools[0].read_slots(0, slots[a: a + 500])
        assert all(torch.equal(x[a: a + 500], y) for x, y in zip(whole, part))
    assert not whole[0][4321].any() and whole[0][4320].any()


def test_out_of_range_slots_are_skipped_and_reported(cuda):
    pool = Fp4PagedPool(1, 2, 16, 2, 64, dtype=torch.float16, device=cuda)
    rows = torch.randn(4, 2, 64).half().cuda()
    pool.write_slots(0, torch.tensor([3, 32, -1, 5], device=cuda), rows, rows)
    with pytest.raises(IndexError, match="token [12] of"):
        pool.check_writes()
    pool.check_writes()  # read and cleared
    k, v = pool.read_slots(0, torch.tensor([3, 5], device=cuda))
    assert torch.equal(k.double().cpu(), oracle.held(rows[[0, 3]])) and torch.equal(k, v)
    k, v = pool.read_slots(0, torch.tensor([32, 3, -7], device=cuda, dtype=torch.int32))
    assert not k[0].any() and not v[2].any() and k[1].any()
    with pytest.raises(IndexError, match="token [02] of"):
        pool.check_writes()
    strict = Fp4PagedPool(1, 2, 16, 2, 64, dtype=torch.float16, device=cuda, strict_writes=True)
    with pytest.raises(IndexError, match="token 0 of"):
        strict.write_slots(0, torch.tensor([99], device=cuda), rows[:1], rows[:1])


def test_write_and_read_refusals(cuda):
    pool = Fp4PagedPool(1, 2, 16, 2, 64, dtype=torch.bfloat16, device=cuda)
    rows = torch.zeros(2, 2, 64, dtype=torch.bfloat16, device=cuda)
    with pytest.raises(ValueError, match="one entry per token"):
        pool.write_slots(0, torch.zeros(3, dtype=torch.long, device=cuda), rows, rows)
    with pytest.raises(ValueError, match="head shape"):
        pool.write_slots(0, torch.zeros(2, dtype=torch.long, device=cuda), rows[..., :32], rows[..., :32])
    with pytest.raises(RuntimeError, match="takes k/v there"):
        pool.write_slots(0, torch.zeros(2, dtype=torch.long, device=cuda), rows.cpu(), rows.cpu())
    with pytest.raises(ValueError, match="slot_ids are on cpu"):
        pool.read_slots(0, torch.zeros(2, dtype=torch.long))
    with pytest.raises(ValueError, match="integer tensor"):
        pool.read_slots(0, torch.zeros(2, device=cuda))
    with pytest.raises(ValueError, match="must be 1-D"):
        pool.read_slots(0, torch.zeros(2, 1, dtype=torch.long, device=cuda))
    with pytest.raises(IndexError, match="layer 1 is outside"):
        pool.read_slots(1, torch.zeros(2, dtype=torch.long, device=cuda))


# ------------------------------------------------------------------ the fused epilogue
def _epilogue_case(B, H, H_kv, D, rotary, dt, seed, n_pos=4000):
    g = torch.Generator().manual_seed(seed)
    qkv = (torch.randn(B, (H + 2 * H_kv) * D, generator=g) * 2.0).to(dt)
    qw, kw = ((1.0 + 0.1 * torch.randn(D, generator=g)).to(dt) for _ in range(2))
    angle = torch.outer(torch.arange(n_pos).double(), 1e6 ** -(torch.arange(0, rotary, 2).double() / rotary))
    pos = torch.randint(0, n_pos, (B,), generator=g)
    return qkv, qw, kw, angle.cos().to(dt), angle.sin().to(dt), pos


def _epilogue_exact(x, w, cos, sin, rotary, eps, zero_centred):
    """(rotated, size) of heads ``(B, heads, D)`` in float64; size bounds the terms of each element's sum."""
    x, w = x.double(), w.double()
    y = x / torch.sqrt(x.pow(2).mean(-1, True) + eps) * (1 + w if zero_centred else w)
    a, b, rest = y[..., : rotary // 2], y[..., rotary // 2: rotary], y[..., rotary:]
    c, s = cos.double().unsqueeze(1), sin.double().unsqueeze(1)
    out = torch.cat([a * c - b * s, b * c + a * s, rest], -1)
    size = torch.cat([(a * c).abs() + (b * s).abs(), (b * c).abs() + (a * s).abs(), rest.abs()], -1)
    return out, size


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("B,H,H_kv,D,rotary,zero_centred", [
    (1, 16, 8, 128, 128, False), (33, 16, 8, 128, 128, False), (5, 8, 2, 256, 64, True), (7, 3, 3, 64, 64, False),
    (1500, 4, 2, 128, 64, False), (9, 5, 1, 256, 256, True), (6, 8, 2, 256, 128, False)])
def test_epilogue_rounds_once_and_stores_what_a_write_of_its_k_would(dtype, B, H, H_kv, D, rotary, zero_centred, cuda):
    dt, eps = DTYPES[dtype], 1e-6
    qkv, qw, kw, cos, sin, pos = _epilogue_case(B, H, H_kv, D, rotary, dt, seed=B + D)
    pool = Fp4PagedPool(1, -(-B // 16) + 2, 16, H_kv, D, dtype=dt, device=cuda, n_head=H, strict_writes=True)
    other = Fp4PagedPool(1, pool.n_blocks, 16, H_kv, D, dtype=dt, device=cuda, n_head=H, strict_writes=True)
    slots = torch.randperm(pool.n_slots, generator=torch.Generator().manual_seed(B))[:B].cuda()
    k_out, v_out = (torch.empty(B, H_kv, D, dtype=dt, device=cuda) for _ in range(2))
    args = [t.cuda() for t in (qw, kw, cos, sin, pos)]
    q = pool.write_qk_norm_rope(0, slots, qkv.cuda(), *args, eps, k_out=k_out, v_out=v_out, rotary_dim=rotary,
                                zero_centred_norm=zero_centred)
    heads = qkv.view(B, H + 2 * H_kv, D)
    for got, x, w in ((q, heads[:, :H], qw), (k_out, heads[:, H: H + H_kv], kw)):
        want, size = _epilogue_exact(x, w, cos[pos], sin[pos], rotary, eps, zero_centred)
        # the norm's sum (8 + 5 levels), root, reciprocal and products: below 2^-19 of the terms; then one rounding
        bound = _half_step(want.abs(), dt) + 2.0 ** -19 * size * (1 + torch.finfo(dt).eps)
        _assert_within(got, want, bound)
    assert torch.equal(v_out.cpu(), heads[:, H + H_kv:])
    other.write_slots(0, slots, k_out, v_out)
    assert torch.equal(pool.keys[0], other.keys[0]) and torch.equal(pool.values[0], other.values[0])
    # without the packed copies, from int32 slots: the same q and pool
    third = Fp4PagedPool(1, pool.n_blocks, 16, H_kv, D, dtype=dt, device=cuda, n_head=H, strict_writes=True)
    q2 = third.write_qk_norm_rope(0, slots.int(), qkv.cuda(), *args, eps, rotary_dim=rotary,
                                  zero_centred_norm=zero_centred)
    assert torch.equal(q, q2) and torch.equal(third.keys[0], pool.keys[0]) and torch.equal(third.values[0], pool.values[0])


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("B,H,H_kv,D,rotary,zero_centred", [
    (3, 16, 8, 128, 128, False), (700, 8, 2, 256, 64, True), (700, 16, 16, 64, 64, False), (7, 24, 2, 128, 64, False)])
def test_epilogue_gives_the_bits_of_fp32_tensor_operations(dtype, B, H, H_kv, D, rotary, zero_centred, cuda):
    """So a k next to a border between two 4-bit levels is stored as the level that those operations give."""
    dt, eps = DTYPES[dtype], 1e-6
    qkv, qw, kw, cos, sin, pos = (t.cuda() for t in _epilogue_case(B, H, H_kv, D, rotary, dt, seed=7 * B + D))
    pool = Fp4PagedPool(1, -(-B // 16), 16, H_kv, D, dtype=dt, device=cuda, n_head=H, strict_writes=True)
    k_out = torch.empty(B, H_kv, D, dtype=dt, device=cuda)
    q = pool.write_qk_norm_rope(0, torch.arange(B, device=cuda), qkv, qw, kw, cos, sin, pos, eps, k_out=k_out,
                                rotary_dim=rotary, zero_centred_norm=zero_centred)
    heads = qkv.view(B, H + 2 * H_kv, D)
    c, s = cos[pos].float().unsqueeze(1), sin[pos].float().unsqueeze(1)
    for got, x, w in ((q, heads[:, :H].float(), qw.float()), (k_out, heads[:, H: H + H_kv].float(), kw.float())):
        y = x * torch.rsqrt(x.pow(2).mean(-1, True) + eps) * (1 + w if zero_centred else w)
        a, b, rest = y[..., : rotary // 2], y[..., rotary // 2: rotary], y[..., rotary:]
        assert torch.equal(got, torch.cat([a * c - b * s, a * s + b * c, rest], -1).to(dt))


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("parts", [1, 2, 3, 9])
def test_epilogue_of_partial_sums_is_that_of_their_rounded_sum(dtype, parts, cuda):
    dt, B, H, H_kv, D = DTYPES[dtype], 6, 4, 2, 128
    _, *rest = _epilogue_case(B, H, H_kv, D, D, dt, seed=parts)
    args = [t.cuda() for t in rest]
    sums = Parts(torch.randn(parts, B, (H + 2 * H_kv) * D, device=cuda), dt)
    slots = torch.arange(B, device=cuda) * 3
    pools = [Fp4PagedPool(1, 2, 16, H_kv, D, dtype=dt, device=cuda, n_head=H, strict_writes=True) for _ in range(2)]
    a = pools[0].write_qk_norm_rope(0, slots, sums, *args, 1e-6)
    b = pools[1].write_qk_norm_rope(0, slots, sums.value(), *args, 1e-6)
    assert torch.equal(a, b) and torch.equal(pools[0].keys[0], pools[1].keys[0])
    assert torch.equal(pools[0].values[0], pools[1].values[0])


def test_epilogue_takes_longer_and_misaligned_rows(cuda):
    B, H, H_kv, D = 5, 4, 2, 128
    qkv, *rest = _epilogue_case(B, H, H_kv, D, D, torch.bfloat16, seed=4)
    args = [t.cuda() for t in rest]
    slots = torch.arange(B, device=cuda)
    outs = []
    for shift, extra in ((0, 0), (0, 64), (0, 3), (1, 0)):
        pool = Fp4PagedPool(1, 1, 16, H_kv, D, dtype=torch.bfloat16, device=cuda, n_head=H)
        flat = torch.full((B * (qkv.shape[1] + extra) + shift,), float("nan"), dtype=torch.bfloat16, device=cuda)
        row = flat[shift:].view(B, -1)[:, : qkv.shape[1]]
        row.copy_(qkv)
        outs.append((pool.write_qk_norm_rope(0, slots, row, *args, 1e-6), pool.keys[0], pool.values[0]))
    for other in outs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(outs[0], other))


def test_epilogue_idle_and_refused_rows_write_nothing_and_return_zeros(cuda):
    B, H, H_kv, D = 6, 4, 2, 64
    qkv, *rest, pos = _epilogue_case(B, H, H_kv, D, D, torch.bfloat16, seed=9, n_pos=50)
    args = [t.cuda() for t in rest]
    pos[1], pos[2] = 50, -1
    slots = torch.tensor([0, 1, 2, -1, 16, 5])
    pool = Fp4PagedPool(1, 1, 16, H_kv, D, dtype=torch.bfloat16, device=cuda, n_head=H)
    pool.keys[0].fill_(0x11)
    k_out, v_out = (torch.full((B, H_kv, D), 7.0, dtype=torch.bfloat16, device=cuda) for _ in range(2))
    q = pool.write_qk_norm_rope(0, slots.cuda(), qkv.cuda(), *args, pos.cuda(), 1e-6, k_out=k_out, v_out=v_out)
    for out in (q, k_out, v_out):
        assert not out[1:5].any() and out[0].any() and out[5].any()
    k, _ = pool.read_slots(0, torch.arange(16, device=cuda))
    untouched = [i for i in range(16) if i not in (0, 5)]
    assert (pool.keys[0].view(1, H_kv, -1)[0, :, : 16 * D // 2].view(H_kv, 16, -1)[:, untouched] == 0x11).all()
    assert torch.equal(k[[0, 5]].cpu().double(), oracle.held(k_out[[0, 5]]))
    with pytest.raises(IndexError, match="token [124] of"):
        pool.check_writes()
    none = pool.write_qk_norm_rope(0, slots[:0].cuda(), qkv[:0].cuda(), *args, pos[:0].cuda(), 1e-6)
    assert none.shape == (0, H, D)
    idle = torch.full((B,), -1, device=cuda)
    assert not pool.write_qk_norm_rope(0, idle, qkv.cuda(), *args, pos.cuda(), 1e-6).any()
    pool.check_writes()  # idle seats report nothing


# ------------------------------------------------------------------ the attention
def _pool_case(lengths, H, H_kv, D, bs, dt, seed, *, spare=3, scale=1.0, garbage=True):
    """A pool whose rows hold N(0, scale) tokens, tables of a random permutation padded with -1, and q.
    Every byte that belongs to no token is garbage, NaN scales among it."""
    g = torch.Generator().manual_seed(seed)
    need = [-(-n // bs) for n in lengths]
    n_blocks = sum(need) + spare
    pool = Fp4PagedPool(1, n_blocks, bs, H_kv, D, dtype=dt, device="cuda", n_head=H)
    if garbage:
        for store in pool.keys + pool.values:
            store.random_(0, 256)
            store[..., bs * D // 2:].fill_(255)
    perm = torch.randperm(n_blocks, generator=g).tolist()
    table = torch.full((len(lengths), max(1, max(need)) + 1), -1, dtype=torch.int32)
    at = 0
    for r, (n, m) in enumerate(zip(lengths, need)):
        ids, at = perm[at: at + m], at + m
        table[r, :m] = torch.tensor(ids, dtype=torch.int32)
        if n:
            k, v = (torch.randn(n, H_kv, D, generator=g) * scale for _ in range(2))
            pool.write_prefill(0, ids, 0, k.to(dt).cuda(), v.to(dt).cuda())
    q = torch.randn(len(lengths), H, D, generator=g).to(dt)
    return pool, q.cuda(), table.cuda(), torch.tensor(lengths, dtype=torch.int32, device="cuda")


def _within(got, q, pool, table, seqlen, scale=None, layer=0):
    want, weight, spread = oracle.paged_attention(q, pool.keys[layer], pool.values[layer], table, seqlen, scale)
    dt, D, n = q.dtype, q.shape[2], max(1, int(seqlen.max()))
    parts = 2.0 ** -22 if dt == torch.float32 else 2.0 ** -14
    each = 2 * (D + 16) * 2.0 ** -24 * spread + 2.0 ** -21 + parts + 2 * n * 2.0 ** -24
    bound = _half_step(want.abs() + each * weight, dt) + each * weight + LOST
    _assert_within(got, want, bound)


# Terms whose p_t is below 2^-126 of the row's largest, the smallest normal fp32 number, count as nothing: at most
# 2^13 tokens of at most 2^13 each here.
LOST = 2.0 ** -100
LENGTHS = [[1], [0, 0, 0], [5, 0, 16, 17, 31, 32, 33, 1], [63, 64, 65, 127, 128, 129, 0, 500], [2047, 3, 700], [4100]]


@pytest.mark.parametrize("lengths", LENGTHS, ids=lambda x: "-".join(map(str, x)))
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("H,H_kv,D,bs", [(16, 8, 128, 16), (8, 2, 256, 32), (4, 4, 64, 16)])
def test_decode_matches_the_oracle(lengths, dtype, H, H_kv, D, bs, cuda):
    pool, q, table, seqlen = _pool_case(lengths, H, H_kv, D, bs, DTYPES[dtype], seed=len(lengths) + D)
    out = paged_decode_fp4(q, pool.keys[0], pool.values[0], table, seqlen)
    _within(out, q, pool, table, seqlen)
    for r, n in enumerate(lengths):
        if n == 0:
            assert not out[r].any()


@pytest.mark.parametrize("H,H_kv", [(1, 1), (3, 1), (5, 1), (7, 1), (8, 1), (9, 1), (12, 2), (16, 1), (17, 1), (40, 2), (64, 1), (10, 5)])
@pytest.mark.parametrize("dtype,D", [("bf16", 128), ("fp16", 64), ("fp32", 128), ("bf16", 256)])
def test_decode_of_every_head_group(H, H_kv, dtype, D, cuda):
    pool, q, table, seqlen = _pool_case([300, 0, 1, 77], H, H_kv, D, 16, DTYPES[dtype], seed=H)
    _within(paged_decode_fp4(q, pool.keys[0], pool.values[0], table, seqlen), q, pool, table, seqlen)


@pytest.mark.parametrize("n", [255, 256, 257, 383, 385, 511, 512, 513, 767, 768, 769, 1023, 1024, 1025, 1537, 2049, 3000])
@pytest.mark.parametrize("H,H_kv,D,dtype", [(16, 8, 128, "bf16"), (8, 2, 256, "fp16"), (16, 1, 256, "bf16"), (4, 4, 64, "fp32")])
def test_decode_around_the_lengths_where_rows_are_cut(n, H, H_kv, D, dtype, cuda):
    """One row alone, and beside others that share the chip with it."""
    for others in ([], [2300, 130, 0, 900]):
        pool, q, table, seqlen = _pool_case([n, *others], H, H_kv, D, 16, DTYPES[dtype], seed=n)
        _within(paged_decode_fp4(q, pool.keys[0], pool.values[0], table, seqlen), q, pool, table, seqlen)


@pytest.mark.parametrize("bs", [16, 32, 64, 128, 512])
def test_decode_of_every_page_size(bs, cuda):
    pool, q, table, seqlen = _pool_case([1, bs - 1, bs, bs + 1, 3 * bs + 5], 8, 4, 128, bs, torch.bfloat16, seed=bs)
    _within(paged_decode_fp4(q, pool.keys[0], pool.values[0], table, seqlen), q, pool, table, seqlen)


@pytest.mark.parametrize("B", [64, 65, 130, 300])
def test_decode_of_many_rows(B, cuda):
    g = torch.Generator().manual_seed(B)
    lengths = torch.randint(0, 200, (B,), generator=g).tolist()
    pool, q, table, seqlen = _pool_case(lengths, 8, 2, 64, 16, torch.bfloat16, seed=B)
    _within(paged_decode_fp4(q, pool.keys[0], pool.values[0], table, seqlen), q, pool, table, seqlen)


@pytest.mark.parametrize("scale", [0.0, 1.0, 30.0, -2.0])
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_decode_with_other_scales(scale, dtype, cuda):
    """No scale (a mean over the tokens), a sharp softmax, and a negative one."""
    pool, q, table, seqlen = _pool_case([200, 33], 4, 2, 128, 16, DTYPES[dtype], seed=7)
    out = paged_decode_fp4(q, pool.keys[0], pool.values[0], table, seqlen, scale=scale)
    want, weight, spread = oracle.paged_attention(q, pool.keys[0], pool.values[0], table, seqlen, scale)
    each = 2 * 144 * 2.0 ** -24 * spread.abs().amax() * 2 + 2.0 ** -13
    _assert_within(out, want, _half_step(want.abs(), q.dtype) + 2 * each * weight + LOST)


def test_decode_scores_that_grow_and_fall_along_the_row(cuda):
    """The running maximum moves up tile after tile, or never again after the first."""
    H, H_kv, D, n = 4, 2, 128, 700
    for flip in (False, True):
        pool, q, table, seqlen = _pool_case([n], H, H_kv, D, 16, torch.bfloat16, seed=3)
        k = torch.randn(n, H_kv, D) * torch.linspace(0.01, 6, n).view(-1, 1, 1)
        k = k + q[0, ::2].float().cpu() * torch.linspace(-3, 3, n).view(-1, 1, 1)
        k = k.flip(0) if flip else k
        ids = table[0][: -(-n // 16)].tolist()
        pool.write_prefill(0, ids, 0, k.bfloat16().cuda(), torch.randn(n, H_kv, D).bfloat16().cuda())
        _within(paged_decode_fp4(q, pool.keys[0], pool.values[0], table, seqlen), q, pool, table, seqlen)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_decode_of_large_and_small_values(dtype, cuda):
    for size in (2.0 ** -14, 2.0 ** 9):
        pool, q, table, seqlen = _pool_case([130, 20], 4, 2, 128, 16, DTYPES[dtype], seed=5, scale=size)
        _within(paged_decode_fp4(q, pool.keys[0], pool.values[0], table, seqlen, scale=1.0 / size / 11), q, pool, table,
                seqlen, scale=1.0 / size / 11)


def test_a_poisoned_token_reaches_only_the_heads_that_read_it(cuda):
    """NaN in a K row makes its KV head's queries NaN, NaN in a V group the elements of that group; other heads
    and rows, and the same token past a row's end, stay as they are."""
    H, H_kv, D, n = 4, 2, 128, 50
    pool, q, table, seqlen = _pool_case([n, n], H, H_kv, D, 16, torch.bfloat16, seed=8)
    clean = paged_decode_fp4(q, pool.keys[0], pool.values[0], table, seqlen)
    ids = table[0][:4].tolist()
    row_k, row_v = pool.read_slots(0, pool.slot_ids(ids, 20, 1))
    bad = row_v.clone()
    bad[0, 1, 70] = float("nan")
    pool.write_prefill(0, ids, 20, row_k, bad)
    out = paged_decode_fp4(q, pool.keys[0], pool.values[0], table, seqlen)
    assert out[0, 2:, 64:96].isnan().all()
    keep = torch.ones_like(out, dtype=torch.bool)
    keep[0, 2:, 64:96] = False
    assert torch.equal(out[keep], clean[keep])
    short = seqlen.clone()
    short[0] = 20
    assert not paged_decode_fp4(q, pool.keys[0], pool.values[0], table, short).isnan().any()
    bad = row_k.clone()
    bad[0, 0, 3] = float("inf")
    pool.write_prefill(0, ids, 20, bad, row_v)
    out = paged_decode_fp4(q, pool.keys[0], pool.values[0], table, seqlen)
    assert out[0, :2].isnan().all() and torch.equal(out[0, 2:], clean[0, 2:]) and torch.equal(out[1], clean[1])


def test_decode_of_strided_inputs(cuda):
    """A query cut from a packed projection, a table with spare columns, int64 lengths, a pool that is a
    slice of a larger one."""
    pool, q, table, seqlen = _pool_case([100, 40, 0], 8, 4, 128, 16, torch.bfloat16, seed=2)
    want = paged_decode_fp4(q, pool.keys[0], pool.values[0], table, seqlen)
    packed = torch.zeros(3, 8 * 128 + 40, dtype=torch.bfloat16, device=cuda)
    packed[:, 8: 8 + 1024] = q.view(3, -1)
    view = packed[:, 8: 8 + 1024].view(3, 8, 128)
    odd = packed.view(-1)[1:1 + 1024].view(1, 8, 128).expand(3, 8, 128).clone()  # misaligned source, cloned by torch
    wide = torch.full((3, 2 * table.shape[1]), -5, dtype=torch.int32, device=cuda)
    wide[:, ::2] = table
    assert torch.equal(paged_decode_fp4(view, pool.keys[0], pool.values[0], table, seqlen.long()), want)
    assert torch.equal(paged_decode_fp4(q, pool.keys[0], pool.values[0], wide[:, ::2], seqlen), want)
    flat = torch.zeros(1025, dtype=torch.bfloat16, device=cuda)
    flat[1:] = q[:1].reshape(-1)
    got = paged_decode_fp4(flat[1:].view(1, 8, 128), pool.keys[0], pool.values[0], table[:1], seqlen[:1])
    assert torch.equal(got, paged_decode_fp4(q[:1], pool.keys[0], pool.values[0], table[:1], seqlen[:1]))
    assert odd.shape == (3, 8, 128)
    heads = torch.zeros(pool.n_blocks, 9, pool.keys[0].shape[2], dtype=torch.uint8, device=cuda)
    heads[:, 2:6] = pool.keys[0]
    values = torch.zeros_like(heads)
    values[:, 2:6] = pool.values[0]
    assert torch.equal(paged_decode_fp4(q, heads[:, 2:6], values[:, 2:6], table, seqlen), want)
    with pytest.raises(ValueError, match="aligned pages"):
        shifted = torch.zeros(pool.keys[0].numel() + 8, dtype=torch.uint8, device=cuda)[8:].view(pool.keys[0].shape)
        paged_decode_fp4(q, shifted, pool.values[0], table, seqlen)
    empty = paged_decode_fp4(q[:0], pool.keys[0], pool.values[0], table[:0], seqlen[:0])
    assert empty.shape == (0, 8, 128)


def test_plan_runs_layers_sees_seqlen_and_refuses_other_queries(cuda):
    pool, q, table, seqlen = _pool_case([90, 0, 33], 8, 4, 128, 16, torch.bfloat16, seed=6)
    plan = paged_decode_fp4_plan(q, [pool.keys[0], pool.values[0]], [pool.values[0], pool.keys[0]], table, seqlen)
    assert torch.equal(plan.run(0, q), paged_decode_fp4(q, pool.keys[0], pool.values[0], table, seqlen))
    assert torch.equal(plan.run(1, q), paged_decode_fp4(q, pool.values[0], pool.keys[0], table, seqlen))
    seqlen.copy_(torch.tensor([17, 0, 2], dtype=torch.int32))
    assert torch.equal(plan.run(0, q), paged_decode_fp4(q, pool.keys[0], pool.values[0], table, seqlen.clone()))
    assert not plan.fused_supported(torch.bfloat16, 128)
    with pytest.raises(IndexError, match="layer 2"):
        plan.run(2, q)
    with pytest.raises(ValueError, match="does not match the validated layout"):
        plan.run(0, q[:, :4])
    with pytest.raises(ValueError, match="int32 seqlen"):
        paged_decode_fp4_plan(q, [pool.keys[0]], [pool.values[0]], table, seqlen.long())
    with pytest.raises(ValueError, match="one pool shape"):
        paged_decode_fp4_plan(q, [pool.keys[0], pool.keys[0][:-1]], [pool.values[0], pool.values[0][:-1]], table, seqlen)
    with pytest.raises(ValueError, match="at least one row"):
        paged_decode_fp4_plan(q[:0], [pool.keys[0]], [pool.values[0]], table[:0], seqlen[:0])


def test_decode_never_leaves_the_table_width(cuda):
    """A plan reads seqlen in place: a length past the table's capacity attends over the capacity only, and a
    negative one over nothing."""
    pool, q, table, seqlen = _pool_case([64, 48], 4, 2, 64, 16, torch.bfloat16, seed=1)
    table = table[:, :4].contiguous()
    table[1, 3] = table[1, 0]
    plan = paged_decode_fp4_plan(q, [pool.keys[0]], [pool.values[0]], table, seqlen)
    seqlen.copy_(torch.tensor([1000, -3], dtype=torch.int32))
    out = plan.run(0, q)
    assert not out[1].any()
    _within(out[:1], q[:1], pool, table[:1], torch.tensor([64], dtype=torch.int32))


@pytest.mark.parametrize("lengths", [[40, 0, 200], [3000, 17, 900, 64]], ids=["short", "long"])
def test_captured_step_replays_with_new_tokens_and_lengths(lengths, cuda):
    """Epilogue and attention in one graph, replayed several times with the program's own eager work and
    synchronisations between; every replay equals the eager calls on a second pool."""
    H, H_kv, D, B = 8, 4, 128, len(lengths)
    room = [n + 8 for n in lengths]
    pool, q, table, _ = _pool_case(room, H, H_kv, D, 16, torch.bfloat16, seed=11, garbage=False)
    twin = Fp4PagedPool(1, pool.n_blocks, 16, H_kv, D, dtype=torch.bfloat16, device=cuda, n_head=H)
    qkv, *rest, _ = _epilogue_case(B, H, H_kv, D, D, torch.bfloat16, seed=2)
    args, qkv = [t.cuda() for t in rest], qkv.cuda()
    pos = torch.tensor(lengths, device=cuda)
    slots = torch.zeros(B, dtype=torch.long, device=cuda)
    seqlen = torch.zeros(B, dtype=torch.int32, device=cuda)
    plan = pool.decode_plan(q, table, seqlen)

    def set_step(i):
        at = [n + i for n in lengths]
        slots.copy_(torch.tensor([int(table[r, p // 16]) * 16 + p % 16 for r, p in enumerate(at)]))
        pos.copy_(torch.tensor(at))
        seqlen.copy_(torch.tensor([p + 1 for p in at], dtype=torch.int32))
        qkv.copy_(torch.randn(qkv.shape, generator=torch.Generator().manual_seed(i)))

    def step():
        return plan.run(0, pool.write_qk_norm_rope(0, slots, qkv, *args, pos, 1e-6))

    set_step(0)
    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    twin.keys[0].copy_(pool.keys[0])
    twin.values[0].copy_(pool.values[0])
    for i in range(1, 7):
        set_step(i)
        graph.replay()
        if i % 2:
            torch.cuda.synchronize()
        eager_q = twin.write_qk_norm_rope(0, slots, qkv, *args, pos, 1e-6)
        want = paged_decode_fp4(eager_q, twin.keys[0], twin.values[0], table, seqlen.clone())
        junk = torch.randn(1 << 20, device=cuda).sum()
        assert torch.equal(out, want) and torch.equal(pool.keys[0], twin.keys[0]) and torch.isfinite(junk)
        _within(out, eager_q, pool, table, seqlen)


def test_captured_one_shot_call_brings_its_own_zeroed_workspace(cuda):
    """Two graphs of the plain call (rows that are cut into splits), replayed several times in turn and at once on
    two streams, with eager calls between: every replay equals the eager call."""
    cases = [_pool_case([2500, 4000, 0, 31], 8, 4, 128, 16, torch.bfloat16, seed=s) for s in (3, 4)]
    graphs, outs = [], []
    for pool, q, table, seqlen in cases:
        paged_decode_fp4(q, pool.keys[0], pool.values[0], table, seqlen)  # the lengths are known to be in range
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(paged_decode_fp4(q, pool.keys[0], pool.values[0], table, seqlen))
        graphs.append(graph)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for i in range(6):
        for j, (pool, q, table, seqlen) in enumerate(cases):
            q.copy_(torch.randn(q.shape, generator=torch.Generator().manual_seed(10 * i + j)))
        torch.cuda.synchronize()
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream if i % 2 else torch.cuda.current_stream()):
                graph.replay()
        torch.cuda.synchronize()
        for out, (pool, q, table, seqlen) in zip(outs, cases):
            assert torch.equal(out, paged_decode_fp4(q, pool.keys[0], pool.values[0], table, seqlen))


def test_a_plan_built_on_a_busy_stream_runs_on_another(cuda):
    """Its workspace, cleared at the build, is clear for the first run, whichever stream that is on."""
    pool, q, table, seqlen = _pool_case([4000, 31], 8, 4, 128, 16, torch.bfloat16, seed=5)
    want = paged_decode_fp4(q, pool.keys[0], pool.values[0], table, seqlen)  # the lengths are known to be in range
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        junk = torch.full((1 << 20,), 0x55, dtype=torch.uint8, device=cuda)  # small enough to share the plan's blocks
        del junk
        torch.cuda._sleep(20_000_000)
        plan = paged_decode_fp4_plan(q, pool.keys, pool.values, table, seqlen)
    for _ in range(3):
        assert torch.equal(plan.run(0, q), want)


def test_a_plan_is_not_built_inside_a_capture(cuda):
    pool, q, table, seqlen = _pool_case([40], 8, 4, 128, 16, torch.bfloat16, seed=5)
    want = paged_decode_fp4(q, pool.keys[0], pool.values[0], table, seqlen)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(RuntimeError, match="before the capture"):
            paged_decode_fp4_plan(q, pool.keys, pool.values, table, seqlen)
        out = paged_decode_fp4(q, pool.keys[0], pool.values[0], table, seqlen)
    for _ in range(3):
        graph.replay()
        assert torch.equal(out, want)


def test_copy_blocks_refuses_pools_that_are_not_contiguous(cuda):
    pool = PagedPool(1, 8, 16, 2, 64, dtype=torch.bfloat16, device=cuda)
    pool.keys[0] = torch.zeros(8, 16, 4, 64, dtype=torch.bfloat16, device=cuda)[:, :, :2]
    with pytest.raises(ValueError, match="contiguous"):
        pool.copy_blocks([0], [1])


def test_calls_on_two_streams_and_repeated_calls_give_the_same_bits(cuda):
    """The same call twice gives the same bits, and two plans may run at once on two streams."""
    cases = [_pool_case([2500, 400, 31], 16, 8, 128, 16, torch.bfloat16, seed=s) for s in (1, 2)]
    plans = [paged_decode_fp4_plan(q, p.keys, p.values, t, n) for p, q, t, n in cases]
    want = [plan.run(0, c[1]).clone() for plan, c in zip(plans, cases)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for i in (0, 1):
            with torch.cuda.stream(streams[i]):
                got[i].append(plans[i].run(0, cases[i][1]))
    torch.cuda.synchronize()
    for i in (0, 1):
        assert all(torch.equal(x, want[i]) for x in got[i])


def test_offsets_past_32_bits(cuda):
    """A pool of more than 4 GiB per side: rows written, read and attended over at its far end."""
    H_kv, D, bs = 8, 128, 16
    n_blocks = (1 << 32) // (H_kv * page_bytes(bs, D)) + 64
    pool = Fp4PagedPool(1, n_blocks, bs, H_kv, D, dtype=torch.bfloat16, device=cuda, n_head=16)
    ids = [n_blocks - 1, 0, n_blocks - 7, n_blocks - 30]
    k, v = torch.randn(60, H_kv, D).bfloat16().cuda(), torch.randn(60, H_kv, D).bfloat16().cuda()
    pool.write_prefill(0, ids, 0, k, v)
    pool.check_writes()
    slots = pool.slot_ids(ids, 0, 60)
    assert torch.equal(pool.read_slots(0, slots)[0].cpu().double(), oracle.held(k))
    q = torch.randn(1, 16, D).bfloat16().cuda()
    small = Fp4PagedPool(1, 4, bs, H_kv, D, dtype=torch.bfloat16, device=cuda, n_head=16)
    small.write_prefill(0, [0, 1, 2, 3], 0, k, v)
    seqlen = torch.tensor([60], dtype=torch.int32, device=cuda)
    got = paged_decode_fp4(q, pool.keys[0], pool.values[0], torch.tensor([ids], dtype=torch.int32, device=cuda), seqlen)
    want = paged_decode_fp4(q, small.keys[0], small.values[0], torch.arange(4, dtype=torch.int32, device=cuda)[None], seqlen)
    assert torch.equal(got, want)
    pool.copy_blocks([n_blocks - 1], [n_blocks - 2])
    assert torch.equal(pool.keys[0][n_blocks - 2], pool.keys[0][n_blocks - 1])


# ------------------------------------------------------------------ page copies
@pytest.mark.parametrize("make", [
    lambda d: PagedPool(3, 40, 16, 8, 128, dtype=torch.bfloat16, device=d),
    lambda d: Fp4PagedPool(2, 40, 16, 2, 64, dtype=torch.bfloat16, device=d),
    lambda d: PagedPool(1, 40, 1, 1, 1, dtype=torch.float16, device=d),
    lambda d: PagedPool(2, 40, 4, 3, 5, dtype=torch.bfloat16, device=d),
    lambda d: PagedPool(1, 40, 64, 8, 256, dtype=torch.float32, device=d),
    lambda d: PagedPool(70, 40, 16, 1, 8, dtype=torch.bfloat16, device=d),
], ids=["bf16", "fp4", "2-byte pages", "120-byte pages", "512-KiB pages", "140 pools"])
@pytest.mark.parametrize("moves", [1, 19])
def test_copy_blocks_moves_every_layers_pages(make, moves, cuda):
    pool = make(cuda)
    for store in pool.keys + pool.values:
        store.view(torch.uint8).random_(0, 100)
    before = [s.clone() for s in pool.keys + pool.values]
    perm = torch.randperm(40, generator=torch.Generator().manual_seed(moves)).tolist()
    dst, src = perm[:moves], [perm[moves + i % 20] for i in range(moves)]
    pool.copy_blocks(src, dst)
    for old, new in zip(before, pool.keys + pool.values):
        want = old.clone()
        want[torch.tensor(dst)] = old[torch.tensor(src)]
        assert torch.equal(new, want)


def test_copy_blocks_of_more_pairs_than_one_launch_takes_and_captured(cuda):
    pool = PagedPool(1, 1000, 16, 1, 64, dtype=torch.bfloat16, device=cuda)
    for store in pool.keys + pool.values:
        store.copy_(torch.randn_like(store))
    start = pool.keys[0].clone()
    src, dst = list(range(500, 1000)), list(range(499, -1, -1))
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        pool.copy_blocks(src, dst)
    assert torch.equal(pool.keys[0], start)
    src.clear()  # the captured copy keeps its own ids
    for i in range(3):
        pool.keys[0].copy_(start * (i + 1))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(pool.keys[0][:500], (start * (i + 1))[500:].flip(0))
        assert torch.equal(pool.keys[0][500:], (start * (i + 1))[500:])


# ------------------------------------------------------------------ together
SMALL = Qwen3Config(vocab=512, hidden=256, inter=512, n_layer=3, n_head=4, n_kv_head=2, head_dim=128)


def test_prefill_fork_decode_and_compaction_of_one_conversation(cuda):
    """A prompt is prefilled, forked, both continue with their own tokens, the pool is compacted and they
    continue: every step's attention is that of the oracle over the pool, and the compaction changes no bit."""
    H, H_kv, D, bs, L, n0 = 4, 2, 128, 16, 2, 37
    pool = Fp4PagedPool(L, 24, bs, H_kv, D, dtype=torch.bfloat16, device=cuda, n_head=H, strict_writes=True)
    blocks = BlockFreeList(24, bs)
    other = blocks.take(5)  # another request, gone before the compaction
    first = blocks.take(blocks.blocks_for(n0 + 20))
    packed, _ = PackedPrefill.upload([list(range(n0))], pool, [first], cuda)
    for i in range(L):
        packed.write(i, torch.randn(1, n0, H_kv, D).bfloat16().cuda(), torch.randn(1, n0, H_kv, D).bfloat16().cuda())
    second, src, dst = blocks.fork(first, n0, capacity=n0 + 20)
    pool.copy_blocks(src, dst)
    tables = [first, second]
    assert second[:2] == first[:2] and second[2] != first[2]

    def steps(kv, count, seed):
        g = torch.Generator().manual_seed(seed)
        got = []
        for _ in range(count):
            kv.build_mask(next_token=True)
            for i in range(L):
                k, v, q = (torch.randn(2, h, 1, D, generator=g).bfloat16().cuda() for h in (H_kv, H_kv, H))
                kv.write(i, k, v)
                got.append((i, q, kv.attend(i, q), kv._seqlen.clone()))
            kv.advance()
        return got

    kv = PagedKV(pool, tables, [n0, n0], rope_len=100, n_head=H)
    for i, q, out, seqlen in steps(kv, 3, 1)[-L:]:
        _within(out.squeeze(2), q.squeeze(2), pool, kv._block_table_tensor, seqlen, layer=i)
    blocks.give_back(other)
    copy = [s.clone() for s in pool.keys + pool.values]
    old_tables = [list(t) for t in tables]
    src, dst = blocks.compact(tables)
    assert src and tables != old_tables and max(max(t) for t in tables) < 24 - blocks.n_free
    pool.copy_blocks(src, dst)
    moved = steps(PagedKV(pool, tables, [n0 + 3] * 2, rope_len=100, n_head=H), 2, 2)
    for s, old in zip(pool.keys + pool.values, copy):
        s.copy_(old)
    stayed = steps(PagedKV(pool, old_tables, [n0 + 3] * 2, rope_len=100, n_head=H), 2, 2)
    assert all(torch.equal(a[2], b[2]) for a, b in zip(moved, stayed))


def test_model_decodes_over_a_4_bit_pool(cuda):
    """A small model's prefill and captured greedy steps on a 4-bit pool: the captured decoder and the eager
    container agree bit by bit, and the tokens' logits are those of the same model on a 16-bit pool that holds
    the 4-bit pool's rows."""
    model = Qwen3(SMALL, random_weights(SMALL, 0), cuda, max_pos=256)
    prompts, tables, new = [list(range(5, 40)), list(range(100, 117))], [[0, 5, 2, 7], [1, 4, 3, 6]], 8
    pool = model.new_pool(8, 16, kv_bits=4)
    assert isinstance(pool, Fp4PagedPool) and pool.bytes() * 64 == 17 * model.new_pool(8, 16).bytes()
    first = model.prefill(prompts, pool, tables).argmax(-1)
    lengths = [len(p) for p in prompts]
    start = [s.clone() for s in pool.keys + pool.values]
    dec = GraphDecoder(model, pool, tables, lengths, first, new)
    dec.capture()
    for _ in range(new):
        dec.step()
    dec.check()
    torch.cuda.synchronize()
    for s, old in zip(pool.keys + pool.values, start):
        s.copy_(old)
    kv = PagedKV(pool, tables, lengths, rope_len=200, n_head=SMALL.n_head)
    wide = model.new_pool(8, 16)
    everywhere = torch.arange(128, device=cuda)
    tokens, picks = first, []
    for _ in range(new):
        logits = model.decode(kv, tokens)
        for i in range(SMALL.n_layer):  # the 16-bit pool with the same contents, this step's token among them
            wide.write_slots(i, everywhere, *pool.read_slots(i, everywhere))
        tokens = logits.argmax(-1)
        picks.append(tokens)
    pool.check_writes()
    assert torch.equal(torch.stack(picks, 1), dec.history)
    # the last step once more: the wide pool holds what the 4-bit pool held, except that it writes its own row
    # in 16 bits; the logits agree within the noise of 16-bit activations plus one row's rounding out of 40
    kv16 = PagedKV(wide, tables, [n + new - 1 for n in lengths], rope_len=200, n_head=SMALL.n_head)
    again = model.decode(kv16, picks[-2])
    assert (again - logits).float().norm() <= 0.1 * logits.float().norm()


def test_server_runs_a_trace_on_a_4_bit_pool(cuda):
    model = Qwen3(SMALL, random_weights(SMALL, 1), cuda, max_pos=256)
    server = ContinuousServer(model, max_batch=4, n_blocks=64, max_prompt=64, max_new=6, max_prefill_tokens=128, kv_bits=4)
    server.warm()
    trace = poisson_trace(9, rate=100.0, vocab=SMALL.vocab, median=24, lo=2, hi=60, max_new=6, seed=3)
    records, _ = server.run(trace, realtime=False, step_s=0.01)
    assert all(len(r.tokens) == 6 for r in records) and server.blocks.n_free == 64
    with pytest.raises(ValueError, match="kv_bits must be 4 or 16"):
        ContinuousServer(model, n_blocks=8, kv_bits=8)


def test_decode_of_lengths_past_24_bits(cuda):
    """Rows of more than 2^24 tokens, where fp32 no longer counts tokens one by one: a mean (scale 0) over one and
    over two such rows, with all weight of V on a few tokens at the rows' ends and at odd places."""
    D, bs, n = 64, 512, (1 << 24) + 1_234_567
    pool = Fp4PagedPool(1, -(-n // bs), bs, 1, D, dtype=torch.float32, device=cuda)
    table = torch.arange(pool.n_blocks, dtype=torch.int32, device=cuda).flip(0).repeat(2, 1).contiguous()
    lengths = [n, n - (1 << 23) + 17]
    marks = sorted({0, 5, 777_777, 1 << 24, *(m - i for m in lengths for i in (1, 2, 300))})
    slots = torch.tensor([int(table[0, t // bs]) * bs + t % bs for t in marks], device=cuda)
    rows = torch.full((len(marks), 1, D), 4.0, device=cuda)
    pool.write_slots(0, slots, torch.zeros_like(rows), rows)
    for count in (1, 2):
        seqlen = torch.tensor(lengths[:count], dtype=torch.int32, device=cuda)
        out = paged_decode_fp4(torch.randn(count, 2, D, device=cuda), pool.keys[0], pool.values[0], table[:count], seqlen,
                               scale=0.0)
        for r in range(count):
            want = 4.0 * sum(t < lengths[r] for t in marks) / lengths[r]
            # fp32 sums of n ones over some hundred waves, a few thousand each: well inside 2^-18
            assert (out[r].double() / want - 1).abs().max() <= 2.0 ** -18


def test_decode_gives_nearly_always_the_nearest_value_of_its_type(cuda):
    """Weights and V of one sign, so that what the weights are off by does not cancel in the output. Each p is off by at
    most 2^-17, to either side: over some hundred tokens 2^-20 of an output, and the fp32 sums and scores 2^-19 at most
    (n = 600 terms of 2^-24 in a random walk, scores of a few units): 2^-18.4 together. An output of fp16 has steps of
    2^-11 of its value at least, so at most 2^-7.4 of them, 0.6%, round to the other side of a border. (Weights cut to 16 bits
    are 2^-17 too small on average, one output in 100.)"""
    lengths = torch.randint(300, 600, (32,), generator=torch.Generator().manual_seed(1)).tolist()
    pool, q, table, seqlen = _pool_case(lengths, 16, 8, 128, 16, torch.float16, seed=21)
    for r, n in enumerate(lengths):
        ids = table[r, : -(-n // 16)].tolist()
        k, v = pool.read_slots(0, pool.slot_ids(ids, 0, n))
        pool.write_prefill(0, ids, 0, k, v.abs())
    out = paged_decode_fp4(q, pool.keys[0], pool.values[0], table, seqlen)
    want, _, _ = oracle.paged_attention(q, pool.keys[0], pool.values[0], table, seqlen)
    off = (out.cpu() != want.to(torch.float16))
    assert off.double().mean() <= 2.0 ** -7.4, f"{int(off.sum())} of {off.numel()}"


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("n", [320, 5000])
def test_decode_of_the_largest_values_stays_finite(n, D, dtype, cuda):
    """Tokens whose scores lie a little above those before them, with V near the format's largest (1.5 * 2^127): weights of
    the row's own largest or less, the products stay in fp32, and the result is V's size."""
    H, H_kv, dt = 4, 2, DTYPES[dtype]
    pool, _, table, seqlen = _pool_case([n], H, H_kv, D, 16, dt, seed=13)
    q = torch.ones(1, H, D, dtype=dt, device=cuda)
    k, v = torch.zeros(n, H_kv, D, dtype=dt), torch.randn(n, H_kv, D).to(dt)
    for t, size in ((300, 1.5), (n - 1, -0.75)):
        k[t], v[t] = 1.0, size * 2.0 ** 126
    v[300, 1] = 1.5 * 2.0 ** 127
    pool.write_prefill(0, table[0][: -(-n // 16)].tolist(), 0, k.cuda(), v.cuda())
    # 7.5 binary orders above the scores of 0, and 100
    for above in (7.5, 100.0):
        scale = above * math.log(2.0) / D
        out = paged_decode_fp4(q, pool.keys[0], pool.values[0], table, seqlen, scale=scale)
        assert out.isfinite().all() and out.abs().max() > 2.0 ** 120
        _within(out, q, pool, table, seqlen, scale=scale)


def test_decode_of_one_row_or_head_whose_stride_is_odd(cuda):
    """A dimension of one has whatever stride its tensor was cut with: a row of a packed projection whose rows are no
    multiple of 16 bytes, one head, one KV head."""
    pool, q, table, seqlen = _pool_case([100, 40, 0], 8, 4, 128, 16, torch.bfloat16, seed=2)
    packed = torch.zeros(3, 8 * 128 + 4, dtype=torch.bfloat16, device=cuda)
    packed[:, :1024] = q.view(3, -1)
    row = packed[:, :1024].view(3, 8, 128)[:1]
    assert row.stride() == (1028, 128, 1) and row.contiguous().stride() == row.stride()
    want = paged_decode_fp4(q[:1].clone(), pool.keys[0], pool.values[0], table[:1], seqlen[:1])
    assert torch.equal(paged_decode_fp4(row, pool.keys[0], pool.values[0], table[:1], seqlen[:1]), want)
    plan = paged_decode_fp4_plan(row, pool.keys, pool.values, table[:1], seqlen[:1])
    assert torch.equal(plan.run(0, row), want)
    single, q1, table1, seqlen1 = _pool_case([100, 40], 1, 1, 128, 16, torch.bfloat16, seed=3)
    want = paged_decode_fp4(q1, single.keys[0], single.values[0], table1, seqlen1)
    odd = q1.as_strided(q1.shape, (128, 3, 1))
    pages = [s.as_strided(s.shape, (s.stride(0), 7, 1)) for s in (single.keys[0], single.values[0])]
    assert torch.equal(paged_decode_fp4(odd, *pages, table1, seqlen1), want)
    assert torch.equal(paged_decode_fp4_plan(odd, pages[:1], pages[1:], table1, seqlen1).run(0, odd), want)


def test_runs_that_overlapped_by_mistake_leave_the_plan_right(cuda):
    """Two graphs of one plan's runs replayed at once, against its contract: those outputs are unspecified, but the runs
    after them, in order again, are right."""
    pool, q, table, seqlen = _pool_case([6000, 2500, 31, 4000], 4, 2, 128, 16, torch.bfloat16, seed=4)
    plan = paged_decode_fp4_plan(q, pool.keys, pool.values, table, seqlen)
    others = [torch.randn(q.shape, device=cuda).bfloat16() for _ in range(2)]  # no split's partial is left from the run before
    want = [plan.run(0, x).clone() for x in others]
    torch.cuda.synchronize()
    graphs = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()]
    for graph in graphs:
        with torch.cuda.graph(graph):
            for _ in range(50):
                plan.run(0, q)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(20):
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for x, y in zip(others, want):
            assert torch.equal(plan.run(0, x), y)


def test_a_refused_read_is_not_reported_as_a_write(cuda):
    pool = Fp4PagedPool(1, 2, 16, 2, 64, dtype=torch.bfloat16, device=cuda)
    pool.read_slots(0, torch.tensor([3, 32], device=cuda))
    with pytest.raises(IndexError, match="token 1 of a write or read .* a read returned zeros"):
        pool.check_writes()


def test_fp16_decode_of_values_past_its_range(cuda):
    """Pages written from bf16 hold more than fp16 does: such outputs come out as fp16's largest value, the others as ever."""
    pool, _, table, seqlen = _pool_case([40], 4, 2, 64, 16, torch.bfloat16, seed=6)
    k, v = torch.zeros(40, 2, 64), torch.randn(40, 2, 64)
    v[:, 0, :32], v[:, 1, 32:] = 2.0 ** 20, -2.0 ** 100
    pool.write_prefill(0, table[0][:3].tolist(), 0, k.bfloat16().cuda(), v.bfloat16().cuda())
    q = torch.randn(1, 4, 64).half().cuda()
    out = paged_decode_fp4(q, pool.keys[0], pool.values[0], table, seqlen)
    want, weight, _ = oracle.paged_attention(q, pool.keys[0], pool.values[0], table, seqlen)
    _assert_within(out, want.clamp(-65504, 65504), _half_step(want.abs(), q.dtype) + 2.0 ** -13 * weight)
    assert (out[0, :2, :32] == 65504).all() and (out[0, 2:, 32:] == -65504).all()


def test_a_pool_stays_on_the_device_it_was_built_on(cuda):
    """Built on "cuda", it names the device that was current then: tensors that its calls make later (q of the epilogue, slot
    maps) belong to that one, whichever is current."""
    pool = Fp4PagedPool(1, 2, 16, 2, 64, dtype=torch.bfloat16, device="cuda", n_head=4)
    assert pool.device == pool.keys[0].device and pool.device.index is not None
    assert pool.slot_ids([1, 0], 0, 20).device == pool.device
    kv = PagedKV(pool, [[0, 1]], [3], rope_len=30, n_head=4)
    assert kv.device == pool.device and kv.pos.device == pool.device


def test_copy_blocks_looks_at_stores_put_in_place_of_the_pools(cuda):
    """Stores of the pool's own layout may take the place of its own at any time, others are refused each time."""
    pool = PagedPool(2, 8, 16, 2, 64, dtype=torch.bfloat16, device=cuda)
    for store in pool.keys + pool.values:
        store.copy_(torch.randn_like(store))
    for _ in range(3):
        pool.copy_blocks([0, 1], [5, 6])
        assert all(torch.equal(s[:2], s[5:7]) for s in pool.keys + pool.values)
        kept, pool.keys[1] = pool.keys[1], torch.randn_like(pool.keys[1])
        pool.copy_blocks([2], [7])
        assert all(torch.equal(s[2], s[7]) for s in pool.keys + pool.values) and not torch.equal(kept[7], pool.keys[1][7])
        good, pool.values[0] = pool.values[0], pool.values[0][:4].clone()
        with pytest.raises(ValueError, match="keys and values of shape"):
            pool.copy_blocks([0], [7])
        pool.values[0] = good
        moved = torch.randn_like(good)
        pool.values[0].data = moved  # the same tensor, elsewhere
        pool.copy_blocks([3], [4])
        assert torch.equal(moved[3], moved[4])
        pool.values[0].data = torch.zeros(4, 16, 2, 64, dtype=torch.bfloat16, device=cuda)
        with pytest.raises(ValueError, match="keys and values of shape"):
            pool.copy_blocks([0], [7])
        pool.values[0].data = moved


# ------------------------------------------------------------------ every kernel variant, and its borders
def _waves(B, H, H_kv, D, bs, width, dtype):
    """Waves per workgroup that a decode of these sizes takes, from its workspace: counters of each row and column (a KV head
    and up to 8 of its query heads, 4 in fp32), then a partial per column for each of target + B splits."""
    heads = 4 if dtype == torch.float32 else 8
    group = H // H_kv
    cols, nh = H_kv * -(-group // heads), min(group, heads)
    partial = 4 * (nh * D + -(-2 * nh // 4) * 4)
    size = _lib.lib.mi_paged_decode_fp4_workspace_size(B, H, H_kv, D, bs, width, _lib.dtype_code(dtype))
    target, rest = divmod(size - -(-B * cols * 4 // 256) * 256, partial * cols)
    assert rest == 0
    return {max(1, 256 // cols): 8, max(1, 512 // cols): 4}[target - B]


def _lengths_with(B, special, seed, most=150):
    """``special`` (row -> length) among rows of 0 to ``most`` tokens."""
    lengths = torch.randint(0, most, (B,), generator=torch.Generator().manual_seed(seed)).tolist()
    for row, n in special.items():
        lengths[row % B] = n
    return lengths


LONG = {0: 1100, 2: 2500, 3: 0, 5: 1, 7: 700, -1: 1500}


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("B,H,H_kv,D,waves", [
    (16, 16, 8, 128, 8), (17, 16, 8, 128, 4), (32, 16, 8, 128, 4), (33, 16, 8, 128, 8),
    (128, 2, 1, 128, 8), (129, 2, 1, 128, 4), (256, 2, 1, 128, 4), (257, 2, 1, 128, 8),
    (8, 16, 16, 64, 8), (16, 16, 16, 64, 4), (257, 1, 1, 64, 8),
    (16, 4, 2, 256, 4), (17, 4, 2, 256, 8), (33, 4, 1, 256, 8), (64, 4, 2, 256, 8), (65, 4, 2, 256, 4), (129, 4, 2, 256, 8)])
def test_decode_in_every_variant_with_rows_that_are_cut(B, H, H_kv, D, waves, dtype, cuda):
    """Both workgroup sizes of every type and head_dim, at the borders between them, with rows of several splits, whole ones and
    empty ones; the same plan twice, so that a counter left behind would show."""
    dt = DTYPES[dtype]
    pool, q, table, seqlen = _pool_case(_lengths_with(B, LONG, B + D), H, H_kv, D, 16, dt, seed=B)
    assert _waves(B, H, H_kv, D, 16, table.shape[1], dt) == waves
    plan = paged_decode_fp4_plan(q, pool.keys, pool.values, table, seqlen)
    out = plan.run(0, q)
    _within(out, q, pool, table, seqlen)
    assert torch.equal(plan.run(0, q), out)
    assert torch.equal(paged_decode_fp4(q, pool.keys[0], pool.values[0], table, seqlen), out)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("B,H,H_kv", [(17, 16, 1), (20, 16, 1), (34, 8, 1), (17, 14, 1)])
def test_decode_of_eight_wide_heads_per_column(B, H, H_kv, dtype, cuda):
    """head_dim 256 in workgroups of 8 waves with 7 or 8 query heads per column: their states take more than 64 KiB of LDS."""
    dt = DTYPES[dtype]
    pool, q, table, seqlen = _pool_case(_lengths_with(B, LONG, B), H, H_kv, 256, 16, dt, seed=B)
    assert _waves(B, H, H_kv, 256, 16, table.shape[1], dt) == 8
    _within(paged_decode_fp4(q, pool.keys[0], pool.values[0], table, seqlen), q, pool, table, seqlen)


@pytest.mark.parametrize("H,H_kv,D,dtype", [(2, 1, 128, "bf16"), (4, 2, 64, "fp16"), (2, 1, 256, "fp32")])
@pytest.mark.parametrize("B", [65, 130, 200])
def test_decode_of_long_rows_past_the_first_64(B, H, H_kv, D, dtype, cuda):
    """The plan counts splits 64 rows at a time: long rows on both sides of such a border and last, run twice, then with the
    lengths of the rows turned round."""
    special = {62: 2100, 63: 5000, 64: 3000, 65: 2000, 66: 0, 128: 2200, 129: 4100, B - 1: 6000}
    pool, q, table, seqlen = _pool_case(_lengths_with(B, {r: n for r, n in special.items() if r < B}, B, 40), H, H_kv, D, 16,
                                        DTYPES[dtype], seed=B)
    plan = paged_decode_fp4_plan(q, pool.keys, pool.values, table, seqlen)
    for _ in range(2):
        out = plan.run(0, q)
        _within(out, q, pool, table, seqlen)
        assert torch.equal(plan.run(0, q), out)
        order = torch.arange(B - 1, -1, -1, device=cuda)
        table.copy_(table[order])
        seqlen.copy_(seqlen[order])


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("H_kv,D", [(2, 64), (3, 128), (1, 256)])
@pytest.mark.parametrize("layout", ["contiguous", "permuted", "strided", "misaligned"])
def test_large_calls_store_and_read_what_small_ones_do(dtype, H_kv, D, layout, cuda):
    """One call on either side of the size from which a lane works on two rows, against calls of 500 tokens, whose bytes the
    oracle's are compared with above."""
    dt, border = DTYPES[dtype], -(-4096 * 64 // (H_kv * (D // 8)))
    for n in (border - 1, border, border + 5):
        g = torch.Generator(device=cuda).manual_seed(n)
        rows = [torch.randn(n, H_kv, D, generator=g, device=cuda).to(dt) for _ in range(2)]
        rows[0][n // 2, 0, 5], rows[1][n - 1, -1, -1] = math.nan, math.inf

        def placed(x):
            if layout == "permuted":
                return x.permute(1, 0, 2).contiguous().permute(1, 0, 2)
            if layout == "strided":
                return torch.stack([x, x], -1)[..., 0]
            if layout == "misaligned":
                return torch.cat([x.new_zeros(1), x.flatten()])[1:].view(x.shape)
            return x

        pools = [Fp4PagedPool(1, n // 16 + 2, 16, H_kv, D, dtype=dt, device=cuda) for _ in range(2)]
        slots = torch.randperm(pools[0].n_slots, generator=g, device=cuda)[:n]
        slots = slots.int() if layout == "permuted" else slots
        pools[0].write_slots(0, slots, *map(placed, rows))
        for a in range(0, n, 500):
            pools[1].write_slots(0, slots[a: a + 500], *(x[a: a + 500] for x in rows))
        assert torch.equal(pools[0].keys[0], pools[1].keys[0]) and torch.equal(pools[0].values[0], pools[1].values[0])
        whole = pools[0].read_slots(0, slots)
        for a in range(0, n, 500):
            part = pools[0].read_slots(0, slots[a: a + 500])
            assert all(torch.equal(x[a: a + 500].nan_to_num(7.0), y.nan_to_num(7.0)) for x, y in zip(whole, part))
        assert whole[0][n // 2, 0, :32].isnan().all() and int(whole[0].isnan().sum()) == 32
        for pool in pools:
            pool.check_writes()


def test_decode_of_a_query_shared_by_rows_and_of_a_misaligned_one(cuda):
    pool, q, table, seqlen = _pool_case([100, 40, 0], 8, 4, 128, 16, torch.bfloat16, seed=2)
    shared = q[:1].expand(3, 8, 128)
    want = paged_decode_fp4(shared.contiguous(), pool.keys[0], pool.values[0], table, seqlen)
    assert torch.equal(paged_decode_fp4(shared, pool.keys[0], pool.values[0], table, seqlen), want)
    flat = torch.zeros(2 * 3 * 1024 + 1, dtype=torch.bfloat16, device=cuda)
    odd = flat[1:].view(3, 2, 8, 128)[:, 1]  # rows apart, and no address a multiple of 16 bytes
    odd.copy_(shared)
    assert torch.equal(paged_decode_fp4(odd, pool.keys[0], pool.values[0], table, seqlen), want)


def test_fp32_decode_rounds_its_exponents_finely(cuda):
    """Rows of two tokens whose scores are 0 and c q (one element of q, so the score is exact), V 0 and 1: the output is
    1 / (1 + 2^-cq), off by what its weights are. The exponents lie above -8 (4 for the reference, 4 at most for the score):
    rounded by 2^-22 at most, times ln 2, over sqrt(3) in the mean square, 9.5e-8; the exponential's ulp 2^-23 / sqrt(3) = 6.9e-8; the
    sum, the reciprocal and the product 2^-24 / sqrt(3) each. Together 1.33e-7."""
    B, H, D = 64, 16, 64
    pool, _, table, seqlen = _pool_case([2] * B, H, 1, D, 16, torch.float32, seed=1, garbage=False)
    k, v = torch.zeros(2, 1, D, device=cuda), torch.zeros(2, 1, D, device=cuda)
    k[1, 0, 0], v[1] = 1.0, 1.0
    for ids in table[:, :1].tolist():
        pool.write_prefill(0, ids, 0, k, v)
    q = torch.zeros(B, H, D, device=cuda)
    q[..., 0] = -3.9 * torch.rand(B, H, generator=torch.Generator().manual_seed(2)).cuda()
    scale = math.log(2.0)
    c = float(torch.tensor(scale) * torch.tensor(1.4426950408889634))  # the scale in fp32, as the exponents' unit
    got = paged_decode_fp4(q, pool.keys[0], pool.values[0], table, seqlen, scale=scale)
    want = 1.0 / (1.0 + 2.0 ** (-c * q[..., :1].double()))
    assert (got.double() / want - 1).pow(2).mean().sqrt() <= 1.33e-7
