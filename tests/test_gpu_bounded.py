"""Attention under a window with sinks, accounts of attention weights and eviction by them on the GPU, against
``oracle/bounded.py`` (float64). Its ``*_bound`` values are derived there; what an eviction moves is compared bit for
bit, and so are two ways to the same arithmetic (an eager call and a replay, a window past the row and none)."""

from __future__ import annotations

import math

import pytest
import torch

from miattn import Fp4PagedPool, HipVarlen, PagedPool, paged_decode, paged_decode_plan
from miattn.packed import PackedPrefill
from miattn.qwen3 import BudgetDecoder, GraphDecoder, Qwen3, Qwen3Config, random_weights
from miattn.serve import ContinuousServer, TraceRequest
from oracle import bounded

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def _within(got, want, bound, what=""):
    got, want = got.double().cpu(), want.double()
    share = torch.where(got == want, 0.0, (got - want).abs() / bound).nan_to_num(nan=math.inf)  # 0 <= 0: empty rows
    assert share.max() <= 1, f"{what} {share.max().item():.3g} of the bound at {share.argmax().item()}"


def _rows(lengths, H, H_kv, D, dt, bs, width=None, seed=0, spare=3):
    """A pool with the rows' blocks in a random order: q, k, v, table, seqlen on the host."""
    g = torch.Generator().manual_seed(seed)
    width = width or max(1, max(-(-n // bs) for n in lengths))
    need = [max(1, -(-n // bs)) for n in lengths]
    perm = torch.randperm(sum(need) + spare, generator=g).int()
    table = torch.full((len(lengths), width), -1, dtype=torch.int32)
    at = 0
    for r, n in enumerate(need):
        table[r, :n] = perm[at: at + n]
        at += n
    k, v = ((torch.randn(len(perm), bs, H_kv, D, generator=g)).to(dt) for _ in range(2))
    return torch.randn(len(lengths), H, D, generator=g).to(dt), k, v, table, torch.tensor(lengths, dtype=torch.int32)


def _cuda(*tensors):
    return tuple(t.cuda() for t in tensors)


def _cu(lengths):
    cu = [0]
    for n in lengths:
        cu.append(cu[-1] + n)
    return cu


# ------------------------------------------------------------------ decode under a window
HEADS = [(16, 8, 128, BF16, 16), (8, 2, 256, F16, 32), (16, 16, 64, BF16, 16), (24, 2, 128, F16, 64), (4, 4, 32, F32, 1),
         (8, 1, 128, F32, 16), (2, 2, 16, BF16, 8), (32, 4, 128, BF16, 16)]


@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("window,sinks", [(1, 0), (64, 4), (37, 50), (300, 1)])
def test_decode_under_a_window(heads, window, sinks, cuda):
    H, H_kv, D, dt, bs = heads
    edge = window + sinks
    lengths = [0, 1, window, window + 1, edge, edge + 1, edge + bs, 2 * edge + 3, 700, 1001]
    q, k, v, table, seqlen = _rows(lengths, H, H_kv, D, dt, bs)
    out, bound, _, _ = bounded.decode_rows(q, k, v, table, seqlen, window=window, sinks=sinks)
    dq, dk, dv, dt_, ds = _cuda(q, k, v, table, seqlen)
    got = paged_decode(dq, dk, dv, dt_, ds, window=window, sinks=sinks)
    _within(got, out, bound)
    plan = paged_decode_plan(dq, [dk], [dv], dt_, ds, window=window, sinks=sinks)
    assert torch.equal(plan.run(0, dq), got) and not got[0].any()


def test_decode_of_many_long_rows_under_a_window(cuda):
    lengths = [(37 * i) % 4000 for i in range(90)]  # past the 64 rows that a lane each holds
    q, k, v, table, seqlen = _rows(lengths, 4, 2, 64, BF16, 16)
    out, bound, _, _ = bounded.decode_rows(q, k, v, table, seqlen, window=500, sinks=20)
    _within(paged_decode(*_cuda(q, k, v, table, seqlen), window=500, sinks=20), out, bound)


def test_hidden_tokens_and_their_table_entries_are_not_read(cuda):
    """Blocks that hold no seen token may be anything: their entries name no block, hidden tokens hold NaN."""
    H, H_kv, D, bs, window, sinks = 16, 8, 128, 16, 100, 20
    lengths = [1000, 121, 130, 600]
    q, k, v, table, seqlen = _rows(lengths, H, H_kv, D, BF16, bs)
    clean = paged_decode(*_cuda(q, k, v, table, seqlen), window=window, sinks=sinks)
    for r, n in enumerate(lengths):
        mask = bounded.seen(n, window, sinks)
        for t in (~mask).nonzero().flatten().tolist():
            k[table[r, t // bs], t % bs] = v[table[r, t // bs], t % bs] = math.nan
        for j in range(-(-n // bs)):
            if not mask[j * bs: (j + 1) * bs].any():
                table[r, j] = -7
    got = paged_decode(*_cuda(q, k, v, table, seqlen), window=window, sinks=sinks)
    assert torch.equal(got, clean)


@pytest.mark.parametrize("lengths", [[5, 0, 90], [700, 33, 2000], [64] * 20])
def test_a_window_past_every_row_is_none(lengths, cuda):
    q, k, v, table, seqlen = _cuda(*_rows(lengths, 16, 8, 128, BF16, 16))
    plain = paged_decode(q, k, v, table, seqlen)
    for window, sinks in ((max(lengths), 0), (2**40, 0), (1, 2**35)):
        assert torch.equal(paged_decode(q, k, v, table, seqlen, window=window, sinks=sinks), plain)


def test_windowed_decode_follows_growing_rows_in_a_graph(cuda):
    q, k, v, table, seqlen = _rows([250, 17, 512, 0], 16, 8, 128, BF16, 16, width=41)
    for r in range(4):
        table[r, table[r] < 0] = 0
    q, k, v, table, seqlen = _cuda(q, k, v, table, seqlen)
    plan = paged_decode_plan(q, [k], [v], table, seqlen, window=64, sinks=4)
    plan.run(0, q)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = plan.run(0, q)
    for step in range(5):
        seqlen += 13 * step
        graph.replay()
        want = paged_decode(q, k, v, table, seqlen, window=64, sinks=4)
        torch.cuda.synchronize()
        assert torch.equal(out, want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = paged_decode(q, k, v, table, seqlen, window=64, sinks=4)
    side.synchronize()
    assert torch.equal(other, want)


@pytest.mark.parametrize("heads", [(16, 8), (16, 16), (8, 2), (64, 8)])
def test_fused_decode_under_a_window_equals_the_two_launches(heads, cuda):
    (H, H_kv), D, bs, window, sinks = heads, 128, 16, 50, 3
    lengths = [1, 2, 50, 53, 54, 400, 1200, 0]  # with the new token; the last row is idle
    q, k, v, table, seqlen = _rows(lengths, H, H_kv, D, BF16, bs)
    pools = [PagedPool(1, k.shape[0], bs, H_kv, D, dtype=BF16, device=cuda, n_head=H) for _ in range(2)]
    for p in pools:
        p.keys[0].copy_(k)
        p.values[0].copy_(v)
    qkv = torch.randn(8, (H + 2 * H_kv) * D).bfloat16().cuda()
    w = [(1 + 0.1 * torch.randn(D)).bfloat16().cuda() for _ in range(2)]
    angle = torch.outer(torch.arange(2000).float(), 1e6 ** -(torch.arange(0, D, 2).float() / D))
    cos, sin = angle.cos().bfloat16().cuda(), angle.sin().bfloat16().cuda()
    pos = (seqlen.long() - 1).cuda()
    at = (seqlen.long() - 1).clamp(min=0)
    slots = torch.where(seqlen > 0, table[torch.arange(8), at // bs].long() * bs + at % bs, torch.tensor(-1)).cuda()
    table, seqlen = _cuda(table, seqlen)
    plans = [p.decode_plan(torch.empty(8, H, D, dtype=BF16, device=cuda), table, seqlen, window=window, sinks=sinks) for p in pools]
    fused = plans[0].run_fused(0, qkv, *w, cos, sin, pos, slots, 1e-6)
    two = plans[1].run(0, pools[1].write_qk_norm_rope(0, slots, qkv, *w, cos, sin, pos, 1e-6))
    assert torch.equal(fused, two) and torch.equal(pools[0].keys[0], pools[1].keys[0])
    assert torch.equal(pools[0].values[0], pools[1].values[0]) and not fused[7].any()


# ------------------------------------------------------------------ prompts under a window
@pytest.mark.parametrize("heads", [(16, 8, 128, BF16), (8, 2, 256, F16), (4, 4, 64, BF16), (6, 1, 128, F16)])
@pytest.mark.parametrize("lengths,window,sinks", [([1, 64, 65, 300, 2], 1, 0), ([700, 130], 64, 4), ([333], 100, 70),
                                                  ([513, 5], 63, 129), ([1500], 200, 0), ([128, 129], 1000, 3),
                                                  ([1300], 1100, 4), ([1], 1, 9), ([900, 400], 500, 17)])
def test_prompts_under_a_window(heads, lengths, window, sinks, cuda):
    H, H_kv, D, dt = heads
    cu = _cu(lengths)
    q, k, v = (torch.randn(cu[-1], h, D).to(dt) for h in (H, H_kv, H_kv))
    want, bound = bounded.varlen(q, k, v, cu, window, sinks)
    arm = HipVarlen(strict=True)
    args = dict(cu_seqlens=cu, max_seqlen=max(lengths), window=window, sinks=sinks)
    got = arm.prefill_varlen(*_cuda(q, k, v), **args)
    _within(got, want, bound)
    # strided, unaligned operands are taken as well
    odd = [torch.empty(t.numel() + 1, dtype=dt, device=cuda)[1:].view(t.shape).copy_(t) for t in (q, k, v)]
    assert torch.equal(arm.prefill_varlen(*odd, **args), got)
    wide = [torch.stack([t, t], 1).cuda()[:, 0] for t in (q, k, v)]
    assert torch.equal(arm.prefill_varlen(*wide, **args), got)


def test_prompts_under_a_window_with_as_many_heads_as_an_item_names(cuda):
    cu = _cu([130, 70])
    q, k, v = (torch.randn(200, h, 64).bfloat16() for h in (255, 85, 85))
    want, bound = bounded.varlen(q, k, v, cu, 40, 3)
    _within(HipVarlen().prefill_varlen(*_cuda(q, k, v), cu_seqlens=cu, max_seqlen=130, window=40, sinks=3), want, bound)


@pytest.mark.parametrize("D", [64, 128, 256])
def test_a_window_past_every_prompt_gives_the_plain_kernels_bits(D, cuda):
    cu = _cu([300, 1000, 17])
    q, k, v = (torch.randn(cu[-1], h, D).bfloat16().cuda() for h in (8, 2, 2))
    plain = HipVarlen(kernel="duo").prefill_varlen(q, k, v, cu_seqlens=cu, max_seqlen=1000)
    for window, sinks in ((1000, 0), (2**40, 5), (1, 1000)):
        assert torch.equal(HipVarlen().prefill_varlen(q, k, v, cu_seqlens=cu, max_seqlen=1000, window=window, sinks=sinks), plain)


def test_keys_that_no_query_sees_do_not_reach_it(cuda):
    """Scores of hidden keys are dropped whatever they are, and tiles without a seen key are not read at all."""
    cu = [0, 900]
    q, k, v = (torch.randn(900, h, 128).bfloat16().cuda() for h in (4, 2, 2))
    args = dict(cu_seqlens=cu, max_seqlen=900, window=100, sinks=0)
    clean = HipVarlen().prefill_varlen(q, k, v, **args)
    bad = k.clone()
    bad[10], bad[200] = math.nan, math.inf
    got = HipVarlen().prefill_varlen(q, bad, v, **args)
    reached = torch.zeros(900, dtype=torch.bool)
    reached[10:110] = reached[200:300] = True
    assert torch.equal(got[~reached], clean[~reached])
    worse = v.clone()
    worse[:64] = math.nan  # the first tile: seen by no query of the tiles from 192 on
    assert torch.equal(HipVarlen().prefill_varlen(q, k, worse, **args)[192:], clean[192:])


def test_windowed_prompts_captured_and_on_two_streams(cuda):
    """A lone short prompt is cut into pieces and merged: every call has partials of its own."""
    cu = [0, 1200]
    sets = [[torch.randn(1200, h, 128).bfloat16().cuda() for h in (2, 1, 1)] for _ in range(2)]
    args = dict(cu_seqlens=cu, max_seqlen=1200, window=1100, sinks=4)
    arm = HipVarlen()
    want = [arm.prefill_varlen(*x, **args) for x in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    for _ in range(3):
        got = []
        for stream, x in zip(streams, sets):
            with torch.cuda.stream(stream):
                got.append(arm.prefill_varlen(*x, **args))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = arm.prefill_varlen(*sets[0], **args)
    for _ in range(3):
        arm.prefill_varlen(*sets[1], **args)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want[0])


def test_windowed_prefill_refusals(cuda):
    q = torch.zeros(4, 2, 128, dtype=BF16, device=cuda)
    arm = HipVarlen()
    for scale in (0.0, -1.0):
        with pytest.raises(ValueError, match="scale must be positive"):
            arm.prefill_varlen(q, q, q, cu_seqlens=[0, 4], max_seqlen=4, window=2, softmax_scale=scale)
    with pytest.raises(RuntimeError, match="fp16/bf16"):
        arm.prefill_varlen(q.float(), q.float(), q.float(), cu_seqlens=[0, 4], max_seqlen=4, window=2)
    with pytest.raises(ValueError, match="head_dim"):
        x = torch.zeros(4, 2, 32, dtype=BF16, device=cuda)
        arm.prefill_varlen(x, x, x, cu_seqlens=[0, 4], max_seqlen=4, window=2)
    with pytest.raises(ValueError, match="at most 255 heads"):
        x = torch.zeros(4, 256, 64, dtype=BF16, device=cuda)
        arm.prefill_varlen(x, x, x, cu_seqlens=[0, 4], max_seqlen=4, window=2)
    with pytest.raises(ValueError, match="whole rows"):
        pool = Fp4PagedPool(1, 2, 16, 2, 64, dtype=BF16, device=cuda)
        pool.decode_plan(torch.zeros(1, 2, 64, dtype=BF16, device=cuda), torch.zeros(1, 1, dtype=torch.int32, device=cuda),
                         torch.zeros(1, dtype=torch.int32, device=cuda), window=4)


# ------------------------------------------------------------------ accounts
@pytest.mark.parametrize("heads", [h for h in HEADS if h[2] > 16])
@pytest.mark.parametrize("lengths", [[0, 1, 2, 17, 300], [1500, 64, 800], [5000], [64, 0, 1, 128, 31, 127, 9, 100], [3]])
def test_weighed_decode(heads, lengths, cuda):
    H, H_kv, D, dt, bs = heads
    q, k, v, table, seqlen = _rows(lengths, H, H_kv, D, dt, bs)
    out, bound, w, w_bound = bounded.decode_rows(q, k, v, table, seqlen)
    dq, dk, dv, dtab, ds = _cuda(q, k, v, table, seqlen)
    plan = paged_decode_plan(dq, [dk], [dv], dtab, ds)
    before = torch.rand(len(lengths), H_kv, table.shape[1] * bs)
    account = before.cuda()
    _within(plan.run_weighed(0, dq, account), out, bound, "out")
    # the sum is rounded once per query head
    _within(account, before.double() + w, w_bound + (H // H_kv + 1) * 2.0 ** -24 * (before + w), "weights")
    for b, n in enumerate(lengths):
        assert torch.equal(account[b, :, n:].cpu(), before[b, :, n:])
    # an account inside a wider tensor, twice the same bits
    wide = torch.zeros(len(lengths), 2, H_kv, account.shape[2] + 3, device=cuda)
    part = wide[:, 1, :, : account.shape[2]]
    part.copy_(before)
    plan.run_weighed(0, dq, part)
    assert torch.equal(part, account) and not wide[:, 0].any() and not wide[:, 1, :, account.shape[2]:].any()


def test_weighed_decode_of_equal_keys(cuda):
    """Every token of a row weighs the same: 1/n per query head."""
    q, k, v, table, seqlen = _rows([256, 1000, 3], 16, 8, 128, BF16, 16)
    k[:] = k[0, 0]
    q, k, v, table, seqlen = _cuda(q, k, v, table, seqlen)
    account = torch.zeros(3, 8, table.shape[1] * 16, device=cuda)
    paged_decode_plan(q, [k], [v], table, seqlen).run_weighed(0, q, account)
    for b, n in enumerate((256, 1000, 3)):
        assert torch.allclose(account[b, :, :n], torch.full((8, n), 2.0 / n, device=cuda), rtol=2e-6, atol=0)


@pytest.mark.parametrize("H,H_kv,D", [(4, 2, 64), (16, 8, 128), (32, 16, 128)])
def test_weighed_decode_with_scores_that_are_not_finite(H, H_kv, D, cuda):
    q, k, v, table, seqlen = _rows([40, 40], H, H_kv, D, F16, 16)
    k[table[1, 0], 3, 0] = math.nan
    q, k, v, table, seqlen = _cuda(q, k, v, table, seqlen)
    account = torch.zeros(2, H_kv, table.shape[1] * 16, device=cuda)
    out = paged_decode_plan(q, [k], [v], table, seqlen).run_weighed(0, q, account)
    assert torch.isfinite(out[0]).all() and torch.isfinite(account[0]).all()
    assert torch.isnan(account[1, 0, :40]).all() and torch.isfinite(account[1, 1:]).all() and torch.isfinite(out[1, 2:]).all()


@pytest.mark.parametrize("lengths,width", [([700, 9, 130], 60), ([70, 0, 55], 8)])
def test_weighed_decode_captured_with_growing_rows(lengths, width, cuda):
    q, k, v, table, seqlen = _rows(lengths, 16, 8, 128, BF16, 16, width=width)
    table[table < 0] = 0
    q, k, v, table, seqlen = _cuda(q, k, v, table, seqlen)
    plan, other = (paged_decode_plan(q, [k], [v], table, seqlen) for _ in range(2))
    account, want = (torch.zeros(3, 8, 16 * width, device=cuda) for _ in range(2))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):  # the workspace is taken inside the capture
        out = plan.run_weighed(0, q, account)
    for step in range(4):
        graph.replay()
        eager = other.run_weighed(0, q, want)
        torch.cuda.synchronize()
        assert torch.equal(out, eager) and torch.equal(account, want)
        seqlen += 11


def test_weighed_decode_refusals(cuda):
    q, k, v, table, seqlen = _cuda(*_rows([40], 4, 2, 64, BF16, 16))
    plan = paged_decode_plan(q, [k], [v], table, seqlen)
    good = torch.zeros(1, 2, 48, device=cuda)
    for bad in (good[..., :47], good.double(), good.cpu(), good[:, :1], torch.zeros(1, 48, 2, device=cuda).transpose(1, 2),
                good[:, :1].expand(1, 2, 48), good[0]):
        with pytest.raises(ValueError, match="weights must be"):
            plan.run_weighed(0, q, bad)
    with pytest.raises(IndexError, match="outside the plan"):
        plan.run_weighed(1, q, good)
    with pytest.raises(ValueError, match="validated layout"):
        plan.run_weighed(0, q.half(), good)
    with pytest.raises(ValueError, match="under a window"):
        paged_decode_plan(q, [k], [v], table, seqlen, window=8).run_weighed(0, q, good)
    q, k, v, table, seqlen = _cuda(*_rows([40], 4, 2, 16, BF16, 16))
    with pytest.raises(ValueError, match="head_dim 16"):
        paged_decode_plan(q, [k], [v], table, seqlen).run_weighed(0, q, good)


@pytest.mark.parametrize("heads", [(16, 8, 128, BF16), (8, 2, 256, F16), (4, 4, 64, BF16), (12, 1, 128, F16), (3, 3, 64, F16),
                                   (64, 1, 64, BF16)])
@pytest.mark.parametrize("lengths,observe", [([1, 2, 31, 64, 65, 300], 1), ([700, 5, 129], 32), ([200, 33], None),
                                             ([1000], 77), ([400, 90], 1000)])
def test_account_of_prompts(heads, lengths, observe, cuda):
    H, H_kv, D, dt = heads
    cu = _cu(lengths)
    q, k = torch.randn(cu[-1], H, D).to(dt), torch.randn(cu[-1], H_kv, D).to(dt)
    want, bound = bounded.prompt_weights(q, k, cu, observe)
    args = dict(cu_seqlens=cu, max_seqlen=max(lengths), observe=observe)
    got = HipVarlen().prompt_weights(*_cuda(q, k), **args)
    _within(got, want, bound)
    for s, n in enumerate(lengths):
        assert not got[s, :, n:].any()
    wide = torch.full((2, len(lengths), H_kv, max(lengths) + 70), math.nan, device=cuda)
    odd = torch.empty(q.numel() + 1, dtype=dt, device=cuda)[1:].view(q.shape).copy_(q)
    HipVarlen().prompt_weights(odd, k.cuda(), out=wide[1], **args)
    assert torch.equal(wide[1][..., : max(lengths)], got) and not wide[1][..., max(lengths):].any()
    assert torch.isnan(wide[0]).all()


def test_account_of_a_long_prompt_in_pieces(cuda):
    """Few rows over many keys: the row block's keys are cut into as many pieces as there may be."""
    q, k = torch.randn(6000, 2, 64).bfloat16(), torch.randn(6000, 1, 64).bfloat16()
    want, bound = bounded.prompt_weights(q, k, [0, 6000], 40)
    got = HipVarlen().prompt_weights(*_cuda(q, k), cu_seqlens=[0, 6000], max_seqlen=6000, observe=40)
    _within(got, want, bound)


@pytest.mark.parametrize("heads", [(16, 8, 128, BF16), (8, 2, 256, F16), (4, 4, 64, BF16), (6, 1, 128, F16)])
@pytest.mark.parametrize("observe", [None, 37])
@pytest.mark.parametrize("value", [math.inf, -math.inf, math.nan])
def test_account_of_keys_behind_a_query_that_is_not_finite(heads, observe, value, cuda):
    """Such a query's weights are NaN, for the keys that it sees; keys behind it, other segments and other KV heads keep their bits."""
    H, H_kv, D, dtype = heads
    g = torch.Generator().manual_seed(7)
    cu = [0, 100, 263, 266]
    q, k = (torch.randn(266, h, D, generator=g).to(dtype).to(cuda) for h in (H, H_kv))
    args = dict(cu_seqlens=cu, max_seqlen=163, observe=observe)
    good = HipVarlen().prompt_weights(q, k, **args)
    for at in (130, 162):  # of the second segment
        bad = q.clone()
        bad[100 + at, 0, 1] = value
        got = HipVarlen().prompt_weights(bad, k, **args)
        assert got[1, 0, : at + 1].isnan().all()
        got[1, 0, : at + 1] = good[1, 0, : at + 1]
        assert torch.equal(got, good), (at, (got != good).nonzero()[:4].tolist())


@pytest.mark.parametrize("heads", [(16, 8, 128, BF16), (8, 2, 256, F16), (4, 4, 64, BF16), (6, 1, 128, F16)])
@pytest.mark.parametrize("observe", [None, 5, 37])
def test_account_of_a_key_of_minus_infinity(heads, observe, cuda):
    """A key whose every score is -infinity weighs nothing, like one at a score whose exponential is 0, in a prompt whose last 32
    rows are not all there."""
    H, H_kv, D, dtype = heads
    g = torch.Generator().manual_seed(8)
    q, k = (torch.randn(170, h, D, generator=g).to(dtype).to(cuda) for h in (H, H_kv))
    q[..., 3] = 2.0
    k[[20, 163], :, 3] = -30000.0  # times 2 / 16 at least: far below the exponents of fp32
    args = dict(cu_seqlens=[0, 103, 170], max_seqlen=103, observe=observe)
    far = HipVarlen().prompt_weights(q, k, **args)
    assert not far[0, :, 20].any() and not far[1, :, 60].any() and far.isfinite().all()
    k[[20, 163], :, 3] = -math.inf
    assert torch.equal(HipVarlen().prompt_weights(q, k, **args), far)


def test_account_of_prompts_captured(cuda):
    cu = _cu([500, 60])
    sets = [[torch.randn(560, h, 128).bfloat16().cuda() for h in (4, 2)] for _ in range(2)]
    args = dict(cu_seqlens=cu, max_seqlen=500, observe=48)
    want = [HipVarlen().prompt_weights(*x, **args) for x in sets]
    live = [t.clone() for t in sets[0]]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = HipVarlen().prompt_weights(*live, **args)
    for i in (0, 1, 0, 1):
        for a, b in zip(live, sets[i]):
            a.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want[i])


# ------------------------------------------------------------------ eviction
def _account(n_layer, B, H_kv, capacity, lengths, seed=0):
    g = torch.Generator().manual_seed(seed)
    w = torch.rand(n_layer, B, H_kv, capacity, generator=g)
    w = torch.where(torch.rand(w.shape, generator=g) < 0.3, (w * 4).floor() / 4, w)  # ties, zeros among them
    for b, n in enumerate(lengths):
        w[:, b, :, n:] = 0
    return w


def _evict_case(lengths, budget, recent, sinks, H_kv, D, dt, bs, n_layer=2, moved=False, weights=None, width=None, seed=0):
    _, k, v, table, seqlen = _rows(lengths, H_kv, H_kv, D, dt, bs, seed=seed, width=width,
                                   spare=len(lengths) * -(-budget // bs) + 2)
    g = torch.Generator().manual_seed(seed + 1)
    ks = [torch.randn(k.shape, generator=g).to(dt) for _ in range(n_layer)]
    vs = [torch.randn(k.shape, generator=g).to(dt) for _ in range(n_layer)]
    to = None
    if moved:
        cols = -(-min(budget, table.shape[1] * bs) // bs)
        free = torch.tensor(sorted(set(range(k.shape[0])) - set(table.flatten().tolist())), dtype=torch.int32)
        to = free[torch.randperm(len(free), generator=g)[: len(lengths) * cols]].view(len(lengths), cols)
    w = _account(n_layer, len(lengths), H_kv, table.shape[1] * bs, lengths) if weights is None else weights(table.shape[1] * bs)
    want = bounded.evicted(ks, vs, table, seqlen, w, budget, recent, sinks, to)
    pool = PagedPool(n_layer, k.shape[0], bs, H_kv, D, dtype=dt, device="cuda")
    pool.keys, pool.values = [x.cuda() for x in ks], [x.cuda() for x in vs]
    dtab, ds, dw = _cuda(table, seqlen, w)
    return pool, dtab, ds, dw, None if to is None else to.cuda(), want


def _check_evicted(pool, seqlen, weights, want):
    for i, (a, b) in enumerate(zip(pool.keys + pool.values, want[0] + want[1])):
        assert torch.equal(a.cpu(), b), f"store {i}"
    assert torch.equal(weights.cpu().nan_to_num(9.0, 8.0, -8.0), want[2].nan_to_num(9.0, 8.0, -8.0))
    assert torch.equal(seqlen.cpu(), want[3])
    pool.check_writes()


@pytest.mark.parametrize("shape", [(2, 128, BF16, 16), (3, 64, F16, 8), (1, 256, F32, 32), (2, 16, BF16, 1), (2, 4, F32, 16)])
@pytest.mark.parametrize("budget,recent,sinks", [(1, 0, 0), (16, 4, 2), (37, 37, 0), (50, 0, 50), (100, 30, 0), (130, 60, 7), (5000, 9, 9)])
@pytest.mark.parametrize("moved", [False, True])
def test_eviction(shape, budget, recent, sinks, moved, cuda):
    H_kv, D, dt, bs = shape
    pool, table, seqlen, w, to, want = _evict_case([0, 1, budget % 90 + 1, 131, 257, 100], budget, recent, sinks, H_kv, D, dt,
                                                   bs, moved=moved)
    pool.evict(table, seqlen, w, budget=budget, recent=recent, sinks=sinks, **({} if to is None else {"to": to}))
    _check_evicted(pool, seqlen, w, want)


@pytest.mark.parametrize("lengths,budget", [([4090, 4096], 700), ([5000, 16384], 2000), ([20011, 300], 1234),
                                            ([32768, 16385], 5000), ([65536, 40001], 9000), ([70003], 3000)])
@pytest.mark.parametrize("moved", [False, True])
def test_eviction_of_long_rows(lengths, budget, moved, cuda):
    """Accounts in the registers of 512 and 1024 threads, to the last of them, and past them."""
    pool, table, seqlen, w, to, want = _evict_case(lengths, budget, 100, 4, 1, 16, BF16, 64, n_layer=1, moved=moved)
    pool.evict(table, seqlen, w, budget=budget, recent=100, sinks=4, **({} if to is None else {"to": to}))
    _check_evicted(pool, seqlen, w, want)


@pytest.mark.parametrize("n", [4096, 16384, 32768, 65536])
def test_eviction_of_long_rows_of_equal_weights(n, cuda):
    """Every weight is at the threshold, as many as the counts hold."""
    for recent, sinks in ((0, 0), (5, 2)):
        pool, table, seqlen, w, _, want = _evict_case([n], n // 2 + 1, recent, sinks, 1, 16, BF16, 64, n_layer=1,
                                                      weights=lambda capacity: torch.full((1, 1, 1, capacity), 0.25))
        pool.evict(table, seqlen, w, budget=n // 2 + 1, recent=recent, sinks=sinks)
        _check_evicted(pool, seqlen, w, want)


@pytest.mark.parametrize("kind", ["equal", "nan", "inf", "zeros", "negative", "tiny"])
def test_eviction_by_odd_weights(kind, cuda):
    def weights(capacity):
        w = torch.rand(1, 2, 2, capacity, generator=torch.Generator().manual_seed(3))
        if kind == "equal":
            w.fill_(0.5)
        elif kind == "nan":
            w[..., ::3] = math.nan
        elif kind == "inf":
            w[..., ::5], w[..., 1::7] = math.inf, -math.inf
        elif kind == "zeros":
            w[..., ::2], w[..., 1::2] = 0.0, -0.0
        elif kind == "negative":
            w -= 0.5
        else:
            w *= 2.0 ** -140
        return w
    pool, table, seqlen, w, _, want = _evict_case([200, 333], 64, 10, 3, 2, 64, BF16, 16, n_layer=1, weights=weights)
    pool.evict(table, seqlen, w, budget=64, recent=10, sinks=3)
    _check_evicted(pool, seqlen, w, want)


def test_eviction_of_more_layers_than_a_launch_takes(cuda):
    pool, table, seqlen, w, _, want = _evict_case([90, 20, 33], 24, 8, 1, 2, 16, BF16, 16, n_layer=70)
    pool.evict(table, seqlen, w, budget=24, recent=8, sinks=1)
    _check_evicted(pool, seqlen, w, want)


def test_eviction_twice_and_captured(cuda):
    """The second eviction finds rows at their budget (nothing to do), and a replay goes by the rows of its time."""
    pool, table, seqlen, w, _, want = _evict_case([300, 100, 40], 64, 16, 4, 2, 128, BF16, 16)
    start = [t.clone() for t in pool.keys + pool.values + [seqlen, w]]

    def restore():
        for t, was in zip(pool.keys + pool.values + [seqlen, w], start):
            t.copy_(was)
    pool.evict(table, seqlen, w, budget=64, recent=16, sinks=4)
    pool.evict(table, seqlen, w, budget=64, recent=16, sinks=4)
    _check_evicted(pool, seqlen, w, want)
    restore()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        pool.evict(table, seqlen, w, budget=64, recent=16, sinks=4)
    for _ in range(3):
        restore()
        graph.replay()
        torch.cuda.synchronize()
        _check_evicted(pool, seqlen, w, want)
        graph.replay()
        torch.cuda.synchronize()
        _check_evicted(pool, seqlen, w, want)


def test_eviction_with_a_wide_account_and_table(cuda):
    """Rows of tables and accounts inside larger tensors; entries past a row's blocks name none."""
    pool, table, seqlen, w, _, want = _evict_case([130, 70], 32, 5, 0, 2, 64, F16, 16, width=12)
    tables = torch.full((2, 3, 12), -1, dtype=torch.int32, device=cuda)
    tables[:, 1] = table
    accounts = torch.full((2, 2, 5, 12 * 16 + 8), 3.0, device=cuda)
    part = accounts[:, :, 1:4:2, : 12 * 16]
    part.copy_(w)
    pool.evict(tables[:, 1], seqlen, part, budget=32, recent=5)
    _check_evicted(pool, seqlen, part, want)
    assert (accounts[:, :, ::2] == 3).all() and (accounts[..., 12 * 16:] == 3).all()


def test_eviction_reports_tables_that_leave_the_pool(cuda):
    pool, table, seqlen, w, _, want = _evict_case([100, 100], 40, 10, 2, 1, 64, BF16, 16, n_layer=1)
    good_k = want[0][0]
    table[1, 0] = pool.n_blocks + 5
    pool.evict(table, seqlen, w, budget=40, recent=10, sinks=2)
    with pytest.raises(IndexError, match="token 1 of"):
        pool.check_writes()
    row = table[0, :3].long()
    assert torch.equal(pool.keys[0][row].cpu(), good_k[row.cpu()]) and torch.equal(seqlen.cpu(), want[3])


def test_eviction_refusals(cuda):
    with pytest.raises(ValueError, match="4-bit pool"):
        pool = Fp4PagedPool(1, 4, 16, 2, 64, dtype=BF16, device=cuda)
        pool.evict(torch.zeros(1, 2, dtype=torch.int32, device=cuda), torch.zeros(1, dtype=torch.int32, device=cuda),
                   torch.zeros(1, 1, 2, 32, device=cuda), budget=4, recent=1)
    pool = PagedPool(1, 4, 16, 2, 64, dtype=BF16, device=cuda)
    args = [torch.zeros(1, 2, dtype=torch.int32, device=cuda), torch.zeros(1, dtype=torch.int32, device=cuda),
            torch.zeros(1, 1, 2, 32, device=cuda)]
    for i in range(3):
        with pytest.raises(ValueError, match="the pool is on"):
            pool.evict(*[t.cpu() if j == i else t for j, t in enumerate(args)], budget=4, recent=1)
    pool.keys = [pool.keys[0][:, :, :, ::2]]
    with pytest.raises(ValueError, match="evict needs keys and values"):
        pool.evict(*args, budget=4, recent=1)
    odd = PagedPool(1, 4, 16, 2, 24, dtype=BF16, device=cuda)
    with pytest.raises(ValueError, match="power of two"):
        odd.evict(*args, budget=4, recent=1)


# ------------------------------------------------------------------ together
def test_prompts_are_weighed_cut_and_decoded(cuda):
    """A packed prompt's account, the rows cut by it, steps that add to it, cut again: each stage against the oracle."""
    H, H_kv, D, bs, budget, recent, sinks = 8, 4, 64, 16, 48, 12, 4
    lengths = [100, 30, 77]
    g = torch.Generator().manual_seed(5)
    pool = PagedPool(1, 40, bs, H_kv, D, dtype=BF16, device=cuda, n_head=H)
    tables = torch.randperm(40, generator=g)[:21].view(3, 7).int()
    packed, _ = PackedPrefill.upload([[1] * n for n in lengths], pool, tables.tolist(), cuda)
    q, k, v = (torch.randn(1, sum(lengths), h, D, generator=g).bfloat16().cuda() for h in (H, H_kv, H_kv))
    packed.write(0, k, v)
    account = torch.full((1, 3, H_kv, 7 * bs), math.nan, device=cuda)
    packed.weigh(q, k, observe=16, out=account[0])
    want, bound = bounded.prompt_weights(q[0].cpu(), k[0].cpu(), packed.cu_seqlens, 16)
    _within(account[0, :, :, :100], want, bound)
    seqlen = torch.tensor(lengths, dtype=torch.int32, device=cuda)
    table = tables.cuda()
    plan = pool.decode_plan(torch.empty(3, H, D, dtype=BF16, device=cuda), table, seqlen)
    for _ in range(3):
        after = bounded.evicted([pool.keys[0].cpu()], [pool.values[0].cpu()], tables, seqlen.cpu(), account.cpu(), budget, recent, sinks)
        pool.evict(table, seqlen, account, budget=budget, recent=recent, sinks=sinks)
        _check_evicted(pool, seqlen, account, after)
        for _ in range(9):
            at = seqlen.long()
            slots = table[torch.arange(3, device=cuda), at // bs].long() * bs + at % bs
            pool.write_slots(0, slots, *(torch.randn(3, H_kv, D, generator=g).bfloat16().cuda() for _ in range(2)))
            seqlen += 1
            qs = torch.randn(3, H, D, generator=g).bfloat16()
            out, bound, w, w_bound = bounded.decode_rows(qs, pool.keys[0].cpu(), pool.values[0].cpu(), tables, seqlen.cpu())
            before = account[0].cpu()
            _within(plan.run_weighed(0, qs.cuda(), account[0]), out, bound)
            _within(account[0], before.double() + w, w_bound + 3 * 2.0 ** -24 * (before + w))


TINY = dict(vocab=512, hidden=256, inter=512, n_layer=2, n_head=4, n_kv_head=2, head_dim=128)


def _tiny(cuda, **kw):
    cfg = Qwen3Config(**TINY, **kw)
    return Qwen3(cfg, random_weights(cfg, 3), cuda, max_pos=1024)


def test_a_model_within_its_budget_decodes_as_without_one(cuda):
    """No row passes the budget: nothing is cut, and the account of a step over n tokens is one unit per head and layer."""
    m = _tiny(cuda)
    prompts = [[(7 * i + 3 * j) % 512 for j in range(n)] for i, n in enumerate((40, 25))]
    pools = [m.new_pool(32) for _ in range(2)]
    tables = [[list(range(8)), list(range(8, 16))] for _ in range(2)]
    account = torch.zeros(2, 2, 2, 8 * 16, device=cuda)
    logits = [m.prefill(prompts, pools[0], tables[0]), m.prefill(prompts, pools[1], tables[1], weights=account, observe=None)]
    assert torch.equal(*logits)
    first = logits[0].argmax(-1)
    plain = GraphDecoder(m, pools[0], tables[0], [40, 25], first, 20)
    cut = BudgetDecoder(m, pools[1], tables[1], [40, 25], first, 20, account, budget=80, recent=16, sinks=2)
    total = account.sum(-1)
    assert torch.allclose(total, torch.tensor([[80.0] * 2, [50.0] * 2], device=cuda).expand(2, 2, 2), rtol=1e-5)
    for d in (plain, cut):
        d.capture()
        for _ in range(20):
            d.step()
        d.check()
    assert torch.equal(cut.pos, plain.pos) and torch.equal(cut.held, plain.pos)
    assert torch.allclose(account.sum(-1) - total, torch.full_like(total, 40.0), rtol=1e-4)
    same = (plain.history == cut.history).float().mean()
    assert same == 1, plain.history


def test_a_model_past_its_budget_replays_what_it_does_eagerly(cuda):
    m = _tiny(cuda)
    prompts = [[(5 * i + j) % 512 for j in range(n)] for i, n in enumerate((150, 25, 60))]
    runs = []
    for captured in (False, True):
        pool = m.new_pool(64)
        tables = [list(range(12 * r, 12 * r + 12)) for r in range(3)]
        account = torch.zeros(2, 3, 2, 12 * 16, device=cuda)
        first = m.prefill(prompts, pool, tables, weights=account, observe=16).argmax(-1)
        d = BudgetDecoder(m, pool, tables, [150, 25, 60], first, 60, account, budget=64, recent=16, sinks=4, every=10)
        assert d.seqlen.tolist() == [64, 25, 60]
        if captured:
            d.capture()
        for _ in range(60):
            d.step()
        d.check()
        assert d.pos.tolist() == [210, 85, 120] and max(d.held.tolist()) <= 74
        runs.append((d.history, account, d.held))
    assert all(torch.equal(a, b) for a, b in zip(*runs))


def test_budget_decoder_refusals(cuda):
    m = _tiny(cuda)
    pool = m.new_pool(16)
    account = torch.zeros(2, 1, 2, 64, device=cuda)
    args = (m, pool, [[0, 1, 2, 3]], [20], torch.zeros(1, dtype=torch.long), 100, account)
    with pytest.raises(ValueError, match="cannot hold the 70"):
        BudgetDecoder(*args, budget=60, recent=10, every=10)
    with pytest.raises(ValueError, match="every must be"):
        BudgetDecoder(*args, budget=30, recent=10, every=0)
    with pytest.raises(ValueError, match="by itself"):
        BudgetDecoder(_tiny(cuda, window=8), *args[1:], budget=30, recent=10)
    with pytest.raises(ValueError, match="must be positive and hold"):
        BudgetDecoder(*args, budget=30, recent=28, sinks=4, every=10)
    with pytest.raises(ValueError, match="weights must be"):
        BudgetDecoder(*args[:6], account[:1], budget=30, recent=10, every=10)
    with pytest.raises(ValueError, match="4-bit pool"):
        four = Fp4PagedPool(2, 16, 16, 2, 128, dtype=BF16, device=cuda, n_head=4)
        BudgetDecoder(m, four, *args[2:], budget=30, recent=10, every=10)
    with pytest.raises(ValueError, match="under a window"):
        _tiny(cuda, window=8).prefill([[1, 2]], pool, [[0]], weights=account)


def test_budget_decoder_captured_with_its_rows_full(cuda):
    """The step that is recorded needs a free place: a decoder whose rows have grown to the end of their tables cuts them."""
    m = _tiny(cuda)
    pool, account = m.new_pool(8), torch.zeros(2, 1, 2, 48, device=cuda)
    first = m.prefill([list(range(20))], pool, [[5, 1, 2]], weights=account).argmax(-1)
    d = BudgetDecoder(m, pool, [[5, 1, 2]], [20], first, 90, account, budget=38, recent=8, sinks=2, every=10)
    for _ in range(28):
        d.step()
    assert d.seqlen.tolist() == [48]
    d.capture()
    assert d.held.tolist() == [38]
    for _ in range(40):
        d.step()
    d.check()
    assert d.pos.tolist() == [88] and d.held.tolist() == [48]


def test_budget_decoder_refuses_to_cut_shared_blocks(cuda):
    """An eviction in place would move one row's tokens under the other's; rows that stay within the budget may share."""
    m = _tiny(cuda)
    pool, account = m.new_pool(16), torch.zeros(2, 2, 2, 64, device=cuda)
    first = torch.zeros(2, dtype=torch.long)
    good = dict(budget=40, recent=8, every=10)
    for tables, lengths, max_new in (([[0, 1, 2, 3], [0, 4, 5, 6]], [20, 20], 21), ([[0, 1, 2, 3], [0, 4, 5, 6]], [4, 30], 11),
                                     ([[0, 1, 2, 3], [4, 5, 6, 4]], [1, 41], 0)):
        with pytest.raises(ValueError, match="in the tables twice"):
            BudgetDecoder(m, pool, tables, lengths, first, max_new, account, **good)
    d = BudgetDecoder(m, pool, [[0, 1, 2, 3], [0, 4, 5, 6]], [20, 17], first, 20, account, **good)
    for _ in range(20):
        d.step()
    d.check()
    assert d.held.tolist() == [40, 37]


def test_budget_decoder_stays_inside_the_rope_table(cuda):
    """Past the table no K/V could be written, so a text that would get there is refused, and so is the step that does."""
    cfg = Qwen3Config(**TINY)
    m = Qwen3(cfg, random_weights(cfg, 3), cuda, max_pos=64)
    pool, account = m.new_pool(16), torch.zeros(2, 2, 2, 64, device=cuda)
    tables = [[5, 1, 2, 9], [3, 4, 0, 7]]
    first = m.prefill([list(range(20)), list(range(9))], pool, tables, weights=account).argmax(-1)
    args = dict(budget=30, recent=8, sinks=2, every=10)
    with pytest.raises(ValueError, match="20 \\+ 45 tokens run past the RoPE table's 64"):
        BudgetDecoder(m, pool, tables, [20, 9], first, 45, account, **args)
    d = BudgetDecoder(m, pool, tables, [20, 9], first, 44, account, **args)
    d.capture()
    for _ in range(44):
        d.step()
    d.check()
    assert d.pos.tolist() == [64, 53]
    before = [t.clone() for t in (*pool.keys, *pool.values, account, d.pos, d.held, d.seqlen, d.tokens, d.history)]
    with pytest.raises(IndexError, match="position 64"):
        d.step()
    d.check()
    assert all(torch.equal(a, b) for a, b in zip((*pool.keys, *pool.values, account, d.pos, d.held, d.seqlen, d.tokens, d.history), before))


@pytest.mark.parametrize("captured", [False, True])
def test_a_row_that_a_step_skips_holds_what_it_held(captured, cuda):
    """A token outside the vocabulary: the row is reported and skipped, keeps its tokens through an eviction right after, and
    its next token goes behind them."""
    m = _tiny(cuda)
    pool, account = m.new_pool(32), torch.zeros(2, 2, 2, 128, device=cuda)
    tables = [list(range(8)), list(range(8, 16))]
    first = m.prefill([list(range(50)), list(range(25))], pool, tables, weights=account).argmax(-1)
    d = BudgetDecoder(m, pool, tables, [50, 25], first, 60, account, budget=40, recent=10, sinks=2, every=12)
    if captured:
        d.capture()
    d.tokens[1] = 512
    row = torch.tensor([8, 9], device=cuda)
    before = [s[row].view(32, 2, 128)[:25].clone() for s in pool.keys + pool.values]
    kept = account[:, 1].clone()
    d.step()
    assert d.held.tolist() == [41, 25]
    with pytest.raises(IndexError, match="row 1"):
        d.check()
    d.evict()
    assert d.held.tolist() == [40, 25] and d.seqlen.tolist() == [40, 25] and torch.equal(account[:, 1], kept)
    d.step()
    d.check()
    assert d.held.tolist() == [41, 26] and d.seqlen.tolist() == [41, 26]
    assert all(torch.equal(s[row].view(32, 2, 128)[:25], x) for s, x in zip(pool.keys + pool.values, before))
    for _ in range(29):
        d.step()
    d.check()
    assert d.held.tolist() == [46, 46] and d.pos.tolist() == [81, 56]  # cut 12 and 24 steps after the first cut


def test_calls_beside_each_other_on_two_streams(cuda):
    """Two plans, two packed groups and two pools, one on a stream each, among other calls that push the groups' schedules
    out: what each gives is what it gives alone."""
    g = torch.Generator().manual_seed(11)
    sides = []
    for i in range(2):
        q, k, v, table, seqlen = _cuda(*_rows([900 + 31 * i, 40, 300], 16, 8, 128, BF16, 16, seed=i))
        prompt = [torch.randn(700 + i, h, 128, generator=g).bfloat16().cuda() for h in (16, 8, 8)]
        pool = PagedPool(1, 64, 16, 8, 128, dtype=BF16, device=cuda, n_head=16)
        rows = torch.randperm(64, generator=g).int().view(2, 32).cuda()
        start = [torch.randn(64, 16, 8, 128, generator=g).bfloat16().cuda() for _ in range(2)]
        weights = torch.rand(1, 2, 8, 512, generator=g).cuda()
        sides.append((q, k, v, table, seqlen, prompt, pool, rows, start, weights, torch.cuda.Stream()))
    torch.cuda.synchronize()

    def go(q, k, v, table, seqlen, prompt, pool, rows, start, weights, stream):
        account = torch.zeros(3, 8, table.shape[1] * 16, device=cuda)
        outs = [paged_decode_plan(q, [k], [v], table, seqlen, window=200, sinks=3).run(0, q),
                paged_decode_plan(q, [k], [v], table, seqlen).run_weighed(0, q, account), account]
        args = dict(cu_seqlens=[0, prompt[0].shape[0]], max_seqlen=prompt[0].shape[0])
        for j in range(10):  # more groups than are kept
            x = prompt[0][: 40 + j]
            HipVarlen().prefill_varlen(x, prompt[1][: 40 + j], prompt[2][: 40 + j], cu_seqlens=[0, 40 + j],
                                       max_seqlen=40 + j, window=9)
            outs.append(HipVarlen().prefill_varlen(*prompt, **args, window=90, sinks=5))
            outs.append(HipVarlen().prompt_weights(*prompt[:2], **args))
        pool.keys[0].copy_(start[0])
        pool.values[0].copy_(start[1])
        w, n = weights.clone(), torch.tensor([500, 200], dtype=torch.int32).to(cuda)
        pool.evict(rows, n, w, budget=100, recent=30, sinks=4)
        return outs + [pool.keys[0].clone(), pool.values[0].clone(), w, n]

    alone = [go(*s) for s in sides]
    torch.cuda.synchronize()
    for _ in range(3):
        both = []
        for s in sides:
            with torch.cuda.stream(s[-1]):
                both.append(go(*s))
        torch.cuda.synchronize()
        for a, b in zip(alone, both):
            assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_a_windowed_model_served_from_a_pool_that_holds_its_windows_only(cuda):
    """Blocks that leave a seat's window go back to the pool: a second request runs beside the first in a pool that
    could not hold both whole, and gets the tokens that it gets from a large one."""
    trace = [TraceRequest(0, 0.0, tuple((11 * j) % 512 for j in range(100)), 70),
             TraceRequest(1, 0.0005, tuple((7 * j + 1) % 512 for j in range(20)), 70)]
    got = {}
    for window, n_blocks in ((32, 96), (32, 14), (None, 14)):
        server = ContinuousServer(_tiny(cuda, window=window, sinks=4 if window else 0), max_batch=2, n_blocks=n_blocks,
                                  max_prompt=100, max_new=70)
        server.warm()
        records, _ = server.run(trace, realtime=False, step_s=1e-3)
        assert server.blocks.n_free == n_blocks
        got[window, n_blocks] = [r.tokens for r in records], server.max_active
    assert got[32, 14] == got[32, 96] and got[32, 14][1] == 2 and got[None, 14][1] == 1


def test_a_windowed_model_decodes_what_its_prefill_computes(cuda):
    """The step after a prompt and the last row of the prompt with its token appended: the same attention on two ways."""
    m = _tiny(cuda, window=40, sinks=3)
    prompt = [(11 * j) % 512 for j in range(120)]
    pool = m.new_pool(32)
    first = m.prefill([prompt], pool, [list(range(10))]).argmax(-1)
    from miattn.paged import PagedKV

    kv = PagedKV(pool, [list(range(10))], [120], rope_len=160, n_head=4, window=40, sinks=3)
    step = m.decode(kv, first)
    whole = m.prefill([prompt + first.tolist()], m.new_pool(32), [list(range(10))])
    # both are bf16 passes of two layers: each of the stream's 12 roundings moves a logit by at most 2^-8 of its largest
    assert (step.float() - whole.float()).abs().max() <= 12 * 2.0 ** -8 * whole.float().abs().max()
    with pytest.raises(ValueError, match="build the PagedKV with the model's"):
        m.decode(PagedKV(pool, [list(range(10))], [120], rope_len=160, n_head=4), first)


# ------------------------------------------------------------------ far ends
def test_rows_at_the_far_end_of_a_large_pool(cuda):
    """Pools and accounts whose offsets pass 32 bits give the bits that small ones do."""
    H, H_kv, D, bs, far = 16, 8, 128, 16, 140000  # 2.3e9 elements of K
    lengths = [700, 90]
    q, k, v, table, seqlen = _cuda(*_rows(lengths, H, H_kv, D, BF16, bs))
    n, width = k.shape[0], table.shape[1] * bs
    small, large = (PagedPool(1, m, bs, H_kv, D, dtype=BF16, device=cuda, n_head=H) for m in (n, far))
    for store, part in ((small.keys, k), (small.values, v)):
        store[0].copy_(part)
    for store, part in ((large.keys, k), (large.values, v)):
        store[0][far - n:].copy_(part)
    room = torch.empty(2**31 + H_kv * width, device=cuda)
    far_account = room.as_strided((1, 2, H_kv, width), (0, 2**31, width, 1))
    near = torch.rand(1, 2, H_kv, width, device=cuda)
    far_account.copy_(near)
    got = []
    for pool, at, account in ((small, table, near), (large, torch.where(table < 0, table, table + far - n), far_account)):
        left = seqlen.clone()
        outs = [pool.decode_plan(q, at, left, window=100, sinks=4).run(0, q),
                pool.decode_plan(q, at, left).run_weighed(0, q, account[0])]
        pool.evict(at, left, account, budget=64, recent=10, sinks=4)
        outs += [account.clone(), left, pool.decode_plan(q, at, left).run(0, q)]
        pool.check_writes()
        got.append(outs)
    assert got[0][3].tolist() == [64, 64] and all(torch.equal(a, b) for a, b in zip(*got))


def test_a_group_whose_offsets_pass_32_bits(cuda):
    """The last of 66 long prompts gets what it gets alone."""
    L, n, H, H_kv, D = 16384, 66, 16, 8, 128  # 2.2e9 elements of q
    q, k, v = (torch.empty(n * L, h, D, dtype=BF16, device=cuda).normal_() for h in (H, H_kv, H_kv))
    last = [t[(n - 1) * L:].clone() for t in (q, k, v)]
    one, all_of = dict(cu_seqlens=[0, L], max_seqlen=L), dict(cu_seqlens=list(range(0, n * L + 1, L)), max_seqlen=L)
    out = HipVarlen().prefill_varlen(q, k, v, **all_of, window=300, sinks=4)[(n - 1) * L:]
    assert torch.equal(out, HipVarlen().prefill_varlen(*last, **one, window=300, sinks=4))
    w = HipVarlen().prompt_weights(q, k, **all_of)[-1]
    # cut into fewer pieces than alone, so against other reference maxima: exponents below 2^6 are rounded by up to 2^-19 each in a
    # weight and in its sum's terms, ln 2 of which a weight moves by, and 512 additions in a row add 2^-24 each
    assert torch.allclose(w, HipVarlen().prompt_weights(*last[:2], **one)[0], rtol=2 * 0.7 * 2.0 ** -19 + 512 * 2.0 ** -24 + 2.0 ** -20, atol=0)
