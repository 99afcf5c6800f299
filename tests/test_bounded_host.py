"""Windows, accounts and eviction without a GPU: the oracle against closed forms, the host arms against the
oracle, and the refusals of the Python and C entry points."""

from __future__ import annotations

import ctypes
import math
import os
import random
import subprocess
import sys

import pytest
import torch

from miattn import PagedPool, SdpaVarlen, _lib, paged_decode, paged_decode_plan
from miattn._contract import rows_apart
from miattn.decode import check_window
from miattn.qwen3 import Qwen3Config
from miattn.serve import BlockFreeList, ContinuousServer
from oracle import bounded


def _cu(lengths):
    cu = [0]
    for n in lengths:
        cu.append(cu[-1] + n)
    return cu


# ------------------------------------------------------------------ the oracle
def test_a_query_sees_its_window_and_the_sinks():
    assert bounded.seen(7, 2, 0).tolist() == [False] * 5 + [True] * 2
    assert bounded.seen(7, 2, 1).tolist() == [True] + [False] * 4 + [True] * 2
    assert bounded.seen(3, 8, 0).all() and bounded.seen(3, 2, 5).all() and bounded.seen(4, None, 0).all()


def test_decode_oracle_closed_forms():
    k = torch.randn(4, 16, 2, 32)
    v = torch.randn(4, 16, 2, 32)
    table, seqlen = torch.tensor([[2, 0, 3, 1]], dtype=torch.int32), torch.tensor([50])
    q = torch.randn(1, 4, 32)
    out, _, w, _ = bounded.decode_rows(q, k, v, table, seqlen, window=1)
    assert torch.allclose(out[0, 3], v[1, 1, 1].double())  # token 49: page 1, slot 1
    assert w[0, 0].nonzero().flatten().tolist() == [49] and w[0, 0, 49] == 2.0
    out, _, w, _ = bounded.decode_rows(torch.zeros_like(q), k, v, table, seqlen, window=3, sinks=2)
    want = torch.stack([v[2, 0, 0], v[2, 1, 0], v[3, 15, 0], v[1, 0, 0], v[1, 1, 0]]).double().mean(0)
    assert torch.allclose(out[0, 0], want) and torch.allclose(w[0, 1, [0, 1, 47, 48, 49]], torch.full((5,), 0.4).double())


def test_varlen_and_account_oracles_agree_with_the_plain_ones():
    from oracle.varlen import varlen_error_bound

    cu = _cu([37, 5, 20])
    q, k, v = (torch.randn(62, h, 16).bfloat16() for h in (4, 2, 2))
    out, bound = bounded.varlen(q, k, v, cu, 64, 0)
    ref, plain = varlen_error_bound(q, k, v, cu)
    assert torch.allclose(out.float(), ref) and torch.allclose(bound.float(), plain)
    w, _ = bounded.prompt_weights(q, k, cu, None)
    assert torch.allclose(w.sum(-1), torch.tensor([[74.0] * 2, [10.0] * 2, [40.0] * 2]).double())
    last, _ = bounded.prompt_weights(q, k, cu, 1)
    one = torch.softmax(q[36, 2].double() @ k[:37, 1].double().T / 4, 0) + \
        torch.softmax(q[36, 3].double() @ k[:37, 1].double().T / 4, 0)
    assert torch.allclose(last[0, 1, :37], one)


# ------------------------------------------------------------------ the host arms
@pytest.mark.parametrize("lengths,window,sinks", [([37, 1, 90], 8, 0), ([64], 5, 3), ([20, 33], 100, 7), ([16], 1, 0)])
def test_sdpa_arm_under_a_window(lengths, window, sinks):
    cu = _cu(lengths)
    q, k, v = (torch.randn(cu[-1], h, 32) for h in (4, 2, 2))
    got = SdpaVarlen().prefill_varlen(q, k, v, cu_seqlens=cu, max_seqlen=max(lengths), window=window, sinks=sinks)
    out, _ = bounded.varlen(q.bfloat16(), k.bfloat16(), v.bfloat16(), cu, window, sinks)  # only its mask matters here
    exact, _ = bounded.varlen(q.half(), k.half(), v.half(), cu, window, sinks)
    assert (got - exact.float()).abs().max() < 2e-2 and (got - out.float()).abs().max() < 2e-1
    got64 = SdpaVarlen().prefill_varlen(q.half().double(), k.half().double(), v.half().double(), cu_seqlens=cu,
                                        max_seqlen=max(lengths), window=window, sinks=sinks)
    assert torch.allclose(got64, exact, atol=1e-12)


@pytest.mark.parametrize("observe", [1, 7, None])
def test_sdpa_arm_of_the_account(observe):
    cu = _cu([30, 1, 12])
    q, k = torch.randn(43, 6, 16), torch.randn(43, 2, 16)
    out = torch.full((3, 2, 40), math.nan)
    got = SdpaVarlen().prompt_weights(q, k, cu_seqlens=cu, max_seqlen=30, observe=observe, out=out)
    want, _ = bounded.prompt_weights(q, k, cu, observe)
    assert got is out and torch.allclose(got[..., :30].double(), want, atol=1e-5) and not got[..., 30:].any()


@pytest.mark.parametrize("observe", [None, 9])
@pytest.mark.parametrize("value", [math.inf, math.nan])
def test_sdpa_arm_of_the_account_behind_a_query_that_is_not_finite(observe, value):
    q, k = torch.randn(30, 6, 16), torch.randn(30, 2, 16)
    args = dict(cu_seqlens=[0, 12, 30], max_seqlen=18, observe=observe)
    want = SdpaVarlen().prompt_weights(q, k, **args)
    q[25, 1, 3] = value
    got = SdpaVarlen().prompt_weights(q, k, **args)
    assert got[1, 0, :14].isnan().all()
    got[1, 0, :14] = want[1, 0, :14]
    assert torch.equal(got, want)


def _pool(n_layer=2, n_blocks=12, bs=4, H_kv=2, D=4, dtype=torch.float32):
    pool = PagedPool(n_layer, n_blocks, bs, H_kv, D, dtype=dtype)
    for store in pool.keys + pool.values:
        store.copy_(torch.randn(store.shape))
    return pool


@pytest.mark.parametrize("budget,recent,sinks", [(5, 2, 1), (7, 0, 0), (4, 4, 0), (3, 1, 2), (40, 3, 3), (1, 0, 0)])
@pytest.mark.parametrize("moved", [False, True])
def test_host_eviction_against_the_oracle(budget, recent, sinks, moved):
    pool = _pool(n_blocks=20)
    table = torch.randperm(20)[:9].view(3, 3).int()
    to = torch.tensor(sorted(set(range(20)) - set(table.flatten().tolist())))[torch.randperm(11)][:9].view(3, 3).int()
    seqlen = torch.tensor([11, 0, 6], dtype=torch.int32)
    weights = torch.rand(2, 3, 2, 12)
    weights[0, 0, 0, 2:6] = 0.25  # ties
    weights[1, 0, 1, 3], weights[1, 2, 0, 1], weights[0, 2, 1, :4] = math.nan, math.inf, torch.tensor([0.0, -0.0, 0.0, -1.0])
    want = bounded.evicted(pool.keys, pool.values, table, seqlen, weights, budget, recent, sinks, to if moved else None)
    pool.evict(table, seqlen, weights, budget=budget, recent=recent, sinks=sinks, **({"to": to} if moved else {}))
    assert all(torch.equal(a, b) for a, b in zip(pool.keys + pool.values, want[0] + want[1]))
    assert torch.equal(weights.nan_to_num(7), want[2].nan_to_num(7)) and torch.equal(seqlen, want[3])


@pytest.mark.parametrize("moved", [False, True])
@pytest.mark.parametrize("page", [-1, 12, -13, 2**31 - 1])
def test_host_eviction_refuses_tables_that_leave_the_pool(page, moved):
    """A row's kept tokens in no block of the pool, or bound for none: refused before any row is moved."""
    pool = _pool()
    table = torch.tensor([[0, 1, 2], [3, 4, 5]], dtype=torch.int32)
    to = torch.tensor([[6, 7], [8, 9]], dtype=torch.int32)
    seqlen, weights = torch.tensor([12, 11], dtype=torch.int32), torch.rand(2, 2, 2, 12)
    before = [t.clone() for t in (*pool.keys, *pool.values, weights, seqlen)]
    args = dict(budget=7, recent=3, sinks=1, **({"to": to} if moved else {}))
    for at, place in [(table, (1, 2)), (table, (1, 0)), *([(to, (1, 1))] if moved else [])]:
        was = int(at[place])
        at[place] = page
        with pytest.raises(IndexError, match="row 1.*outside the pool"):
            pool.evict(table, seqlen, weights, **args)
        at[place] = was
        assert all(torch.equal(a, b) for a, b in zip((*pool.keys, *pool.values, weights, seqlen), before))
    # entries behind a row's tokens, and of a block that keeps none of them, name what they like
    table[1, 2], weights[:, 1, :, 4:8] = page, -1.0
    table[1, 1], seqlen[1] = page, 8
    weights[:, 1, :, :4] = 1.0
    one = torch.tensor([[6, page], [7, page]], dtype=torch.int32)
    want = bounded.evicted(pool.keys, pool.values, table, seqlen, weights, 4, 0, 0, one if moved else None)
    pool.evict(table, seqlen, weights, budget=4, recent=0, **({"to": one} if moved else {}))
    assert all(torch.equal(a, b) for a, b in zip(pool.keys + pool.values, want[0] + want[1]))
    assert torch.equal(weights, want[2]) and seqlen.tolist() == [4, 4]


# ------------------------------------------------------------------ refusals
@pytest.mark.parametrize("window,sinks", [(0, 0), (-3, 0), (True, 0), (1.5, 0), (4, -1), (None, 2), ("4", 0), (4, 0.5)])
def test_windows_that_are_refused(window, sinks):
    q = torch.zeros(1, 2, 32)
    pools = [torch.zeros(1, 16, 1, 32)]
    table, seqlen = torch.zeros(1, 1, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    with pytest.raises(ValueError, match="window|sinks"):
        paged_decode(q, pools[0], pools[0], table, seqlen, window=window, sinks=sinks)
    with pytest.raises(ValueError, match="window|sinks"):
        paged_decode_plan(q, pools, pools, table, seqlen, window=window, sinks=sinks)
    with pytest.raises(ValueError, match="window|sinks"):
        SdpaVarlen().prefill_varlen(q, pools[0][0, :1], pools[0][0, :1], cu_seqlens=[0, 1], max_seqlen=1, window=window,
                                    sinks=sinks)


def test_a_window_is_held_to_32_bits_and_causal():
    assert check_window(2**40, 2**33) == (2**31 - 1, 2**31 - 1) and check_window(None, 0) is None
    x = torch.zeros(2, 1, 8)
    with pytest.raises(ValueError, match="causal"):
        SdpaVarlen().prefill_varlen(x, x, x, cu_seqlens=[0, 2], max_seqlen=2, window=1, causal=False)


def test_account_refusals():
    q, k = torch.zeros(5, 4, 8), torch.zeros(5, 2, 8)
    arm = SdpaVarlen()
    for observe in (0, -1, True, 2.0):
        with pytest.raises(ValueError, match="observe"):
            arm.prompt_weights(q, k, cu_seqlens=[0, 5], max_seqlen=5, observe=observe)
    for out in (torch.zeros(1, 2, 4), torch.zeros(1, 4, 5), torch.zeros(1, 2, 5).double(), torch.zeros(1, 5, 2).transpose(1, 2),
                torch.zeros(1, 1, 5).expand(1, 2, 5), torch.zeros(9).as_strided((1, 2, 5), (9, 4, 1))):
        with pytest.raises(ValueError, match="out must be"):
            arm.prompt_weights(q, k, cu_seqlens=[0, 5], max_seqlen=5, out=out)
    with pytest.raises(ValueError, match="3-D"):
        arm.prompt_weights(q[0], k, cu_seqlens=[0, 5], max_seqlen=5)


def test_rows_that_are_written_lie_apart():
    t = torch.zeros(3, 4, 5, 6)
    for ok in (t, t.transpose(0, 2), t[:, ::2, 1:, :4], t[:1].expand(1, 4, 5, 6), t[:0], t[:, 0], t[0, 0, 0]):
        assert rows_apart(ok)
    for bad in (t[:1].expand(3, 4, 5, 6), t[:, :, :1].expand(3, 4, 5, 6), torch.zeros(20).as_strided((2, 6), (5, 1)),
                torch.zeros(99).as_strided((3, 4, 6), (12, 6, 1))):
        assert not rows_apart(bad)


def test_eviction_refusals():
    pool = _pool()
    table, seqlen = torch.zeros(2, 3, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    weights = torch.zeros(2, 2, 2, 12)
    good = dict(budget=4, recent=1, sinks=1)
    for bad in (dict(budget=0, recent=0), dict(budget=4, recent=3, sinks=2), dict(budget=4, recent=-1), dict(budget=4, recent=0, sinks=-1)):
        with pytest.raises(ValueError, match="budget"):
            pool.evict(table, seqlen, weights, **bad)
    with pytest.raises(ValueError, match="must be an int"):
        pool.evict(table, seqlen, weights, budget=4.0, recent=1)
    with pytest.raises(ValueError, match="int32"):
        pool.evict(table.long(), seqlen, weights, **good)
    with pytest.raises(ValueError, match="seqlen"):
        pool.evict(table, seqlen.long(), weights, **good)
    with pytest.raises(ValueError, match="seqlen"):
        pool.evict(table, torch.zeros(3, dtype=torch.int32), weights, **good)
    for w in (weights.double(), weights[:1], weights[..., :11], torch.zeros(2, 2, 12, 2).transpose(2, 3),
              weights[:, :1].expand(2, 2, 2, 12), weights[:1].expand(2, 2, 2, 12)):
        with pytest.raises(ValueError, match="weights must be"):
            pool.evict(table, seqlen, w, **good)
    with pytest.raises(ValueError, match="a row for each"):
        pool.evict(table, seqlen, weights, to=table[:1], **good)
    with pytest.raises(ValueError, match="too few"):
        pool.evict(table, seqlen, weights, to=table[:, :1], budget=5, recent=1)
    pool.evict(table[:0], seqlen[:0], weights[:, :0], **good)  # no rows: nothing to do


def test_c_entries_refuse_before_any_launch():
    lib, s15 = _lib.lib, _lib.int64_array([1] * 15)
    decode = (None, None, None, None, None, None, 1, 4, 2, 128, 16, 4, s15, 1.0, 2)
    for window, sinks in ((0, 0), (-1, 0), (4, -1)):
        assert lib.mi_paged_decode_window(*decode, window, sinks, None, 0, None) == _lib.MI_ERR_INVALID
        assert "window must be" in _lib.last_error()
    assert lib.mi_paged_decode_window(None, None, None, None, None, None, 1, 3, 2, *decode[9:], 4, 0, None, 0, None) == _lib.MI_ERR_INVALID
    assert lib.mi_paged_decode_weigh(*decode, None, 0, 0, None, 0, None) == _lib.MI_ERR_INVALID
    assert lib.mi_paged_decode_weigh(*decode, 64, 0, 0, None, 0, None) == _lib.MI_ERR_WORKSPACE
    assert lib.mi_paged_decode_weigh(None, None, None, None, None, None, 1, 4, 2, 16, 16, 4, s15, 1.0, 2, 64, 0, 0, None, 0,
                                     None) == _lib.MI_ERR_UNSUPPORTED
    assert lib.mi_paged_decode_weigh_workspace_size(2, 4, 2, 128, 16, 4, 2) == \
        lib.mi_paged_decode_workspace_size(2, 4, 2, 128, 16, 4, 2) + 2 * 4 * 64 * 4
    cu = (ctypes.c_int32 * 3)(0, 100, 230)
    assert lib.mi_varlen_schedule_window(cu, 2, 4, 2, 128, 0, 0, None, 0) == _lib.MI_ERR_INVALID
    assert lib.mi_varlen_schedule_window(cu, 2, 256, 2, 128, 8, 0, None, 0) == _lib.MI_ERR_UNSUPPORTED
    assert lib.mi_varlen_schedule_window(cu, 2, 4, 2, 80, 8, 0, None, 0) == _lib.MI_ERR_UNSUPPORTED
    n = lib.mi_varlen_schedule_window(cu, 2, 4, 2, 128, 8, 0, None, 0)
    words = (ctypes.c_int32 * n)()
    assert n > 0 and lib.mi_varlen_schedule_window(cu, 2, 4, 2, 128, 8, 0, words, n) == n
    assert lib.mi_varlen_schedule_window(cu, 2, 4, 2, 128, 8, 0, words, n - 1) == _lib.MI_ERR_INVALID
    launch = (64, 64, 64, 64, 64, 2, 230, 130, 64, *words[:4])
    tail = (None, 0, None, None)
    # a plain schedule's layout, the windowed one's on the plain entry, a scale that is not positive
    assert lib.mi_varlen_prefill_window(*launch[:-1], (3 << 20) | (128 << 8) | 64, 4, 2, 128, 1.0, 8, 0, 2, *tail) == _lib.MI_ERR_INVALID
    assert lib.mi_varlen_prefill(*launch, 4, 2, 128, 1.0, 1, 2, *tail) == _lib.MI_ERR_INVALID
    for scale in (0.0, -1.0, math.nan):
        assert lib.mi_varlen_prefill_window(*launch, 4, 2, 128, scale, 8, 0, 2, *tail) == _lib.MI_ERR_INVALID
    assert lib.mi_varlen_prefill_window(*launch, 4, 2, 128, 1.0, 8, 0, 0, *tail) == _lib.MI_ERR_UNSUPPORTED
    assert lib.mi_prompt_weights_schedule(cu, 2, 4, 2, 128, 0, None, 0) == _lib.MI_ERR_INVALID
    n = lib.mi_prompt_weights_schedule(cu, 2, 4, 2, 128, 32, None, 0)
    words = (ctypes.c_int32 * n)()
    assert lib.mi_prompt_weights_schedule(cu, 2, 4, 2, 128, 32, words, n) == n
    head = (ctypes.c_int32 * 8)(*words[:8])
    assert lib.mi_prompt_weights(64, 64, 64, head, 4, 2, 128, 1.0, 2, 64, 1, 1, 130, None, 0, None) == _lib.MI_ERR_WORKSPACE
    assert lib.mi_prompt_weights(64, 64, 64, head, 4, 2, 128, -1.0, 2, 64, 1, 1, 130, 64, 1 << 30, None) == _lib.MI_ERR_INVALID
    assert lib.mi_prompt_weights(64, 64, 64, head, 4, 2, 96, 1.0, 2, 64, 1, 1, 130, 64, 1 << 30, None) == _lib.MI_ERR_UNSUPPORTED
    pools = (ctypes.c_void_p * 1)(64)
    s3 = _lib.int64_array([1] * 3)

    def evict(n_blocks=8, bs=16, row_bytes=256, to_blocks=4, B=1, budget=8, recent=2, sinks=1, ws=1 << 20, store=pools):
        return lib.mi_cache_evict(store, store, 1, n_blocks, bs, 2, row_bytes, 64, 4, 4, 64, 4, to_blocks, 64, 64, s3, B,
                                  budget, recent, sinks, 64, ws, None, None)
    assert evict(budget=0) == evict(recent=8) == evict(sinks=-1) == evict(to_blocks=0) == _lib.MI_ERR_INVALID
    assert evict(row_bytes=48) == evict(row_bytes=2048) == evict(n_blocks=2**30) == _lib.MI_ERR_UNSUPPORTED
    assert evict(budget=33, to_blocks=2) == _lib.MI_ERR_INVALID and evict(ws=8) == _lib.MI_ERR_WORKSPACE
    assert evict(store=(ctypes.c_void_p * 1)(None)) == _lib.MI_ERR_INVALID and evict(B=0) == _lib.MI_OK


def test_accounts_refuse_a_schedule_of_another_call():
    """Other heads, or an account narrower than the longest segment, before any launch (the workspace holds all that they ask for)."""
    lib, cu = _lib.lib, (ctypes.c_int32 * 3)(0, 300, 310)
    n = lib.mi_prompt_weights_schedule(cu, 2, 4, 2, 128, 300, None, 0)
    words = (ctypes.c_int32 * n)()
    assert lib.mi_prompt_weights_schedule(cu, 2, 4, 2, 128, 300, words, n) == n
    head = (ctypes.c_int32 * 8)(*words[:8])

    def account(H, H_kv, width, workspace=None, ws_bytes=0):
        return lib.mi_prompt_weights(64, 64, 64, head, H, H_kv, 128, 1.0, 2, 64, H_kv * width, width, width, workspace,
                                     ws_bytes, None)
    for H, H_kv, width in ((8, 2, 300), (4, 4, 300), (2, 2, 300), (8, 4, 300), (2, 1, 300), (4, 2, 299), (4, 2, 10)):
        assert account(H, H_kv, width) == _lib.MI_ERR_INVALID and "does not fit" in _lib.last_error()
    for width in (300, 4096):  # the call that it was made for gets as far as its workspace
        assert account(4, 2, width) == _lib.MI_ERR_WORKSPACE


# ------------------------------------------------------------------ schedules and blocks
@pytest.mark.parametrize("lengths,window,sinks,D", [([700, 1, 64, 65], 100, 0, 128), ([4096], 512, 4, 128),
                                                    ([3000, 100], 64, 200, 64), ([129], 10**6, 0, 256)])
def test_windowed_items_cover_every_seen_key_once(lengths, window, sinks, D):
    cu = _cu(lengths)
    host = (ctypes.c_int32 * len(cu))(*cu)
    args = (host, len(lengths), 4, 2, D, window, sinks)
    n = _lib.lib.mi_varlen_schedule_window(*args, None, 0)
    words = (ctypes.c_int32 * n)()
    assert _lib.lib.mi_varlen_schedule_window(*args, words, n) == n
    n_wg, n_merge = words[0], words[1]
    assert words[3] == (5 << 20) | (D << 8) | 64
    pieces = {}
    for w in range(n_wg):
        first, count = words[4 + 8 * w], words[5 + 8 * w]
        for i in range(count):
            seq0, L, w2, w3 = (words[first + 4 * i + j] & 0xFFFFFFFF for j in range(4))
            pieces.setdefault((seq0, w2 >> 16, w3 >> 24), []).append(((w2 >> 8) & 0xFF, (w2 & 0xFF) + 1))
    want = {(a, t, h) for a, b in zip(cu, cu[1:]) for t in range(-(-(b - a) // 64)) for h in range(4)}
    assert set(pieces) == want
    for got in pieces.values():
        assert sorted(got) == [(i, got[0][1]) for i in range(got[0][1])]


@pytest.fixture(scope="module")
def band_tiles(tmp_path_factory):
    """The key tiles of a query tile, by the header that the schedule and the kernel include, built for the host."""
    out = tmp_path_factory.mktemp("band")
    csrc = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "llm-serving_amd", "csrc")
    (out / "band.cpp").write_text('''
#include "window_band.h"
extern "C" int tiles(int row0, int q_end, int window, int sinks, int* out) {
  const miattn::Band b = miattn::band_of(row0, q_end, window, sinks, 64);
  for (int t = 0; t < b.n; ++t) out[t] = miattn::band_tile(t, b.ts, b.jump);
  return b.n;
}
''')
    subprocess.run(["g++", "-O1", "-shared", "-fPIC", "-D__host__=", "-D__device__=", "-I", csrc, "-o", str(out / "band.so"),
                    str(out / "band.cpp")], check=True)
    lib = ctypes.CDLL(str(out / "band.so"))

    def tiles(row0, q_end, window, sinks):
        words = (ctypes.c_int * (q_end // 64 + 2))()
        return words[:lib.tiles(row0, q_end, window, sinks, words)]
    return tiles


def _tiles_seen(row0, q_end, window, sinks):
    """The 64-key tiles that hold a key which one of the rows sees, by the mask over all of their keys."""
    i, j = torch.arange(row0, q_end).unsqueeze(1), torch.arange(q_end)
    seen = ((j <= i) & ((i - j < window) | (j < sinks))).any(0)
    return sorted({t // 64 for t in seen.nonzero().flatten().tolist()})


def test_windowed_key_tiles_are_those_with_a_seen_key(band_tiles):
    rng = random.Random(4)
    draws = [(row0, rows, window, sinks) for row0 in (0, 64, 640) for rows in (1, 63, 64) for window in (1, 2, 64, 65, 10**6)
             for sinks in (0, 1, 64, 65, 700, 2**31 - 1)]
    draws += [(64 * rng.randrange(60), rng.randrange(1, 65), round(2 ** rng.uniform(0, 13)), rng.choice((0, round(2 ** rng.uniform(0, 13)))))
              for _ in range(1500)]
    for row0, rows, window, sinks in draws:
        assert band_tiles(row0, row0 + rows, window, sinks) == _tiles_seen(row0, row0 + rows, window, sinks), (row0, rows, window, sinks)


@pytest.mark.parametrize("lengths,window,sinks", [([700, 1, 64, 65], 100, 0), ([4096], 512, 4), ([3000, 100], 64, 200), ([129], 10**6, 0),
                                                  ([2500], 1, 0), ([1000, 333], 300, 70), ([2000], 1500, 0)])
def test_windowed_pieces_take_each_seen_key_tile_once(band_tiles, lengths, window, sinks):
    """The tiles that the pieces of a query tile walk, each its share of the numbers, and no other ones."""
    cu = _cu(lengths)
    args = ((ctypes.c_int32 * len(cu))(*cu), len(lengths), 2, 1, 128, window, sinks)
    n = _lib.lib.mi_varlen_schedule_window(*args, None, 0)
    words = (ctypes.c_int32 * n)()
    assert _lib.lib.mi_varlen_schedule_window(*args, words, n) == n
    walked, cut = {}, 0
    for w in range(words[0]):
        first, count = words[4 + 8 * w], words[5 + 8 * w]
        for i in range(count):
            seq0, L, w2, w3 = (words[first + 4 * i + j] & 0xFFFFFFFF for j in range(4))
            row0, split, n_split = 64 * (w2 >> 16), (w2 >> 8) & 0xFF, (w2 & 0xFF) + 1
            assert L == dict(zip(cu, lengths))[seq0]
            tiles = band_tiles(row0, min(L, row0 + 64), window, sinks)
            piece = tiles[split * len(tiles) // n_split: (split + 1) * len(tiles) // n_split]
            assert piece  # an item has at least one step
            cut += n_split > 1
            walked.setdefault((seq0, L, row0, w3 >> 24), []).extend(piece)
    assert (cut > 0) == (max(map(len, walked.values())) > 8)  # few items: those of more than 8 tiles are cut
    assert len(walked) == 2 * sum(-(-n // 64) for n in lengths)
    for (seq0, L, row0, _), tiles in walked.items():
        assert sorted(tiles) == _tiles_seen(row0, min(L, row0 + 64), window, sinks)


def test_hidden_blocks_of_a_seat():
    server = ContinuousServer.__new__(ContinuousServer)
    server.blocks = BlockFreeList(64, 16)
    server.window, server.sinks = 40, 4
    for n in range(1, 200):
        hidden = set(server._hidden(n))
        for j in range(0, n // 16 + 1):
            tokens = range(16 * j, min(16 * j + 16, n))
            unseen = len(tokens) == 16 and not any(t >= n - 40 or t < 4 for t in tokens)
            assert (j in hidden) == unseen, (n, j)
    server.window = None
    assert not list(server._hidden(10**6))


def test_config_defaults_see_everything():
    assert Qwen3Config().window is None and Qwen3Config().sinks == 0


def test_schedules_past_the_hosts_memory_are_errors():
    """A schedule that the host cannot hold comes back as an error code: no exception crosses the C entries."""
    script = """
import ctypes, resource, sys
from miattn import _lib
import torch
sizes = [(_lib.lib.mi_varlen_schedule_window, 64, 65535 * 64, (64, 0)), (_lib.lib.mi_prompt_weights_schedule, 1, 1 << 29, (1 << 29,))]
if __name__ == "__main__":
    held = int(open("/proc/self/statm").read().split()[0]) * resource.getpagesize()
    resource.setrlimit(resource.RLIMIT_AS, (held + (24 << 20),) * 2)
    for schedule, n, length, args in sizes:
        cu = (ctypes.c_int32 * (n + 1))(*(i * min(length, (1 << 31) // (n + 1)) for i in range(n + 1)))
        print(schedule(cu, n, 1, 1, 64, *args, None, 0), "out of host memory" in _lib.last_error(), flush=True)
"""
    done = subprocess.run([sys.executable, "-c", script], capture_output=True, text=True, timeout=100,
                          env={**os.environ, "PYTHONPATH": os.pathsep.join(sys.path)})
    assert done.returncode == 0 and done.stdout.split() == ["-2", "True"] * 2, done.stdout + done.stderr
