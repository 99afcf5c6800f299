"""The 4-bit cache and the page copies on a CPU-only host: the oracle's rounding, argument checks,
refusals at the C ABI, host pools' page copies, and the block bookkeeping of forks and compactions."""

from __future__ import annotations

import ctypes
import random

import pytest
import torch

from miattn import Fp4PagedPool, PagedPool, _lib, paged_decode_fp4, paged_decode_fp4_plan
from miattn import fp4 as fp4_mod
from miattn.serve import BlockFreeList
from oracle import fp4 as oracle


# ------------------------------------------------------------------ the format
def test_oracle_rounds_to_the_nearest_level_ties_to_even_and_saturates():
    x = torch.zeros(1, 64)
    x[0, :14] = torch.tensor([7.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, -0.2, -0.3, 6.5, 0.26, -5.1, 1e-9])
    x[0, 32:] = 0.0
    got = oracle.held(x)[0]
    want = [6.0, 0.0, 1.0, 1.0, 2.0, 2.0, 4.0, 4.0, 0.0, -0.5, 6.0, 0.5, -6.0, 0.0]
    assert got[:14].tolist() == want and not got[14:].any()
    codes, scales = oracle.encode(x)
    assert scales.tolist() == [[127, 7]]  # 7 * 2^0 holds the first group, an empty group has the least scale
    assert codes[0, 8].item() == 8  # a negative value that rounds to zero keeps its sign


def test_oracle_scale_is_the_smallest_that_holds_the_group():
    for most, byte in ((7.0, 127), (7.0000005, 128), (3.5, 126), (1.75, 125), (2.0 ** -118, 7), (1e-40, 7), (3e38, 252)):
        x = torch.zeros(1, 32)
        x[0, 5] = most
        assert oracle.encode(x)[1].item() == byte, most
    x[0, 5] = float("inf")
    assert oracle.encode(x)[1].item() == 255 and oracle.held(x).isnan().all()


# ------------------------------------------------------------------ refusals
@pytest.mark.parametrize("kw,error,match", [
    (dict(head_dim=96), ValueError, "head_dim 64, 128 or 256"),
    (dict(head_dim=32), ValueError, "head_dim 64, 128 or 256"),
    (dict(block_size=8), ValueError, "at least 16"),
    (dict(block_size=48), ValueError, "power of two"),
    (dict(dtype=torch.float64), ValueError, "fp16, bf16 or fp32"),
    (dict(device="cpu"), RuntimeError, "needs a CUDA"),
])
def test_pool_refuses_what_the_format_does_not_hold(kw, error, match):
    args = dict(n_layer=1, n_blocks=4, block_size=16, n_kv_head=2, head_dim=64, dtype=torch.bfloat16, device="cpu")
    with pytest.raises(error, match=match):
        Fp4PagedPool(**{**args, **kw})


def _inputs(H=4, H_kv=2, D=64, bs=16, lengths=(17, 5)):
    B = len(lengths)
    pages = torch.zeros(4, H_kv, fp4_mod.page_bytes(bs, D), dtype=torch.uint8)
    return [torch.randn(B, H, D), pages, pages.clone(), torch.zeros(B, 2, dtype=torch.int32),
            torch.tensor(lengths, dtype=torch.int32)]


def test_decode_never_falls_back_to_the_cpu():
    with pytest.raises(RuntimeError, match="CUDA"):
        paged_decode_fp4(*_inputs())
    with pytest.raises(RuntimeError, match="CUDA"):
        q, k, v, table, seqlen = _inputs()
        paged_decode_fp4_plan(q, [k], [v], table, seqlen)


@pytest.mark.parametrize("mutate,match", [
    (lambda a: a.__setitem__(0, a[0][0]), "must be \\(B, H, D\\)"),
    (lambda a: a.__setitem__(1, a[1][0]), "page_bytes"),
    (lambda a: a.__setitem__(1, a[1][:3]), "shapes differ"),
    (lambda a: a.__setitem__(0, a[0].double()), "fp16, bf16 or fp32"),
    (lambda a: (a.__setitem__(1, a[1].short()), a.__setitem__(2, a[2].short())), "uint8"),
    (lambda a: a.__setitem__(0, torch.randn(2, 4, 96)), "head_dim 64, 128 or 256"),
    (lambda a: a.__setitem__(0, a[0][:, :3]), "multiple of n_kv_head"),
    (lambda a: a.__setitem__(0, a[0][:, :0]), "multiple of n_kv_head"),
    (lambda a: (a.__setitem__(1, a[1][..., :272].contiguous()), a.__setitem__(2, a[2][..., :272].contiguous())), "at least 16"),
    (lambda a: (a.__setitem__(1, a[1][..., :100].contiguous()), a.__setitem__(2, a[2][..., :100].contiguous())), "at least 16"),
    (lambda a: a.__setitem__(3, a[3].long()), "int32"),
    (lambda a: a.__setitem__(3, a[3][:1]), "does not match q batch"),
    (lambda a: a.__setitem__(4, a[4].float()), "int32 or int64"),
    (lambda a: a.__setitem__(4, torch.tensor([33, 1], dtype=torch.int32)), "capacity"),
    (lambda a: a.__setitem__(4, torch.tensor([-1, 1], dtype=torch.int32)), ">= 0"),
])
def test_decode_validation_errors_are_value_errors(mutate, match):
    args = _inputs()
    mutate(args)
    with pytest.raises(ValueError, match=match):
        fp4_mod._check(*args)


def test_c_entries_refuse_bad_sizes_before_any_launch():
    lib, st = _lib.lib, _lib.int64_array([0] * 10)
    assert lib.mi_fp4_page_bytes(16, 128) == 1088 and lib.mi_fp4_page_bytes(0, 128) == 0

    def write(n=1, H_kv=2, D=64, blocks=4, bs=16, dtype=2, bits=64, strides=st):
        return lib.mi_kv_slot_write_fp4(None, None, None, bits, None, None, n, H_kv, D, blocks, bs, strides, dtype, None, None)

    def read(n=1, H_kv=2, D=64, blocks=4, bs=16, dtype=2, bits=64):
        return lib.mi_kv_slot_read_fp4(None, None, None, bits, None, None, n, H_kv, D, blocks, bs, dtype, None, None)

    for call in (write, read):
        assert call(D=32) == _lib.MI_ERR_UNSUPPORTED and "head_dim 32" in _lib.last_error()
        assert call(bs=8) == _lib.MI_ERR_UNSUPPORTED and call(bs=24) == _lib.MI_ERR_UNSUPPORTED
        assert call(dtype=7) == _lib.MI_ERR_INVALID and call(bits=16) == _lib.MI_ERR_INVALID
        assert call(n=-1) == _lib.MI_ERR_INVALID and call(H_kv=0) == _lib.MI_ERR_INVALID
        assert call() == _lib.MI_ERR_INVALID and "NULL" in _lib.last_error()
        assert call(n=0) == _lib.MI_OK
    assert write(strides=None) == _lib.MI_ERR_INVALID

    def decode(B=1, H=4, H_kv=2, D=64, bs=16, width=2, strides=st, dtype=2):
        return lib.mi_paged_decode_fp4(None, None, None, None, None, None, B, H, H_kv, D, bs, width, strides, 1.0, dtype,
                                       None, 0, None)

    assert decode(H=3) == _lib.MI_ERR_INVALID and decode(dtype=9) == _lib.MI_ERR_INVALID
    assert decode(D=512) == _lib.MI_ERR_UNSUPPORTED and decode(bs=4) == _lib.MI_ERR_UNSUPPORTED
    assert decode(width=0) == _lib.MI_ERR_INVALID and decode(strides=None) == _lib.MI_ERR_INVALID
    assert decode() == _lib.MI_ERR_INVALID and "NULL" in _lib.last_error()
    assert decode(B=0) == _lib.MI_OK
    # sizes and the workspace are looked at before any pointer is used
    dense = _lib.int64_array([256, 64, 1088, 544, 1088, 544, 256, 64, 2, 0])

    def placed(width=2, strides=dense, q=4096, workspace=4096, size=1 << 30):
        return lib.mi_paged_decode_fp4(q, 4096, 4096, 4096, 4096, 4096, 1, 4, 2, 64, 16, width, strides, 1.0, 2, workspace,
                                       size, None)

    need = lib.mi_paged_decode_fp4_workspace_size(1, 4, 2, 64, 16, 2, 2)
    assert need > 0 and lib.mi_paged_decode_fp4_workspace_size(1, 3, 2, 64, 16, 2, 2) == 0
    assert placed(workspace=None) == _lib.MI_ERR_WORKSPACE and placed(workspace=4100) == _lib.MI_ERR_WORKSPACE
    assert placed(size=need - 1) == _lib.MI_ERR_WORKSPACE
    assert placed(width=(1 << 26) + 1) == _lib.MI_ERR_UNSUPPORTED and "2^30" in _lib.last_error()
    assert placed(q=4104) == _lib.MI_ERR_UNSUPPORTED and "aligned" in _lib.last_error()
    assert placed(strides=_lib.int64_array([256, 60, 1088, 544, 1088, 544, 256, 64, 2, 0])) == _lib.MI_ERR_UNSUPPORTED
    assert placed(strides=_lib.int64_array([256, 64, 1080, 544, 1088, 544, 256, 64, 2, 0])) == _lib.MI_ERR_UNSUPPORTED

    def epilogue(B=1, H=4, H_kv=2, D=64, bs=16, rotary=64, row=512, n_pos=8, mode=0, parts=0):
        return lib.mi_qk_norm_rope_write_fp4(None, row, parts, None, None, None, None, n_pos, rotary, None, None, 64, None,
                                             None, None, None, None, B, H, H_kv, D, 4, bs, 1e-6, mode, 2, None, None)

    assert epilogue(row=511) == _lib.MI_ERR_INVALID and epilogue(n_pos=0) == _lib.MI_ERR_INVALID
    assert epilogue(mode=2) == _lib.MI_ERR_INVALID and epilogue(parts=-1) == _lib.MI_ERR_INVALID
    assert epilogue(rotary=128) == _lib.MI_ERR_UNSUPPORTED and epilogue(H=5) == _lib.MI_ERR_INVALID
    assert epilogue() == _lib.MI_ERR_INVALID and "NULL" in _lib.last_error()
    assert epilogue(B=0) == _lib.MI_OK


def test_c_page_copy_refuses_ids_outside_the_pool():
    pools = (ctypes.c_void_p * 1)(4096)
    ids = lambda *x: (ctypes.c_int32 * len(x))(*x)  # noqa: E731
    copy = _lib.lib.mi_copy_pages
    assert copy(pools, 1, 64, 4, ids(0, 4), ids(1, 2), 2, None) == _lib.MI_ERR_INVALID
    assert "move 1 (4 -> 2)" in _lib.last_error()
    assert copy(pools, 1, 64, 4, ids(0), ids(-1), 1, None) == _lib.MI_ERR_INVALID
    assert copy(pools, 1, 0, 4, ids(0), ids(1), 1, None) == _lib.MI_ERR_INVALID
    assert copy((ctypes.c_void_p * 1)(), 1, 64, 4, ids(0), ids(1), 1, None) == _lib.MI_ERR_INVALID
    assert copy(None, 0, 64, 4, None, None, 0, None) == _lib.MI_OK


# ------------------------------------------------------------------ page copies on a host pool
def test_host_pool_copies_blocks_and_refuses_ambiguous_copies():
    pool = PagedPool(2, 6, 4, 2, 8)
    for store in pool.keys + pool.values:
        store.copy_(torch.randn_like(store))
    before = [s.clone() for s in pool.keys + pool.values]
    pool.copy_blocks([1, 1, 4], [0, 3, 5])
    for old, new in zip(before, pool.keys + pool.values):
        want = old.clone()
        want[0], want[3], want[5] = old[1], old[1], old[4]
        assert torch.equal(new, want)
    pool.copy_blocks([], [])
    for src, dst, error, match in (([0], [6], IndexError, "outside the pool"), ([-1], [0], IndexError, "outside"),
                                   ([0, 1], [2], ValueError, "one destination per source"),
                                   ([0, 1], [2, 2], ValueError, "named twice"),
                                   ([0, 1], [1, 2], ValueError, "both a source and a destination"),
                                   ([0], [0], ValueError, "both a source and a destination"),
                                   ([0.5], [1], ValueError, "must be ints"), ([True], [2], ValueError, "must be ints")):
        with pytest.raises(error, match=match):
            pool.copy_blocks(src, dst)


# ------------------------------------------------------------------ block bookkeeping
def test_fork_shares_full_blocks_and_copies_the_partial_one():
    blocks = BlockFreeList(10, 16)
    a = blocks.take(4)
    table, src, dst = blocks.fork(a, 37)
    assert table[:2] == a[:2] and src == [a[2]] and dst == [table[2]] and len(table) == 4
    assert not set(table[2:]) & set(a) and blocks.n_free == 4
    again, src, dst = blocks.fork(table, 32, capacity=33)  # at a block boundary nothing is copied
    assert again[:2] == a[:2] and src == [] and dst == [] and len(again) == 3
    assert blocks.fork(a, 64, capacity=200) is None and blocks.n_free == 3  # too few blocks: nothing taken or shared
    blocks.give_back(a)
    assert blocks.n_free == 5  # the two shared blocks stay
    blocks.give_back(table)
    assert blocks.n_free == 7
    blocks.give_back(again)
    assert blocks.n_free == 10 and sorted(blocks.take(10)) == list(range(10))


def test_fork_refuses_lengths_that_the_tables_do_not_hold():
    blocks = BlockFreeList(10, 16)
    a = blocks.take(2)
    for length, capacity in ((33, None), (-1, None), (20, 15)):
        with pytest.raises(ValueError, match="hold"):
            blocks.fork(a, length, capacity)
    table, src, dst = blocks.fork(a, 0)
    assert not set(table) & set(a) and src == [] and dst == []


def test_blocks_come_back_in_the_order_they_did_without_sharing():
    blocks = BlockFreeList(6, 16)
    a, b = blocks.take(2), blocks.take(2)
    blocks.give_back(a)
    assert blocks.take(3) == [0, 1, 4] and b == [2, 3]


@pytest.mark.parametrize("seed", range(20))
def test_compact_keeps_every_table_reading_the_same_tokens(seed):
    """Random takes, forks and returns; the pool's blocks hold a tag each, and after a compaction every
    table still reads the tags it read before, on a packed pool."""
    rng = random.Random(seed)
    n = rng.randint(8, 60)
    blocks, pool = BlockFreeList(n, 4), PagedPool(1, n, 4, 1, 2)
    pool.keys[0][:] = torch.arange(n).view(n, 1, 1, 1)
    tables = []
    for _ in range(40):
        what = rng.random()
        if what < 0.5:
            got = blocks.take(rng.randint(1, 6))
            if got is not None:
                tables.append(got)
        elif what < 0.75 and tables:
            table = rng.choice(tables)
            got = blocks.fork(table, rng.randint(0, 4 * len(table)))
            if got is not None:
                if got[1]:
                    pool.copy_blocks(got[1], got[2])
                tables.append(got[0])
        elif tables:
            blocks.give_back(tables.pop(rng.randrange(len(tables))))
    read = [pool.keys[0][t].clone() for t in tables]
    free = blocks.n_free
    src, dst = blocks.compact(tables)
    assert not set(src) & set(dst)
    pool.copy_blocks(src, dst)
    used = {b for t in tables for b in t}
    assert used == set(range(len(used))) and blocks.n_free == free == n - len(used)
    for t, want in zip(tables, read):
        assert torch.equal(pool.keys[0][t], want)
    for t in tables:
        blocks.give_back(t)
    assert sorted(blocks.take(n)) == list(range(n))


def test_compact_refuses_tables_that_are_not_all_of_them():
    blocks = BlockFreeList(8, 16)
    a, b = blocks.take(3), blocks.take(2)
    with pytest.raises(ValueError, match="every live request"):
        blocks.compact([a])
    with pytest.raises(ValueError, match="every live request"):
        blocks.compact([a, b, [7]])
    with pytest.raises(ValueError, match="every live request"):
        blocks.compact([a, b, list(a)])  # not shared, yet in two tables
    for outside in (-1, 8):
        with pytest.raises(ValueError, match="every live request"):
            blocks.compact([a, [b[0], outside]])  # as many blocks as are held, one of them not the pool's
    assert blocks.compact([a, b]) == ([], [])


@pytest.mark.parametrize("D,most", [(64, 1 << 25), (128, 1 << 24), (256, 1 << 23)])
def test_decode_refuses_pages_past_its_32_bit_offsets(D, most):
    """Offsets inside a page of one KV head are 32 bits: the largest block sizes that fit are taken, the next is refused
    before anything is read."""
    lib, dense = _lib.lib, _lib.int64_array([512, 256, 1 << 34, 1 << 33, 1 << 34, 1 << 33, 512, 256, 1])
    assert lib.mi_fp4_page_bytes(most, D) < 1 << 31 <= lib.mi_fp4_page_bytes(2 * most, D)
    assert lib.mi_paged_decode_fp4_workspace_size(1, 4, 2, D, most, 1, 2) > 0
    assert lib.mi_paged_decode_fp4_workspace_size(1, 4, 2, D, 2 * most, 1, 2) == 0

    def call(bs):  # without a workspace, so a call of sizes that are taken ends there
        return lib.mi_paged_decode_fp4(4096, 4096, 4096, 4096, 4096, 4096, 1, 4, 2, D, bs, 1, dense, 1.0, 2, None, 0, None)

    assert call(most) == _lib.MI_ERR_WORKSPACE
    assert call(2 * most) == _lib.MI_ERR_UNSUPPORTED and "2^31" in _lib.last_error()
    q, table, seqlen = torch.zeros(1, 4, D), torch.zeros(1, 1, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    page = torch.zeros(1, dtype=torch.uint8).expand(1, 2, fp4_mod.page_bytes(2 * most, D))  # no memory behind it
    with pytest.raises(ValueError, match="below 2\\^31 bytes"):
        fp4_mod._check(q, page, page, table, seqlen)
    page = page[..., : fp4_mod.page_bytes(most, D)]
    assert fp4_mod._check(q, page, page, table, seqlen).page == most


def test_decode_counts_tokens_past_64_bits():
    """B * max_blocks * block_size = 2^64: refused, not taken for 0."""
    dense = _lib.int64_array([256, 64, 1 << 34, 1 << 33, 1 << 34, 1 << 33, 256, 64, 1])
    for B, width in ((1 << 20, 1 << 19), (1, 1 << 19), (1 << 20, 1)):
        rc = _lib.lib.mi_paged_decode_fp4(4096, 4096, 4096, 4096, 4096, 4096, B, 4, 2, 64, 1 << 25, width, dense, 1.0, 2,
                                          None, 0, None)
        assert rc == _lib.MI_ERR_UNSUPPORTED and "2^30" in _lib.last_error(), (B, width)


def test_decode_looks_at_the_strides_it_uses_only():
    page = 1088
    for H, H_kv, B, strides, taken in (
            (4, 2, 1, [1028, 128, 2 * page, page, 2 * page, page, 1028, 128, 1], True),
            (4, 2, 2, [1028, 128, 2 * page, page, 2 * page, page, 1028, 128, 1], False),
            (1, 1, 2, [128, 3, page, 7, page, 9, 128, 5, 1], True),
            (2, 1, 2, [256, 3, page, 7, page, 9, 256, 5, 1], False),
            (4, 2, 1, [512, 128, 2 * page, 8, 2 * page, page, 512, 128, 1], False),
            (4, 2, 1, [512, 128, 8, page, 2 * page, page, 512, 128, 1], False)):
        rc = _lib.lib.mi_paged_decode_fp4(4096, 4096, 4096, 4096, 4096, 4096, B, H, H_kv, 128, 16, 1,
                                          _lib.int64_array(strides), 1.0, 2, None, 0, None)
        # without a workspace, so a call whose strides are taken ends there
        assert rc == (_lib.MI_ERR_WORKSPACE if taken else _lib.MI_ERR_UNSUPPORTED), (H, H_kv, B, strides)


def test_page_copies_on_a_device_refuse_stores_that_are_not_the_pools():
    """The device's copy takes addresses, so a store put in the pool's place has to have its layout. The stores here are on
    the host: the checks come before anything is launched."""
    for i, wrong in ((0, lambda t: t[:4].clone()), (1, lambda t: t.double()), (2, lambda t: t.flatten(2))):
        pool = PagedPool(2, 8, 4, 2, 8)
        pool._on_device = True
        stores = pool.keys if i < 2 else pool.values
        stores[i % 2] = wrong(stores[i % 2])
        with pytest.raises(ValueError, match="keys and values of shape \\(8, 4, 2, 8\\)"):
            pool.copy_blocks([0], [5])
    pool = PagedPool(2, 8, 4, 2, 8)
    pool._on_device = True
    pool.keys[1] = torch.zeros(8, 4, 4, 8)[:, :, :2]
    with pytest.raises(ValueError, match="contiguous"):
        pool.copy_blocks([0], [5])


def test_fork_takes_any_sequence_of_blocks():
    """A table kept as a tuple forks as a list does, and no block is taken or shared by a call that fails."""
    blocks = BlockFreeList(10, 16)
    a = tuple(blocks.take(3))
    table, src, dst = blocks.fork(a, 37)
    assert table[:2] == list(a[:2]) and src == [a[2]] and dst == [table[2]] and blocks.n_free == 6
    blocks.give_back(list(a))
    blocks.give_back(table)
    assert blocks.n_free == 10


def test_compact_changes_nothing_when_a_table_cannot_be_rewritten():
    blocks = BlockFreeList(8, 16)
    gone, a, b = blocks.take(2), blocks.take(2), blocks.take(2)
    blocks.give_back(gone)
    with pytest.raises(TypeError, match="needs lists"):
        blocks.compact([a, tuple(b)])
    assert a == [2, 3] and b == [4, 5] and blocks.n_free == 4
    src, dst = blocks.compact([a, b])
    assert src == [4, 5] and dst == [0, 1] and a == [2, 3] and b == [0, 1]


def test_page_copies_on_a_device_refuse_stores_on_the_host():
    """The pool's own layout, but host memory: its addresses are nothing a device may read."""
    pool = PagedPool(2, 8, 4, 2, 8)
    pool._on_device = True
    with pytest.raises(ValueError, match="every store on its device, got one on cpu"):
        pool.copy_blocks([0], [5])
