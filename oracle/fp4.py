"""The 4-bit cache in 64 bits: its rounding, its page layout and the attention over it.

Written from the format's definition alone (groups of 32 elements under a scale 2^e, e the
smallest integer with max|x| <= 7 * 2^e in [-120, 125]; levels 0, 0.5, 1, 1.5, 2, 3, 4, 6 with a sign; nearest
level, ties to the even code; a group that is not finite reads as NaN), in float64 on the host.
"""

from __future__ import annotations

import math

import torch

LEVELS = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)
GROUP = 32


def encode(rows: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """(codes 0..15 ``(.., D)``, scale bytes ``(.., D / 32)``) of rows ``(.., D)``, one group at a time."""
    flat = rows.detach().double().cpu().reshape(-1, GROUP)
    codes = torch.zeros(flat.shape, dtype=torch.uint8)
    scales = torch.zeros(flat.shape[0], dtype=torch.uint8)
    for i, g in enumerate(flat):
        if not torch.isfinite(g).all():
            scales[i] = 255
            continue
        most = float(g.abs().max())
        e = -120
        while e < 125 and most > 7.0 * 2.0 ** e:
            e += 1
        scales[i] = e + 127
        dist = ((g.abs() * 2.0 ** -e).unsqueeze(1) - LEVELS).abs()
        best = dist.min(1).values
        near = dist == best.unsqueeze(1)  # one level, or the two of a tie: take the even code
        even_first = torch.tensor([0, 2, 4, 6, 1, 3, 5, 7])
        code = even_first[near[:, even_first].to(torch.uint8).argmax(1)]
        codes[i] = (code + 8 * torch.signbit(g)).to(torch.uint8)
    return codes.view(rows.shape), scales.view(*rows.shape[:-1], -1)


def decode(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """float64 values of :func:`encode`'s output."""
    value = LEVELS[(codes & 7).long()] * torch.where(codes >= 8, -1.0, 1.0).double()
    by = torch.where(scales == 255, torch.tensor(math.nan, dtype=torch.float64), 2.0 ** (scales.double() - 127))
    return value * by.repeat_interleave(GROUP, -1)


def held(rows: torch.Tensor) -> torch.Tensor:
    """What the cache holds of ``rows``, in float64."""
    return decode(*encode(rows))


def page_rows(pages: torch.Tensor, head_dim: int) -> torch.Tensor:
    """float64 rows ``(n_blocks, H_kv, block_size, head_dim)`` of uint8 pages ``(n_blocks, H_kv, page_bytes)``."""
    pages = pages.cpu()
    bs = pages.shape[-1] // (head_dim // 2 + head_dim // GROUP)
    n, h = pages.shape[:2]
    byte = pages[..., : bs * head_dim // 2].reshape(n, h, bs, head_dim // 2)
    codes = torch.empty(n, h, bs, head_dim, dtype=torch.uint8)
    codes[..., 0::2], codes[..., 1::2] = byte & 15, byte >> 4
    scales = pages[..., bs * head_dim // 2:].reshape(n, h, head_dim // GROUP, bs).permute(0, 1, 3, 2)
    return decode(codes, scales)


def paged_attention(q, k_pages, v_pages, table, seqlen, scale=None):
    """``(out, weight, spread)`` in float64: the attention, ``sum_t p_t |v_t|`` per output element (what a relative
    error of a term scales with) and the largest ``scale * sum_d |q_d k_d|`` per (row, head) (what the
    rounding of a score scales with)."""
    B, H, D = q.shape
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    q = q.detach().double().cpu()
    out, weight, spread = torch.zeros(B, H, D).double(), torch.zeros(B, H, D).double(), torch.zeros(B, H, 1).double()
    for b, n in enumerate(seqlen.tolist()):
        if n <= 0:
            continue
        ids = table[b].cpu().long()
        used = ids[: -(-n // (k_pages.shape[2] // (D // 2 + D // GROUP)))]
        k, v = (page_rows(p[used.to(p.device)], D).permute(1, 0, 2, 3).reshape(p.shape[1], -1, D)[:, :n]
                for p in (k_pages, v_pages))
        group = H // k.shape[0]
        for h in range(H):
            kh, vh = k[h // group], v[h // group]
            p = torch.softmax(scale * (kh @ q[b, h]), 0)
            out[b, h], weight[b, h] = p @ vh, p @ vh.abs()
            spread[b, h] = scale * (kh.abs() @ q[b, h].abs()).max()
    return out, weight, spread
