"""Attention under a window with sinks, accounts of attention weights and eviction by them, in float64 on the
CPU. Test infrastructure only.

Each function works from the definition: a mask over all of a row's tokens (no tile, split or page
appears), one softmax per query head, and for the eviction a sort of the row's tokens. ``*_bound`` values
are the largest error that a kernel may show which computes as the docstrings say; ``gamma(n)`` bounds the
relative error of an fp32 sum of ``n`` terms in any order.
"""

from __future__ import annotations

import math

import torch

from .decode import dense_kv
from .varlen import UNIT_ROUNDOFF

__all__ = ["seen", "decode_rows", "varlen", "prompt_weights", "evicted"]


def gamma(n):
    return n * 2.0 ** -24 / (1.0 - n * 2.0 ** -24)


def seen(n: int, window: int | None, sinks: int) -> torch.Tensor:
    """Which of a row's ``n`` tokens its query (the last one) sees."""
    at = torch.arange(n)
    return torch.ones(n, dtype=torch.bool) if window is None else (at >= n - window) | (at < sinks)


def _half_step(x: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    """Half a step of ``dtype`` around ``x`` (its smallest subnormal step included)."""
    return torch.finfo(dtype).eps / 2 * x.abs() + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def decode_rows(q, k_cache, v_cache, table, seqlen, *, window=None, sinks=0, scale=None):
    """``(out, out_bound, weights, weights_bound)``: float64 attention of one query per row over the tokens it sees
    and its weights summed over each KV head's query heads, ``(B, H_kv, capacity)``.

    The bounds are of fp32 arithmetic over the exact products of the inputs. A score ``s = scale q.k`` is a sum of D
    products (gamma(D)), scaled and shifted by the running maximum (six roundings more, counted generously, each
    relative to at most ``scale |q| |k|``), so a weight ``exp(s - m) / l`` and the sum ``l`` are each off by a
    relative ``d = gamma(D + 6) scale |q| max|k| + 2^-21``, the exp2 unit's few ulp included; sums over the
    row's n tokens, their rescaling and the merge of splits add ``gamma(2 n + 64)`` each."""
    B, H, D = q.shape
    H_kv, capacity = k_cache.shape[2], table.shape[1] * k_cache.shape[1]
    G = H // H_kv
    scale = 1.0 / math.sqrt(D) if scale is None else float(scale)
    out, bound = torch.zeros(B, H, D, dtype=torch.float64), torch.zeros(B, H, D, dtype=torch.float64)
    weights, w_bound = (torch.zeros(B, H_kv, capacity, dtype=torch.float64) for _ in range(2))
    for b in range(B):
        n = int(seqlen[b])
        if n == 0:
            continue
        mask = seen(n, window, sinks)
        at = mask.nonzero().flatten()
        bs = k_cache.shape[1]
        page = table[b].long()[at // bs]
        k, v = (c[page, at % bs].double() for c in (k_cache, v_cache))  # (seen, H_kv, D)
        for h in range(H):
            x = scale * (k[:, h // G] @ q[b, h].double())
            pi = torch.softmax(x, 0)
            o, a = pi @ v[:, h // G], pi @ v[:, h // G].abs()
            d = gamma(D + 6) * abs(scale) * float(q[b, h].double().norm() * k[:, h // G].norm(dim=-1).max()) + 2.0 ** -21
            rel = 2 * d + 2 * gamma(2 * len(at) + 64)
            out[b, h] = o
            bound[b, h] = _half_step(o.abs() + rel * (a + o.abs()), q.dtype) + rel * (a + o.abs())
            weights[b, h // G, at] += pi
            w_bound[b, h // G, at] += (rel + gamma(G + 2)) * pi + 2.0 ** -126
    return out, bound, weights, w_bound


def varlen(q, k, v, cu_seqlens, window: int, sinks: int, *, scale: float | None = None):
    """``(out, bound)`` of packed causal attention under a window with sinks; the bound is
    :func:`oracle.varlen.varlen_error_bound`'s, over the keys that each query sees."""
    scale = 1.0 / math.sqrt(q.shape[-1]) if scale is None else float(scale)
    u, D, group = UNIT_ROUNDOFF[q.dtype], q.shape[-1], q.shape[1] // k.shape[1]
    outs, bounds = [], []
    for a0, b0 in zip(cu_seqlens, cu_seqlens[1:]):
        qs = q[a0:b0].double().transpose(0, 1)
        ks, vs = (t[a0:b0].double().transpose(0, 1).repeat_interleave(group, 0) for t in (k, v))
        at = torch.arange(b0 - a0)
        back = at.unsqueeze(1) - at
        mask = (back >= 0) & ((back < window) | (at < sinks))
        pi = torch.softmax((torch.matmul(qs, ks.transpose(1, 2)) * scale).masked_fill(~mask, -math.inf), -1)
        o, a = torch.matmul(pi, vs), torch.matmul(pi, vs.abs())
        spread = (torch.matmul(pi, vs * vs) - o * o).clamp_min(0.0).sqrt()
        delta = gamma(D) * scale * qs.norm(dim=-1, keepdim=True) * ks.norm(dim=-1).amax(-1)[:, None, None]
        rest = (2 * delta + 2 * gamma(mask.sum(-1)[None, :, None] + 1.0) + 2.0 ** -20) * (a + o.abs())
        bound = u * o.abs() + u * (1 + 2 * u) * torch.maximum(a, spread) + rest
        outs.append(o.transpose(0, 1))
        bounds.append(bound.transpose(0, 1))
    return torch.cat(outs), torch.cat(bounds)


def prompt_weights(q, k, cu_seqlens, observe: int | None, *, scale: float | None = None):
    """``(weights, bound)``, ``(n_seqs, H_kv, longest)``: what each segment's last ``observe`` queries give its keys. The
    bound is :func:`decode_rows`'s for a weight, and ``gamma`` of the number of weights that a sum has."""
    D, group = q.shape[-1], q.shape[1] // k.shape[1]
    scale = 1.0 / math.sqrt(D) if scale is None else float(scale)
    longest = max(b - a for a, b in zip(cu_seqlens, cu_seqlens[1:]))
    out, bound = (torch.zeros(len(cu_seqlens) - 1, k.shape[1], longest, dtype=torch.float64) for _ in range(2))
    for s, (a, b) in enumerate(zip(cu_seqlens, cu_seqlens[1:])):
        n = b - a
        first = 0 if observe is None else max(0, n - observe)
        qs = q[a + first: b].double().transpose(0, 1)
        ks = k[a:b].double().transpose(0, 1).repeat_interleave(group, 0)
        mask = torch.arange(n) <= torch.arange(first, n).unsqueeze(1)
        pi = torch.softmax((torch.matmul(qs, ks.transpose(1, 2)) * scale).masked_fill(~mask, -math.inf), -1)
        d = gamma(D + 6) * scale * qs.norm(dim=-1, keepdim=True) * ks.norm(dim=-1).amax(-1)[:, None, None] + 2.0 ** -21
        rel = 2 * d + 2 * gamma(2 * n + 64)
        out[s, :, :n] = pi.sum(1).view(-1, group, n).sum(1)
        terms = gamma((n - first) * group + 2)
        bound[s, :, :n] = ((rel + terms) * pi).sum(1).view(-1, group, n).sum(1) + 2.0 ** -120
    return out, bound


def evicted(keys, values, table, seqlen, weights, budget: int, recent: int, sinks: int, to=None):
    """The pools, accounts and lengths after an eviction, from copies of what there was: tokens sorted one row
    and head at a time, then moved one by one. ``to``: the destination table, None for in place."""
    n_layer, H_kv, bs = len(keys), keys[0].shape[2], keys[0].shape[1]
    after_k, after_v = [x.clone() for x in keys], [x.clone() for x in values]
    after_w, lengths = weights.clone(), seqlen.clone()
    target = table if to is None else to
    for b in range(table.shape[0]):
        n = int(seqlen[b])
        if n <= budget and to is None:
            continue
        for i in range(n_layer):
            for h in range(H_kv):
                kept = list(range(n))
                if n > budget:
                    def place(t):
                        w = float(weights[i, b, h, t])
                        protected = t < sinks or t >= n - recent
                        return (not protected, not math.isnan(w), 0.0 if math.isnan(w) else -w, t)
                    kept = sorted(sorted(kept, key=place)[:budget])
                    after_w[i, b, h, :n] = 0
                    after_w[i, b, h, :budget] = weights[i, b, h, kept]
                for p, t in enumerate(kept):
                    src = (int(table[b, t // bs]), t % bs, h)
                    dst = (int(target[b, p // bs]), p % bs, h)
                    after_k[i][dst], after_v[i][dst] = keys[i][src], values[i][src]
        lengths[b] = min(n, budget)
    return after_k, after_v, after_w, lengths
