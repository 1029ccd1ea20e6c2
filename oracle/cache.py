"""A key and value cache in MX formats in 64 bits: the values of its rows, and attention over them query by query, with the
bound that float32 sums, rounded weights and the one rounding of the output allow."""
import math

import numpy as np
import torch

from .packed import FORMATS, code_table, e8m0_decode

BLOCK = 32


def values(codes, scales, fmt, D):
    """Code bytes (..., bytes) and E8M0 bytes (..., blocks) as torch float64 (..., D) on the codes' device."""
    e, m = FORMATS[fmt]
    if fmt == "MXFP4":
        codes = torch.stack([codes & 15, codes >> 4], -1).flatten(-2)
    table = torch.from_numpy(code_table(e, m).astype(np.float64)).to(codes.device)
    powers = torch.from_numpy(e8m0_decode(np.arange(256)).astype(np.float64)).to(codes.device)
    return (table[codes.long() & (len(table) - 1)] * powers[scales.long()].repeat_interleave(BLOCK, -1))[..., :D]


def rows(cache, slots):
    """(k, v) float64, T x heads x D, zeros for slots that the cache does not have."""
    P, G, S, _ = cache.k_codes.shape
    slots = slots.long()
    there = (slots >= 0) & (slots < P * S)
    at = torch.where(there, slots, 0)
    out = []
    for codes, scales in ((cache.k_codes, cache.k_scales), (cache.v_codes, cache.v_scales)):
        x = values(codes[at // S, :, at % S], scales[at // S, :, at % S], cache.fmt, cache.head_dim)
        out.append(torch.where(there[:, None, None], x, 0.0))
    return out


#: how far a weight of bfloat16, float16 and float32 queries may be from exp's value by its rounding alone: half a step of
#: bfloat16; two bfloat16, the weight to the nearest and what that leaves, 2^-8 of it at most, to the nearest; three, which
#: hold all of a float32
ROUNDED = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -16, torch.float32: 0.0}


def attend(q, cache, table, lengths, starts=None, scale=None, causal=True, window=None, rounded=None):
    """(out, lse, bound of out, bound of lse), float64, T x heads x D and T x heads.

    A score is a float32 sum of D exact products, then scaled: off by (D + 8) half steps of the sum of magnitudes.  Such an
    error e of all scores' exponents is at most 2 e of a normalised weight, beside the weight's own rounding, exp2's unit
    and the sums of L terms of numerator and denominator, joined from 64 parts at most in as many steps.  A weight is taken
    relative to a maximum that is no larger than the scores', so that the weights' sum is 1 or more, and the hardware's exp2
    makes those below float32's smallest normal zero: 2^-126 of each value at most.  rounded: the weights' rounding, where it
    is not ROUNDED's."""
    D, G, S = cache.head_dim, cache.k_codes.shape[1], cache.page_size
    if starts is None:
        starts = [i * q.shape[1] for i in range(q.shape[0] + 1)]
    else:
        starts = starts.tolist()
    flat = q.reshape(-1, *q.shape[-2:]).double()
    T, H, _ = flat.shape
    scale = D ** -0.5 if scale is None else scale
    half = 2.0 ** -24
    out, off = torch.zeros_like(flat), torch.zeros_like(flat)
    lse, lse_off = (torch.full(flat.shape[:2], fill, dtype=torch.float64, device=q.device) for fill in (-math.inf, 0.0))
    for b, length in enumerate(lengths.tolist()):
        low, high = (min(max(x, 0), T) for x in starts[b:b + 2])
        length = min(max(length, 0), table.shape[1] * S)
        if high <= low or not length:
            continue
        at = torch.arange(length, device=q.device)
        page = table[b].long()[at // S]
        there = (page >= 0) & (page < cache.k_codes.shape[0])
        k, v = rows(cache, torch.where(there, page * S + at % S, -1))
        for t in range(low, high):
            p = length - (high - low) + t - low
            last = p if causal else length - 1
            first = 0 if window is None else p - window + 1
            seen = ((at >= first) & (at <= last) & there).nonzero()[:, 0]
            if not len(seen):
                continue
            L = len(seen)
            for g in range(G):
                heads = slice(g * (H // G), (g + 1) * (H // G))
                x, kk, vv = flat[t, heads], k[seen, g], v[seen, g]
                s = scale * (x @ kk.t())
                total = torch.logsumexp(s, -1, keepdim=True)
                w = torch.exp(s - total)
                size = scale * (x.abs() @ kk.abs().t()).amax(-1, keepdim=True)
                e = (D + 8) * half * size + 16 * half
                each = 2 * e + 2 * (ROUNDED[q.dtype] if rounded is None else rounded) + (2 * min(L, 4096) + 200) * half
                out[t, heads] = w @ vv
                off[t, heads] = each * (w @ vv.abs()) + 2.0 ** -126 * vv.abs().sum(0)
                lse[t, heads] = total[:, 0]
                lse_off[t, heads] = (e + (min(L, 4096) + 200) * half)[:, 0] + 4 * half * total[:, 0].abs()
    info = torch.finfo(q.dtype)
    off = off + info.eps / 2 * (out.abs() + off) + info.smallest_normal * info.eps
    return out.reshape(q.shape), lse.reshape(q.shape[:-1]), off.reshape(q.shape), lse_off.reshape(q.shape[:-1])
