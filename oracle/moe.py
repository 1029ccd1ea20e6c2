"""A mixture-of-experts layer's operators in 64 bits: routing and its gradient by enumeration, the slots' order, the
weighted sum, the product with packed weights and its epilogue, each with the bound its float32 sum and its one
rounding allow."""
import numpy as np
import torch

from .packed import FORMATS, code_table, e8m0_decode

F64 = np.float64


def route(logits, k, score="softmax", bias=None, groups=1, top_groups=1, renormalize=True, scale=1.0):
    """logits (T, E) -> weights (T, k) float64, experts (T, k), scores (T, E); a row with no scores has NaN weights."""
    logits = np.asarray(logits, dtype=F64)
    T, E = logits.shape
    weights, experts, scores = np.zeros((T, k)), np.full((T, k), -1, dtype=np.int64), np.zeros((T, E))
    for t in range(T):
        l = logits[t]
        with np.errstate(all="ignore"):
            if score == "softmax":
                top = l.max()
                p = np.exp(l - (top if top > -np.inf else 0.0))
                s = p / (p.sum() if p.sum() != 0 else 1.0)
            else:
                s = 1 / (1 + np.exp(-l))
            r = s if bias is None else s + np.asarray(bias, dtype=F64)
            r = np.where(l == -np.inf, -np.inf, r)
        scores[t] = s
        if np.isnan(r).any():
            weights[t] = np.nan
            continue
        per = E // groups
        if groups > 1:
            of_group = []
            for g in range(groups):
                two = sorted(r[g * per:(g + 1) * per], reverse=True)[:2]
                of_group.append(two[0] + (two[1] if len(two) > 1 and two[1] > -np.inf else 0.0))
            kept = sorted(range(groups), key=lambda g: (-of_group[g], g))[:top_groups]
            r = np.where(np.isin(np.arange(E) // per, kept), r, -np.inf)
        chosen = [e for e in sorted(range(E), key=lambda e: (-r[e], e))[:k] if r[e] > -np.inf]
        w = s[chosen]
        if renormalize and w.sum() != 0:
            w = w / w.sum()
        weights[t, :len(chosen)], experts[t, :len(chosen)] = w * scale, chosen
    return weights, experts, scores


def route_grad(scores, experts, grad, score="softmax", renormalize=True, scale=1.0):
    """The gradient of the logits by the formulas."""
    out = np.zeros_like(scores)
    for t in range(scores.shape[0]):
        s, e = scores[t], experts[t][experts[t] >= 0]
        g, u = np.asarray(grad[t], dtype=F64)[experts[t] >= 0] * scale, scores[t][e]
        if renormalize and u.sum() != 0:
            g = (g - (g * u).sum() / u.sum()) / u.sum()
        d = np.zeros_like(s)
        d[e] = g
        out[t] = s * (d - (d * s).sum()) if score == "softmax" else d * s * (1 - s)
    return out


def dispatch(experts, E):
    """order, offsets, positions by Python's stable sort."""
    flat = [int(e) if 0 <= int(e) < E else E for e in np.asarray(experts).reshape(-1)]
    order = sorted(range(len(flat)), key=lambda i: flat[i])
    offsets = np.concatenate([[0], np.cumsum([flat.count(e) for e in range(E)])])
    positions = np.empty(len(flat), dtype=np.int64)
    for row, slot in enumerate(order):
        positions[slot] = row if flat[slot] < E else -1 - row
    return np.array(order, dtype=np.int64), offsets, positions.reshape(np.shape(experts))


def weight(codes, scales, fmt, K):
    """Code bytes (..., K), or MXFP4 pairs (..., ceil(K / 2)), and E8M0 bytes -> float64 values (..., K)."""
    e, m = FORMATS[fmt]
    codes = np.asarray(codes).astype(np.int64)
    if fmt == "MXFP4" and codes.shape[-1] != K:
        codes = np.stack([codes & 15, codes >> 4], -1).reshape(*codes.shape[:-1], -1)[..., :K]
    table = code_table(e, m).astype(F64)
    spread = np.repeat(e8m0_decode(scales).astype(F64), 32, axis=-1)[..., :K]
    return table[codes & (len(table) - 1)] * spread


def activate(z, name):
    if name == "silu":
        return z * torch.sigmoid(z)
    if name == "gelu":
        return z * torch.special.ndtr(z)
    if name == "gelu_tanh":
        return 0.5 * z * (1 + torch.tanh((2 / np.pi) ** 0.5 * (z + 0.044715 * z ** 3)))
    if name == "relu":
        return torch.clamp_min(z, 0)
    return z


#: the largest slope of the activations (gelu_tanh's and gelu's is 1.13), and how far from its value one may be
#: evaluated, relative to its argument: sixteen of float32's half steps
SLOPE, EVALUATION = 1.14, 2.0 ** -20


def linear(x, W, bias=None, activation=None, gated=False, residual=None, y_dtype=torch.float32):
    """(y, bound) float64: x (M, K) torch, W (rows, K) float64 torch.  The contraction's float32 sum of K products is off
    by at most K half steps of the sum of their magnitudes, bias and residual add one each, the activation carries the
    contraction's error with its slope, y's rounding is half a step of y."""
    x = x.double()
    z, size = x @ W.t(), x.abs() @ W.abs().t()
    half = torch.finfo(torch.float32).eps / 2
    off = (x.shape[1] + 2) * half * size
    if bias is not None:
        z = z + bias.double()
        off = off + half * (size + bias.double().abs())
    if gated:
        n = z.shape[1] // 2
        z, u, off, off_u = z[:, :n], z[:, n:], off[:, :n], off[:, n:]
    y = activate(z, activation)
    off = SLOPE * off + (EVALUATION * z.abs() if activation else 0)
    if gated:
        off = off * u.abs() + off_u * (y.abs() + off) + half * (y * u).abs()
        y = y * u
    if residual is not None:
        y = y + residual.double()
        off = off + half * y.abs()
    return y, off + torch.finfo(y_dtype).eps / 2 * (y.abs() + off) + torch.finfo(y_dtype).smallest_normal * torch.finfo(y_dtype).eps
