"""A plain 64-bit restatement of the MX cache (write, rotate, read, attend) for its tests."""

import math

import numpy as np
import torch

from oracle import fused_rmsnorm as ora

CODES = {"e4m3": torch.float8_e4m3fn, "e2m1": torch.float4_e2m1fn_x2}


def as_bytes(cache):
    return [t.view(torch.uint8).cpu().numpy() for t in cache]


def from_bytes(parts, fmt, device):
    dtypes = (CODES[fmt], torch.float8_e8m0fnu) * 2
    return tuple(torch.from_numpy(np.ascontiguousarray(p)).to(device).view(d) for p, d in zip(parts, dtypes))


def quantise(x, fmt):
    """(codes [tokens, heads, bytes], scales [tokens, heads, blocks]) of float32 x."""
    n, h, d = x.shape
    codes, scales = ora.mx_quantize_rows(np.ascontiguousarray(x.reshape(n * h, d)), fmt)
    return codes.reshape(n, h, -1), scales.reshape(n, h, -1)


def values(codes, scales, fmt):
    """Float64 values of codes [..., bytes] with scales [..., blocks]."""
    if fmt == "e2m1":
        codes = np.stack((codes & 15, codes >> 4), -1).reshape(codes.shape[:-1] + (2 * codes.shape[-1],))
        v = ora.e2m1_decode(codes).astype(np.float64)
    else:
        v = torch.from_numpy(codes.copy()).view(torch.float8_e4m3fn).double().numpy()
    return v * np.repeat(ora.e8m0_decode(scales).astype(np.float64), 32, -1)


def write(parts, k, v, slots, page, fmt):
    """parts (numpy bytes) with k, v (float32 numpy [tokens, heads, dim]) in their slots."""
    kc, ks, vc, vs = parts
    for x, c, s in ((k, kc, ks), (v, vc, vs)):
        codes, scales = quantise(x, fmt)
        for t, slot in enumerate(slots):
            if 0 <= slot < c.shape[0] * page:
                c[slot // page, :, slot % page] = codes[t]
                s[slot // page, :, :, slot % page] = scales[t]


def rotate(x, cos_sin, positions):
    """Rotate half of float32 x [tokens, heads, dim], every product and sum rounded to float32."""
    half = x.shape[-1] // 2
    row = cos_sin[positions][:, None]
    c, s = row[..., :half], row[..., half:]
    a, b = x[..., :half], x[..., half:]
    return np.concatenate((a * c - b * s, a * s + b * c), -1)


def attention(q, parts, table, lengths, starts, page, fmt, scale, causal, out_eps, p_eps):
    """(out, lse, how far a right result may be off for each, out of [tokens, heads, dim]) in float64.

    The bound counts: the output's own rounding (out_eps relative to it), the probabilities' (p_eps
    relative to each, so p_eps * A with A = sum p|v| / sum p), the scores' (a sum of dim float32 products
    has an error of at most (dim + 8) 2^-24 S, S the sum of the products' magnitudes; scaling and the base
    of the exponential add 4 2^-24 |s|; a score off by e moves p by a factor within 1 + 2 e), the
    hardware's exponential (2 ulps: 2^-22), and the float32 sums over n keys and their rescaling and
    joining ((n + 64) 2^-24 A)."""
    kc, ks, vc, vs = parts
    tokens, heads, dim = q.shape
    group = heads // kc.shape[1]
    out, lse = np.zeros(q.shape), np.full((tokens, heads), -np.inf)
    off, lse_off = np.zeros(q.shape), np.zeros((tokens, heads))
    u = 2.0 ** -24
    for b, held in enumerate(lengths):
        first, last = (b, b + 1) if starts is None else (starts[b], starts[b + 1])
        t = np.arange(held)
        pages = table[b][t // page] if held else np.zeros(0, np.int64)
        there = (pages >= 0) & (pages < kc.shape[0])
        pages = np.where(there, pages, 0)
        k = values(kc[pages, :, t % page], ks[pages, :, :, t % page], fmt)
        v = values(vc[pages, :, t % page], vs[pages, :, :, t % page], fmt)
        if last == first or not held:
            continue
        limit = np.maximum(held - (last - first) + np.arange(last - first) + 1, 0) if causal else \
            np.full(last - first, held)
        hidden = ~there | (t >= limit[:, None])                       # [rows, keys]
        seen = (~hidden).sum(-1)
        rows = np.nonzero(seen)[0]
        for h in range(heads):
            kk, vv, qq = k[:, h // group], v[:, h // group], q[first:last, h][rows]
            kk, vv = (np.where(there[:, None], x, 0.0) for x in (kk, vv))   # leftovers, NaN among them
            s = np.where(hidden[rows], -np.inf, qq @ kk.T * scale)
            m = s.max(-1, keepdims=True)
            p = np.exp(s - m)
            total = p.sum(-1, keepdims=True)
            o = p @ vv / total
            at = first + rows
            out[at, h] = o
            lse[at, h] = (m + np.log(total))[:, 0]
            weight = p @ np.abs(vv) / total
            size = np.where(hidden[rows], 0.0, np.abs(qq) @ np.abs(kk).T).max(-1) * abs(scale)
            score = ((dim + 12) * u * size)[:, None]
            sums = (seen[rows][:, None] + 64) * u
            off[at, h] = out_eps * np.abs(o) + weight * (p_eps + 2 * score + 4 * u + sums)
            lse_off[at, h] = (2 * u * np.abs(m + np.log(total)) + score + 4 * u + sums)[:, 0]
    return out, lse, off, lse_off
