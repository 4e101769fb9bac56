"""Rotary positions, KV append and attention over a paged cache, restated in 64
bits on the CPU straight from their definitions (loops over tokens and rows)."""
import math

import torch


def pair_axes(mode, pairs, sections):
    """(axis, place among the frequencies) of each pair"""
    out = []
    s = list(sections)
    for i in range(pairs):
        if mode in ("norm", "neox"):
            out.append((0, i))
            continue
        j = i % sum(s)
        if mode == "imrope":
            out.append((j % 3 if j < 3 * s[j % 3] else 3, i))
            continue
        axis = 0
        while j >= s[axis]:
            j -= s[axis]
            axis += 1
        out.append((axis, j if mode == "vision" else i))
    return out


def yarn_mix(i, n_dims, base, n_ctx, fast, slow):
    """share of the unscaled frequency that pair i keeps"""
    dim = lambda beta: n_dims * math.log(n_ctx / (beta * 2 * math.pi)) / (2 * math.log(base))
    lo, hi = max(0, math.floor(dim(fast))), min(n_dims - 1, math.ceil(dim(slow)))
    return 1.0 - min(1.0, max(0.0, (i - lo) / max(0.001, hi - lo)))


def rope(x, pos, mode, n_dims, base, sections=(0, 0, 0, 0), factors=None, scale=1.0, ext=0.0, attn=1.0, n_ctx=0, fast=32.0,
         slow=1.0):
    """x [T, H, D] any float type, pos [axes, T] -> (y, |x0| + |x1| of each element's pair), 64 bits"""
    x = x.double()
    y, mag = x.clone(), torch.zeros_like(x)
    pairs = n_dims if mode == "vision" else n_dims // 2
    mscale = attn * (1 + 0.1 * math.log(1 / scale)) if ext else attn
    for i, (axis, place) in enumerate(pair_axes(mode, pairs, sections)):
        f = base ** (-2.0 * place / n_dims)
        f = f / (float(factors[i]) if factors is not None else 1.0)
        mix = yarn_mix(i, n_dims, base, n_ctx, fast, slow) * ext if ext else 0.0
        a = pos[axis].double() * (f * (scale * (1 - mix) + mix))
        c, s = (a.cos() * mscale).unsqueeze(1), (a.sin() * mscale).unsqueeze(1)
        e0, e1 = (2 * i, 2 * i + 1) if mode == "norm" else (i, i + pairs)
        x0, x1 = x[..., e0], x[..., e1]
        y[..., e0], y[..., e1] = x0 * c - x1 * s, x0 * s + x1 * c
        mag[..., e0] = mag[..., e1] = (x0.abs() + x1.abs()) * abs(mscale)
    return y, mag


def attention(q, kv, seqs, scale, sinks=None, window=0, n_first=0):
    """q [T, H, D], kv [pages, page, H_kv, 2 D], seqs: lists (q0, nq, nkv, pages ..).
    -> (out, score magnitude max_j scale sum |q k|, sum p |v| / sum p), each 64 bits;
    rows that no sequence names are NaN in `out`."""
    T, H, D = q.shape
    pages, page, Hkv, _ = kv.shape
    G = H // Hkv
    q, kvd = q.double(), kv.double()
    out = torch.full((T, H, D), float("nan"), dtype=torch.float64)
    mag, wgt = torch.zeros((T, H, 1), dtype=torch.float64), torch.zeros((T, H, D), dtype=torch.float64)
    for row in seqs:
        q0, nq, nkv = (int(v) for v in row[:3])
        for i in range(nq):
            t, p = q0 + i, nkv - nq + i
            seen = [j for j in range(max(0, p + 1)) if not window or j > p - window or j < n_first]
            if not seen:
                out[t] = 0.0
                continue
            js = torch.tensor(seen)
            table = torch.as_tensor([int(v) for v in row[3:]])
            rows = kvd[table[js // page], js % page]  # [n, H_kv, 2 D]
            for h in range(H):
                k, v = rows[:, h // G, :D], rows[:, h // G, D:]
                s = (k * q[t, h]).sum(-1) * scale
                mag[t, h] = (k.abs() * q[t, h].abs()).sum(-1).max() * abs(scale)
                m = s.max() if sinks is None else torch.maximum(s.max(), sinks[h].double())
                e = (s - m).exp()
                l = e.sum() + (0 if sinks is None else (sinks[h].double() - m).exp())
                out[t, h] = (e[:, None] * v).sum(0) / l
                wgt[t, h] = (e[:, None] * v.abs()).sum(0) / l
    return out, mag, wgt


def attention_tol(mag, wgt, D):
    """How far a row may be off.  A score is a sum of D products in 32 bits of q in
    at least 17 bits (bf16 cache: two roundings of 2^-9 each; f16: 22 bits), off by
    (D 2^-24 + 2^-17) of its magnitude; p and the sum both take that, p is held in
    17 bits too, and exp, the sums' rescalings and the quotient add 2^-18."""
    return (2 * (D * 2.0 ** -24 + 2.0 ** -17) * mag + 2.0 ** -17 + 2.0 ** -18) * wgt + 1e-30
