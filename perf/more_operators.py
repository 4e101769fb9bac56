"""The operators of a quantized paged KV cache that performance is measured on:
appending keys and values as 8-bit or 4-bit codes with the rotation on the way,
reading rows back, and attention over such a cache.

A cache is two tensors: codes [pages, page, H_kv, 2 D] (E4M3, or pairs of E2M1 in
a byte, the first in the low bits) and scales [pages, page, H_kv, 2 S], a byte
(E8M0: 2^(byte - 127)) for each 32 codes of the key, then of the value; S is D / 32
rounded up to a power of two.  A block's scale is the least power of two from
2^-100 on that brings its largest element to at most 448 (E4M3) or 7 (E2M1, where
6 is the largest code); elements are rounded to the nearest code, ties to the even one.

`run` computes them in elementary torch operations, or, with `own` set, through
the Python binding (llama.rust_amd/ghip.py)."""
import math
import os
import sys

import torch

own = False
DEV = "cuda"
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # generation: one new token for each of 32 sequences
        {"name": "append_tokens", "kind": "append", "bits": 8, "mode": "neox", "T": 32, "B": 32, "H_kv": 8, "D": 128, "n_dims": 128,
         "sections": "0,0,0,0", "base": 5e5, "start": 9000, "grid": 1, "type": "f32", "page": 64, "factors": True, "pad": 0},
        # three prompts of a vision-language model in one batch, a few rows of padding, and
        # what later tokens will see of them
        {"name": "append_prompts", "kind": "append", "bits": 4, "mode": "mrope", "T": 2011, "B": 3, "H_kv": 4, "D": 128, "n_dims": 128,
         "sections": "16,24,24,0", "base": 1e6, "start": 500, "grid": 27, "type": "bf16", "page": 16, "factors": False, "pad": 5},
        # a large prefill batch
        {"name": "append_prefill", "kind": "append", "bits": 8, "mode": "norm", "T": 8192, "B": 8, "H_kv": 8, "D": 128, "n_dims": 128,
         "sections": "0,0,0,0", "base": 1e4, "start": 0, "grid": 1, "type": "f32", "page": 64, "factors": False, "pad": 0},
        # the last page of a conversation, whose keys are to be rotated to new positions
        {"name": "read_page", "kind": "read", "bits": 4, "T": 61, "H_kv": 8, "D": 64, "type": "f32", "page": 64, "pad": 0},
        # a long conversation leaves the cache for the host
        {"name": "read_sequence", "kind": "read", "bits": 8, "T": 16000, "H_kv": 8, "D": 128, "type": "bf16", "page": 16, "pad": 7},
        # one new token of one conversation
        {"name": "token", "kind": "attn", "bits": 8, "B": 1, "q_lo": 1, "q_hi": 1, "kv_lo": 1061, "kv_hi": 1061, "H": 64, "H_kv": 8,
         "D": 64, "page": 16, "window": 0, "n_first": 0, "shared": 0, "sinks": True},
        # generation of 24 sequences of very different length
        {"name": "batch", "kind": "attn", "bits": 8, "B": 24, "q_lo": 1, "q_hi": 1, "kv_lo": 500, "kv_hi": 16384, "H": 32, "H_kv": 8,
         "D": 128, "page": 64, "window": 0, "n_first": 0, "shared": 0, "sinks": False},
        # the same of 64 sequences in 4 bits
        {"name": "batch_4bit", "kind": "attn", "bits": 4, "B": 64, "q_lo": 1, "q_hi": 1, "kv_lo": 2000, "kv_hi": 12000, "H": 32, "H_kv": 8,
         "D": 128, "page": 64, "window": 0, "n_first": 0, "shared": 0, "sinks": False},
        # five or six drafted tokens for each of 12 sequences
        {"name": "drafts", "kind": "attn", "bits": 8, "B": 12, "q_lo": 5, "q_hi": 6, "kv_lo": 900, "kv_hi": 8192, "H": 32, "H_kv": 8,
         "D": 128, "page": 64, "window": 0, "n_first": 0, "shared": 0, "sinks": False},
        # prefill chunks of two long prompts
        {"name": "chunk", "kind": "attn", "bits": 8, "B": 2, "q_lo": 701, "q_hi": 1001, "kv_lo": 4000, "kv_hi": 8192, "H": 32, "H_kv": 8,
         "D": 128, "page": 16, "window": 0, "n_first": 0, "shared": 0, "sinks": False},
        # the same under a window, heads of 64, 4 bits
        {"name": "chunk_4bit", "kind": "attn", "bits": 4, "B": 3, "q_lo": 333, "q_hi": 512, "kv_lo": 1500, "kv_hi": 6000, "H": 64, "H_kv": 8,
         "D": 64, "page": 16, "window": 1024, "n_first": 4, "shared": 0, "sinks": True},
        # generation of 64 requests under one long system prompt
        {"name": "shared_tokens", "kind": "attn", "bits": 8, "B": 64, "q_lo": 1, "q_hi": 1, "kv_lo": 8232, "kv_hi": 8792, "H": 32, "H_kv": 8,
         "D": 128, "page": 64, "window": 0, "n_first": 0, "shared": 8192, "sinks": False},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    most, large = max(_cost(c) for c in listed()), max(_size(c) for c in listed())
    while True:
        kind = rng.choice(["append", "read", "attn", "attn", "shared"])
        bits = rng.choice([8, 4])
        D = rng.choice([64, 64, 80, 96, 128, 128, 128, 256])
        page = rng.choice([1, 16, 24, 64, 256])
        if kind == "append":
            mode = rng.choice(["norm", "neox", "mrope", "imrope"])
            n = D if rng.random() < 0.7 else 2 * (D // 8)
            p, sec = n // 2, (0, 0, 0, 0)
            if mode == "mrope":
                a = rng.randint(1, p // 2)
                sec = (a, (p - a) // 2, p - a - (p - a) // 2, 0)
            elif mode == "imrope":
                sec = (p - 2 * (p // 3), p // 3, p // 3, 0)
            T = _log_int(rng, 1, 8192)
            return {"kind": "append", "bits": bits, "mode": mode, "T": T, "B": rng.randint(1, min(T, 40)), "H_kv": rng.choice([1, 2, 4, 8]),
                    "D": D, "n_dims": n, "sections": "%d,%d,%d,%d" % sec, "base": rng.choice([1e4, 5e5, 1e6]),
                    "start": rng.randint(0, 20000), "grid": rng.randint(2, 80), "type": rng.choice(["f32", "f32", "f16", "bf16"]),
                    "page": page, "factors": rng.random() < 0.3, "pad": rng.randint(0, T // 8)}
        if kind == "read":
            T = _log_int(rng, 1, 16000)
            return {"kind": "read", "bits": bits, "T": T, "H_kv": rng.choice([1, 2, 4, 8]), "D": D,
                    "type": rng.choice(["f32", "f16", "bf16"]), "page": page, "pad": rng.randint(0, T // 8)}
        H_kv = rng.choice([1, 2, 4, 8])
        c = {"kind": "attn", "bits": bits, "B": _log_int(rng, 1, 96), "q_lo": 1, "q_hi": 1, "kv_lo": 0, "kv_hi": 0,
             "H": H_kv * rng.choice([1, 3, 4, 5, 8, 16]), "H_kv": H_kv, "D": D, "page": page, "window": 0, "n_first": 0, "shared": 0,
             "sinks": rng.random() < 0.3}
        if rng.random() < 0.5:
            c["q_hi"] = _log_int(rng, 2, 1200)
            c["q_lo"] = rng.randint(1, c["q_hi"])
        c["kv_hi"] = c["q_hi"] + _log_int(rng, 1, 16384)
        if kind == "attn":
            c["kv_lo"] = rng.randint(c["q_lo"], c["kv_hi"])
            if rng.random() < 0.4:
                c["window"] = _log_int(rng, 1, 8192)
                c["n_first"] = rng.choice([0, 1, 4, 130])
        else:
            c["B"] = max(2, c["B"])
            c["shared"] = rng.randint(1, c["kv_hi"] - c["q_hi"])
            c["kv_lo"] = rng.randint(c["shared"] + 1, c["kv_hi"])
        if _cost(c) <= most and _size(c) <= large:
            return c


def _size(c):
    w = work(c)
    return max(w["bytes"], w["flops"] / 50)


def _cost(c):
    """what bounds a case's time: the work, and the keys and scores that the plain form lays out"""
    if c["kind"] != "attn":
        return 0.0
    w = work(c)
    return max(w["bytes"] / 5e12, w["flops"] / 5e14, c["B"] * c["kv_hi"] * c["H_kv"] * c["D"] * 4e-12,
               c["B"] * c["q_hi"] * c["kv_hi"] * c["H"] * 4e-12)


# ------------------------------------------------------------------- inputs

def _spread(lo, hi, n):
    """n whole numbers from lo to hi in no order; the first is hi"""
    return [hi - int((hi - lo) * ((i * 0.6180339887498949) % 1.0)) for i in range(n)]


def _lengths(c):
    """(query rows, cached keys) of each sequence"""
    q = _spread(c["q_lo"], c["q_hi"], c["B"])
    return q, [max(a, b) for a, b in zip(q, _spread(c["kv_lo"], c["kv_hi"], c["B"]))]


def _scale_bytes(D):
    """scale bytes of a key (or a value)"""
    n = 1
    while 32 * n < D:
        n *= 2
    return n


def _positions(c, T, start):
    """positions of T tokens, [axes, T]: text, then an image of `grid` columns"""
    i = torch.arange(T, device=DEV)
    if c["mode"] in ("norm", "neox"):
        return (start + i).to(torch.int32).reshape(1, T)
    text = T // 3
    j = (i - text).clamp(min=0)
    img = i >= text
    base = start + torch.where(img, text, i)
    return torch.stack([base, base + torch.where(img, j // c["grid"], 0), base + torch.where(img, j % c["grid"], 0),
                        torch.zeros_like(i)]).to(torch.int32)


def _heads(shape, g):
    """rows as a projection leaves them: a few strong channels"""
    x = torch.randn(shape, generator=g, device=DEV)
    return x.mul_(0.5 + torch.rand(shape[-2:], generator=g, device=DEV)).add_(0.3 * torch.randn(shape[-2:], generator=g, device=DEV))


def _cache(c, pages, g):
    """a cache in use: codes as blocks of normal values have them, scales that differ from block to block"""
    rows = (pages, c["page"], c["H_kv"])
    if c["bits"] == 8:
        kv = torch.randn(rows + (2 * c["D"],), generator=g, device=DEV).mul_(150).clamp_(-448, 448).to(torch.float8_e4m3fn)
        low = 118
    else:
        # sixteen equally frequent parts of a normal distribution -> codes
        nib = torch.tensor([15, 14, 14, 13, 12, 11, 10, 9, 1, 2, 3, 4, 5, 6, 6, 7], dtype=torch.uint8, device=DEV)
        pair = (nib.view(1, 16) | (nib.view(16, 1) << 4)).reshape(256)
        kv = pair[torch.randint(0, 256, rows + (c["D"],), generator=g, device=DEV, dtype=torch.int32)]
        low = 124
    scales = torch.randint(low, low + 3, rows + (2 * _scale_bytes(c["D"]),), generator=g, device=DEV, dtype=torch.uint8)
    return kv, scales


def _inputs(case, seed):
    c = case
    g = torch.Generator(device=DEV).manual_seed(seed)
    s = {"case": c}
    page, D, Hkv, T = c["page"], c["D"], c["H_kv"], c.get("T", 0)
    if c["kind"] == "read":
        n = T - c["pad"]
        need = (n + page - 1) // page
        perm = torch.randperm(need + max(8, need // 2), generator=g, device=DEV)
        i = torch.arange(n, device=DEV)
        s["slots"] = torch.cat([perm[i // page] * page + i % page, torch.full((c["pad"],), -1, dtype=torch.int64, device=DEV)])
        s["real"] = n
        s["kv"], s["scales"] = _cache(c, perm.numel(), g)
        return s
    if c["kind"] == "append":
        real, B = T - c["pad"], c["B"]
        n = [real // B + (i < real % B) for i in range(B)]
        s["k"], s["v"] = (_heads((T, Hkv, D), g).to(TYPES[c["type"]]) for _ in range(2))
        first = [(c["start"] + 37 * i + seed) % page for i in range(B)]  # the row of its page each sequence goes on at
        need = [(2 * page - 2 + m) // page for m in n]  # wherever it starts
        pages = sum(need) + max(8, sum(need) // 2)
        perm = torch.randperm(pages, generator=g, device=DEV)
        slots, pos, at = [], [], 0
        for f, m, k in zip(first, n, need):
            i = f + torch.arange(m, device=DEV)
            slots.append(perm[at + i // page] * page + i % page)
            pos.append(_positions(c, m, c["start"] + seed % 97 + f))
            at += k
        slots.append(torch.full((c["pad"],), -1, dtype=torch.int64, device=DEV))
        pos.append(torch.zeros((pos[0].shape[0], c["pad"]), dtype=torch.int32, device=DEV))
        s["slots"], s["pos"], s["real"] = torch.cat(slots), torch.cat(pos, 1).contiguous(), real
        s["kv"], s["scales"] = _cache(c, pages, g)
        # longer wavelengths for the low frequencies, as long-context models ship them
        s["factors"] = torch.linspace(1.0, 8.0, c["n_dims"] // 2, device=DEV) if c["factors"] else None
        return s
    nq, nkv = _lengths(c)
    T, per = sum(nq), (max(nkv) + page - 1) // page
    common, rest = divmod(c["shared"], page)  # pages that all sequences have, and rows of the next one, copied for each
    need = [(m + page - 1) // page for m in nkv]
    pages = sum(max(0, m - common) for m in need) + common + 4
    perm = torch.randperm(pages, generator=g, device=DEV).to(torch.int32)
    seqs = torch.zeros((c["B"], 3 + per), dtype=torch.int32, device=DEV)
    head, q0, at = [], 0, common
    for b in range(c["B"]):
        head.append([q0, nq[b], nkv[b]])
        k = min(common, need[b])
        seqs[b, 3:3 + k] = perm[:k]
        seqs[b, 3 + k:3 + need[b]] = perm[at:at + need[b] - k]
        at += need[b] - k
        q0 += nq[b]
    seqs[:, :3] = torch.tensor(head, dtype=torch.int32, device=DEV)
    s["seqs"], s["T"], s["q_max"], s["kv_max"] = seqs, T, max(nq), max(nkv)
    s["q"] = _heads((T, c["H"], D), g)
    s["kv"], s["scales"] = _cache(c, pages, g)
    if rest:
        a, b = seqs[0, 3 + common].long(), seqs[1:, 3 + common].long()
        for t in (s["kv"].view(torch.uint8), s["scales"]):
            t[b, :rest] = t[a, :rest]
    s["sinks"] = torch.randn(c["H"], generator=g, device=DEV) if c["sinks"] else None
    s["scale"] = 1.0 / math.sqrt(D)
    return s


def prepare(case, seed):
    s, c = _inputs(case, seed), case
    if c["kind"] == "attn":
        s["out"] = torch.empty((s["T"], c["H"], c["D"]), device=DEV)
    elif c["kind"] == "read" or c["bits"] == 4:
        # (bfloat16 holds a 4-bit code's value as it is)
        s["out"] = torch.zeros((c["T"], c["H_kv"], 2 * c["D"]), device=DEV, dtype=TYPES[c["type"]] if c["kind"] == "read" else torch.bfloat16)
    return s


# --------------------------------------------------------------- plain forms

E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _power(e, double=False):
    """2^e, exactly"""
    if double:
        return ((e.long() + 1023) << 52).view(torch.float64)
    return ((e.int() + 127) << 23).view(torch.float32)


def _values(codes, scales, c):
    """what the codes [.., 2 D] (or D bytes) and their scales stand for, in 32 bits (exact)"""
    D, S = c["D"], scales.shape[-1] // 2
    if c["bits"] == 8:
        x = codes.float()
    else:
        table = torch.tensor(E2M1 + tuple(-v for v in E2M1), device=DEV)
        x = torch.stack([table[(codes & 15).int()], table[(codes >> 4).int()]], -1).flatten(-2)
    e = _power(scales.int() - 127).unflatten(-1, (2, S))
    return x * e.repeat_interleave(32, -1)[..., :D].flatten(-2)


def _encoded(x, c):
    """rows x [.., D] in 64 bits -> codes, scale bytes"""
    D, S = x.shape[-1], _scale_bytes(x.shape[-1])
    x = torch.nn.functional.pad(x, (0, 32 * S - D)).unflatten(-1, (S, 32))
    m, e = torch.frexp(x.abs().amax(-1, keepdim=True))
    e = torch.where(m > 0, e - (9 if c["bits"] == 8 else 3) + (m > 0.875), -100).clamp(min=-100)
    y = x * _power(-e, True)
    low, digits = (-6, 3) if c["bits"] == 8 else (0, 1)
    step = (torch.frexp(y)[1] - 1).clamp(min=low) - digits
    y = (torch.round(y * _power(-step, True)) * _power(step, True)).flatten(-2)[..., :D]
    if c["bits"] == 8:
        codes = y.to(torch.float8_e4m3fn)
    else:
        n = torch.bucketize(y.abs().clamp(max=6.0), torch.tensor(E2M1, device=DEV, dtype=torch.float64)) + 8 * torch.signbit(y)
        codes = (n[..., 0::2] | (n[..., 1::2] << 4)).to(torch.uint8)
    return codes, (e.squeeze(-1) + 127).to(torch.uint8)


def _axis_of_pairs(mode, n_pairs, sections):
    """for each pair: its position's axis"""
    i = torch.arange(n_pairs, device=DEV)
    s = [int(x) for x in sections.split(",")]
    if mode in ("norm", "neox"):
        return torch.zeros_like(i)
    j = i % sum(s)
    if mode == "imrope":
        r = j % 3
        return torch.where(j < 3 * torch.where(r == 0, s[0], torch.where(r == 1, s[1], s[2])), r, 3)
    return (j >= s[0]).long() + (j >= s[0] + s[1]).long() + (j >= s[0] + s[1] + s[2]).long()


def _rotate(x, pos, c, factors):
    """x [T, heads, D] rotated, in 64 bits (positions are far, and a code is a rounding)"""
    n = c["n_dims"]
    pairs = n // 2
    i = torch.arange(pairs, device=DEV)
    f = torch.pow(torch.tensor(c["base"], dtype=torch.float64, device=DEV), -2.0 * i.double() / n)
    if factors is not None:
        f = f / factors.double()
    a = pos[_axis_of_pairs(c["mode"], pairs, c["sections"])].t().double() * f
    cos, sin = a.cos().unsqueeze(1), a.sin().unsqueeze(1)
    x = x.double()
    y = x.clone()
    if c["mode"] == "norm":
        x0, x1 = x[..., 0:n:2], x[..., 1:n:2]
        y[..., 0:n:2], y[..., 1:n:2] = x0 * cos - x1 * sin, x0 * sin + x1 * cos
    else:
        x0, x1 = x[..., :pairs], x[..., pairs:n]
        y[..., :pairs], y[..., pairs:n] = x0 * cos - x1 * sin, x0 * sin + x1 * cos
    return y


def _plain_append(s):
    c, n, kv = s["case"], s["real"], s["kv"]
    kc, ks = _encoded(_rotate(s["k"][:n], s["pos"][:, :n], c, s["factors"]), c)
    vc, vs = _encoded(s["v"][:n].double(), c)
    at = s["slots"][:n]
    codes, scales = torch.cat([kc, vc], -1), torch.cat([ks, vs], -1)
    kv.view(torch.uint8).view(-1, *kv.shape[2:])[at] = codes.view(torch.uint8)
    s["scales"].view(-1, *s["scales"].shape[2:])[at] = scales
    if c["bits"] == 8:
        return [kv, s["scales"]]
    s["out"][:n] = _values(codes, scales, c).to(s["out"].dtype)
    return s["out"]


def _plain_read(s):
    c, n = s["case"], s["real"]
    at = s["slots"][:n]
    codes = s["kv"].view(torch.uint8).view(-1, *s["kv"].shape[2:])[at].view(s["kv"].dtype)
    s["out"][:n] = _values(codes, s["scales"].view(-1, *s["scales"].shape[2:])[at], c).to(s["out"].dtype)
    return s["out"]


def _plain_attention(s):
    c = s["case"]
    seqs, page = s["seqs"].long(), c["page"]
    B, S, Q, D, Hkv, G = c["B"], s["kv_max"], s["q_max"], c["D"], c["H_kv"], c["H"] // c["H_kv"]
    q0, nq, nkv = seqs[:, 0:1], seqs[:, 1:2], seqs[:, 2:3]
    key = torch.arange(S, device=DEV)
    pages, row = seqs[:, 3 + key // page], key % page
    rows = _values(s["kv"].view(torch.uint8)[pages, row].view(s["kv"].dtype), s["scales"][pages, row], c)  # [B, S, H_kv, 2D]
    k = rows[..., :D].permute(0, 2, 3, 1).contiguous()
    v = rows[..., D:].permute(0, 2, 1, 3).contiguous()
    i = torch.arange(Q, device=DEV)
    at = q0 + torch.minimum(i, nq - 1)
    q = s["q"][at].view(B, Q, Hkv, G, D).permute(0, 2, 1, 3, 4).reshape(B, Hkv, Q * G, D)
    score = torch.matmul(q, k).view(B, Hkv, Q, G, S).mul_(s["scale"])
    pos = (nkv - nq + i).unsqueeze(2)
    seen = key <= pos
    if c["window"]:
        seen = seen & ((key > pos - c["window"]) | (key < c["n_first"]))
    score = score.masked_fill_(~seen.view(B, 1, Q, 1, S), -math.inf)
    top = score.amax(-1, keepdim=True)
    if s["sinks"] is not None:
        sink = s["sinks"].view(1, Hkv, 1, G, 1)
        top = torch.maximum(top, sink)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    p = score.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    if s["sinks"] is not None:
        total = total + (sink - top).exp()
    o = torch.matmul(p.view(B, Hkv, Q * G, S), v).view(B, Hkv, Q, G, D) / total
    o = torch.where(total > 0, o, torch.zeros_like(o)).permute(0, 2, 1, 3, 4).reshape(B, Q, c["H"], D)
    out = torch.zeros((s["T"], c["H"], D), device=DEV)
    out[at] = o[torch.arange(B, device=DEV).unsqueeze(1), torch.minimum(i, nq - 1)]
    return out


# -------------------------------------------------------- the framework's calls

_BE = None


def _backend():
    global _BE
    if _BE is None:
        sys.path.insert(0, os.path.join(os.getcwd(), "llama.rust_amd"))
        import ghip
        _BE = (ghip, ghip.Backend(0))
    return _BE


def _rope_of(ghip, c):
    mode = {"norm": ghip.ROPE_NORM, "neox": ghip.ROPE_NEOX, "mrope": ghip.ROPE_MROPE, "imrope": ghip.ROPE_IMROPE}[c["mode"]]
    return ghip.Rope(c["n_dims"], mode, freq_base=c["base"], sections=tuple(int(x) for x in c["sections"].split(",")))


def run(state):
    s, c = state, state["case"]
    if own:
        ghip, be = _backend()
        if c["kind"] == "attn":
            return be.flash_attn_paged(s["q"], s["kv"], s["seqs"], scales=s["scales"], scale=s["scale"], sinks=s["sinks"],
                                       window=c["window"], n_first=c["n_first"], n_shared=c["shared"], max_q=s["q_max"], out=s["out"])
        if c["kind"] == "append":
            if "rope" not in s:
                s["rope"] = _rope_of(ghip, c)
            be.kv_append(s["k"], s["v"], s["slots"], s["kv"], scales=s["scales"], pos=s["pos"], rope=s["rope"], factors=s["factors"])
            if c["bits"] == 8:
                return [s["kv"], s["scales"]]
        return be.kv_read(s["kv"], s["slots"], scales=s["scales"], out=s["out"])
    return {"append": _plain_append, "read": _plain_read, "attn": _plain_attention}[c["kind"]](s)


# ---------------------------------------------------------------------- work

def _seen(p, window, first):
    """keys that a row at position p sees"""
    n = p + 1
    if window and n > window:
        n = window + min(first, n - window)
    return max(0, n)


def work(case):
    c = case
    row = 2 * c["D"] * c["bits"] // 8 + 2 * ((c["D"] + 31) // 32)  # bytes of a head's key and value
    if c["kind"] == "read":
        n = (c["T"] - c["pad"]) * c["H_kv"]
        return {"bytes": n * (row + 2 * c["D"] * (4 if c["type"] == "f32" else 2)) + 8 * c["T"], "flops": n * 2 * c["D"]}
    if c["kind"] == "append":
        n = (c["T"] - c["pad"]) * c["H_kv"]
        back = 0 if c["bits"] == 8 else 2 * c["D"] * 2 + row
        return {"bytes": n * (row + 2 * c["D"] * (4 if c["type"] == "f32" else 2) + back) + 12 * c["T"], "flops": 7 * n * c["D"]}
    nq, nkv = _lengths(c)
    pairs = keys = 0
    for q, kv in zip(nq, nkv):
        ends = range(kv - q, kv)
        pairs += sum(_seen(p, c["window"], c["n_first"]) for p in (ends if q <= 64 or c["window"] else (ends[0], ends[-1]))) \
            * (1 if q <= 64 or c["window"] else q / 2)
        own_keys = kv
        if c["window"] and kv - q + 1 > c["window"]:
            low = kv - q - c["window"] + 1
            own_keys = kv - low + min(c["n_first"], low)
        keys += own_keys - min(c["shared"], kv)
    keys += c["shared"]
    return {"bytes": keys * c["H_kv"] * row + sum(nq) * c["H"] * c["D"] * 8, "flops": 4.0 * c["D"] * c["H"] * pairs}


# --------------------------------------------------------------------- exact

def _grid(bits):
    """the values that codes without a sign stand for, in order"""
    if bits == 4:
        return list(E2M1)
    return [(1 + m / 8 if e else m / 8) * 2.0 ** max(e - 7, -6) for e in range(16) for m in range(8)][:127]


def _two_to(e):
    """2^e of whole numbers in 64 bits, from a table"""
    return torch.tensor([2.0 ** i for i in range(-200, 201)], dtype=torch.float64, device=DEV)[e.long() + 200]


def _decoded64(kv, scales, c):
    """the cache's rows [n, H_kv, 2 D] in 64 bits, code by code from a table"""
    D, S = c["D"], scales.shape[-1] // 2
    grid = torch.tensor(_grid(c["bits"]), dtype=torch.float64, device=DEV)
    b = kv.view(torch.uint8).long()
    if c["bits"] == 4:
        b = torch.stack([b % 16, b // 16], -1).flatten(-2)
    half = 128 if c["bits"] == 8 else 8
    v = torch.where(b >= half, -grid[(b % half).clamp(max=len(grid) - 1)], grid[(b % half).clamp(max=len(grid) - 1)])
    j = torch.arange(2 * D, device=DEV)
    return v * _two_to(scales[..., (j // D) * S + j % D // 32].long() - 127)


def _rounded64(x, c):
    """rows [n, H, D] in 64 bits -> the values that their codes stand for (without the scale), the scales' exponents"""
    grid = torch.tensor(_grid(c["bits"]), dtype=torch.float64, device=DEV)
    top = 448.0 if c["bits"] == 8 else 7.0
    D = x.shape[-1]
    codes, exps = torch.empty_like(x), []
    mid = (grid[1:] + grid[:-1]) / 2
    for d in range(0, 32 * _scale_bytes(D), 32):
        y = x[..., d:d + 32]
        if d >= D:
            exps.append(torch.full(x.shape[:-1], -100.0, dtype=torch.float64, device=DEV))
            continue
        big = y.abs().max(-1).values
        e = torch.ceil(torch.log2(big / top)).clamp(min=-100)
        e = e + (big > top * _two_to(e)).double()  # (the logarithm's own rounding)
        e = e - ((big <= top * _two_to(e - 1)) & (e > -100)).double()
        y = y / _two_to(e.unsqueeze(-1))
        i = torch.bucketize(y.abs(), mid)  # mid[i - 1] < |y| <= mid[i]
        tie = (i < len(mid)) & (y.abs() == mid[i.clamp(max=len(mid) - 1)]) & (i % 2 == 1)
        codes[..., d:d + 32] = grid[i + tie.long()].copysign(y)
        exps.append(e)
    return codes, torch.stack(exps, -1)


def _rotated64(c, x, pos, factors):
    """pair by pair, as products of complex numbers"""
    n, s = c["n_dims"], [int(v) for v in c["sections"].split(",")]
    x, cols = x.double(), []
    for i in range(n // 2):
        axis = 0
        if c["mode"] == "mrope":
            place = i % sum(s)
            while place >= s[axis]:
                place, axis = place - s[axis], axis + 1
        elif c["mode"] == "imrope":
            j = i % sum(s)
            axis = j % 3 if j < 3 * s[j % 3] else 3
        f = c["base"] ** (-2.0 * i / n)
        cols.append(pos[axis].double() * (f if factors is None else f / factors[i].double()))
    a = torch.stack(cols, 1)
    z = torch.polar(torch.ones_like(a), a).unsqueeze(1)
    P = n // 2
    if c["mode"] == "norm":
        y = torch.view_as_real(torch.view_as_complex(x[..., :n].reshape(*x.shape[:-1], P, 2).contiguous()) * z).flatten(-2)
    else:
        y = torch.complex(x[..., :P].contiguous(), x[..., P:n].contiguous()) * z
        y = torch.cat([y.real, y.imag], -1)
    return torch.cat([y, x[..., n:]], -1)


def exact(case, seed):
    c, s = case, _inputs(case, seed)
    D, page, Hkv = c["D"], c["page"], c["H_kv"]
    if c["kind"] == "read":
        out, n = torch.zeros((c["T"], Hkv, 2 * D), dtype=torch.float64, device=DEV), s["real"]
        at = s["slots"][:n]
        out[:n] = _decoded64(s["kv"][at // page, at % page] if c["bits"] == 4 else s["kv"].view(torch.uint8)[at // page, at % page],
                             s["scales"][at // page, at % page], c)
        return out
    if c["kind"] == "append":
        n, at = s["real"], s["slots"][:s["real"]]
        kc, ke = _rounded64(_rotated64(c, s["k"][:n], s["pos"][:, :n], s["factors"]), c)
        vc, ve = _rounded64(s["v"][:n].double(), c)
        codes, exps = torch.cat([kc, vc], -1), torch.cat([ke, ve], -1)
        if c["bits"] == 8:
            kv = s["kv"].double()
            kv[at // page, at % page] = codes
            return [kv, None]
        j = torch.arange(2 * D, device=DEV)
        out = torch.zeros((c["T"], Hkv, 2 * D), dtype=torch.float64, device=DEV)
        out[:n] = codes * _two_to(exps)[..., (j // D) * _scale_bytes(D) + j % D // 32]
        return out
    nq, nkv = _lengths(c)
    G = c["H"] // Hkv
    out = torch.zeros((s["T"], c["H"], D), dtype=torch.float64, device=DEV)
    q0 = 0
    for b, (n, m) in enumerate(zip(nq, nkv)):
        pages = s["seqs"][b, 3:3 + (m + page - 1) // page].long()
        rows = _decoded64(s["kv"].view(torch.uint8)[pages].flatten(0, 1)[:m], s["scales"][pages].flatten(0, 1)[:m], c)
        for t0 in range(0, n, 64):
            t1 = min(n, t0 + 64)
            p = (m - n + torch.arange(t0, t1, device=DEV)).view(-1, 1)
            j = torch.arange(m, device=DEV).view(1, -1)
            hidden = j > p
            if c["window"]:
                hidden = hidden | ((j <= p - c["window"]) & (j >= c["n_first"]))
            for h in range(Hkv):
                q = s["q"][q0 + t0:q0 + t1, h * G:(h + 1) * G].double().reshape(-1, D)
                x = (q @ rows[:, h, :D].t().contiguous() * s["scale"]).view(t1 - t0, G, m)
                x = x.masked_fill(hidden.unsqueeze(1), -math.inf)
                if s["sinks"] is not None:
                    x = torch.cat([x, s["sinks"][h * G:(h + 1) * G].double().view(1, G, 1).expand(t1 - t0, G, 1)], -1)
                w = torch.softmax(x, -1)[..., :m].reshape(-1, m)
                out[q0 + t0:q0 + t1, h * G:(h + 1) * G] = (w @ rows[:, h, D:]).view(t1 - t0, G, D)
        q0 += n
    return out
