"""The serving operators that performance is measured on: rotary positions with
several axes, appending to a paged KV cache with the rotation on the way, and
attention over that cache with a sliding window and first tokens that stay
visible, or with a prefix that the whole batch shares.

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
        # generation: the query rows of one new token of a vision-language model
        {"name": "rope_token", "kind": "rope", "mode": "mrope", "T": 1, "H": 32, "D": 128, "n_dims": 128,
         "sections": "16,24,24,0", "base": 1e6, "start": 4000, "grid": 40, "type": "f32"},
        # the queries of a prompt with an image in it, axes interleaved
        {"name": "rope_prompt", "kind": "rope", "mode": "imrope", "T": 1500, "H": 32, "D": 128, "n_dims": 128,
         "sections": "24,20,20,0", "base": 5e6, "start": 100000, "grid": 33, "type": "f32"},
        # a vision encoder's queries: 70 x 70 patches, rows and columns
        {"name": "rope_vision", "kind": "rope", "mode": "vision", "T": 4900, "H": 16, "D": 80, "n_dims": 40,
         "sections": "20,20,0,0", "base": 1e4, "start": 0, "grid": 70, "type": "f16"},
        # generation: one new token for each of 32 sequences
        {"name": "append_tokens", "kind": "append", "mode": "neox", "T": 32, "B": 32, "H_kv": 8, "D": 128, "n_dims": 128,
         "sections": "0,0,0,0", "base": 5e5, "start": 9000, "grid": 1, "type": "f16", "page": 64, "factors": True, "pad": 0},
        # three prompts of a vision-language model in one batch, small pages, a few rows of padding
        {"name": "append_prompts", "kind": "append", "mode": "mrope", "T": 2011, "B": 3, "H_kv": 4, "D": 128, "n_dims": 128,
         "sections": "16,24,24,0", "base": 1e6, "start": 500, "grid": 27, "type": "bf16", "page": 16, "factors": False, "pad": 5},
        # a large prefill batch
        {"name": "append_prefill", "kind": "append", "mode": "norm", "T": 8192, "B": 8, "H_kv": 8, "D": 128, "n_dims": 128,
         "sections": "0,0,0,0", "base": 1e4, "start": 0, "grid": 1, "type": "f16", "page": 64, "factors": False, "pad": 0},
        # one new token of one conversation, a layer with a short window and learned sinks
        {"name": "window_token", "kind": "attn", "B": 1, "q_lo": 1, "q_hi": 1, "kv_lo": 1061, "kv_hi": 1061, "H": 64, "H_kv": 8,
         "D": 64, "type": "f16", "page": 16, "window": 128, "n_first": 4, "shared": 0, "sinks": True},
        # generation of 24 sequences of very different length under a long window
        {"name": "window_batch", "kind": "attn", "B": 24, "q_lo": 1, "q_hi": 1, "kv_lo": 500, "kv_hi": 16384, "H": 32, "H_kv": 8,
         "D": 128, "type": "bf16", "page": 64, "window": 4096, "n_first": 4, "shared": 0, "sinks": False},
        # prefill chunks of two long prompts
        {"name": "window_prompt", "kind": "attn", "B": 2, "q_lo": 701, "q_hi": 1001, "kv_lo": 4000, "kv_hi": 8192, "H": 32, "H_kv": 8,
         "D": 128, "type": "f16", "page": 16, "window": 2048, "n_first": 4, "shared": 0, "sinks": False},
        # five samples of one answer, shortly after the prompt
        {"name": "shared_samples", "kind": "attn", "B": 5, "q_lo": 1, "q_hi": 1, "kv_lo": 1062, "kv_hi": 1400, "H": 64, "H_kv": 8,
         "D": 64, "type": "f16", "page": 16, "window": 0, "n_first": 0, "shared": 1061, "sinks": False},
        # generation of 64 requests under one long system prompt
        {"name": "shared_tokens", "kind": "attn", "B": 64, "q_lo": 1, "q_hi": 1, "kv_lo": 8232, "kv_hi": 8792, "H": 32, "H_kv": 8,
         "D": 128, "type": "f16", "page": 64, "window": 0, "n_first": 0, "shared": 8192, "sinks": False},
        # twelve short user turns under one document
        {"name": "shared_turns", "kind": "attn", "B": 12, "q_lo": 20, "q_hi": 60, "kv_lo": 4061, "kv_hi": 4300, "H": 32, "H_kv": 8,
         "D": 128, "type": "bf16", "page": 64, "window": 0, "n_first": 0, "shared": 4001, "sinks": False},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _rotation(rng):
    """mode, n_dims, sections for a head size"""
    D = rng.choice([64, 80, 96, 128, 256])
    mode = rng.choice(["norm", "neox", "mrope", "imrope"])
    n = D if rng.random() < 0.7 else 2 * (D // 8)
    p = n // 2
    if mode == "mrope":
        a = rng.randint(1, p // 2)
        b = (p - a) // 2
        sec = (a, b, p - a - b, 0)
    elif mode == "imrope":
        sec = (p - 2 * (p // 3), p // 3, p // 3, 0)
    else:
        sec = (0, 0, 0, 0)
    return D, mode, n, "%d,%d,%d,%d" % sec


def draw(rng):
    most, large = max(_cost(c) for c in listed()), max(_size(c) for c in listed())
    while True:
        kind = rng.choice(["rope", "append", "window", "shared"])
        if kind == "rope":
            if rng.random() < 0.3:
                D = rng.choice([64, 72, 80, 128])
                mode, n, sec = "vision", D // 2, "%d,%d,0,0" % (D // 4, D // 4)
            else:
                D, mode, n, sec = _rotation(rng)
            return {"kind": "rope", "mode": mode, "T": _log_int(rng, 1, 8192), "H": rng.choice([1, 7, 12, 16, 32]), "D": D,
                    "n_dims": n, "sections": sec, "base": rng.choice([1e4, 5e5, 1e6]), "start": rng.randint(0, 200000),
                    "grid": rng.randint(2, 80), "type": rng.choice(["f32", "f32", "f16", "bf16"])}
        if kind == "append":
            D, mode, n, sec = _rotation(rng)
            T = _log_int(rng, 1, 8192)
            return {"kind": "append", "mode": mode, "T": T, "B": rng.randint(1, min(T, 40)), "H_kv": rng.choice([1, 2, 4, 8]), "D": D,
                    "n_dims": n, "sections": sec, "base": rng.choice([1e4, 5e5, 1e6]), "start": rng.randint(0, 20000),
                    "grid": rng.randint(2, 80), "type": rng.choice(["f16", "bf16"]), "page": rng.choice([1, 16, 24, 64, 256]),
                    "factors": rng.random() < 0.3, "pad": rng.randint(0, T // 8)}
        H_kv = rng.choice([1, 2, 4, 8])
        D = rng.choice([64, 64, 80, 128, 128, 128, 256])
        c = {"kind": "attn", "B": _log_int(rng, 1, 96), "q_lo": 1, "q_hi": 1, "kv_lo": 0, "kv_hi": 0,
             "H": H_kv * rng.choice([1, 3, 4, 5, 8, 16]), "H_kv": H_kv, "D": D, "type": rng.choice(["f16", "bf16"]),
             "page": rng.choice([1, 16, 24, 64, 256]), "window": 0, "n_first": 0, "shared": 0, "sinks": rng.random() < 0.3}
        if rng.random() < 0.5:
            c["q_hi"] = _log_int(rng, 2, 1200)
            c["q_lo"] = rng.randint(1, c["q_hi"])
        c["kv_hi"] = c["q_hi"] + _log_int(rng, 1, 16384)
        if kind == "window":
            c["kv_lo"] = rng.randint(c["q_lo"], c["kv_hi"])
            c["window"] = rng.choice([0, _log_int(rng, 1, 8192), _log_int(rng, 64, 4096)])
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


def _share(T, B):
    """T tokens over B sequences"""
    return [T // B + (i < T % B) for i in range(B)]


def _positions(c, T, start):
    """positions of T tokens, [axes, T]: text, then an image of `grid` columns"""
    i = torch.arange(T, device=DEV)
    if c["mode"] in ("norm", "neox"):
        return (start + i).to(torch.int32).reshape(1, T)
    if c["mode"] == "vision":
        y, x = i // c["grid"], i % c["grid"]
        return torch.stack([y, x, y, x]).to(torch.int32)
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


def _inputs(case, seed):
    c = case
    g = torch.Generator(device=DEV).manual_seed(seed)
    s = {"case": c}
    if c["kind"] == "rope":
        s["x"] = _heads((c["T"], c["H"], c["D"]), g).to(TYPES[c["type"]])
        s["pos"] = _positions(c, c["T"], c["start"] + seed % 97)
        s["factors"] = None
        return s
    ty = TYPES[c["type"]]
    page, D, Hkv = c["page"], c["D"], c["H_kv"]
    if c["kind"] == "append":
        T, real = c["T"], c["T"] - c["pad"]
        n = _share(real, c["B"])
        s["k"], s["v"] = _heads((T, Hkv, D), g), _heads((T, Hkv, D), g)
        first = [(c["start"] + 37 * i + seed) % page for i in range(c["B"])]  # the row of its page each sequence goes on at
        need = [(2 * page - 2 + m) // page for m in n]  # wherever it starts
        s["pages"] = sum(need) + max(8, sum(need) // 2)
        perm = torch.randperm(s["pages"], generator=g, device=DEV)
        slots, pos, at = [], [], 0
        for f, m, k in zip(first, n, need):
            i = f + torch.arange(m, device=DEV)
            slots.append(perm[at + i // page] * page + i % page)
            pos.append(_positions(c, m, c["start"] + seed % 97 + f))
            at += k
        slots.append(torch.full((c["pad"],), -1, dtype=torch.int64, device=DEV))
        pos.append(torch.zeros((pos[0].shape[0], c["pad"]), dtype=torch.int32, device=DEV))
        s["slots"], s["pos"], s["real"] = torch.cat(slots), torch.cat(pos, 1).contiguous(), real
        s["kv"] = torch.randn((s["pages"], page, Hkv, 2 * D), generator=g, device=DEV).to(ty)
        # longer wavelengths for the low frequencies, as long-context models ship them
        s["factors"] = torch.linspace(1.0, 8.0, c["n_dims"] // 2, device=DEV) if c["factors"] else None
        return s
    nq, nkv = _lengths(c)
    T, per = sum(nq), (max(nkv) + page - 1) // page
    common, rest = divmod(c["shared"], page)  # pages that all sequences have, and rows of the next one, copied for each
    need = [(m + page - 1) // page for m in nkv]
    s["pages"] = sum(max(0, m - common) for m in need) + common + 4
    perm = torch.randperm(s["pages"], generator=g, device=DEV).to(torch.int32)
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
    s["kv"] = torch.randn((s["pages"], page, Hkv, 2 * D), generator=g, device=DEV).to(ty)
    if rest:
        s["kv"][seqs[1:, 3 + common].long(), :rest] = s["kv"][seqs[0, 3 + common].long(), :rest]
    s["sinks"] = torch.randn(c["H"], generator=g, device=DEV) if c["sinks"] else None
    s["scale"] = 1.0 / math.sqrt(D)
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if case["kind"] == "rope":
        s["out"] = torch.empty_like(s["x"])
    elif case["kind"] == "attn":
        s["out"] = torch.empty((s["T"], case["H"], case["D"]), device=DEV)
    return s


# --------------------------------------------------------------- plain forms

def _axis_of_pairs(mode, n_pairs, sections):
    """for each pair: its position's axis, and its place in the frequencies"""
    i = torch.arange(n_pairs, device=DEV)
    s = [int(x) for x in sections.split(",")]
    if mode in ("norm", "neox"):
        return torch.zeros_like(i), i
    j = i % sum(s)
    if mode == "imrope":
        r = j % 3
        ok = j < 3 * torch.where(r == 0, s[0], torch.where(r == 1, s[1], s[2]))
        return torch.where(ok, r, 3), i
    b = [0, s[0], s[0] + s[1], s[0] + s[1] + s[2]]
    axis = (j >= b[1]).long() + (j >= b[2]).long() + (j >= b[3]).long()
    return axis, (j - torch.tensor(b, device=DEV)[axis] if mode == "vision" else i)


def _rotate(x, pos, c, factors):
    """x [T, heads, D] in 32 bits, rotated; the angles in 64 bits (positions are far)"""
    n = c["n_dims"]
    pairs = n if c["mode"] == "vision" else n // 2
    axis, i = _axis_of_pairs(c["mode"], pairs, c["sections"])
    f = torch.pow(torch.tensor(c["base"], dtype=torch.float64, device=DEV), -2.0 * i.double() / n)
    if factors is not None:
        f = f / factors.double()
    a = pos[axis].t().double() * f
    cos, sin = a.cos().float().unsqueeze(1), a.sin().float().unsqueeze(1)
    y = x.float().clone()
    if c["mode"] == "norm":
        x0, x1 = x[..., 0:2 * pairs:2].float(), x[..., 1:2 * pairs:2].float()
        y[..., 0:2 * pairs:2], y[..., 1:2 * pairs:2] = x0 * cos - x1 * sin, x0 * sin + x1 * cos
    else:
        x0, x1 = x[..., :pairs].float(), x[..., pairs:2 * pairs].float()
        y[..., :pairs], y[..., pairs:2 * pairs] = x0 * cos - x1 * sin, x0 * sin + x1 * cos
    return y


def _plain_attention(s):
    c = s["case"]
    seqs, kv, page = s["seqs"].long(), s["kv"], c["page"]
    B, S, Q, D, Hkv, G = c["B"], s["kv_max"], s["q_max"], c["D"], c["H_kv"], c["H"] // c["H_kv"]
    q0, nq, nkv = seqs[:, 0:1], seqs[:, 1:2], seqs[:, 2:3]
    key = torch.arange(S, device=DEV)
    rows = kv[seqs[:, 3 + key // page], key % page]  # [B, S, H_kv, 2D]
    k = rows[..., :D].float().permute(0, 2, 3, 1).contiguous()
    v = rows[..., D:].float().permute(0, 2, 1, 3).contiguous()
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
    mode = {"norm": ghip.ROPE_NORM, "neox": ghip.ROPE_NEOX, "mrope": ghip.ROPE_MROPE, "imrope": ghip.ROPE_IMROPE,
            "vision": ghip.ROPE_VISION}[c["mode"]]
    return ghip.Rope(c["n_dims"], mode, freq_base=c["base"], sections=tuple(int(x) for x in c["sections"].split(",")))


def run(state):
    s, c = state, state["case"]
    if own:
        ghip, be = _backend()
        if c["kind"] == "attn":
            return be.flash_attn_paged(s["q"], s["kv"], s["seqs"], scale=s["scale"], sinks=s["sinks"], window=c["window"],
                                       n_first=c["n_first"], n_shared=c["shared"], max_q=s["q_max"], out=s["out"])
        if "rope" not in s:
            s["rope"] = _rope_of(ghip, c)
        if c["kind"] == "rope":
            return be.rope(s["x"], s["pos"], s["rope"], out=s["out"])
        be.kv_append(s["k"], s["v"], s["slots"], s["kv"], pos=s["pos"], rope=s["rope"], factors=s["factors"])
        return s["kv"]
    if c["kind"] == "attn":
        return _plain_attention(s)
    if c["kind"] == "rope":
        return _rotate(s["x"], s["pos"], c, None).to(s["x"].dtype)
    n, D, kv = s["real"], c["D"], s["kv"]
    k = _rotate(s["k"][:n], s["pos"][:, :n], c, s["factors"])
    kv.view(-1, c["H_kv"], 2 * D)[s["slots"][:n]] = torch.cat([k, s["v"][:n]], -1).to(kv.dtype)
    return kv


# ---------------------------------------------------------------------- work

def _seen(p, window, first):
    """keys that a row at position p sees"""
    n = p + 1
    if window and n > window:
        n = window + min(first, n - window)
    return max(0, n)


def work(case):
    c = case
    if c["kind"] == "rope":
        e = 4 if c["type"] == "f32" else 2
        return {"bytes": 2 * e * c["T"] * c["H"] * c["D"] + 4 * c["T"] * (1 if c["mode"] in ("norm", "neox") else 4),
                "flops": 3 * c["T"] * c["H"] * c["D"]}
    if c["kind"] == "append":
        n = (c["T"] - c["pad"]) * c["H_kv"] * 2 * c["D"]
        return {"bytes": 6 * n + 12 * c["T"], "flops": 1.5 * n}
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
    return {"bytes": keys * c["H_kv"] * 2 * c["D"] * 2 + sum(nq) * c["H"] * c["D"] * 8,
            "flops": 4.0 * c["D"] * c["H"] * pairs}


# --------------------------------------------------------------------- exact

def _angles64(c, pos, factors):
    """angle of every token's every pair, pair by pair"""
    n, s = c["n_dims"], [int(x) for x in c["sections"].split(",")]
    cols = []
    for i in range(n if c["mode"] == "vision" else n // 2):
        axis, place = 0, i
        if c["mode"] in ("mrope", "vision"):
            place, axis = i % sum(s), 0
            while place >= s[axis]:
                place, axis = place - s[axis], axis + 1
            place = place if c["mode"] == "vision" else i
        elif c["mode"] == "imrope":
            j = i % sum(s)
            axis = j % 3 if j < 3 * s[j % 3] else 3
        f = c["base"] ** (-2.0 * place / n)
        cols.append(pos[axis].double() * (f if factors is None else f / factors[i].double()))
    return torch.stack(cols, 1)


def _rotated64(c, x, pos, factors):
    x, a = x.double(), _angles64(c, pos, factors)
    z = torch.polar(torch.ones_like(a), a).unsqueeze(1)
    P = a.shape[1]
    if c["mode"] == "norm":
        y = torch.view_as_real(torch.view_as_complex(x[..., :2 * P].reshape(*x.shape[:-1], P, 2).contiguous()) * z).flatten(-2)
    else:
        y = torch.complex(x[..., :P].contiguous(), x[..., P:2 * P].contiguous()) * z
        y = torch.cat([y.real, y.imag], -1)
    return torch.cat([y, x[..., 2 * P:]], -1)


def exact(case, seed):
    c, s = case, _inputs(case, seed)
    if c["kind"] == "rope":
        return _rotated64(c, s["x"], s["pos"], None)
    if c["kind"] == "append":
        kv, n = s["kv"].double(), s["real"]
        flat = kv.view(-1, c["H_kv"], 2 * c["D"])
        flat[s["slots"][:n], :, :c["D"]] = _rotated64(c, s["k"][:n], s["pos"][:, :n], s["factors"])
        flat[s["slots"][:n], :, c["D"]:] = s["v"][:n].double()
        return kv
    nq, nkv = _lengths(c)
    D, page, G = c["D"], c["page"], c["H"] // c["H_kv"]
    out = torch.zeros((s["T"], c["H"], D), dtype=torch.float64, device=DEV)
    q0 = 0
    for b, (n, m) in enumerate(zip(nq, nkv)):
        pages = s["seqs"][b, 3:3 + (m + page - 1) // page].long()
        rows = s["kv"][pages].reshape(-1, c["H_kv"], 2 * D)[:m].double()
        for t0 in range(0, n, 64):
            t1 = min(n, t0 + 64)
            p = (m - n + torch.arange(t0, t1, device=DEV)).view(-1, 1)
            j = torch.arange(m, device=DEV).view(1, -1)
            hidden = j > p
            if c["window"]:
                hidden = hidden | ((j <= p - c["window"]) & (j >= c["n_first"]))
            for h in range(c["H_kv"]):
                q = s["q"][q0 + t0:q0 + t1, h * G:(h + 1) * G].double().reshape(-1, D)
                x = (q @ rows[:, h, :D].t().contiguous() * s["scale"]).view(t1 - t0, G, m)
                x = x.masked_fill(hidden.unsqueeze(1), -math.inf)
                if s["sinks"] is not None:
                    x = torch.cat([x, s["sinks"][h * G:(h + 1) * G].double().view(1, G, 1).expand(t1 - t0, G, 1)], -1)
                w = torch.softmax(x, -1)[..., :m].reshape(-1, m)
                out[q0 + t0:q0 + t1, h * G:(h + 1) * G] = (w @ rows[:, h, D:]).view(t1 - t0, G, D)
        q0 += n
    return out
