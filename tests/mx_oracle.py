"""A quantized KV cache restated in 64 bits on the CPU, code by code from tables:
blocks of 32 elements, E4M3 or E2M1 codes, a power of two for each."""
import torch

TOP = {8: 448.0, 4: 7.0}


def grid(bits):
    """the values that codes without a sign stand for, in order (8 bits: code 127 is NaN)"""
    if bits == 4:
        v = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
    else:
        v = [(1 + m / 8 if e else m / 8) * 2.0 ** max(e - 7, -6) for e in range(16) for m in range(8)][:127]
    return torch.tensor(v, dtype=torch.float64)


def scale_bytes(D):
    return 1 if D <= 32 else 2 if D <= 64 else 4 if D <= 128 else 8


def two_to(e):
    return torch.tensor([2.0 ** i for i in range(-160, 161)], dtype=torch.float64)[e.long() + 160]


def encode(x, bits):
    """rows x [.., D] in 64 bits -> (codes as whole numbers [.., D], scale bytes [.., S], how far each
    element is from where its code would change, relative to its block's largest)"""
    g, top, D = grid(bits), TOP[bits], x.shape[-1]
    mid = (g[1:] + g[:-1]) / 2
    codes, room = torch.zeros(x.shape, dtype=torch.int64), torch.full(x.shape, float("inf"), dtype=torch.float64)
    sb = torch.full(x.shape[:-1] + (scale_bytes(D),), 27, dtype=torch.int64)
    for b in range((D + 31) // 32):
        y = x[..., 32 * b:32 * b + 32]
        big = y.abs().amax(-1)
        ok = big < float("inf")  # no infinity, no NaN
        m, e = torch.frexp(torch.where(ok & (big > 0), big, torch.ones_like(big)))
        exps = torch.stack([e.long() + k for k in range(-12, 2)], -1)  # the least one that will do
        will = big.unsqueeze(-1) <= top * two_to(exps.clamp(-159, 159))
        e = exps.gather(-1, will.to(torch.int8).argmax(-1, keepdim=True)).squeeze(-1)
        e = torch.where(big == 0, torch.full_like(e, -100), e).clamp(min=-100)
        sb[..., b] = torch.where(ok, e + 127, torch.full_like(e, 255))
        z = torch.where(ok.unsqueeze(-1), y / two_to(e).unsqueeze(-1), torch.zeros_like(y))
        i = torch.bucketize(z.abs(), mid)  # mid[i - 1] < |z| <= mid[i]
        tie = (i < len(mid)) & (z.abs() == mid[i.clamp(max=len(mid) - 1)]) & (i % 2 == 1)
        i = i + tie.long()
        half = 128 if bits == 8 else 8
        codes[..., 32 * b:32 * b + 32] = torch.where(ok.unsqueeze(-1), i + half * torch.signbit(y).long(), torch.zeros_like(i))
        far = torch.minimum((z.abs() - mid[(i - 1).clamp(min=0)]).abs(), (z.abs() - mid[i.clamp(max=len(mid) - 1)]).abs())
        lim = top * two_to(e)  # where the scale would change
        edge = torch.minimum((big - lim).abs(), (big - lim / 2).abs()) / big.clamp(min=1e-300)
        room[..., 32 * b:32 * b + 32] = torch.minimum(far * (two_to(e) / big.clamp(min=1e-300)).unsqueeze(-1), edge.unsqueeze(-1))
    return codes, sb, room


def pack(codes, bits):
    """whole numbers [.., n] -> the cache's bytes"""
    if bits == 8:
        return codes.to(torch.uint8)
    return (codes[..., 0::2] | (codes[..., 1::2] << 4)).to(torch.uint8)


def unpack(kv, bits):
    """the cache's bytes -> whole numbers"""
    b = kv.view(torch.uint8).long()
    return b if bits == 8 else torch.stack([b % 16, b // 16], -1).flatten(-2)


def decode(codes, scales, D, bits):
    """codes [.., 2 D] as whole numbers, scale bytes [.., 2 S] -> values in 64 bits"""
    g, half = grid(bits), 128 if bits == 8 else 8
    if bits == 8:
        g = torch.cat([g, torch.full((1,), float("nan"), dtype=torch.float64)])
    v = torch.where(codes >= half, -g[codes % half], g[codes % half])
    j = torch.arange(2 * D)
    s = scales.long()[..., (j // D) * (scales.shape[-1] // 2) + j % D // 32]
    return torch.where(s == 255, torch.full_like(v, float("nan")), v * two_to(s - 127))


def values(kv, scales, bits):
    """a cache's values in 64 bits"""
    D = kv.shape[-1] * (1 if bits == 8 else 2) // 2
    return decode(unpack(kv.cpu(), bits), scales.cpu(), D, bits)


def cache(pages, page, Hkv, D, bits, g, spread=3):
    """a cache in use: codes of normal values, scales of 1 / 16 and around"""
    x = torch.randn((pages, page, Hkv, 2 * D), generator=g, dtype=torch.float64)
    c, sb, _ = encode(x.view(pages, page, Hkv, 2, D), bits)
    sb = sb + torch.randint(-spread, spread + 1, sb.shape, generator=g)
    kv = pack(c.flatten(-2), bits)
    return (kv.view(torch.float8_e4m3fn) if bits == 8 else kv), sb.flatten(-2).to(torch.uint8)
