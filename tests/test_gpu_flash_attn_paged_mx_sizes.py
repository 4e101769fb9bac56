"""Attention over a quantized cache whose blocks differ widely in size, all of them in what
float16 holds, against 64 bits.  Tiles of many rows may be computed as float16 only where q's
second term and p's keep what 32 bits would: the bounds are those of
test_gpu_flash_attn_paged_mx.py (five roundings of at most 2^-22 in 2-norm, and 2^-24 of
the largest score), here too."""
import math

import pytest

import mx_oracle as M
import paged_oracle as P
from test_gpu_flash_attn_paged import ways
from test_gpu_flash_attn_paged_mx import compare, make

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu
BITS = pytest.mark.parametrize("bits", [8, 4])

# scale bytes of blocks that float16 holds in full; where blocks of normal values are
ENDS = {8: (106, 128), 4: (104, 140)}
HOME = {8: 120, 4: 126}


@pytest.fixture(scope="module")
def be():
    import ghip
    b = ghip.Backend(0)
    yield b
    b.close()


def run(be, q, kv, sc, table, bits, nq, n_shared=0, what=""):
    D = q.shape[-1]
    want, mag, wgt = P.attention(q, M.values(kv, sc, bits), table.tolist(), D ** -0.5)
    for how in ways(n_shared):
        print(what, bits, D, nq, how, flush=True)
        got = be.flash_attn_paged(q.cuda(), kv.cuda(), table.cuda(), scale=D ** -0.5, n_shared=n_shared, max_q=nq, scales=sc.cuda()).cpu()
        compare(got, want, mag, wgt, D)


SHAPES = pytest.mark.parametrize("D,nq,n_shared", [(64, 40, 0), (128, 40, 0), (128, 150, 0), (256, 20, 0), (128, 1, 128), (64, 24, 128)])


def batch(nq, n_shared):
    return [(nq, 300), (nq, 220)] if nq > 1 else [(1, 300 - 9 * i) for i in range(8)]


@BITS
@SHAPES
@pytest.mark.parametrize("apart", [1.0, 0.75, 0.5])
def test_keys_apart_and_q_undoing_it(be, D, nq, n_shared, apart, bits):
    """Blocks of keys as far apart as float16's range goes (or part of it), every other one small,
    against channels of q that make up for it: each block has its share of the scores."""
    q, kv, sc, table = make(batch(nq, n_shared), 4, 2, D, bits, 16, n_shared, seed=3)
    lo, hi = ENDS[bits]
    mid = (lo + hi) / 2
    for b in range(D // 32):
        byte = round(mid + apart * ((hi if b % 2 else lo) - mid))
        sc[..., b] = byte
        q[..., 32 * b:32 * b + 32] *= 2.0 ** (HOME[bits] - byte)
    run(be, q, kv, sc, table, bits, nq, n_shared, f"keys {apart}")


@BITS
@SHAPES
def test_zeros_under_large_q(be, D, nq, n_shared, bits):
    """Channels whose keys are all 0 under a q 2^28 times the others': it has no part in the scores."""
    q, kv, sc, table = make(batch(nq, n_shared), 4, 2, D, bits, 16, n_shared, seed=4)
    kv.view(torch.uint8)[..., :32 * bits // 8] = 0
    q[..., :32] *= 2.0 ** 14
    q[..., 32:] *= 2.0 ** -14
    for byte in (27, HOME[bits]):  # as they are written; a scale like the others'
        sc[..., 0] = byte
        for b in range(1, D // 32):
            sc[..., b] = min(HOME[bits] + 14, ENDS[bits][1])
        q2 = q.clone()
        q2[..., 32:] *= 2.0 ** (HOME[bits] + 14 - min(HOME[bits] + 14, ENDS[bits][1]))
        run(be, q2, kv, sc, table, bits, nq, n_shared, f"zeros {byte}")


def three_weights(kv, sc, q, table, bits, D):
    """Scores so that keys have one of three sizes of weight, about 1 (0), 2^-8 (1) and 2^-25 (2): of every 64 keys the first 32
    the first two, the others the last two.  -> which one each row of the cache is"""
    kind = torch.zeros(kv.shape[:2], dtype=torch.long)
    for b in range(table.shape[0]):
        for j in range(int(table[b, 2])):
            kind[int(table[b, 3 + j // 16]), j % 16] = (0 if j % 64 in (5, 17) else 1) if j % 64 < 32 else 1 if j % 8 == 0 else 2
    u = kv.view(torch.uint8)
    u[..., :D * bits // 8] = 0
    u[..., 0] = torch.tensor({8: (0, 0x71, 0x7e), 4: (0, 4, 7)}[bits], dtype=torch.uint8)[kind].unsqueeze(-1)  # 0, 144, 448; 0, 2, 6
    sc[..., :M.scale_bytes(D)] = 118
    q[..., 0] = -17.1 * math.sqrt(D) / ({8: 448.0, 4: 6.0}[bits] * 2.0 ** -9) * torch.linspace(1.0, 1.02, q.shape[0] * q.shape[1]).view(q.shape[:2])
    return kind


@BITS
@SHAPES
def test_light_keys_with_large_values(be, D, nq, n_shared, bits):
    """Keys of weight 2^-25 beside some of 2^-8, with values 2^20 (2^24) times the others': a part of the output is theirs."""
    q, kv, sc, table = make(batch(nq, n_shared), 2, 1, D, bits, 16, n_shared, seed=5)
    S = M.scale_bytes(D)
    kind = three_weights(kv, sc, q, table, bits, D)
    lo, hi = {8: (107, 127), 4: (115, 139)}[bits]
    sc[..., S:] = torch.where(kind == 2, hi, lo).to(torch.uint8).view(*kind.shape, 1, 1)
    run(be, q, kv, sc, table, bits, nq, n_shared, "light")


@BITS
@SHAPES
def test_weak_values_under_the_weight(be, D, nq, n_shared, bits):
    """The heavier keys' values are 0 in one block, or have codes far below what their scale allows."""
    q, kv, sc, table = make(batch(nq, n_shared), 2, 1, D, bits, 16, n_shared, seed=6)
    S = M.scale_bytes(D)
    kind = three_weights(kv, sc, q, table, bits, D)
    sc[..., S:] = HOME[bits]
    for code in ((0, 1) if bits == 8 else (0, 0x11)):  # 2^-9; 0.5
        w = kv.view(torch.uint8).clone()
        w[..., D * bits // 8:(D + 32) * bits // 8][kind < 2] = code
        run(be, q, w.view(torch.float8_e4m3fn) if bits == 8 else w, sc, table, bits, nq, n_shared, f"weak {code}")


@BITS
@SHAPES
@pytest.mark.parametrize("end", [0, 1])
def test_ends_of_the_range(be, D, nq, n_shared, end, bits):
    """All blocks at the smallest or largest scale that float16 holds all codes of."""
    for keys, values in ((end, end), (end, 1 - end)):
        q, kv, sc, table = make(batch(nq, n_shared), 4, 2, D, bits, 16, n_shared, seed=7)
        S = M.scale_bytes(D)
        sc[..., :S], sc[..., S:] = ENDS[bits][keys], ENDS[bits][values]
        q *= 2.0 ** (HOME[bits] - ENDS[bits][keys])
        run(be, q, kv, sc, table, bits, nq, n_shared, f"end {keys} {values}")


@BITS
@pytest.mark.parametrize("D,nq", [(64, 150), (128, 150), (128, 40), (256, 40)])
def test_out_of_range_keeps_all_terms(be, D, nq, bits):
    """Blocks that float16 does not hold: bfloat16 with all three terms of q and p, in 2-norm for each
    block of dims (the values' sizes differ between them)."""
    S = M.scale_bytes(D)
    for n_shared, seqs in ((0, [(nq, 1500), (20, 300)]), (256, [(nq, 600), (nq, 500)])):
        for what in ("key", "zeros", "keys", "values", "last"):
            q, kv, sc, table = make(seqs, 4, 2, D, bits, 16, n_shared, seed=8)
            if what == "key":       # one block of keys
                q[..., 32:64] *= 2.0 ** -44
                sc[int(table[0, 3 + 200 // 16]), 200 % 16, 1, 1] += 40
            elif what == "values":  # one block of all values
                sc[..., S + 1] -= 40
            elif what == "last":    # ... of a sequence's last key
                j = seqs[0][1] - 1
                sc[int(table[0, 3 + j // 16]), j % 16, :, S] -= 40
            elif what == "keys":
                q[..., :32] *= 2.0 ** 40
                sc[..., 0] -= 40
            else:
                kv.view(torch.uint8)[..., 32 * bits // 8:64 * bits // 8] = 0
                sc[..., 1] = 27
            want, mag, wgt = P.attention(q, M.values(kv, sc, bits), table.tolist(), D ** -0.5)
            size = float(mag.max())
            for how in ways(n_shared):
                print(what, bits, D, nq, n_shared, how, flush=True)
                got = be.flash_attn_paged(q.cuda(), kv.cuda(), table.cuda(), scale=D ** -0.5, n_shared=n_shared, max_q=nq, scales=sc.cuda()).cpu()
                off, n = ((x.double().unflatten(-1, (D // 32, 32)).pow(2).sum((0, 1, 3)).sqrt()) for x in (got.double() - want, want))
                assert (off <= (5 * 2.0 ** -22 + 2.0 ** -24 * size) * n).all(), (off / n).tolist()


@BITS
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("what", ["key", "value", "weak"])
@pytest.mark.parametrize("late", [1859, 1210, 701])
def test_one_key_far_into_the_keys(be, D, late, what, bits):
    """A workgroup goes through many tiles before the one key whose block is far from all others in size,
    (key) one of q's small channels draws nearly all weight to it, (value, weak) it has next to none and most of
    the output."""
    seqs = [(40, 1900), (40, 1700)] + [(1, 5)] * 30
    q, kv, sc, table = make(seqs, 8, 8, D, bits, 16, seed=9)
    S = M.scale_bytes(D)
    at = int(table[0, 3 + late // 16]), late % 16
    u = kv.view(torch.uint8)
    if what == "key":
        lo, hi = {8: (106, 128), 4: (110, 132)}[bits]
        sc[..., :S] = lo
        sc[at][:, 1] = hi
        q *= 2.0 ** (HOME[bits] - lo)
        # (as large as they may be towards the key's codes)
        c = M.values(kv, sc, bits)[at][:, 32:64].float() * 2.0 ** (HOME[bits] - hi)
        g = torch.Generator().manual_seed(3)
        q[..., 32:64] = 8 * math.sqrt(D) / 32 * 2.0 ** (HOME[bits] - hi) * torch.sign(c) * (0.8 + 0.4 * torch.rand((q.shape[0], 8, 1), generator=g))
    else:
        u[..., :D * bits // 8] = 0
        u[at][:, 0] = {8: 0x7e, 4: 7}[bits]
        sc[..., :S] = 118
        q[..., 0] = -math.sqrt(D) / ({8: 448.0, 4: 6.0}[bits] * 2.0 ** -9)
        q[..., 0] *= (17.1 if what == "weak" else 13.2) * torch.linspace(1.0, 1.03, q.shape[0] * 8).view(-1, 8)
        if what == "value":
            lo, hi = {8: (106, 128), 4: (106, 136)}[bits]
            sc[..., S:] = lo
            sc[at][:, S:] = hi
        else:
            sc[..., S:] = HOME[bits]
            u[..., D * bits // 8:] = 0
            u[at][:, D * bits // 8:] = torch.randint(0, 128 if bits == 4 else 126, (8, D * bits // 8), generator=torch.Generator().manual_seed(2)).to(torch.uint8)
    run(be, q, kv, sc, table, bits, 40, 0, f"late {what} {late}")
