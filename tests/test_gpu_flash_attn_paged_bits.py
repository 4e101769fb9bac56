"""How many bits ghip_flash_attn_paged keeps: against the formula in 64 bits, in
2-norm over a call's outputs.

q and p are held in 22 bits at least (two terms of 11 for F16, three of 8 for
BF16), a score's sum, 2^x and the row's sum in 24: five roundings of at most 2^-22
of what they round, which are what a value is off by where its scores are near the
row's largest.  A score that lies g powers of two below it is rounded at that
distance: 2^-24 g more.  (One term fewer of q or p is 2^-16 or more, 3e-6 in norm.)"""
import math

import pytest

import paged_oracle as P
from test_gpu_flash_attn_paged import make, ways

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

NEAR = 5 * 2.0 ** -22


@pytest.fixture(scope="module")
def be():
    import ghip
    b = ghip.Backend(0)
    yield b
    b.close()


def check(be, q, kv, table, scale, gap=0.0, want=None, **kw):
    if want is None:
        want, _, _ = P.attention(q, kv, table.tolist(), scale)
    for how in ways(kw.get("n_shared", 0)):
        got = be.flash_attn_paged(q.cuda(), kv.cuda(), table.cuda(), scale=scale, max_q=int(table[:, 1].max()), **kw).cpu().double()
        off = torch.linalg.vector_norm(got - want) / torch.linalg.vector_norm(want)
        print(f"{tuple(q.shape)} {kv.dtype} {how} {kw}: {float(off):.2e}", flush=True)
        assert off <= NEAR + 2.0 ** -24 * gap, (how, float(off))


@pytest.mark.parametrize("ctype", ["f16", "bf16"])
@pytest.mark.parametrize("H,Hkv,D", [(8, 2, 128), (4, 4, 64), (3, 1, 96), (2, 1, 256)])
@pytest.mark.parametrize("seqs,n_shared", [([(1, 900), (1, 33)], 0), ([(40, 300), (3, 200)], 0), ([(1, 700), (1, 660), (1, 690)], 640)])
def test_every_term_counts(be, seqs, n_shared, H, Hkv, D, ctype):
    q, kv, table = make(seqs, H, Hkv, D, ctype, 16, n_shared)
    check(be, q, kv, table, D ** -0.5, n_shared=n_shared)


@pytest.mark.parametrize("ctype", ["f16", "bf16"])
@pytest.mark.parametrize("nq,keys", [(1, 300), (5, 700), (40, 300)])
@pytest.mark.parametrize("nats", [6, 12, 18, 40])
def test_first_key_that_draws_the_weight(be, nats, nq, keys, ctype):
    """One key far above the others, its value 0: the others, e^-nats each, make the output."""
    H, Hkv, D = 4, 2, 64
    q, kv, table = make([(nq, keys)], H, Hkv, D, ctype, 16)
    u = torch.randn(D, generator=torch.Generator().manual_seed(9))
    u /= u.norm()
    q += 8 * u - (q @ u)[..., None] * u  # every row has 8 along u, and the other keys nothing
    for j in range(keys):
        k = kv[int(table[0, 3 + j // 16]), j % 16, :, :D]
        k.copy_(k.float() - (k.float() @ u)[:, None] * u + (0 if j else nats / (8 * D ** -0.5)) * u)
    kv[int(table[0, 3]), 0, :, D:] = 0
    check(be, q, kv, table, D ** -0.5, gap=nats / math.log(2) + 16)


def test_weight_that_moves_down_and_up(be):
    """Runs of keys whose scores step up and down by up to 2^60."""
    H, Hkv, D = 4, 2, 64
    for nq in (1, 30):
        q, kv, table = make([(nq, 1500)], H, Hkv, D, "f16", 16)
        u = torch.randn(D, generator=torch.Generator().manual_seed(9))
        u /= u.norm()
        q += 8 * u - (q @ u)[..., None] * u
        for j in range(1500):
            rows = kv[int(table[0, 3 + j // 16]), j % 16]
            at = (40, 0, 20, -2, 39, 1, 30)[j // 64 % 7]
            rows[:, :D] = (rows[:, :D].float() - (rows[:, :D].float() @ u)[:, None] * u + at * u).half()
            if at > 1:
                rows[:, D:] = 0
        check(be, q, kv, table, D ** -0.5, gap=76)


@pytest.mark.parametrize("ctype", ["f16", "bf16"])
@pytest.mark.parametrize("nq", [1, 40])
@pytest.mark.parametrize("of_q,of_k", [(0.1, 10.0), (1e-2, 100.0), (1e-4, 1e4), (1e-30, 1.0), (1e6, 1e-6), (3e4, 1e-4)])
def test_sizes_of_q(be, of_q, of_k, nq, ctype):
    q, kv, table = make([(nq, 300)], 4, 2, 64, ctype, 16)
    kv[..., :64] *= of_k
    check(be, q * of_q, kv, table, 0.125)


@pytest.mark.parametrize("ctype", ["f16", "bf16"])
@pytest.mark.parametrize("nq", [1, 40])
def test_channels_of_different_size(be, nq, ctype):
    """Strong channels of q against weak ones of the keys, each adding as much to a score."""
    for D in (64, 128, 256):
        q, kv, table = make([(nq, 300)], 4, 2, D, ctype, 16)
        size = 10.0 ** torch.linspace(-2, 2, D)
        kv[..., :D] = (kv[..., :D].float() / size).to(kv.dtype)
        check(be, q * size, kv, table, D ** -0.5)


@pytest.mark.parametrize("ctype", ["f16", "bf16"])
def test_rows_of_different_size(be, ctype):
    for nq in (3, 40):
        q, kv, table = make([(nq, 300)], 4, 2, 128, ctype, 16)
        check(be, q * 10.0 ** -(torch.arange(nq * 4).view(nq, 4, 1) % 7), kv, table, 128 ** -0.5)
