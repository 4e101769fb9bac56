"""Infinities and NaN among the keys and values of ghip_flash_attn_paged's cache:
what the formula gives for them, whatever tile or split they lie in."""
import math

import pytest

import paged_oracle as P
from test_gpu_flash_attn_paged import compare, make, ways

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu
INF, NAN = math.inf, math.nan


@pytest.fixture(scope="module")
def be():
    import ghip
    b = ghip.Backend(0)
    yield b
    b.close()


def expect(be, seqs, H, Hkv, D, ctype, put, n_shared=0, window=0, n_first=0):
    """put(rows of the cache by (sequence, key)): where infinities and NaN go; the
    elements that the formula leaves finite are compared, the others have to be the
    same infinity or NaN"""
    q, kv, table = make(seqs, H, Hkv, D, ctype, 16, n_shared)
    put(lambda b, j: kv[int(table[b, 3 + j // 16]), j % 16], q)
    want, mag, wgt = P.attention(q, kv, table.tolist(), D ** -0.5, None, window, n_first)
    finite = torch.isfinite(want)
    mag = torch.where(torch.isfinite(mag), mag, torch.full_like(mag, 30.0))
    for how in ways(n_shared):
        print(f"odd {seqs} H={H}/{Hkv} D={D} {ctype} shared={n_shared} window={window} {how}", flush=True)
        got = be.flash_attn_paged(q.cuda(), kv.cuda(), table.cuda(), scale=D ** -0.5, n_shared=n_shared, window=window, n_first=n_first,
                                  max_q=max(n for n, _ in seqs)).cpu().double()
        assert torch.equal(torch.isnan(got), torch.isnan(want))
        assert torch.equal(got[~finite].nan_to_num(5.0), want[~finite].nan_to_num(5.0))
        tol = P.attention_tol(mag, torch.where(finite, wgt, torch.zeros_like(wgt)), D)
        assert ((got - want).abs().expand_as(got)[finite] <= tol.expand_as(got)[finite]).all()


SIZES = [(4, 2, 64), (8, 2, 128), (3, 1, 96), (2, 1, 256)]


@pytest.mark.parametrize("ctype", ["f16", "bf16"])
@pytest.mark.parametrize("H,Hkv,D", SIZES)
@pytest.mark.parametrize("nq", [1, 3, 40])
def test_values(be, nq, H, Hkv, D, ctype):
    def put(at, q):
        at(0, 7)[:, D + 3] = INF                  # every row sees it
        at(0, 100)[:, D + 4] = -INF
        at(0, 9)[:, D + 5], at(0, 130)[:, D + 5] = INF, -INF
        at(0, 64)[:, D + 6] = NAN
        at(0, 198)[:, D + 1] = INF                # among the last rows' own keys
        at(0, 199)[:, D + 2] = -INF
        at(1, 60)[0, D:] = INF
    expect(be, [(nq, 200), (nq, 90)], H, Hkv, D, ctype, put)
    expect(be, [(nq, 200), (nq, 90)], H, Hkv, D, ctype, put, window=120, n_first=8)
    expect(be, [(nq, 200), (nq, 120)], H, Hkv, D, ctype, put, n_shared=80)


@pytest.mark.parametrize("ctype", ["f16", "bf16"])
@pytest.mark.parametrize("H,Hkv,D", SIZES)
@pytest.mark.parametrize("nq", [1, 3, 40])
def test_keys(be, nq, H, Hkv, D, ctype):
    """A key with an infinite element scores an infinity for every row: without weight
    where it is the lower one, NaN where it is the upper one or both come together."""
    def put(at, q):
        q[:, :, 1], q[:, :, 2] = q[:, :, 1].abs(), q[:, :, 2].abs()
        at(0, 7)[:, 1] = -INF
        at(0, 150)[0, 2] = -INF
        at(0, 199)[:, 1] = -INF
        at(1, 30)[0, 1] = INF
    expect(be, [(nq, 200), (nq, 90)], H, Hkv, D, ctype, put)

    def both(at, q):
        q[:, :, 1], q[:, :, 2] = q[:, :, 1].abs(), -q[:, :, 2].abs()
        at(0, 50)[:, 1] = at(0, 50)[:, 2] = -INF
        at(1, 20)[:, 1], at(1, 20)[:, 2] = -INF, INF
        at(2, 60)[:, 3] = NAN
    expect(be, [(nq, 200), (nq, 90), (nq, 70)], H, Hkv, D, ctype, both)


# sizes where several rows at different positions share a workgroup of up to 16

@pytest.mark.parametrize("nq", [2, 3, 4])
@pytest.mark.parametrize("what", [INF, NAN])
def test_few_rows_and_what_they_do_not_see(be, nq, what):
    import test_gpu_flash_attn_paged as A
    A.test_what_unseen_places_hold(be, nq, what)


@pytest.mark.parametrize("n_shared", [0, 32])
@pytest.mark.parametrize("nq", [3, 8])
def test_few_rows_and_missing_pages(be, nq, n_shared):
    import test_gpu_flash_attn_paged as A
    A.test_bad_pages_give_nan(be, nq, n_shared)


@pytest.mark.parametrize("ctype", ["f16", "bf16"])
@pytest.mark.parametrize("H,Hkv,D,nq", [(4, 2, 64, 8), (3, 1, 96, 5), (8, 2, 128, 4), (2, 2, 256, 16), (1, 1, 8, 3)])
def test_few_rows_and_later_values(be, H, Hkv, D, nq, ctype):
    """Values of the last keys, which only some of the rows see."""
    def put(at, q):
        for i, x in enumerate((INF, -INF, NAN)):
            at(0, 100 - nq + 1 + i % (nq - 1))[:, D + i] = x
            at(1, 200 - 1 - i % nq)[:, D + 3 + i] = x
    expect(be, [(nq, 100), (nq, 200)], H, Hkv, D, ctype, put)
    expect(be, [(nq, 100), (nq, 200)], H, Hkv, D, ctype, put, window=50, n_first=3)
