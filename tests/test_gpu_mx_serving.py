"""The serving example over a quantized cache, step by step against 64 bits: prompts, shared
pages, generated tokens, a conversation forked inside a page."""
import os
import sys

import pytest

import mx_oracle as M
import paged_oracle as P

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu
sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))


@pytest.fixture(scope="module")
def be():
    import ghip
    b = ghip.Backend(0)
    yield b
    b.close()


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("window,n_first,head", [(0, 0, 128), (40, 4, 64)])
def test_serving(be, window, n_first, head, bits):
    import paged_serving as S
    layer, pages = S.make(be, window=window, n_first=n_first, head=head, bits=bits)
    D = layer.D

    def step(todo, n_shared=0):
        x = torch.randn((sum(n for _, n in todo), 1024), device="cuda")
        b = pages.batch(todo)
        y, q, o = layer(x, b, n_shared=n_shared)
        T = x.shape[0]
        values = M.values(layer.kv, layer.scales, bits)  # [pages, page, Hkv, 2 D]
        rows = values.flatten(0, 1)[b["slots"].cpu()]
        # what is read back: the codes' values; in 32 bits they are exact
        assert torch.equal(be.kv_read(layer.kv, b["slots"], layer.scales).cpu().double(), rows)
        # what was written: the projections, keys rotated, within half a step of their codes: of 1/8 (1/2) of their
        # binade, below the least normal one of 2^-9 (1/2) of the scale.  6 to 7 becomes 6: less than 1/4 of it.
        # (a product of three matrices in one launch may differ in its sum's last bits, 2^-20 of the key)
        sb = layer.scales.cpu().flatten(0, 1)[b["slots"].cpu()].long()
        S2 = sb.shape[-1] // 2
        for name, at in (("k", 0), ("v", 1)):
            raw = be.mul_mat(layer.w[name], layer.ty, 1024, x).view(T, layer.Hkv, D).cpu()
            if name == "k":
                want, mag = P.rope(raw, b["pos"].cpu().view(1, T), "neox", D, 500000.0)
            else:
                want, mag = raw.double(), raw.double().abs()
            scale = M.two_to(sb[..., at * S2:at * S2 + D // 32] - 127).repeat_interleave(32, -1)
            rel, least = (2.0 ** -4, 2.0 ** -10) if bits == 8 else (2.0 ** -2, 2.0 ** -2)
            off = (rows[..., at * D:(at + 1) * D] - want).abs()
            assert (off <= torch.maximum(rel * want.abs(), least * scale) + mag * 2.0 ** -19).all()
        want, mag, wgt = P.attention(q.cpu(), values, b["seqs"].tolist(), D ** -0.5, None, window, n_first)
        assert ((o.cpu().double() - want).abs() <= P.attention_tol(mag, wgt, D)).all()
        assert y.shape == (T, 1024) and torch.isfinite(y).all()

    pages.open("system")
    step([("system", 48)])
    for u in "abc":
        pages.open(u, like="system", shared=48)
    step([("a", 20), ("b", 1), ("c", 33)], n_shared=48)
    for _ in range(3):
        step([("c", 1), ("a", 1), ("b", 1)], n_shared=48)
    src, dst = pages.fork("d", "a", 60)
    assert len(src) == 12 and not set(src) & set(dst)
    layer.copy(src, dst)
    values = M.values(layer.kv, layer.scales, bits).flatten(0, 1)
    assert torch.equal(values[src], values[dst])
    step([("d", 1), ("a", 1)], n_shared=48)
    step([("a", 1), ("c", 5), ("d", 7)])
    step([("c", 30), ("d", 25)])
