"""Appending to a quantized cache: every scale byte and every element's value for itself.

The rotation is off by t of a pair (test_gpu_kv_mx.py has the sum), so a key block's largest element is known to 2 t of
itself: its scale has to be one of the two that the largest elements 2 t smaller and larger have, which are the same but next
to a border.  An element's value is within half a step of its code, and 2 t of the block's largest, of the value in 64 bits.
Everything else is equal: values' scales and codes, rows of other heads, padding."""
import pytest

import mx_oracle as M
import paged_oracle as P
from test_gpu_kv_mx import rope_of, tokens

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def be():
    import ghip
    b = ghip.Backend(0)
    yield b
    b.close()


def steps(x, scale, bits):
    """how far a rounding to codes of these scales may move x: half a step; from 6 to 7 times the scale (4 bits) to 6"""
    z = (x / scale).abs()
    if bits == 8:
        low = torch.frexp(z)[1].clamp(min=-5) - 1  # the binade's power of two, 2^-6 for all below it
        half = M.two_to(low - 4)
    else:
        half = torch.where(z < 2, 0.25, torch.where(z < 4, 0.5, 1.0))
    return half.double() * scale


def check(be, bits, ty, T, H, D, mode, n, base=10000.0, start=0, sections=(0, 0, 0, 0), strided=False, layers=2, page=16):
    g = torch.Generator().manual_seed(7)
    k, v = tokens(T, H, D, ty, g, strided), tokens(T, H, D, ty, g, strided)
    pages = (T + page - 1) // page + 2
    whole = [M.cache(pages, page, H * layers, D, bits, g)[i].cuda() for i in (0, 1)]
    h0 = H * (layers - 1)
    kv, sc = (t[:, :, h0:] for t in whole)
    before = [t.cpu().clone() for t in whole]
    slots = torch.randperm(pages * page, generator=g)[:T]
    slots[T // 3::7] = -1 - slots[T // 3::7]
    slots[2 % T] = pages * page
    axes = 4 if sum(sections) else 1
    pos = (start + torch.arange(T) * 3 + 50 * torch.arange(axes).view(-1, 1)).to(torch.int32)
    print(f"append {bits} {ty} T={T} H={H} D={D} {mode} n={n} start={start}", flush=True)
    be.kv_append(k, v, slots.cuda(), kv, pos=pos.cuda() if axes > 1 else pos[0].cuda(), rope=rope_of(mode, n, base, sections), scales=sc)
    want, mag = P.rope(k.cpu(), pos, mode, n, base, sections, None)
    far = pos.double().abs().amax(0)
    t = (far * 3 * 2.0 ** -53 * 6.3 + 2.0 ** -43 * (far > 0)).view(T, 1, 1)
    t = torch.where((mag > 0).any(-1, keepdim=True), t, torch.zeros_like(t))

    got, gsc = M.unpack(whole[0].cpu(), bits).flatten(0, 1), whole[1].cpu().long().flatten(0, 1)
    wc, wsc = M.unpack(before[0], bits).flatten(0, 1), before[1].long().flatten(0, 1)
    S = M.scale_bytes(D)
    named = (slots >= 0) & (slots < pages * page)
    at = slots[named]
    # values, and all that no token names: equal
    c, sb, _ = M.encode(v.cpu().double(), bits)
    wc[at, h0:, D:], wsc[at, h0:, S:] = c[named], sb[named]
    mine = torch.zeros(wc.shape[0], dtype=torch.bool)
    mine[at] = True
    for a, b, width in ((got, wc, D), (gsc, wsc, S)):
        assert torch.equal(a[~mine], b[~mine]) and torch.equal(a[:, :h0], b[:, :h0]) and torch.equal(a[:, h0:, width:], b[:, h0:, width:])
    # keys: the scale of the block, or that of one 2 t smaller or larger
    _, less, _ = M.encode(want * (1 - 2 * t), bits)
    _, more, _ = M.encode(want * (1 + 2 * t), bits)
    ks = gsc[at][:, h0:, :S]
    assert ((ks == less[named]) | (ks == more[named])).all()
    assert (less == more).double().mean() > 0.98  # (16-bit keys at position 0 or past the pairs lie on a border now and then)
    val = M.decode(got[at][:, h0:], gsc[at][:, h0:], D, bits)[..., :D]
    w, scale = want[named], M.two_to(ks - 127)
    scale = scale.repeat_interleave(32, -1)[..., :D]
    big = torch.nn.functional.pad(w.abs(), (0, -D % 32)).unflatten(-1, (-1, 32)).amax(-1).repeat_interleave(32, -1)[..., :D]
    off = (val - w).abs()
    assert (off <= steps(w, scale, bits) + 2 * t[named] * big).all(), float((off / (steps(w, scale, bits) + 2 * t[named] * big)).max())


BITS = pytest.mark.parametrize("bits", [8, 4])


@BITS
@pytest.mark.parametrize("ty", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("mode,D,n,sections", [
    ("neox", 128, 128, (0, 0, 0, 0)), ("norm", 128, 128, (0, 0, 0, 0)), ("neox", 80, 20, (0, 0, 0, 0)), ("norm", 96, 22, (0, 0, 0, 0)),
    ("neox", 16, 16, (0, 0, 0, 0)), ("norm", 256, 250, (0, 0, 0, 0)), ("mrope", 128, 128, (16, 24, 24, 0)), ("vision", 80, 40, (20, 20, 0, 0)),
    ("imrope", 64, 64, (12, 10, 10, 0))])
def test_every_scale(be, mode, D, n, sections, ty, bits):
    check(be, bits, ty, 41, 3, D, mode, n, 500000.0, 9000, sections)


@BITS
@pytest.mark.parametrize("ty", ["f32", "f16", "bf16"])
def test_every_scale_of_four_heads_a_thread(be, ty, bits):
    for H in (4, 5, 7):
        check(be, bits, ty, 2600, H, 64, "neox", 64, start=100, layers=1)
        check(be, bits, ty, 2600, H, 64, "norm", 60, start=100, layers=1)
    check(be, bits, ty, 2600, 5, 80, "neox", 20, start=100, layers=1)


@BITS
def test_every_scale_far_positions_and_slices(be, bits):
    check(be, bits, "f32", 23, 2, 128, "neox", 128, 1e6, 2 ** 24)
    check(be, bits, "f32", 23, 2, 128, "norm", 128, 1e4, -500)
    check(be, bits, "bf16", 23, 2, 128, "norm", 128, strided=True)
    check(be, bits, "f32", 1, 1, 64, "neox", 64, start=5)
