"""ghip_flash_attn_paged_mx against attention's formula in 64 bits over the values
that a quantized cache's codes stand for (mx_oracle, paged_oracle).  A code's
value is a bfloat16 (of most caches a float16 too), so the bounds are those of such a cache: every element
within attention_tol, and the whole within 5 * 2^-22 in 2-norm (q and p as three
terms of 8 bits or two of 11, a score's sum, 2^x and the row's sum in 24: five roundings of at most 2^-22) for
scores of about 1.  A score of size s is a 32-bit number too, whose last place is 2^-24 s:
that much of its p, and of what the row sums, 2^-24 s is added for the largest s
(these caches' scales spread over 2^6, scores reach 40)."""
import math

import pytest

import mx_oracle as M
import paged_oracle as P
import test_gpu_flash_attn_paged as A
from test_gpu_flash_attn_paged import ways

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu
NAN = math.nan


@pytest.fixture(scope="module")
def be():
    import ghip
    b = ghip.Backend(0)
    yield b
    b.close()


def make(seqs, H, Hkv, D, bits, page, n_shared=0, seed=0, order=None):
    """A.make's batch with a quantized cache -> q, codes, scales, table"""
    q, kv, table = A.make(seqs, H, Hkv, D, "bf16", page, n_shared, seed, order=order)
    g = torch.Generator().manual_seed(seed + 7)
    codes, sc = M.cache(*kv.shape[:3], D, bits, g)
    common, rest = divmod(n_shared, page)
    if rest:  # the cut page's rows, copied for each
        for b in range(1, len(seqs)):
            if seqs[b][1] > common * page:
                for t in (codes.view(torch.uint8), sc):
                    t[table[b, 3 + common].long(), :rest] = t[table[0, 3 + common].long(), :rest]
    return q, codes, sc, table


def compare(got, want, mag, wgt, D):
    A.compare(got, want, mag, wgt, D)
    named = ~torch.isnan(want)
    n, off = torch.linalg.vector_norm(want[named]), torch.linalg.vector_norm((got.double() - want)[named])
    size = float(mag[torch.isfinite(mag)].max()) if mag.numel() else 0.0
    assert off <= (5 * 2.0 ** -22 + 2.0 ** -24 * size) * n, float(off / n)


def check(be, seqs, H, Hkv, D, bits, page=16, window=0, n_first=0, n_shared=0, sinks=False, seed=0, max_q=None, order=None):
    q, codes, sc, table = make(seqs, H, Hkv, D, bits, page, n_shared, seed, order)
    sk = torch.randn(H, generator=torch.Generator().manual_seed(seed + 1)) if sinks else None
    scale = 1 / math.sqrt(D)
    want, mag, wgt = P.attention(q, M.values(codes, sc, bits), table.tolist(), scale, sk, window, n_first)
    print(f"mx{bits} {seqs[:4]} H={H}/{Hkv} D={D} page={page} window={window}+{n_first} shared={n_shared} sinks={sinks}", flush=True)
    for how in ways(n_shared):
        got = be.flash_attn_paged(q.cuda(), codes.cuda(), table.cuda(), scale=scale, sinks=sk.cuda() if sinks else None, window=window,
                                  n_first=n_first, n_shared=n_shared, max_q=max_q or max([a for a, _ in seqs] + [1]), scales=sc.cuda())
        compare(got.cpu(), want, mag, wgt, D)


BITS = pytest.mark.parametrize("bits", [8, 4])


@BITS
@pytest.mark.parametrize("H,Hkv,D", [(8, 2, 64), (8, 2, 128), (5, 1, 80), (4, 4, 96), (16, 1, 64), (6, 2, 256), (3, 1, 16), (2, 2, 112), (2, 1, 32),
                                     (2, 1, 48), (1, 1, 144), (2, 1, 240)])
@pytest.mark.parametrize("page", [1, 16, 24, 64, 256])
def test_decode(be, H, Hkv, D, page, bits):
    check(be, [(1, 1), (1, 63), (1, 64), (1, 65), (1, 700), (1, 17)], H, Hkv, D, bits, page)


@BITS
@pytest.mark.parametrize("H,Hkv,D", [(4, 1, 128), (2, 2, 64), (3, 1, 80), (2, 1, 256), (10, 2, 64), (2, 1, 16), (2, 1, 176), (2, 1, 48)])
def test_prompts(be, H, Hkv, D, bits):
    check(be, [(33, 33), (70, 200), (1, 90), (17, 300), (2, 2)], H, Hkv, D, bits, 16)


@BITS
@pytest.mark.parametrize("H,Hkv,D,nq", [(4, 2, 64, 8), (3, 1, 96, 5), (8, 2, 128, 4), (2, 2, 256, 16), (1, 1, 16, 3), (4, 1, 128, 6)])
def test_drafted_tokens(be, H, Hkv, D, nq, bits):
    """A few new rows of each sequence, as many as 16 rows of a KV head and a little over."""
    check(be, [(nq, nq), (nq - 1, 500), (1, 77), (nq, 131)], H, Hkv, D, bits, 24)


@BITS
@pytest.mark.parametrize("window,n_first", [(1, 0), (7, 0), (64, 4), (100, 1), (100, 130), (64, 64), (1, 1), (5000, 4)])
@pytest.mark.parametrize("nq", [1, 9, 40])
def test_window(be, window, n_first, nq, bits):
    check(be, [(nq, nq), (nq, 64 + nq), (nq, 257), (nq, 400), (nq, nq + 1)], 8, 2, 64, bits, 16, window, n_first, sinks=True)


@BITS
@pytest.mark.parametrize("n_shared,page", [(1, 16), (64, 64), (200, 16), (333, 24), (300, 1), (320, 64)])
def test_shared_prefix(be, n_shared, page, bits):
    lens = [n_shared + 1, n_shared + 63, n_shared + 200, n_shared + 7, n_shared + 64]
    check(be, [(1, n) for n in lens], 8, 2, 128, bits, page, n_shared=n_shared)
    check(be, [(1, n) for n in lens], 16, 1, 64, bits, page, n_shared=n_shared, sinks=True)
    check(be, [(min(n, 1 + 5 * i), n) for i, n in enumerate(lens)], 4, 1, 80, bits, page, n_shared=n_shared)
    check(be, [(1, n) for n in lens[:3]], 4, 1, 256, bits, page, n_shared=n_shared)


@BITS
def test_shared_prefix_of_rows_inside_it(be, bits):
    check(be, [(20, 150), (40, 130), (5, 80), (128, 128)], 4, 2, 64, bits, n_shared=128)
    check(be, [(1, 128), (1, 30), (1, 129), (1, 1)], 4, 2, 64, bits, n_shared=128)
    check(be, [(20, 250), (40, 230), (1, 180)], 4, 2, 64, bits, window=70, n_first=5, n_shared=160)
    check(be, [(1, 250), (1, 230), (1, 180)], 4, 2, 64, bits, window=70, n_first=5, n_shared=160, sinks=True)
    check(be, [(1, 30), (1, 100), (1, 150), (1, 97)], 16, 4, 64, bits, n_shared=96)


@BITS
def test_long_keys(be, bits):
    """Enough keys that one row's are split over workgroups and joined."""
    check(be, [(1, 9000), (1, 100), (1, 5000)], 8, 2, 128, bits, 64)
    check(be, [(1, 9000), (1, 8300), (1, 8200)], 4, 1, 64, bits, 64, n_shared=8192)
    check(be, [(3, 6000), (1, 6100)], 4, 4, 128, bits, 64, window=5000, n_first=100)
    check(be, [(20, 6000), (1, 100)], 4, 2, 256, bits, 64)


@BITS
def test_any_order_of_rows_and_idle_slots(be, bits):
    check(be, [(3, 40), (0, 0), (20, 60), (0, 30), (1, 5)], 4, 2, 64, bits, order=[4, 2, 3, 0, 1])
    check(be, [(1, 40), (0, 90), (1, 60), (1, 100)], 4, 2, 64, bits, n_shared=32, order=[3, 2, 0, 1])
    check(be, [(1 if 30 <= b < 34 else 0, 101 + b % 7) for b in range(40)], 16, 1, 64, bits, n_shared=96)


@BITS
@pytest.mark.parametrize("nq", [1, 30])
def test_rows_that_see_nothing(be, nq, bits):
    for sinks in (False, True):
        check(be, [(nq, 0), (nq, nq), (2 * nq + 3, nq)], 4, 2, 64, bits, sinks=sinks)


@BITS
def test_rows_outside_the_table_are_kept(be, bits):
    q, kv, sc, table = make([(2, 30), (3, 20)], 4, 2, 64, bits, 16)
    q = torch.cat([q, torch.randn((4, 4, 64))])
    for max_q, kept in ((3, 5), (2, 4)):
        out = torch.full(q.shape, 7.0).cuda()
        be.flash_attn_paged(q.cuda(), kv.cuda(), table.cuda(), scale=0.125, max_q=max_q, out=out, scales=sc.cuda())
        assert (out[kept:] == 7).all() and not (out[:kept] == 7).any()


@BITS
@pytest.mark.parametrize("nq", [1, 3, 5, 40])
def test_what_unseen_places_hold(be, nq, bits):
    """NaN blocks in the rows of a page past the last key, in keys before the window, in pages of
    no sequence; pages before the window are gone."""
    for window, n_first, n_shared in [(0, 0, 0), (50, 4, 0), (0, 0, 64)]:
        seqs = [(nq, 150), (nq, 201), (nq, 97)]
        q, kv, sc, table = make(seqs, 8, 2, 64, bits, 16, n_shared)
        want, mag, wgt = P.attention(q, M.values(kv, sc, bits), table.tolist(), 0.125, None, window, n_first)
        seen = torch.zeros(kv.shape[:2], dtype=torch.bool)
        for b, (n, m) in enumerate(seqs):
            for j in range(m):
                if any(j <= p and (not window or j > p - window or j < n_first) for p in range(m - n, m)):
                    seen[table[b, 3 + j // 16].long(), j % 16] = True
        sc[~seen] = 255
        kv.view(torch.uint8)[~seen] = 255
        gone = table.clone()
        for b, (n, m) in enumerate(seqs):
            for i in range((m + 15) // 16):
                if not seen[table[b, 3 + i].long()].any():
                    gone[b, 3 + i] = 10 ** 6
        for how in ways(n_shared):
            got = be.flash_attn_paged(q.cuda(), kv.cuda(), gone.cuda(), scale=0.125, window=window, n_first=n_first, n_shared=n_shared,
                                      max_q=nq, scales=sc.cuda())
            compare(got.cpu(), want, mag, wgt, 64)


@BITS
@pytest.mark.parametrize("H,Hkv,D", [(4, 2, 64), (8, 2, 128), (3, 1, 96), (2, 1, 256)])
@pytest.mark.parametrize("nq", [1, 3, 40])
def test_nan_blocks(be, nq, H, Hkv, D, bits):
    """A key's NaN block makes the rows that see it NaN, a value's its 32 elements of theirs; rows
    before it, and with it out of the window, are as they would be."""
    S = M.scale_bytes(D)
    for window, n_first, n_shared, lens in ((0, 0, 0, (200, 90)), (120, 8, 0, (200, 90)), (0, 0, 80, (200, 120))):
        seqs = [(nq, n) for n in lens]
        q, kv, sc, table = make(seqs, H, Hkv, D, bits, 16, n_shared)
        at = lambda b, j: sc[int(table[b, 3 + j // 16]), j % 16]
        at(0, 7)[:, S] = 255                      # every row sees it (under the window: as a first key)
        at(0, 100)[0, S + (D - 1) // 32] = 255
        at(0, 198)[:, S + (1 if D > 32 else 0)] = 255  # among the last rows' own keys
        at(1, lens[1] - 1)[0, 0] = 255
        want, mag, wgt = P.attention(q, M.values(kv, sc, bits), table.tolist(), D ** -0.5, None, window, n_first)
        nan = torch.isnan(want)
        assert nan.any() and (not nan.all() or (D == 96 and nq == 1))  # (there the three blocks are all of it)
        for how in ways(n_shared):
            got = be.flash_attn_paged(q.cuda(), kv.cuda(), table.cuda(), scale=D ** -0.5, n_shared=n_shared, window=window, n_first=n_first,
                                      max_q=nq, scales=sc.cuda()).cpu().double()
            assert torch.equal(torch.isnan(got), nan)
            mag = torch.where(torch.isfinite(mag), mag, torch.full_like(mag, 30.0))
            tol = P.attention_tol(mag, torch.where(nan, torch.zeros_like(wgt), wgt), D)
            assert ((got - want).abs()[~nan] <= tol.expand_as(got)[~nan]).all()


@BITS
@pytest.mark.parametrize("nq", [1, 40])
def test_strides(be, nq, bits):
    """q inside a wider projection, dst, codes and scales with gaps and in another order of axes."""
    seqs = [(nq, 77), (nq, 130)]
    for D in (64, 80, 128):
        q, kv, sc, table = make(seqs, 4, 2, D, bits, 16)
        want, mag, wgt = P.attention(q, M.values(kv, sc, bits), table.tolist(), 0.125)
        wide = torch.full((q.shape[0], 7, D + 7), 9.0)
        wide[:, 1:5, 5:D + 5] = q
        out = torch.full((q.shape[0], 5, D + 16), 7.0).cuda()
        turned = lambda t: t.permute(0, 2, 1, 3).contiguous().cuda().permute(0, 2, 1, 3)  # [pages, H_kv, page, ..] in memory
        gaps = torch.full((kv.shape[0], 16, 3, kv.shape[3] + 32), 255, dtype=torch.uint8)
        gaps[:, :, 1:, 16:16 + kv.shape[3]] = kv.view(torch.uint8)
        gapped = gaps.cuda()[:, :, 1:, 16:16 + kv.shape[3]].view(kv.dtype)
        S2 = sc.shape[3]
        sgaps = torch.full((kv.shape[0], 17, 2, 3 * S2), 255, dtype=torch.uint8)
        sgaps[:, 1:, :, S2:2 * S2] = sc
        wt = torch.full((2, table.shape[1] + 4), -1, dtype=torch.int32)
        wt[:, :table.shape[1]] = table
        for k, s in ((turned(kv.view(torch.uint8)).view(kv.dtype), turned(sc)), (gapped, sgaps.cuda()[:, 1:, :, S2:2 * S2])):
            for how in ways(0):
                out.fill_(7.0)
                be.flash_attn_paged(wide.cuda()[:, 1:5, 5:D + 5], k, wt.cuda()[:, :table.shape[1]], scale=0.125, max_q=nq, out=out[:, :4, 8:D + 8],
                                    scales=s)
                got = out.cpu()
                compare(got[:, :4, 8:D + 8], want, mag, wgt, D)
                got[:, :4, 8:D + 8] = 7.0
                assert (got == 7.0).all()


@BITS
def test_blocks_of_every_size(be, bits):
    """Scales from 2^-60 to 2^60 beside one another; scores far apart."""
    for nq, D in ((1, 128), (33, 128), (1, 64), (20, 256)):
        q, kv, sc, table = make([(nq, 500)], 4, 2, D, bits, 16)
        S = M.scale_bytes(D)
        sc[..., S:] = (sc[..., S:].long() + torch.randint(-60, 60, sc[..., S:].shape)).to(torch.uint8)
        q *= 6
        want, mag, wgt = P.attention(q, M.values(kv, sc, bits), table.tolist(), 0.125)
        for how in ways(0):
            got = be.flash_attn_paged(q.cuda(), kv.cuda(), table.cuda(), scale=0.125, max_q=nq, scales=sc.cuda()).cpu().double()
            # (a p, or a term of it, below 2^-126 of the largest is 0 in 32 bits, beside values of up to 2^66)
            under = 500 * 2.0 ** -125 * M.values(kv, sc, bits)[..., D:].abs().max()
            assert ((got - want).abs() <= P.attention_tol(mag, wgt, D) + under).all()
        # keys of very different size against channels of q that undo it
        q, kv, sc, table = make([(nq, 300)], 4, 2, D, bits, 16)
        size = 2.0 ** (torch.arange(D) // 32 * 9 - 12)
        q = q / size
        sc[..., :S] = (sc[..., :S].long() + torch.arange(S) * 9 - 12).to(torch.uint8)
        want, mag, wgt = P.attention(q, M.values(kv, sc, bits), table.tolist(), D ** -0.5)
        for how in ways(0):
            got = be.flash_attn_paged(q.cuda(), kv.cuda(), table.cuda(), scale=D ** -0.5, max_q=nq, scales=sc.cuda())
            compare(got.cpu(), want, mag, wgt, D)


@BITS
def test_equal_calls_give_equal_bits(be, bits):
    for seqs, sh in (([(1, 5000), (1, 4990)], 4096), ([(40, 900), (3, 700)], 512), ([(1, 3000)], 0)):
        q, kv, sc, table = make(seqs, 8, 2, 128, bits, 64, sh)
        for how in ways(sh):
            a = [be.flash_attn_paged(q.cuda(), kv.cuda(), table.cuda(), scale=0.1, n_shared=sh, max_q=max(n for n, _ in seqs), scales=sc.cuda())
                 for _ in range(4)]
            assert all(torch.equal(a[0], x) for x in a[1:])


def test_nothing_to_do(be):
    import ghip
    kv, sc = ghip.mx_cache(2, 4, 1, 64, 8)
    t = torch.zeros((0, 5), dtype=torch.int32, device="cuda")
    q = torch.ones((3, 2, 64), device="cuda")
    out = torch.full_like(q, 5)
    be.flash_attn_paged(q, kv, t, out=out, scales=sc)
    assert (out == 5).all()
    assert be.flash_attn_paged(q[:0], kv, torch.zeros((1, 5), dtype=torch.int32, device="cuda"), scales=sc).shape == (0, 2, 64)


@BITS
@pytest.mark.parametrize("rows", [1, 9, 70])
def test_cache_without_pages(be, rows, bits):
    import ghip
    for n_shared in (0, 20):
        flat = torch.randn(2 * rows * 4 * 64 + 3, device="cuda")
        q = flat[3:].view(2 * rows, 4, 64)
        kv, sc = ghip.mx_cache(0, 16, 2, 64, bits)
        seqs = torch.tensor([[0, rows, rows, 0, 1], [rows, rows, rows // 2, 5, -1]], dtype=torch.int32, device="cuda")
        for sinks in (None, torch.zeros(4, device="cuda")):
            got = be.flash_attn_paged(q, kv, seqs, sinks=sinks, n_shared=n_shared, max_q=rows, scales=sc).cpu()
            torch.cuda.synchronize()
            first = rows + rows - rows // 2
            assert torch.isnan(got[:rows]).all() and torch.isnan(got[first:]).all() and (got[rows:first] == 0).all()


@BITS
def test_far_pages(be, bits):
    """Keys past 2^32 bytes of codes, scales past 2^31."""
    import ghip
    D, Hkv, page = 128, 8, 64
    pages = 36000 * 8 // bits  # 4.7 GB
    kv, sc = ghip.mx_cache(pages, page, Hkv, D, bits)
    far = torch.tensor([pages - 1, 3, pages - 500, pages // 2], dtype=torch.int32)
    g = torch.Generator().manual_seed(3)
    codes, scales = M.cache(4, page, Hkv, D, bits, g)
    kv.view(torch.uint8)[far.long().cuda()] = codes.view(torch.uint8).cuda()
    sc[far.long().cuda()] = scales.cuda()
    small = M.values(codes, scales, bits)
    for nq in (1, 20):
        q = torch.randn((nq, 16, D), generator=g)
        head = torch.tensor([0, nq, 250], dtype=torch.int32)
        want, mag, wgt = P.attention(q, small, [torch.cat([head, torch.arange(4)]).tolist()], 0.088)
        got = be.flash_attn_paged(q.cuda(), kv, torch.cat([head, far]).view(1, -1).cuda(), scale=0.088, scales=sc)
        compare(got.cpu(), want, mag, wgt, D)
    slots = (far.long() * page + torch.tensor([1, 63, 0, 5])).cuda()
    back = be.kv_read(kv, slots, sc).cpu()
    assert torch.equal(back.double(), small[torch.arange(4), torch.tensor([1, 63, 0, 5])])
    be.kv_append(back[..., D:].cuda(), back[..., :D].cuda(), slots.flip(0), kv, scales=sc)
    again = be.kv_read(kv, slots.flip(0), sc).cpu()
    assert torch.equal(again, torch.cat([back[..., D:], back[..., :D]], -1))


@BITS
@pytest.mark.parametrize("nq,n_shared", [(1, 0), (1, 64), (24, 0)])
def test_graph_replays_follow_the_table(be, nq, n_shared, bits):
    """Captured once for the largest lengths, with append and read beside it; replays with other
    lengths, pages, rows and codes, and eager calls between them."""
    H, Hkv, D, page, per, B = 8, 2, 64, 16, 80, 4
    g = torch.Generator().manual_seed(1)
    kv, sc = (t.cuda() for t in M.cache(400, page, Hkv, D, bits, g))
    q = torch.randn((B * nq, H, D), device="cuda")
    k, v = (torch.randn((B * nq, Hkv, D), device="cuda") for _ in range(2))
    slots = torch.zeros(B * nq, dtype=torch.int64, device="cuda")
    table = torch.zeros((B, 3 + per), dtype=torch.int32, device="cuda")

    def fill(seed):
        g = torch.Generator().manual_seed(seed)
        t = torch.zeros((B, 3 + per), dtype=torch.int32)
        perm = torch.randperm(400, generator=g).to(torch.int32)
        at = []
        for b in range(B):
            n = int(torch.randint(nq + n_shared + 80, per * page, (1,), generator=g))
            t[b, :3] = torch.tensor([b * nq, nq, n])
            t[b, 3:] = perm[b * per:(b + 1) * per]
            t[b, 3:3 + n_shared // page] = perm[:n_shared // page]
            at += [int(t[b, 3 + j // page]) * page + j % page for j in range(n - nq, n)]
        table.copy_(t)
        slots.copy_(torch.tensor(at))
        for x in (q, k, v):
            x.copy_(torch.randn(x.shape, generator=g))

    def call(o, rows):
        be.kv_append(k, v, slots, kv, scales=sc)
        be.kv_read(kv, slots, sc, out=rows)
        return be.flash_attn_paged(q, kv, table, scale=0.125, n_shared=n_shared, max_q=nq, out=o, scales=sc)

    for how in ways(n_shared):
        out, rows = torch.empty_like(q), torch.empty((B * nq, Hkv, 2 * D), device="cuda")
        fill(0)
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.stream(s):
            call(out, rows)
            torch.cuda.synchronize()
            with torch.cuda.graph(graph, stream=s):
                call(out, rows)
        for i in range(4):
            fill(i)
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            o2, r2 = torch.empty_like(out), torch.empty_like(rows)
            call(o2, r2)
            torch.cuda.synchronize()
            assert torch.equal(out, o2) and torch.equal(rows, r2), i


@BITS
@pytest.mark.parametrize("nq,n_shared", [(1, 0), (3, 0), (30, 0), (1, 32), (8, 32), (30, 32)])
def test_bad_pages_give_nan(be, nq, n_shared, bits):
    seqs = [(nq, 150), (nq, 100), (nq, 64)]
    q, kv, sc, table = make(seqs, 4, 2, 64, bits, 16, n_shared)
    want, mag, wgt = P.attention(q, M.values(kv, sc, bits), table.tolist(), 0.125)
    bad = table.clone()
    bad[0, 3 + 140 // 16] = kv.shape[0]
    bad[1, 3 + 96 // 16] = -1
    for how in ways(n_shared):
        got = be.flash_attn_paged(q.cuda(), kv.cuda(), bad.cuda(), scale=0.125, n_shared=n_shared, max_q=nq, scales=sc.cuda()).cpu()
        for b, first in ((0, 128), (1, 96), (2, 10 ** 6)):
            for i in range(nq):
                t, p = int(table[b, 0]) + i, seqs[b][1] - nq + i
                if p >= first:
                    assert torch.isnan(got[t]).all(), (b, i)
                else:
                    compare(got[t:t + 1], want[t:t + 1], mag[t:t + 1], wgt[t:t + 1], 64)
    # lengths and rows that do not fit: past the table, before or past q
    odd = table.clone()
    odd[0, 2] = 16 * (table.shape[1] - 3) + 5
    odd[1, 0] = q.shape[0]
    odd[2, 0] = -1
    for how in ways(n_shared):
        out = torch.full(q.shape, 7.0).cuda()
        be.flash_attn_paged(q.cuda(), kv.cuda(), odd.cuda(), scale=0.125, n_shared=n_shared, max_q=nq, out=out, scales=sc.cuda())
        out = out.cpu()
        assert torch.isnan(out[nq - 1]).all()
        assert (out[nq:] == 7).all()


@BITS
def test_workspace_of_the_caller(be, bits):
    """With a workspace of the size asked for, holding NaN, attention allocates nothing and gives the
    same bits; with less it is refused with a status.  Two streams take turns at it."""
    import ghip
    g = torch.Generator().manual_seed(2)
    q = torch.randn((6, 8, 128), generator=g).cuda()
    kv, sc = (t.cuda() for t in M.cache(300, 16, 2, 128, bits, g))
    seqs = torch.zeros((6, 3 + 200), dtype=torch.int32)
    for b in range(6):
        seqs[b, :3] = torch.tensor([b, 1, 3000 - b])
        seqs[b, 3:] = torch.randperm(300, generator=g)[:200]
    seqs = seqs.cuda()
    for kw in (dict(max_q=1), dict(max_q=1, window=1000), dict(max_q=3)):
        want = be.flash_attn_paged(q, kv, seqs, scale=0.09, scales=sc, **kw)
        torch.cuda.synchronize()
        need = be.flash_attn_paged_workspace(q, kv, seqs, scales=sc, **kw)
        if not need:
            continue
        own = ghip.Backend(0)
        own.set_workspace(torch.full((need // 4,), NAN, device="cuda").view(torch.uint8))
        assert torch.equal(own.flash_attn_paged(q, kv, seqs, scale=0.09, scales=sc, **kw), want)
        streams = [torch.cuda.Stream() for _ in range(2)]
        torch.cuda.synchronize()
        got = []
        for i in range(6):
            with torch.cuda.stream(streams[i % 2]):
                got.append(own.flash_attn_paged(q, kv, seqs, scale=0.09, scales=sc, **kw))
        torch.cuda.synchronize()
        assert all(torch.equal(x, want) for x in got)
        own.set_workspace(torch.empty(need - 1, dtype=torch.uint8, device="cuda"))
        with pytest.raises(ghip.GhipError, match="workspace"):
            own.flash_attn_paged(q, kv, seqs, scale=0.09, scales=sc, **kw)
        torch.cuda.synchronize()
        own.close()


@BITS
@pytest.mark.parametrize("D,nq", [(64, 150), (128, 150), (128, 40), (256, 40)])
def test_scales_out_of_half_precisions_range(be, D, nq, bits):
    """Tiles of rows are computed with as float16 where that holds a tile's blocks, else as bfloat16:
    a block out of its range in one split of the keys, in all of them, in a shared prefix, and
    blocks of zeros, whose scale is the least there is."""
    S = M.scale_bytes(D)
    for n_shared, seqs in ((0, [(nq, 5000), (20, 300)]), (256, [(nq, 900), (nq, 700)])):
        for what in ("key", "value", "values", "zeros", "keys"):
            q, kv, sc, table = make(seqs, 4, 2, D, bits, 16, n_shared, seed=5)
            at = lambda j: (int(table[0, 3 + j // 16]), j % 16)
            if what == "key":      # one block of keys, of 2^40 (the row's q there as small)
                q[..., 32:64] *= 2.0 ** -44
                sc[at(200)][1, 1] += 40
            elif what == "value":  # values of about 2^30 and 2^-20 in one block each
                sc[at(130)][0, S] += 30
                sc[at(201)][1, S + 1] -= 20
            elif what == "values":
                sc[..., S + 1] -= 40
            elif what == "keys":
                q[..., :32] *= 2.0 ** 40
                sc[..., 0] -= 40
            else:
                kv.view(torch.uint8)[..., 32 * bits // 8:64 * bits // 8] = 0
                kv.view(torch.uint8)[..., D * bits // 8:(D + 32) * bits // 8] = 0
                sc[..., 1], sc[..., S] = 27, 27
            want, mag, wgt = P.attention(q, M.values(kv, sc, bits), table.tolist(), D ** -0.5)
            print(what, D, nq, n_shared, flush=True)
            for how in ways(n_shared):
                got = be.flash_attn_paged(q.cuda(), kv.cuda(), table.cuda(), scale=D ** -0.5, n_shared=n_shared, max_q=nq, scales=sc.cuda()).cpu()
                assert ((got.double() - want).abs() <= P.attention_tol(mag, wgt, D)).all()


@BITS
@pytest.mark.parametrize("D,H,Hkv,nq", [(128, 4, 1, 1), (64, 8, 1, 2), (128, 16, 1, 1), (128, 4, 1, 7), (64, 5, 1, 4), (256, 4, 2, 1)])
def test_many_sequences_share_the_workgroups(be, D, H, Hkv, nq, bits):
    """More sequences than a wavefront has lanes, long and short ones, idle ones among them and at the
    end, whose splits go by length: a workspace full of NaN, rows no sequence has as they were."""
    import ghip
    page, B, pages = 16, 150, 400
    g = torch.Generator().manual_seed(9)
    kv, sc = M.cache(pages, page, Hkv, D, bits, g)
    lens = [3000 if b in (3, 70, 140) else 0 if b % 7 == 5 or b >= 145 else 1 + 13 * b % 190 for b in range(B)]
    table = torch.zeros((B, 3 + 190), dtype=torch.int32)
    rows = []
    for b, n in enumerate(lens):
        m = min(nq, n)
        table[b, :3] = torch.tensor([len(rows), m, n])
        table[b, 3:] = torch.randint(0, pages, (190,), generator=g)
        rows += [b] * m
    for few in (0, 90):  # all, and up to 64 of them
        t = table[few:]
        q = torch.randn((len(rows) + 3, H, D), generator=g)
        for window, n_first, sinks in ((0, 0, None), (1500, 5, torch.randn(H, generator=g))):
            want, mag, wgt = P.attention(q, M.values(kv, sc, bits), t.tolist(), D ** -0.5, sinks, window, n_first)
            print(D, H, nq, few, window, flush=True)
            kw = dict(scale=D ** -0.5, max_q=nq, window=window, n_first=n_first, scales=sc.cuda(), sinks=None if sinks is None else sinks.cuda())
            need = be.flash_attn_paged_workspace(q.cuda(), kv.cuda(), t.cuda(), scales=sc.cuda(), max_q=nq, window=window, n_first=n_first)
            own = ghip.Backend(0)
            if need:
                own.set_workspace(torch.full((need // 4,), NAN, device="cuda").view(torch.uint8))
            out = torch.full(q.shape, 7.0).cuda()
            own.flash_attn_paged(q.cuda(), kv.cuda(), t.cuda(), out=out, **kw)
            got = out.cpu()
            own.close()
            first, last = int(t[0, 0]), len(rows)
            assert (got[:first] == 7).all() and (got[last:] == 7).all()
            compare(got[first:last], want[first:last], mag[first:last], wgt[first:last], D)


@BITS
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("nq,H", [(17, 1), (6, 4), (8, 4), (31, 1), (4, 8)])
def test_up_to_32_rows_of_a_head(be, nq, H, D, bits):
    """Two tiles of 16 rows in a wavefront: long keys in splits, windows, idle sequences between, sinks."""
    check(be, [(nq, 4000), (0, 70), (max(nq - 2, 1), 90), (nq, nq), (1, 2500)], 2 * H, 2, D, bits, 64)
    check(be, [(nq, 900), (nq, 40), (nq - 1, 333)], H, 1, D, bits, 24, window=100, n_first=6, sinks=True)


@pytest.mark.parametrize("dtype", ["bf16", 8, 4])
def test_bad_page_beside_keys_that_overflow(be, dtype):
    """A row that sees a key on no page is NaN whatever the cache holds elsewhere: keys of the first page's first
    row whose product with the row's q is minus infinity."""
    for nq in (1, 3, 40):
        for Hkv in (1, 2):
            q = torch.ones((nq, 4, 64))
            if dtype == "bf16":
                kv, sc = torch.zeros((4, 16, Hkv, 128), dtype=torch.bfloat16), None
                kv[0, 0, :, :64] = -math.inf
            else:
                kv, sc = M.cache(4, 16, Hkv, 64, dtype, torch.Generator().manual_seed(0))
                kv.view(torch.uint8)[0, 0, :, :64 * dtype // 8] = 0xfe if dtype == 8 else 0xff
                sc[0, 0, :, :2] = 254
            t = torch.tensor([[0, nq, 60, 1, -1, 2, 3]], dtype=torch.int32)
            got = be.flash_attn_paged(q.cuda(), kv.cuda(), t.cuda(), scale=1.0, max_q=nq, **({} if sc is None else dict(scales=sc.cuda())))
            assert torch.isnan(got).all(), (dtype, nq, Hkv)
