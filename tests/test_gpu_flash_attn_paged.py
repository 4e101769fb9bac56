"""ghip_flash_attn_paged against attention's formula in 64 bits (paged_oracle):
every element within attention_tol, and the whole within 2^-17 in 2-norm (17 bits
of q and p are the least that a kernel holds; roundings of single elements do not
all point one way)."""
import math
import os

import pytest

import paged_oracle as P

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

TYPES = {"f16": torch.float16, "bf16": torch.bfloat16}


@pytest.fixture(scope="module")
def be():
    import ghip
    b = ghip.Backend(0)
    yield b
    b.close()


def make(seqs, H, Hkv, D, ctype, page, n_shared=0, seed=0, spare=3, order=None):
    """seqs: (nq, nkv) of each.  -> q, kv, table [B, 3 + per] with pages in no order,
    the first n_shared keys' pages common (and a cut page's rows copied)"""
    g = torch.Generator().manual_seed(seed)
    per = max([(n + page - 1) // page for _, n in seqs] + [0])
    common, rest = divmod(n_shared, page)
    total = sum(max(0, (n + page - 1) // page - common) for _, n in seqs) + common + spare
    perm = torch.randperm(total, generator=g).to(torch.int32)
    table = torch.full((len(seqs), 3 + per), -7, dtype=torch.int32)
    T, at, first = sum(a for a, _ in seqs), common, 0
    starts = {}
    for b in (order or range(len(seqs))):
        starts[b] = first
        first += seqs[b][0]
    for b, (nq, nkv) in enumerate(seqs):
        need = (nkv + page - 1) // page
        table[b, :3] = torch.tensor([starts[b], nq, nkv])
        c = min(common, need)
        table[b, 3:3 + c] = perm[:c]
        table[b, 3 + c:3 + need] = perm[at:at + need - c]
        at += need - c
    q = torch.randn((T, H, D), generator=g)
    kv = torch.randn((total, page, Hkv, 2 * D), generator=g).to(TYPES[ctype])
    if rest:
        for b in range(1, len(seqs)):
            if seqs[b][1] > common * page:
                kv[table[b, 3 + common].long(), :rest] = kv[table[0, 3 + common].long(), :rest]
    return q, kv, table


def ways(n_shared):
    """A shared prefix read once for all and read by each sequence, tiles of 64 rows
    and of 128: the sizes of these tests would take one of each by themselves."""
    for shared in ("1", "0") if n_shared else (None,):
        for rows in ("64", "128"):
            os.environ["GHIP_FAP_ROWS"] = rows
            if shared is not None:
                os.environ["GHIP_FAP_SHARED"] = shared
            try:
                yield shared, rows
            finally:
                os.environ.pop("GHIP_FAP_SHARED", None)
                os.environ.pop("GHIP_FAP_ROWS", None)


def compare(got, want, mag, wgt, D):
    got = got.double()
    named = ~torch.isnan(want)
    err, tol = (got - want).abs(), P.attention_tol(mag, wgt, D)
    assert (err[named] <= tol.expand_as(err)[named]).all(), float((err / tol)[named].max())
    n = torch.linalg.vector_norm(want[named])
    off = torch.linalg.vector_norm(err[named])
    assert off <= 2.0 ** -17 * n, float(off / n)


def check(be, seqs, H, Hkv, D, ctype="f16", page=16, window=0, n_first=0, n_shared=0, sinks=False, seed=0, max_q=None, order=None):
    q, kv, table = make(seqs, H, Hkv, D, ctype, page, n_shared, seed, order=order)
    sk = torch.randn(H, generator=torch.Generator().manual_seed(seed + 1)) if sinks else None
    scale = 1 / math.sqrt(D)
    want, mag, wgt = P.attention(q, kv, table.tolist(), scale, sk, window, n_first)
    print(f"paged {seqs[:4]} H={H}/{Hkv} D={D} {ctype} page={page} window={window}+{n_first} shared={n_shared} sinks={sinks}", flush=True)
    for how in ways(n_shared):
        got = be.flash_attn_paged(q.cuda(), kv.cuda(), table.cuda(), scale=scale, sinks=sk.cuda() if sinks else None, window=window,
                                  n_first=n_first, n_shared=n_shared, max_q=max_q or max([a for a, _ in seqs] + [1]))
        compare(got.cpu(), want, mag, wgt, D)


@pytest.mark.parametrize("ctype", ["f16", "bf16"])
@pytest.mark.parametrize("H,Hkv,D", [(8, 2, 64), (8, 2, 128), (5, 1, 80), (4, 4, 96), (16, 1, 64), (6, 2, 256), (3, 1, 8), (2, 2, 120)])
@pytest.mark.parametrize("page", [1, 16, 24, 64, 256])
def test_decode(be, H, Hkv, D, page, ctype):
    check(be, [(1, 1), (1, 63), (1, 64), (1, 65), (1, 700), (1, 17)], H, Hkv, D, ctype, page)


@pytest.mark.parametrize("ctype", ["f16", "bf16"])
@pytest.mark.parametrize("H,Hkv,D", [(4, 1, 128), (2, 2, 64), (3, 1, 80), (2, 1, 256), (10, 2, 64)])
def test_prompts(be, H, Hkv, D, ctype):
    check(be, [(33, 33), (70, 200), (1, 90), (17, 300), (2, 2)], H, Hkv, D, ctype, 16)


@pytest.mark.parametrize("window,n_first", [(1, 0), (7, 0), (64, 4), (100, 1), (100, 130), (64, 64), (1, 1), (5000, 4)])
@pytest.mark.parametrize("nq", [1, 9, 40])
def test_window(be, window, n_first, nq):
    check(be, [(nq, nq), (nq, 64 + nq), (nq, 257), (nq, 400), (nq, nq + 1)], 8, 2, 64, "f16", 16, window, n_first, sinks=True)


@pytest.mark.parametrize("ctype", ["f16", "bf16"])
@pytest.mark.parametrize("n_shared,page", [(1, 16), (64, 64), (200, 16), (333, 24), (300, 1), (320, 64)])
def test_shared_prefix(be, n_shared, page, ctype):
    lens = [n_shared + 1, n_shared + 63, n_shared + 200, n_shared + 7, n_shared + 64]
    check(be, [(1, n) for n in lens], 8, 2, 128, ctype, page, n_shared=n_shared)
    check(be, [(1, n) for n in lens], 16, 1, 64, ctype, page, n_shared=n_shared, sinks=True)
    check(be, [(min(n, 1 + 5 * i), n) for i, n in enumerate(lens)], 4, 1, 80, ctype, page, n_shared=n_shared)


def test_shared_prefix_of_rows_inside_it(be):
    """Rows at positions inside the prefix, sequences that end there, a window over it."""
    check(be, [(20, 150), (40, 130), (5, 80), (128, 128)], 4, 2, 64, "f16", 16, n_shared=128)
    check(be, [(1, 128), (1, 30), (1, 129), (1, 1)], 4, 2, 64, "f16", 16, n_shared=128)
    check(be, [(20, 250), (40, 230), (1, 180)], 4, 2, 64, "f16", 16, window=70, n_first=5, n_shared=160)
    check(be, [(1, 250), (1, 230), (1, 180)], 4, 2, 64, "f16", 16, window=70, n_first=5, n_shared=160, sinks=True)
    check(be, [(1, 250)], 4, 2, 64, "f16", 16, n_shared=240)


def test_long_keys(be):
    """Enough keys that one row's are split over workgroups and joined."""
    check(be, [(1, 9000), (1, 100), (1, 5000)], 8, 2, 128, "bf16", 64)
    check(be, [(1, 9000), (1, 8300), (1, 8200)], 4, 1, 64, "f16", 64, n_shared=8192)
    check(be, [(3, 6000), (1, 6100)], 4, 4, 128, "f16", 64, window=5000, n_first=100)


def test_any_order_of_rows(be):
    """Sequences whose rows lie in another order than the table, some without rows."""
    check(be, [(3, 40), (0, 0), (20, 60), (0, 30), (1, 5)], 4, 2, 64, order=[4, 2, 3, 0, 1])
    check(be, [(1, 40), (0, 90), (1, 60), (1, 100)], 4, 2, 64, order=[3, 2, 0, 1], n_shared=32)


@pytest.mark.parametrize("nq", [1, 30])
def test_rows_that_see_nothing(be, nq):
    """More rows than keys: the rows before key 0 give 0, with sinks too."""
    for sinks in (False, True):
        check(be, [(nq, 0), (nq, nq), (2 * nq + 3, nq)], 4, 2, 64, sinks=sinks)


def test_rows_outside_the_table_are_kept(be):
    q, kv, table = make([(2, 30), (3, 20)], 4, 2, 64, "f16", 16)
    q = torch.cat([q, torch.randn((4, 4, 64))])
    out = torch.full(q.shape, 7.0).cuda()
    be.flash_attn_paged(q.cuda(), kv.cuda(), table.cuda(), scale=0.125, max_q=3, out=out)
    assert (out[5:] == 7).all() and not (out[:5] == 7).any()
    out.fill_(7.0)
    be.flash_attn_paged(q.cuda(), kv.cuda(), table.cuda(), scale=0.125, max_q=2, out=out)
    assert (out[4:] == 7).all() and not (out[:4] == 7).any()


@pytest.mark.parametrize("nq", [1, 5, 40])
@pytest.mark.parametrize("what", [float("nan"), float("inf")])
def test_what_unseen_places_hold(be, nq, what):
    """NaN and infinities in the rows of a page past the last key, in keys before
    the window, in pages of no sequence; pages before the window are gone."""
    for window, n_first, n_shared in [(0, 0, 0), (50, 4, 0), (0, 0, 64)]:
        seqs = [(nq, 150), (nq, 201), (nq, 97)]
        q, kv, table = make(seqs, 8, 2, 64, "f16", 16, n_shared)
        want, mag, wgt = P.attention(q, kv, table.tolist(), 0.125, None, window, n_first)
        seen = torch.zeros(kv.shape[:2], dtype=torch.bool)
        for b, (n, m) in enumerate(seqs):
            for j in range(m):
                if any(j <= p and (not window or j > p - window or j < n_first) for p in range(m - n, m)):
                    seen[table[b, 3 + j // 16].long(), j % 16] = True
        kv[~seen] = what
        gone = table.clone()
        for b, (n, m) in enumerate(seqs):
            for i in range((m + 15) // 16):
                if not seen[table[b, 3 + i].long()].any():
                    gone[b, 3 + i] = 10 ** 6
        for how in ways(n_shared):
            got = be.flash_attn_paged(q.cuda(), kv.cuda(), gone.cuda(), scale=0.125, window=window, n_first=n_first, n_shared=n_shared, max_q=nq)
            compare(got.cpu(), want, mag, wgt, 64)


def test_later_rows_do_not_reach_earlier_ones(be):
    """A NaN or infinite value of key j changes the rows from j on alone."""
    for what in (float("nan"), float("inf")):
        q, kv, table = make([(50, 120)], 4, 2, 64, "f16", 16)
        want, mag, wgt = P.attention(q, kv, table.tolist(), 0.125)
        for j in (80, 100):
            kv[table[0, 3 + j // 16].long(), j % 16, :, 64:] = what
        for how in ways(0):
            got = be.flash_attn_paged(q.cuda(), kv.cuda(), table.cuda(), scale=0.125, max_q=50).cpu()
            compare(got[:10], want[:10], mag[:10], wgt[:10], 64)
            assert not torch.isfinite(got[10:]).any()


@pytest.mark.parametrize("nq", [1, 40])
def test_strides(be, nq):
    """q inside a wider projection, dst and cache with gaps, a cache with heads outside rows."""
    seqs = [(nq, 77), (nq, 130)]
    q, kv, table = make(seqs, 4, 2, 64, "f16", 16)
    want, mag, wgt = P.attention(q, kv, table.tolist(), 0.125)
    wide = torch.full((q.shape[0], 7, 71), 9.0)
    wide[:, 1:5, 5:69] = q
    out = torch.full((q.shape[0], 5, 80), 7.0).cuda()
    kvh = kv.permute(0, 2, 1, 3).contiguous().cuda().permute(0, 2, 1, 3)  # [pages, H_kv, page, 2 D] in memory
    wt = torch.full((2, table.shape[1] + 4), -1, dtype=torch.int32)
    wt[:, :table.shape[1]] = table
    be.flash_attn_paged(wide.cuda()[:, 1:5, 5:69], kvh, wt.cuda()[:, :table.shape[1]], scale=0.125, max_q=nq, out=out[:, :4, 8:72])
    out = out.cpu()
    compare(out[:, :4, 8:72], want, mag, wgt, 64)
    out[:, :4, 8:72] = 7.0
    assert (out == 7.0).all()


def test_large_scores(be):
    """Scores far apart, and rows whose running maximum moves at almost every key."""
    for nq in (1, 33):
        q, kv, table = make([(nq, 500)], 4, 2, 64, "f16", 16)
        q *= 20
        for j in range(500):
            kv[table[0, 3 + j // 16].long(), j % 16, :, :64] *= 0.01 * j
        want, mag, wgt = P.attention(q, kv, table.tolist(), 0.125)
        for how in ways(0):
            got = be.flash_attn_paged(q.cuda(), kv.cuda(), table.cuda(), scale=0.125, max_q=nq).cpu().double()
            assert ((got - want).abs() <= P.attention_tol(mag, wgt, 64)).all()


def test_equal_calls_give_equal_bits(be):
    for seqs, sh in (([(1, 5000), (1, 4990)], 4096), ([(40, 900), (3, 700)], 512), ([(1, 3000)], 0)):
        q, kv, table = make(seqs, 8, 2, 128, "bf16", 64, sh)
        for how in ways(sh):
            a = [be.flash_attn_paged(q.cuda(), kv.cuda(), table.cuda(), scale=0.1, n_shared=sh, max_q=max(n for n, _ in seqs)) for _ in range(4)]
            assert all(torch.equal(a[0], x) for x in a[1:])


def test_nothing_to_do(be):
    kv = torch.zeros((2, 4, 1, 128), dtype=torch.float16, device="cuda")
    t = torch.zeros((0, 5), dtype=torch.int32, device="cuda")
    q = torch.ones((3, 2, 64), device="cuda")
    out = torch.full_like(q, 5)
    be.flash_attn_paged(q, kv, t, out=out)
    assert (out == 5).all()
    assert be.flash_attn_paged(q[:0], kv, torch.zeros((1, 5), dtype=torch.int32, device="cuda")).shape == (0, 2, 64)


def test_far_pages(be):
    """Keys past 2^32 bytes of the cache."""
    D, Hkv, page, pages = 128, 8, 64, 18000  # 4.7 GB
    kv = torch.zeros((pages, page, Hkv, 2 * D), dtype=torch.float16, device="cuda")
    far = torch.tensor([17999, 3, 17500, 16390], dtype=torch.int32)
    small = torch.randn((4, page, Hkv, 2 * D)).half()
    kv[far.long().cuda()] = small.cuda()
    for nq in (1, 20):
        q = torch.randn((nq, 16, D))
        head = torch.tensor([0, nq, 250], dtype=torch.int32)
        want, mag, wgt = P.attention(q, small, [torch.cat([head, torch.arange(4)]).tolist()], 0.088)
        got = be.flash_attn_paged(q.cuda(), kv, torch.cat([head, far]).view(1, -1).cuda(), scale=0.088)
        compare(got.cpu(), want, mag, wgt, D)


def test_graph_replays_follow_the_table(be):
    """Captured once for the largest lengths; replays with other lengths, pages and rows."""
    import ghip
    H, Hkv, D, page, per, B = 8, 2, 64, 16, 80, 4
    for nq, n_shared in ((1, 0), (1, 64), (24, 0)):
        kv = torch.randn((400, page, Hkv, 2 * D), device="cuda").half()
        q = torch.randn((B * nq, H, D), device="cuda")
        out = torch.empty_like(q)
        table = torch.zeros((B, 3 + per), dtype=torch.int32, device="cuda")

        def fill(seed):
            g = torch.Generator().manual_seed(seed)
            t = torch.zeros((B, 3 + per), dtype=torch.int32)
            perm = torch.randperm(400, generator=g).to(torch.int32)
            for b in range(B):
                t[b, :3] = torch.tensor([b * nq, nq, int(torch.randint(80, per * page, (1,), generator=g))])
                t[b, 3:] = perm[b * per:(b + 1) * per]
                t[b, 3:3 + n_shared // page] = perm[:n_shared // page]
            table.copy_(t)
            q.copy_(torch.randn(q.shape, generator=g))

        call = lambda o: be.flash_attn_paged(q, kv, table, scale=0.125, n_shared=n_shared, max_q=nq, out=o)
        for how in ways(n_shared):
            fill(0)
            s = torch.cuda.Stream()
            s.wait_stream(torch.cuda.current_stream())
            g = torch.cuda.CUDAGraph()
            with torch.cuda.stream(s):
                call(out)
                torch.cuda.synchronize()
                with torch.cuda.graph(g, stream=s):
                    call(out)
            for i in range(4):
                fill(i)
                torch.cuda.synchronize()
                g.replay()
                torch.cuda.synchronize()
                assert torch.equal(out, call(torch.empty_like(out))), i
                torch.cuda.synchronize()


@pytest.mark.parametrize("nq,n_shared", [(1, 0), (30, 0), (1, 32), (30, 32)])
def test_bad_pages_give_nan(be, nq, n_shared):
    """A row that sees a key on a page that does not exist is NaN, the others are
    computed; tables that point outside q write nothing."""
    seqs = [(nq, 150), (nq, 100), (nq, 64)]
    q, kv, table = make(seqs, 4, 2, 64, "f16", 16, n_shared)
    want, mag, wgt = P.attention(q, kv, table.tolist(), 0.125)
    bad = table.clone()
    bad[0, 3 + 140 // 16] = kv.shape[0]
    bad[1, 3 + 96 // 16] = -1
    for how in ways(n_shared):
        got = be.flash_attn_paged(q.cuda(), kv.cuda(), bad.cuda(), scale=0.125, n_shared=n_shared, max_q=nq).cpu()
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
        be.flash_attn_paged(q.cuda(), kv.cuda(), odd.cuda(), scale=0.125, n_shared=n_shared, max_q=nq, out=out)
        out = out.cpu()
        assert torch.isnan(out[nq - 1]).all()
        assert (out[nq:] == 7).all()


def test_shared_prefix_is_read_where_it_pays(be):
    """Many sequences under a long prefix: the first sequence's pages are read (the
    others' copies hold something else), few under a short one: each its own."""
    for B, n_shared, once in ((40, 2048, True), (3, 32, False)):
        seqs = [(1, n_shared + 20 + b) for b in range(B)]
        q, kv, table = make(seqs, 8, 2, 128, "f16", 16)
        want, _, _ = P.attention(q[:1], kv, table[:1].tolist(), 0.09)
        first = be.flash_attn_paged(q.cuda(), kv.cuda(), table.cuda(), scale=0.09, n_shared=n_shared, max_q=1).cpu()
        as_first = table.clone()
        as_first[:, 3:3 + n_shared // 16] = table[0, 3:3 + n_shared // 16]
        same = be.flash_attn_paged(q.cuda(), kv.cuda(), as_first.cuda(), scale=0.09, n_shared=n_shared, max_q=1).cpu()
        assert ((first[:1].double() - want).abs() < 1e-4).all()
        assert torch.equal(first, same) == once
