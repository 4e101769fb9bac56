// ghip_fap.hip -- attention over a paged KV cache: a batch of sequences of any
// length, each with its query rows at the end of its keys.
//
// Row i of a sequence with nq rows and nkv keys is at position p = nkv - nq + i
// and sees the keys j <= p with j > p - window or j < n_first (no window: all
// of them):  o = sum_j e^(s_j - m) v_j / sum_j e^(s_j - m),  s_j = scale q . k_j;
// a sink adds e^(sink - m) below the line.  A row that sees nothing gives 0.
// Key j is row j % page of page table[j / page]; a row that sees a key whose
// page does not exist gives NaN.
//
// Both kernels walk the keys once with a running reference and sum, on the matrix
// cores (v_mfma_f32_16x16x32): S^T = K Q^T leaves a query row in 4 lanes (n, n +
// 16, n + 32, n + 48), whose scores are the B operand of O^T += V^T P^T as they
// are.  q is 32-bit and the output too, so q and p are split into terms of the
// cache's type that add up to them (bf16: 3 terms, 24 bits; f16: 2 terms, 22 bits of
// what is brought into its range first, a row's q by a power of two, p by where the
// reference is), each a product of its own on the same K or V fragment; sums are
// 32-bit.  With one term fewer the error against 64 bits is 2e-6 (bf16, p: 2 terms;
// 2.5e-6 with 2 of q) where 32-bit arithmetic has 0.7e-6 and these terms 0.3e-6 to
// 0.5e-6.
//
//  * ghip_fap_few: up to 16 rows of a KV head (generation: the G = H / H_kv query
//    heads that share it, times a few rows).  Bound by reading K and V once: each
//    of the 4 wavefronts streams its own 32-key tiles and they meet at the end.
//    24 sequences of 500 .. 16384 keys under a window of 4096, 32 / 8 heads of 128,
//    bf16: 77 us for 365 MB, 4.7 TB/s, what a large copy reaches.
//  * ghip_fap_tile: 128 or 64 rows; the 4 wavefronts hold 32 or 16 rows each and share
//    64-key tiles, so that a K or V fragment read from LDS serves one or two row
//    tiles times the terms.  Bound by the matrix cores, the softmax's vector work and
//    what of them two wavefronts a SIMD do not overlap (registers: q's terms and the
//    output are 128 of 256): 1001 + 701 rows under a window of 2048, 32 / 8 heads of 128,
//    f16, 128 rows: 125 us, 0.49 PFLOP/s of the formula's, twice that of products.
//  * ghip_fap_both: a prefix shared by the batch as tiles of all its rows, and each
//    sequence's own keys for few rows, in one launch.
//  * ghip_fap_join: the partials of keys split over workgroups, in their order.
//
// K and V go straight from memory into LDS, 16 bytes a lane.  A row's 16-byte
// chunks are swapped about by its number so that the fragment reads meet no bank
// twice (k_swz, v_swz).  The loads are inline assembly: the compiler would wait
// for all of them before any LDS read.  Everything the loops load is counted by
// hand, in the order of issue.
#include "ghip_fap_core.h"

// An infinity in the cache: the terms of q and p make NaN of it (its product with a
// term that is 0, or below it), and so does p = 0 of a row that does not see its key.
// So a row whose result is not finite is computed again here, as the formula says, in
// 32 bits and with the keys that it sees alone: a lane a key for the scores, first their
// maximum, then p and its products with the values, lane l the dims 4 l ... A wavefront
// a row, and hardly ever one: 12 us for 64 keys (512 rows of 32 heads over 2048 keys that
// all see an infinite value: 2.6 ms, 58 us where it is finite); it ends at a score of
// NaN (77 us).
template <typename E>
DEV v4f row_again(const FapParams &p, const int32_t *table, int64_t tok, int h, int64_t pos) {
    const int lane = threadIdx.x & 63;
    const float *q = p.q + tok * p.q_nb2 + h * p.q_nb1;
    const uint16_t *kv = p.kv + h / (p.H / p.H_kv) * p.kv_head;
    const PagedKeys ks = paged_keys(pos, pos, p.window, p.n_first);
    const float nan = __builtin_nanf("");
    const v4f none = {nan, nan, nan, nan};
    float m = p.sinks ? p.sinks[h] * kLog2e : -__builtin_inff(), l = 0.0f;
    v4f o = {0, 0, 0, 0};
    for (int pass = 0; pass < 2; pass++) {
        if (pass) {
            if (m == -__builtin_inff()) m = 0.0f;  // nothing has weight
            if (p.sinks) l = __builtin_amdgcn_exp2f(p.sinks[h] * kLog2e - m);
        }
        for (int64_t j0 = 0; j0 < ks.hi; j0 += 64) {
            if (j0 >= ks.first && j0 + 64 <= ks.lo) {  // to the window
                j0 = (ks.lo & ~(int64_t)63) - 64;
                continue;
            }
            const int64_t j = j0 + lane;
            const bool seen = j < ks.first || (j >= ks.lo && j < ks.hi);
            const uint32_t i = paged_div(seen ? (uint32_t)j : 0, p.by_page);
            const int32_t page = seen ? table[i] : 0;
            if (__ballot(page < 0 || page >= p.n_pages)) return none;
            const uint16_t *at = kv + page * p.kv_page + (seen ? (uint32_t)j - i * (uint32_t)p.page : 0) * p.kv_row;
            float s = 0.0f;
#pragma unroll 2
            for (int d = 0; d < p.D; d += 8) {
                const uint4 x = *(const uint4 *)(at + d);
                const E *k = (const E *)&x;
#pragma unroll
                for (int e = 0; e < 8; e++) s = fmaf(q[d + e], (float)k[e], s);
            }
            s = seen ? s * (p.scale * kLog2e) : -__builtin_inff();
            if (__ballot(!(s < __builtin_inff()))) return none;
            if (!pass) {
#pragma unroll
                for (int t = 32; t; t >>= 1) s = fmaxf(s, __shfl_xor(s, t, 64));
                m = fmaxf(m, s);
                continue;
            }
            const float w = __builtin_amdgcn_exp2f(s - m);
            l += wave_sum(w);
            const float f = seen ? w : -1.0f;
            for (int k0 = 0; k0 < 64; k0 += 8) {
                uint2 x[8];
#pragma unroll
                for (int k = 0; k < 8; k++)
                    x[k] = *(const uint2 *)(__shfl((unsigned long long)(at + p.D), k0 + k, 64) + 2 * min(4 * lane, p.D - 4));
#pragma unroll
                for (int k = 0; k < 8; k++) {
                    const float y = __shfl(f, k0 + k, 64);
                    const E *e = (const E *)&x[k];
#pragma unroll
                    for (int c = 0; c < 4; c++) o[c] = y < 0.0f ? o[c] : fmaf(y, (float)e[c], o[c]);
                }
            }
        }
    }
    return l == 0.0f ? v4f{0, 0, 0, 0} : o / l;
}
template <typename E>
struct Again {
    static __device__ __forceinline__ v4f row(const FapParams &p, const int32_t *table, int64_t tok, int h, int64_t pos) {
        return row_again<E>(p, table, tok, h, pos);
    }
};

// Where the keys of a tile are: page numbers pg[] -> bytes into the cache of each
// key's row, offs[] (a lane a key, once for all the lanes that load its row).
// Keys past the tile's end or on no page: row 0 of page 0, which is not used.
DEV void find_keys(const FapParams &p, const Tile &tl, int kt, const int32_t *pg, int64_t *offs, uint64_t &ok, uint64_t &bad) {
    const int lane = threadIdx.x & 63;
    const uint32_t j = tl.k0 + lane;
    const bool in = lane < kt && (int)j < tl.ke;
    const int page = in ? pg[lane] : 0;
    const bool there = page >= 0 && page < p.n_pages;
    ok = __ballot(in && there);
    bad = __ballot(in && !there);
    const uint32_t r = j - paged_div(j, p.by_page) * (uint32_t)p.page;
    offs[lane] = in && there ? 2 * (page * p.kv_page + r * p.kv_row) : 0;
}
// The 16-byte pieces that a lane loads of a tile's rows: load ii of a wavefront
// fills LDS chunks 64 (from + ii) + lane.  Where 64 chunks are whole rows, the
// load's part of a row's number is bits apart from the lane's, so its part of the
// swizzle is flipped into the lane's.  Chunks past the row's end (D < DP) take its last.
template <int DP>
struct RowLoads {
    static constexpr int CH = DP / 8;
    static constexpr bool WHOLE = 64 % CH == 0;
    int from, row0;
    uint32_t k0, v0, last;
    DEV_M RowLoads(int D, int from_) : from(from_), last(2 * D - 16) {
        const int lane = threadIdx.x & 63;
        row0 = lane / CH;
        k0 = 16 * k_swz<CH>(row0, lane % CH);
        v0 = 16 * v_swz<CH>(row0, lane % CH);
    }
    DEV_M int row(int ii) const {
        return WHOLE ? row0 + 64 / CH * (from + ii) : (64 * (from + ii) + (int)(threadIdx.x & 63)) / CH;
    }
    DEV_M uint32_t k_chunk(int ii) const {
        if (WHOLE) return min(k0 ^ (uint32_t)(16 * k_swz<CH>(64 / CH * (from + ii), 0)), last);
        const int r = row(ii);
        return min((uint32_t)(16 * k_swz<CH>(r, (64 * (from + ii) + (int)(threadIdx.x & 63)) - r * CH)), last);
    }
    DEV_M uint32_t v_chunk(int ii) const {
        if (WHOLE) return min(v0 ^ (uint32_t)(16 * v_swz<CH>(64 / CH * (from + ii), 0)), last);
        const int r = row(ii);
        return min((uint32_t)(16 * v_swz<CH>(r, (64 * (from + ii) + (int)(threadIdx.x & 63)) - r * CH)), last);
    }
};

// ---- up to 16 rows a KV head: 4 wavefronts, each its own 32-key tiles

template <int DP>
struct FewLds {
    uint8_t kvs[4][2][32 * DP * 2];  // each wavefront's K and V tile
    int64_t offs[4][64];
    int32_t te[4][2][64];
    float ws[4][2][16];
};
template <typename E, int DP>
DEV void fap_few(const FapParams &p, FewLds<DP> &lds) {
    constexpr int KT = 32, CH = DP / 8, NI = KT * CH / 64;  // loads of a K (or V) tile
    auto &kvs = lds.kvs;
    auto &offs = lds.offs;
    auto &te = lds.te;
    auto &ws = lds.ws;
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n = lane & 15, g = lane >> 4;
    const int G = p.H / p.H_kv;
    const int64_t table = (int64_t)p.per * p.page;
    const int id = blockIdx.x - p.wg_sh, hk = id % p.H_kv, z = (id / p.H_kv) % p.zs_own, b = id / (p.H_kv * p.zs_own);
    const int32_t *row = p.seqs + (int64_t)b * p.seq_nb1;
    const PagedSeq sq = paged_seq(row[0], row[1], row[2], p.T, p.max_q);
    if (sq.nq == 0) return;
    Pass ps;
    ps.p0 = clip_pos(sq.pos0, table);
    ps.p1 = clip_pos(sq.pos0 + sq.nq - 1, table);
    ps.tl = paged_tiles(ps.p0, ps.p1, p.window, p.n_first, p.n_shared, (int)table, KT);
    const int share = paged_share(ps.tl.n, p.zs_own);
    const int t0 = (int)min((int64_t)z * share, (int64_t)ps.tl.n), t1 = min(ps.tl.n, t0 + share);
    const int i = n / G, hd = hk * G + n % G;
    const bool valid = n < sq.nq * G;
    const int64_t tok = sq.q0 + (valid ? i : 0);
    const int64_t pi = (tok * p.H + hd) * (p.zs_sh + p.zs_own) + p.zs_sh + z;
    if (t0 >= t1 && p.part) {  // nothing in this split
        if (valid && w == 0 && g == 0) stat_none(p, pi, sq.pos0 + i >= table);
        return;
    }
    Rows<E, DP, 1> R;
    RawRow<DP> raw;
    raw_load<DP>(raw, p.q + tok * p.q_nb2 + hd * p.q_nb1, p.D, valid);
    R.pos[0] = valid ? clip_pos(sq.pos0 + i, table) : -1;
    const uint32_t ka = lds_addr(kvs[w][0]), va = lds_addr(kvs[w][1]);

    // page numbers of tile t's keys, a lane each
    auto load_pages = [&](int t) {
        const Tile tl = tile_at(ps.tl, min(t, t1 - 1), KT);
        const int j = min(tl.k0 + lane, tl.ke - 1);
        load4(row + 3 + paged_div((uint32_t)j, p.by_page), lds_addr(te[w][t >> 2 & 1]));
    };
    const RowLoads<DP> rl(p.D, 0);
    uint64_t ok = 0, bad = 0;  // the next tile's keys that are there, those on no page
    auto find_rows = [&](int t) { find_keys(p, tile_at(ps.tl, t, KT), KT, te[w][t >> 2 & 1], offs[w], ok, bad); };
    const uint8_t *kvh = (const uint8_t *)(p.kv + hk * p.kv_head);
    auto load_k = [&]() {
#pragma unroll
        for (int ii = 0; ii < NI; ii++) load16(kvh + offs[w][rl.row(ii)] + rl.k_chunk(ii), ka + 1024 * ii);
    };
    auto load_v = [&]() {
#pragma unroll
        for (int ii = 0; ii < NI; ii++) load16(kvh + offs[w][rl.row(ii)] + 2 * p.D + rl.v_chunk(ii), va + 1024 * ii);
    };
    // in flight at the top of a step, oldest first: pages t + 4, K t, V t
    const int first = t0 + w;
    if (first < t1) load_pages(first);
    wait_loads<0>();
    raw_wait<DP>(raw);
    if (first < t1) {
        find_rows(first);
        load_pages(first + 4);
        load_k();
        load_v();
    }
    rows_start<E, DP, 1>(R, 0, raw, p.scale * kLog2e);
    for (int t = first; t < t1; t += 4) {
        const Tile tile = tile_at(ps.tl, t, KT);
        const uint64_t okc = ok, badc = bad;
        const bool more = t + 4 < t1;
        wait_loads<NI>();
        v4f s[2][1];
        scores<E, DP, 1, 2>(R, ka, s, [](int) {});
        if (more) {
            find_rows(t + 4);
            wait_lds();
            load_pages(t + 8);
            load_k();
        }
        const bool part = !tile_whole(tile, KT, ps, p.window, p.n_first);
        if (part || badc) mask_scores<E, DP, 1, 2>(R, s, tile.k0, tile.ke, badc, p.window, p.n_first);
        auto values_in = [&]() {
            if (more) wait_loads<NI + 1>();
            else wait_loads<0>();
            if (okc != 0xffffffffull) {
                // rows that were not there: no value of theirs may count
#pragma unroll
                for (int ii = 0; ii < NI; ii++) {
                    const int c = 64 * ii + lane;
                    if (!((okc >> (c / CH)) & 1)) *(uint4 *)(kvs[w][1] + 16 * c) = make_uint4(0, 0, 0, 0);
                }
                wait_lds();
            }
        };
        softmax<E, DP, 1, 2>(R, s, va, values_in);
        values_in();
        values<E, DP, 1, 2>(R, va, s);
        if (more) {
            wait_lds();
            load_v();
        }
    }
    static_assert(sizeof(kvs) >= 4 * 16 * (DP + 4) * 4, "the wavefronts' rows fit the tiles");
    few_join<Again<E>, E, DP, 1>(p, R, 0, (float *)&kvs[0][0][0], ws, sq.nq * G, valid, table, tok, hd, pi, row + 3);
}

// How a tile of a cache of 16-bit elements comes into LDS: straight from memory.
template <typename E>
struct Direct {
    typedef ::Again<E> Again;
    static constexpr int HOME_K = 0;
    static constexpr bool NARROW = false, LATE = false;
    struct Lds {
        int64_t offs[4][64];
        int32_t te[4][2][64];
    };
    template <int DP>
    struct Loads {
        static constexpr int KT = 64, CH = DP / 8, NI = KT * CH / 256;  // loads of a K tile by each wavefront
        static_assert(KT * CH % 256 == 0 && 2 * NI == DP / 16, "the wavefronts load alike, one load under each of a half's fragments");
        const FapParams &p;
        Lds &lds;
        uint8_t (&kvs)[2][2][64 * DP * 2];
        const int32_t *row;
        int w, t1;
        const PagedTiles &tl;
        const uint8_t *kvh;
        // Three tiles are under way: t is computed, t + 1 loaded, and at the step's end,
        // where it would wait for those loads, the rows of t + 2 are found (from pages
        // that were loaded a step before).
        uint64_t ok = 0, bad = 0, ok2 = 0, bad2 = 0;  // keys of tiles t + 1, t + 2 that are there, those on no page
        const uint8_t *at[NI];                        // this lane's rows of the tile found last
        const RowLoads<DP> rl;
        DEV_M Loads(const FapParams &p_, Lds &lds_, uint8_t (&kvs_)[2][2][64 * DP * 2], int hk, const int32_t *row_, int w_,
                    const PagedTiles &tl_, int t1_)
            : p(p_), lds(lds_), kvs(kvs_), row(row_), w(w_), t1(t1_), tl(tl_), kvh((const uint8_t *)(p_.kv + hk * p_.kv_head)), rl(p_.D, NI * w_) {}
        DEV_M void load_pages(int t) {
            const Tile tile = tile_at(tl, min(t, t1 - 1), KT);
            const int j = min(tile.k0 + (int)(threadIdx.x & 63), tile.ke - 1);
            load4(row + 3 + paged_div((uint32_t)j, p.by_page), lds_addr(lds.te[w][t & 1]));
        }
        DEV_M void find_tile(int t) {
            find_keys(p, tile_at(tl, t, KT), KT, lds.te[w][t & 1], lds.offs[w], ok2, bad2);
#pragma unroll
            for (int ii = 0; ii < NI; ii++) at[ii] = kvh + lds.offs[w][rl.row(ii)];
        }
        // load f of 2 NI of tile t: one goes out under each fragment's products (bf16, 12
        // turns under 4001 keys, 128 rows: 125 us, and 130 with all of them at the step's
        // start; f16 the same)
        DEV_M void load_part(int t, int f) {
            const int ii = f >> 1, kv = f & 1;
            load16(at[ii] + (kv ? 2 * p.D + rl.v_chunk(ii) : rl.k_chunk(ii)), lds_addr(kvs[t & 1][kv]) + 1024 * (NI * w + ii));
        }
        DEV_M void load_half(int t, int) {
#pragma unroll
            for (int f = 0; f < 2 * NI; f++) load_part(t, f);
        }
        DEV_M void load_first(int t) { load_half(t, 0); }
        DEV_M void middle(int) {}
        // What this wavefront loaded of tile t is in: rows that were not there hold
        // nothing that counts.
        DEV_M void loaded(int t) {
            uint8_t *Vs = kvs[t & 1][1];
            if (ok != ~0ull) {
#pragma unroll
                for (int ii = 0; ii < NI; ii++) {
                    const int c = 64 * (NI * w + ii) + (threadIdx.x & 63);
                    if (!((ok >> (c / CH)) & 1)) *(uint4 *)(Vs + 16 * c) = make_uint4(0, 0, 0, 0);
                }
            }
        }
    };
};

extern "C" __global__ void __launch_bounds__(256) ghip_fap_join_f16(FapParams p) { fap_join<Again<f16>>(p); }
extern "C" __global__ void __launch_bounds__(256) ghip_fap_join_bf16(FapParams p) { fap_join<Again<bf16>>(p); }

// ghip_fap_both: the shared prefix on tiles and each sequence's own keys, for few
// rows each, in one launch, so that the one's loads run under the other's products.
template <typename E, int DP, int RW>
union FapLds {
    FewLds<DP> few;
    TileLds<Direct<E>, DP, RW> tile;
};
#define FAP_FEW(E, DP)                                                                                   \
    extern "C" __global__ void __launch_bounds__(256, 2) ghip_fap_few_##E##_##DP(FapParams p) {          \
        __shared__ __attribute__((aligned(1024))) uint8_t lds[sizeof(FewLds<DP>)];                       \
        fap_few<E, DP>(p, *(FewLds<DP> *)lds);                                                           \
    }
// (R: rows of a workgroup, 64 RW)
#define FAP_TILE(E, DP, RW, R)                                                                           \
    extern "C" __global__ void __launch_bounds__(256, 2) ghip_fap_tile##R##_##E##_##DP(FapParams p) {    \
        __shared__ __attribute__((aligned(1024))) uint8_t lds[sizeof(TileLds<Direct<E>, DP, RW>)];                  \
        fap_tile<Direct<E>, E, DP, RW>(p, *(TileLds<Direct<E>, DP, RW> *)lds);                                                 \
    }                                                                                                    \
    extern "C" __global__ void __launch_bounds__(256, 2) ghip_fap_both##R##_##E##_##DP(FapParams p) {    \
        __shared__ __attribute__((aligned(1024))) uint8_t lds[sizeof(FapLds<E, DP, RW>)];                   \
        if ((int)blockIdx.x < p.wg_sh) fap_tile<Direct<E>, E, DP, RW>(p, *(TileLds<Direct<E>, DP, RW> *)lds);                  \
        else fap_few<E, DP>(p, *(FewLds<DP> *)lds);                                                      \
    }
#define FAP_E(E)                                                                                         \
    FAP_FEW(E, 64) FAP_FEW(E, 96) FAP_FEW(E, 128) FAP_FEW(E, 256)                                        \
    FAP_TILE(E, 64, 1, 64) FAP_TILE(E, 96, 1, 64) FAP_TILE(E, 128, 1, 64) FAP_TILE(E, 256, 1, 64)        \
    FAP_TILE(E, 64, 2, 128) FAP_TILE(E, 96, 2, 128)
FAP_E(f16) FAP_E(bf16)
FAP_TILE(f16, 128, 2, 128)
