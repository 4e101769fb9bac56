// ghip_fapq.hip -- attention over a quantized paged KV cache (codes and scales of ghip_mx.h).
// The formula, tables, masks and partials are those of ghip_fap.hip.
#include "ghip_fap_core.h"
#include "ghip_mx.h"

// (kv_head, kv_row, kv_page count bytes)
struct FapMxParams : FapParams {
    const uint8_t *sc;
    int64_t sc_head, sc_row, sc_page;
    int S;  // scale bytes of a key
};

// One row of q, a wavefront: as the formula says, in 32 bits, a lane a key for the
// scores, first their maximum, then p and its products with the values, lane l the dims 4 l ..
template <int BITS>
DEV v4f row_alone(const FapMxParams &p, const int32_t *table, int64_t tok, int h, int64_t pos) {
    const int lane = threadIdx.x & 63, hk = h / (p.H / p.H_kv);
    const float *q = p.q + tok * p.q_nb2 + h * p.q_nb1;
    const uint8_t *kv = (const uint8_t *)p.kv + hk * p.kv_head, *sc = p.sc + hk * p.sc_head;
    const PagedKeys ks = paged_keys(pos, pos, p.window, p.n_first);
    const float nan = __builtin_nanf("");
    const v4f none = {nan, nan, nan, nan};
    float m = p.sinks ? p.sinks[h] * kLog2e : -__builtin_inff(), l = 0.0f;
    v4f o = {0, 0, 0, 0};
    const int d4 = min(4 * lane, p.D - 4);
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
            const int64_t r = seen ? (uint32_t)j - i * (uint32_t)p.page : 0;
            const uint8_t *at = kv + page * p.kv_page + r * p.kv_row, *sat = sc + page * p.sc_page + r * p.sc_row;
            float s = 0.0f;
            for (int d = 0; d < p.D; d += 16) {
                uint32_t w[BITS / 2];
                __builtin_memcpy(w, at + d * BITS / 8, sizeof w);
                const float f = mx_scale(sat[d >> 5]);
#pragma unroll
                for (int e = 0; e < BITS / 2; e++) {
                    mx_f2 x[16 / BITS];
                    x[0] = mx_pair<BITS, 0>(w[e], f);
                    x[1] = mx_pair<BITS, 1>(w[e], f);
                    if constexpr (BITS == 4) {
                        x[2] = mx_pair<BITS, 2>(w[e], f);
                        x[3] = mx_pair<BITS, 3>(w[e], f);
                    }
#pragma unroll
                    for (int k = 0; k < 32 / BITS; k++) s = fmaf(q[d + e * (32 / BITS) + k], x[k / 2][k & 1], s);
                }
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
                uint32_t x[8], b[8];
#pragma unroll
                for (int k = 0; k < 8; k++) {
                    const uint8_t *va = (const uint8_t *)__shfl((unsigned long long)at, k0 + k, 64);
                    const uint8_t *vs = (const uint8_t *)__shfl((unsigned long long)sat, k0 + k, 64);
                    x[k] = 0;
                    __builtin_memcpy(&x[k], va + (p.D + d4) * BITS / 8, BITS / 2);
                    b[k] = vs[p.S + (d4 >> 5)];
                }
#pragma unroll
                for (int k = 0; k < 8; k++) {
                    const float y = __shfl(f, k0 + k, 64), g = mx_scale(b[k]);
                    const mx_f2 u = mx_pair<BITS, 0>(x[k], g), v = mx_pair<BITS, 1>(x[k], g);
#pragma unroll
                    for (int c = 0; c < 4; c++) {
                        const float e = c < 2 ? u[c] : v[c - 2];
                        o[c] = y < 0.0f ? o[c] : fmaf(y, e, o[c]);
                    }
                }
            }
        }
    }
    return l == 0.0f ? v4f{0, 0, 0, 0} : o / l;
}

template <int BITS>
struct Alone {
    static __device__ __forceinline__ v4f row(const FapParams &p, const int32_t *table, int64_t tok, int h, int64_t pos) {
        return row_alone<BITS>(static_cast<const FapMxParams &>(p), table, tok, h, pos);
    }
};

// Where the keys of a tile are, a lane a key (its page: pg): bytes into the codes and the
// scales of its row.  Keys past the tile's end or on no page: row 0 of page 0, which is not used.
DEV void find_keys_mx(const FapMxParams &p, const Tile &tl, int kt, int pg, int64_t *offs, int64_t *soffs, uint64_t &ok, uint64_t &bad) {
    const int lane = threadIdx.x & 63;
    const uint32_t j = tl.k0 + lane;
    const bool in = lane < kt && (int)j < tl.ke;
    const bool there = in && pg >= 0 && pg < p.n_pages;
    ok = __ballot(there);
    bad = __ballot(in && !there);
    const int64_t r = j - paged_div(j, p.by_page) * (uint32_t)p.page;
    if (lane < kt) {
        offs[lane] = there ? pg * p.kv_page + r * p.kv_row : 0;
        soffs[lane] = there ? pg * p.sc_page + r * p.sc_row : 0;
    }
}
template <int W>
DEV void load_words(uint32_t (&w)[W], const uint8_t *from) {
    __builtin_memcpy(w, from, 4 * W);
}

// ---- up to 16 rows a KV head: 4 wavefronts, each its own 32-key tiles

template <int DP>
struct FewqLds {
    uint8_t v[4 * 64 * (DP + 4)];  // each wavefront's values as bfloat16 [32][DP]; at the end their rows
    int64_t offs[4][2][32];
    float ws[4][2][16];
};
template <int BITS, int DP>
DEV void fapq_few(const FapMxParams &p, FewqLds<DP> &lds) {
    // A lane's codes of a key: NU units of EL elements, unit g + 4 i; fragment kk of the products takes 8 of
    // them, and so does q's.
    constexpr int KT = 32, CH = DP / 8, EL = BITS == 4 && DP >= 128 ? 32 : 16, NU = DP / EL / 4, FU = EL / 8, WK = EL * BITS / 32;
    // ... of the values: unit lane % U of keys lane / U + (64 / U) ii
    constexpr int U = DP / 16, NV = KT * U / 64, WV = BITS / 2;
    auto &offs = lds.offs;
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
    Rows<bf16, DP, 1> R;
    R.pos[0] = valid ? clip_pos(sq.pos0 + i, table) : -1;
    RawRow<DP> raw;
    const float *qr = p.q + tok * p.q_nb2 + hd * p.q_nb1;
#pragma unroll
    for (int kk = 0; kk < DP / 32; kk++) {
        const int d = EL * (g + 4 * (kk / FU)) + 8 * (kk % FU);
#pragma unroll
        for (int e = 0; e < 8; e++) raw.x[kk][e] = 0.0f;
        if (valid && d < p.D) __builtin_memcpy(raw.x[kk], qr + d, 32);
    }
    const uint8_t *kvh = (const uint8_t *)p.kv + hk * p.kv_head, *sch = p.sc + hk * p.sc_head;
    uint8_t *Vs = lds.v + w * (64 * DP);
    const uint32_t va = lds_addr(Vs);

    auto load_page = [&](int t) {  // page number of a key of tile t, a lane each
        const Tile tl = tile_at(ps.tl, min(t, t1 - 1), KT);
        return row[3 + paged_div((uint32_t)min(tl.k0 + lane, tl.ke - 1), p.by_page)];
    };
    uint64_t ok = 0, bad = 0;  // the next tile's keys that are there, those on no page
    const int units = (p.D + EL - 1) / EL, uv = min(lane % U, p.D / 16 - 1);
    uint32_t kw[2][NU][WK], ks[2][NU], vw[NV][WV], vs[NV];
    auto load_k = [&]() {
#pragma unroll
        for (int t = 0; t < 2; t++) {
            const uint8_t *at = kvh + offs[w][0][16 * t + n], *sat = sch + offs[w][1][16 * t + n];
#pragma unroll
            for (int u = 0; u < NU; u++) {
                const int un = min(g + 4 * u, units - 1);
                load_words(kw[t][u], at + un * (EL * BITS / 8));
                ks[t][u] = sat[un * EL / 32];
            }
        }
    };
    auto load_v = [&]() {
#pragma unroll
        for (int ii = 0; ii < NV; ii++) {
            const int key = lane / U + 64 / U * ii;
            load_words(vw[ii], kvh + offs[w][0][key] + (p.D + 16 * uv) * BITS / 8);
            vs[ii] = sch[offs[w][1][key] + p.S + uv / 2];
        }
    };
    const int first = t0 + w;
    int pg = 0;
    if (first < t1) {
        find_keys_mx(p, tile_at(ps.tl, first, KT), KT, load_page(first), offs[w][0], offs[w][1], ok, bad);
        pg = load_page(first + 4);
        load_k();
        load_v();
    }
    rows_start<bf16, DP, 1>(R, 0, raw, p.scale * kLog2e);
    for (int t = first; t < t1; t += 4) {
        const Tile tile = tile_at(ps.tl, t, KT);
        const uint64_t okc = ok, badc = bad;
        const bool more = t + 4 < t1;
        v4f s[2][1];
#pragma unroll
        for (int kk = 0; kk < DP / 32; kk++)
#pragma unroll
            for (int x = 0; x < 2; x++) {
                const mx_bf8 a = mx_eight<BITS>(&kw[x][kk / FU][kk % FU * (BITS / 4)], mx_scale(ks[x][kk / FU]));
#pragma unroll
                for (int j = Frag<bf16>::NQ - 1; j >= 0; j--)
                    s[x][0] = Frag<bf16>::mfma(a, R.q[0][kk][j], kk > 0 || j < Frag<bf16>::NQ - 1 ? s[x][0] : R.start(0));
            }
        if (more) {
            find_keys_mx(p, tile_at(ps.tl, t + 4, KT), KT, pg, offs[w][0], offs[w][1], ok, bad);
            pg = load_page(t + 8);
            load_k();
        }
        __builtin_amdgcn_sched_barrier(0);
        const bool part = !tile_whole(tile, KT, ps, p.window, p.n_first);
        if (part || badc) mask_scores<bf16, DP, 1, 2>(R, s, tile.k0, tile.ke, badc, p.window, p.n_first);
        softmax<bf16, DP, 1, 2>(R, s, va, []() {});
#pragma unroll
        for (int ii = 0; ii < NV; ii++) {
            const int key = lane / U + 64 / U * ii;
            const float f = mx_scale(vs[ii]);
            mx_bf8 lo = mx_eight<BITS>(&vw[ii][0], f), hi = mx_eight<BITS>(&vw[ii][WV / 2], f);
            // rows that were not there: no value of theirs may count
            if (!((okc >> key) & 1)) lo = hi = mx_bf8{};
            mx_bf8 *to = (mx_bf8 *)(Vs + 2 * key * DP + 16 * v_swz<CH>(key, 2 * (lane % U)));
            to[0] = lo;
            to[1] = hi;
        }
        if (more) load_v();
        __builtin_amdgcn_sched_barrier(0);
        values<bf16, DP, 1, 2>(R, va, s);
    }
    few_join<Alone<BITS>, bf16, DP>(p, R, (float *)lds.v, lds.ws, sq.nq * G, valid, table, tok, hd, pi, row + 3);
}

// How a tile comes into LDS: its codes go into registers, 16 elements a lane (load ii of wavefront
// w: unit idx % U of key 16 w + idx / U, idx = 64 ii + lane), and from there as bfloat16 into LDS.
template <int BITS>
struct Decoded {
    typedef Alone<BITS> Again;
    struct Lds {
        int64_t offs[4][2][64];
    };
    template <int DP>
    struct Loads {
        static constexpr int KT = 64, CH = DP / 8, U = DP / 16, NL = 16 * U / 64, W = BITS / 2;
        static_assert(2 * NL <= DP / 16, "one load under each of a half's fragments");
        const FapMxParams &p;
        Lds &lds;
        uint8_t (&kvs)[2][2][64 * DP * 2];
        const int32_t *row;
        int w, t1;
        const PagedTiles &tl;
        const uint8_t *kvh, *sch;
        uint64_t ok = 0, bad = 0, ok2 = 0, bad2 = 0;
        int pg[2];                        // page numbers of the tiles to be found next, a lane a key
        const uint8_t *at[NL], *sat[NL];  // this lane's rows of the tile found last
        uint32_t kw[NL][W], vw[NL][W], ks[NL], vs[NL];
        int unit;
        DEV_M Loads(const FapMxParams &p_, Lds &lds_, uint8_t (&kvs_)[2][2][64 * DP * 2], int hk, const int32_t *row_, int w_,
                    const PagedTiles &tl_, int t1_)
            : p(p_), lds(lds_), kvs(kvs_), row(row_), w(w_), t1(t1_), tl(tl_), kvh((const uint8_t *)p_.kv + hk * p_.kv_head),
              sch(p_.sc + hk * p_.sc_head), unit(min((int)(threadIdx.x & 63) % U, p_.D / 16 - 1)) {}
        DEV_M int key(int ii) const { return 16 * w + (64 * ii + (int)(threadIdx.x & 63)) / U; }
        DEV_M void load_pages(int t) {
            const Tile tile = tile_at(tl, min(t, t1 - 1), KT);
            const int j = min(tile.k0 + (int)(threadIdx.x & 63), tile.ke - 1);
            pg[0] = pg[1];
            pg[1] = row[3 + paged_div((uint32_t)j, p.by_page)];
        }
        DEV_M void find_tile(int t) {
            // (the pages loaded last are those of the tile after t)
            find_keys_mx(p, tile_at(tl, t, KT), KT, pg[0], lds.offs[w][0], lds.offs[w][1], ok2, bad2);
#pragma unroll
            for (int ii = 0; ii < NL; ii++) {
                at[ii] = kvh + lds.offs[w][0][key(ii)] + unit * (2 * BITS);
                sat[ii] = sch + lds.offs[w][1][key(ii)] + unit / 2;
            }
        }
        DEV_M void load_part(int t, int f) {
            if (f < NL) {
                load_words(kw[f], at[f]);
                ks[f] = *sat[f];
            } else if (f < 2 * NL) {
                load_words(vw[f - NL], at[f - NL] + p.D * BITS / 8);
                vs[f - NL] = sat[f - NL][p.S];
            }
        }
        DEV_M void load_tile(int t) {
#pragma unroll
            for (int f = 0; f < 2 * NL; f++) load_part(t, f);
        }
        DEV_M void loaded(int t) {
            const int u = (threadIdx.x & 63) % U;
#pragma unroll
            for (int ii = 0; ii < NL; ii++) {
                const int r = key(ii);
                const float kf = mx_scale(ks[ii]), vf = mx_scale(vs[ii]);
                uint8_t *K = kvs[t & 1][0] + 2 * r * DP, *V = kvs[t & 1][1] + 2 * r * DP;
                *(mx_bf8 *)(K + 16 * k_swz<CH>(r, 2 * u)) = mx_eight<BITS>(&kw[ii][0], kf);
                *(mx_bf8 *)(K + 16 * k_swz<CH>(r, 2 * u + 1)) = mx_eight<BITS>(&kw[ii][W / 2], kf);
                mx_bf8 lo = mx_eight<BITS>(&vw[ii][0], vf), hi = mx_eight<BITS>(&vw[ii][W / 2], vf);
                // rows that were not there: no value of theirs may count
                if (!((ok >> r) & 1)) lo = hi = mx_bf8{};
                *(mx_bf8 *)(V + 16 * v_swz<CH>(r, 2 * u)) = lo;
                *(mx_bf8 *)(V + 16 * v_swz<CH>(r, 2 * u + 1)) = hi;
            }
        }
    };
};

extern "C" __global__ void __launch_bounds__(256) ghip_fapq_join_8(FapMxParams p) { fap_join<Alone<8>>(p); }
extern "C" __global__ void __launch_bounds__(256) ghip_fapq_join_4(FapMxParams p) { fap_join<Alone<4>>(p); }

template <int BITS, int DP, int RW>
union FapqLds {
    FewqLds<DP> few;
    TileLds<Decoded<BITS>, DP, RW> tile;
};
#define FAPQ_FEW(B, DP, WG)                                                                            \
    extern "C" __global__ void __launch_bounds__(256, WG) ghip_fapq_few_##B##_##DP(FapMxParams p) {    \
        __shared__ __attribute__((aligned(1024))) uint8_t lds[sizeof(FewqLds<DP>)];                   \
        fapq_few<B, DP>(p, *(FewqLds<DP> *)lds);                                                      \
    }
// (R: rows of a workgroup, 64 RW)
#define FAPQ_TILE(B, DP, RW, R)                                                                                                 \
    extern "C" __global__ void __launch_bounds__(256, 2) ghip_fapq_tile##R##_##B##_##DP(FapMxParams p) {                         \
        __shared__ __attribute__((aligned(1024))) uint8_t lds[sizeof(TileLds<Decoded<B>, DP, RW>)];                              \
        fap_tile<Decoded<B>, bf16, DP, RW>(p, *(TileLds<Decoded<B>, DP, RW> *)lds);                                              \
    }                                                                                                                           \
    extern "C" __global__ void __launch_bounds__(256, 2) ghip_fapq_both##R##_##B##_##DP(FapMxParams p) {                         \
        __shared__ __attribute__((aligned(1024))) uint8_t lds[sizeof(FapqLds<B, DP, RW>)];                                       \
        if ((int)blockIdx.x < p.wg_sh) fap_tile<Decoded<B>, bf16, DP, RW>(p, *(TileLds<Decoded<B>, DP, RW> *)lds);               \
        else fapq_few<B, DP>(p, *(FewqLds<DP> *)lds);                                                                            \
    }
#define FAPQ_B(B)                                                                                                \
    FAPQ_FEW(B, 64, 2) FAPQ_FEW(B, 128, 2) FAPQ_FEW(B, 256, 1)                                                          \
    FAPQ_TILE(B, 64, 1, 64) FAPQ_TILE(B, 128, 1, 64) FAPQ_TILE(B, 256, 1, 64) FAPQ_TILE(B, 64, 2, 128)
FAPQ_B(8) FAPQ_B(4)
