// ghip_fapq.hip -- attention over a quantized paged KV cache (codes and scales of ghip_mx.h).
// The formula, tables, masks and partials are those of ghip_fap.hip.
//
// A code times its scale is exact in bfloat16, and where the scales are in a range in float16
// too, so the products are those over a 16-bit cache: q and p as three terms or, of float16 and where that
// costs no more than 32-bit arithmetic does (MxHalf), two; the error against 64 bits is that of 32-bit
// arithmetic (0.15 .. 0.8e-6), whatever the codes' own rounding cost.
//
// Up to 32 rows a KV head (decode, drafted tokens): fapq_few, bound by memory, 264 bytes a key and value of
// 128 dims in 8 bits, 136 in 4.  Long runs of keys reach 5.0 TB/s in 8 bits, what a large copy does;
// in 4 bits 3.9, held by the conversions.  A wavefront takes tiles of its own, so
// that nothing waits for the other three until the end, with the next tile's rows in registers.
//   24 sequences of 500 .. 16384 keys, 32 heads over 8 of 128, 8 bits: 101 us, 4.4 TB/s
//   64 sequences of 2000 .. 12000 keys, 4 bits: 125 us, 3.9 TB/s, once the card runs steadily
//   12 sequences of 5 or 6 drafted tokens, 900 .. 8192 keys, 8 bits: 44 us, 2.7 TB/s (20 of them launches, the
//   first tile's latencies and the join)
//
// More rows: tiles of 64 or 128 rows, bound by the products and the vector work beside them.
//   1702 rows of two prompts over 4000 .. 8192 keys, 8 bits: 400 us, 489 TFLOP/s of the formula's (two terms: twice
//   that on the matrix cores); four of 2048 rows over 8192 keys: 580
//   1290 rows of 64 heads over 8 of 64 in a window of 1024, 4 bits: 80 us
// A prefix that the batch shares takes the tiles, the sequences' own keys the other way, in one launch:
//   64 sequences over 8192 shared and 40 .. 600 own keys, 8 bits: 46 us with the join
#include "ghip_fap_core.h"
#include "ghip_mx.h"

// (kv_head, kv_row, kv_page count bytes)
struct FapMxParams : FapParams {
    const uint8_t *sc;
    int64_t sc_head, sc_row, sc_page;
    int S;         // scale bytes of a key
    int together;  // few rows: the heads of the same keys follow one another on one XCD
    int wgs;       // ... workgroups of a head, which share out the sequences' tiles; 0: zs_own a sequence
    int least;     // ... tiles of a workgroup at least
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
DEV void find_keys_mx(const FapMxParams &p, const Tile &tl, int kt, int pg, int64_t *offs, int64_t *soffs, uint64_t &ok, uint64_t &bad,
                      bool any = true) {
    const int lane = threadIdx.x & 63;
    const uint32_t j = tl.k0 + lane;
    const bool in = any && lane < kt && (int)j < tl.ke;
    const bool there = in && pg >= 0 && pg < p.n_pages;
    ok = __ballot(there);
    bad = __ballot(in && !there);
    const int64_t r = j - paged_div(j, p.by_page) * (uint32_t)p.page;
    if (lane < kt) {
        offs[lane] = there ? pg * p.kv_page + r * p.kv_row : 0;
        soffs[lane] = there ? pg * p.sc_page + r * p.sc_row : 0;
    }
}
// Words and bytes of the cache.  The address has been through LDS, and of that the compiler cannot
// tell that it is not LDS itself: said to be global memory, or the loads count as LDS's too
// and each wait for LDS waits for memory (24 sequences of 500 .. 16384 keys: 118 us, 108 without).
typedef const __attribute__((address_space(1))) uint8_t *in_memory;
template <int W>
DEV void load_words(uint32_t (&w)[W], const uint8_t *from) {
    typedef uint32_t words __attribute__((ext_vector_type(W)));
    const words x = *(const __attribute__((address_space(1))) words *)from;
#pragma unroll
    for (int i = 0; i < W; i++) w[i] = x[i];
}
DEV uint32_t load_byte(const uint8_t *from) { return *(in_memory)from; }

// ---- up to 16 RW rows a KV head: 4 wavefronts, each its own tiles of KT keys

// 64 keys a tile are twice the bytes in flight and half the work of finding them; of 8-bit codes
// they are too many registers for three wavefronts a SIMD.
constexpr int few_keys(int bits, int DP) { return DP == 256 || bits == 8 ? 32 : 64; }

// Which part of the keys a workgroup takes: split z (of `of`) of sequence b, its tiles [t0, t1).
// With p.wgs the sequences' tiles are shared out over that many workgroups, each sequence having
// as many splits as its tiles are worth: of splits alike for all, the longest sequence's are the last to
// end (24 sequences of 500 .. 16384 keys: 108 us, 102 so).
struct Part {
    int b, z, of, t0, t1;
};
// sums over the lanes up to and with each; lane 63: over all
DEV int lane_sums(int x) {
    x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false);  // of the lane 1 before in a row of 16, 2, 4, 8
    x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);  // of rows 0 and 2 to the next
    x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);  // of the first two rows to the others
    return x;
}
DEV int lane_sum(int x) { return __builtin_amdgcn_readlane(lane_sums(x), 63); }
// the largest of all lanes, x >= 0
DEV int lane_max(int x) {
    x = max(x, __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false));
    x = max(x, __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false));
    x = max(x, __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false));
    x = max(x, __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false));
    x = max(x, __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false));
    x = max(x, __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false));
    return __builtin_amdgcn_readlane(x, 63);
}
template <int KT>
DEV bool find_part(const FapMxParams &p, int no, Part &w) {
    const int lane = threadIdx.x & 63;
    const int64_t table = (int64_t)p.per * p.page;
    // a sequence's tiles; one at least, whose workgroup says that the rows see nothing
    auto tiles_of = [&](int b) {
        const PagedSeq sq = seq_of(p, b);
        if (sq.nq == 0) return 0;
        return max(1, paged_tiles(clip_pos(sq.pos0, table), clip_pos(sq.pos0 + sq.nq - 1, table), p.window, p.n_first, p.n_shared, (int)table, KT).n);
    };
    if (!p.wgs) {
        w.b = no / p.zs_own;
        w.z = no - w.b * p.zs_own;
        w.of = p.zs_own;
        if (w.b >= p.B) return false;
        const int n = tiles_of(w.b), share = paged_share(n, w.of);
        w.t0 = (int)min((int64_t)w.z * share, (int64_t)n);
        w.t1 = min(n, w.t0 + share);
        return n > 0;
    }
    int64_t total = 0;
    int live = 0;
    const int first = lane < p.B ? tiles_of(lane) : 0;
    for (int b0 = 0; b0 < p.B; b0 += 64) {
        const int n = b0 == 0 ? first : b0 + lane < p.B ? tiles_of(b0 + lane) : 0;
        live += __popcll(__ballot(n > 0));
        total += (uint32_t)lane_sum(n);  // (2^25 tiles each at most)
    }
    // The fewest tiles a part that need no more parts than there are workgroups: with total / (wgs - live)
    // they never do; up to 64 sequences the least is looked for.
    const int64_t room = max(p.wgs - live, 1);
    int64_t each = max((total + room - 1) / room, (int64_t)p.least);
    if (p.B <= 64) {
        int lo = max((int)((total + p.wgs - 1) / p.wgs), p.least), hi = (int)each;
        while (lo < hi) {
            const int mid = (lo + hi) / 2;
            if (lane_sum((first + mid - 1) / mid) <= p.wgs) hi = mid;
            else lo = mid + 1;
        }
        each = hi;
    }
    int base = 0;
    for (int b0 = 0; b0 < p.B && base <= no; b0 += 64) {
        const int n = b0 == 0 ? first : b0 + lane < p.B ? tiles_of(b0 + lane) : 0;
        const int parts = (int)min((n + each - 1) / each, (int64_t)p.zs_own);
        const int to = lane_sums(parts);
        const uint64_t here = __ballot(base + to - parts <= no && no < base + to);
        if (here) {
            const int at = __builtin_ctzll(here), tiles = __builtin_amdgcn_readlane(n, at);
            w.b = b0 + at;
            w.of = __builtin_amdgcn_readlane(parts, at);
            w.z = no - base - __builtin_amdgcn_readlane(to - parts, at);
            const int share = paged_share(tiles, w.of);
            w.t0 = (int)min((int64_t)w.z * share, (int64_t)tiles);
            w.t1 = min(tiles, w.t0 + share);
            return true;
        }
        base += __builtin_amdgcn_readlane(to, 63);
    }
    return false;
}

// The products have 16 columns for rows.  Where there are 16 / CG rows at most, the columns are CG
// groups of them: group j has term j of q and of p, and one product does what takes three (CG 4; its
// fourth group is not used) or two of three (CG 2: the third term in a product of its own, group 1).
// A score is then the sum over the groups, taken pair by pair so that all have the same bits.
template <int CG>
DEV float all_groups(float x) {
    if (CG > 1) x += __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(x), 0x128, 0xf, 0xf, true));  // the lane 8 on, of 16
    if (CG > 2) x += __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(x), 0x124, 0xf, 0xf, true));  // 4 on
    return x;
}
// products for the three terms
template <int CG>
constexpr int few_products() { return CG == 4 ? 1 : CG == 2 ? 2 : 3; }
// x's term for this lane's group in each product; j1, j2: 1 in the groups that leave the first term
// (and the second) to others, else 0
template <int CG>
DEV void group_terms(v2f x, float j1, float j2, Frag<bf16>::v2 (&t)[few_products<CG>()]) {
    typedef Frag<bf16>::v2 v2;
    if constexpr (CG == 1) {
        split_pair<bf16, 3>(x[0], x[1], t);
    } else {
        v2 y = __builtin_convertvector(x, v2);
#pragma unroll
        for (int k = 0; k < 2; k++) x[k] = fmaf((float)y[k], -j1, x[k]);
        y = __builtin_convertvector(x, v2);
        if (CG == 2) t[0] = y;
#pragma unroll
        for (int k = 0; k < 2; k++) x[k] = CG == 2 ? fmaf((float)y[k], -1.0f, x[k]) * j1 : fmaf((float)y[k], -j2, x[k]);
        t[few_products<CG>() - 1] = __builtin_convertvector(x, v2);
    }
}
// O^T += V^T P^T over 32 keys at Vs, p a group's terms
template <int DP, int CG>
DEV void group_values(v4f (&o)[DP / 16], uint32_t Vs, const v4f &s0, const v4f &s1, float j1, float j2) {
    typedef Frag<bf16> F;
    constexpr int NM = few_products<CG>();
    const uint32_t vat = v_at<DP>(Vs);
    F::v8 p[NM];
#pragma unroll
    for (int e = 0; e < 4; e++) {
        const v4f &s = e < 2 ? s0 : s1;
        F::v2 t[NM];
        group_terms<CG>(v2f{s[2 * (e & 1)], s[2 * (e & 1) + 1]}, j1, j2, t);
#pragma unroll
        for (int i = 0; i < NM; i++) {
            p[i][2 * e] = t[i][0];
            p[i][2 * e + 1] = t[i][1];
        }
    }
    F::v8 a[3];
    a[0] = value_frag<bf16, DP>(vat, 0, 0);
    a[1] = value_frag<bf16, DP>(vat, 0, 1);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int dt = 0; dt < DP / 16; dt++) {
        if (dt + 2 < DP / 16) a[(dt + 2) % 3] = value_frag<bf16, DP>(vat, 0, dt + 2);
#pragma unroll
        for (int i = NM - 1; i >= 0; i--) o[dt] = F::mfma(a[dt % 3], p[i], o[dt]);
        __builtin_amdgcn_sched_barrier(0);
    }
}

// A tile's rows (a key's codes, then its value's) as they lie, 16-byte chunk c of row r at place raw_swz of CH:
// reads of one chunk of 16 rows then touch each bank once.
template <int CH>
DEV int raw_swz(int r, int c) {
    return CH == 4 ? c ^ ((r >> 2) & 3) : CH == 8 ? c ^ ((r >> 1) & 7) : c ^ (r & 15);
}
template <int BITS, int DP, int CG, int RW>
struct FewqLds {
    uint8_t v[4][64 * DP + (CG == 1 ? 256 : 0)];         // each wavefront's rows as they lie, then 32 values as bfloat16; at the end its sums
    uint8_t q[RW][DP / 32][few_products<CG>()][1024];    // the fragments of q, the same for all wavefronts
    int64_t offs[4][2][few_keys(BITS, DP)];
    uint8_t sc[4][few_keys(BITS, DP)][DP / 16];  // a tile's scales: a row of 2 S bytes for each key
    float ws[4][2][16];
};
template <int BITS, int DP, int CG, int RW>
DEV void fapq_few(const FapMxParams &p, FewqLds<BITS, DP, CG, RW> &lds) {
    static_assert(RW == 1 || CG == 1, "more than 16 rows have no columns to spare");
    // A lane's codes of a key: NU units of EL elements, unit g + 4 i; fragment kk of the products takes 8 of
    // them, and so does q's.
    constexpr int KT = few_keys(BITS, DP), NT = KT / 16, CH = DP / 8, EL = BITS == 4 && DP >= 128 ? 32 : 16, NU = DP / EL / 4, FU = EL / 8,
                  WK = EL * BITS / 32;
    // ... of the values: unit lane % U of keys lane / U + (64 / U) ii, NVH loads for 32 keys
    constexpr int U = DP / 16, NV = KT * U / 64, NVH = U / 2, WV = BITS / 2;
    constexpr int SB = DP / 16;  // bytes of a key's and its value's scales (of up to 32 dims: half of that)
    constexpr int NM = few_products<CG>(), ROWS = 16 / CG;
    auto &offs = lds.offs;
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n = lane & 15, g = lane >> 4;
    const int G = p.H / p.H_kv;
    const int64_t table = (int64_t)p.per * p.page;
    const int id = blockIdx.x - p.wg_sh, k = p.together ? id >> 3 : id, hk = k % p.H_kv;
    Part part;
    if (!find_part<KT>(p, p.together ? (k / p.H_kv) * 8 + (id & 7) : k / p.H_kv, part)) return;
    const int32_t *row = p.seqs + (int64_t)part.b * p.seq_nb1;
    const PagedSeq sq = paged_seq(row[0], row[1], row[2], p.T, p.max_q);
    Pass ps;
    ps.p0 = clip_pos(sq.pos0, table);
    ps.p1 = clip_pos(sq.pos0 + sq.nq - 1, table);
    ps.tl = paged_tiles(ps.p0, ps.p1, p.window, p.n_first, p.n_shared, (int)table, KT);
    const int t0 = part.t0, t1 = min(part.t1, ps.tl.n);
    // this lane's row of row tile rt
    const int j = n / ROWS;
    struct Row {
        int hd, i;
        bool there, valid;  // is there one; does the lane stand for it
        int64_t tok, pi;
    };
    auto row_of = [&](int rt) {
        Row y;
        const int r = 16 * rt + n % ROWS;
        y.i = r / G;
        y.hd = hk * G + r % G;
        y.there = r < sq.nq * G;
        y.valid = y.there && j == 0;
        y.tok = sq.q0 + (y.there ? y.i : 0);
        y.pi = (y.tok * p.H + y.hd) * (p.zs_sh + p.zs_own) + p.zs_sh + part.z;
        return y;
    };
    Rows<bf16, DP, RW> R;  // (its q: in LDS)
#pragma unroll
    for (int rt = 0; rt < RW; rt++) {
        const Row y = row_of(rt);
        if (part.z == part.of - 1 && y.valid)  // no more splits of this sequence
            for (int z = part.of + 4 * w + g; z < p.zs_own; z += 16) stat_none(p, y.pi - part.z + z, sq.pos0 + y.i >= table);
        if (t0 >= t1 && p.part && y.valid && w == 0 && g == 0) stat_none(p, y.pi, sq.pos0 + y.i >= table);
        R.pos[rt] = y.there ? clip_pos(sq.pos0 + y.i, table) : -1;
        R.mneg[rt] = v4f{0, 0, 0, 0};
        R.l[rt] = 0.0f;
        R.from[rt] = R.pos[rt] < 0 ? -__builtin_inff() : __builtin_inff();
#pragma unroll
        for (int dt = 0; dt < DP / 16; dt++) R.o[rt][dt] = v4f{0, 0, 0, 0};
    }
    if (t0 >= t1 && p.part) return;  // nothing in this split
    const float j1 = j >= 1, j2 = j >= 2;
    // q: loaded here, worked on when the first tile is on its way
    constexpr int NF = RW * DP / 32, QF = (NF + 3) / 4;
    float x[QF][8];
#pragma unroll
    for (int i = 0; i < QF; i++) {
        const int f = min(w + 4 * i, NF - 1), rt = f / (DP / 32), kk = f % (DP / 32), d = EL * (g + 4 * (kk / FU)) + 8 * (kk % FU);
        const Row y = row_of(rt);
#pragma unroll
        for (int e = 0; e < 8; e++) x[i][e] = 0.0f;
        if (y.there && d < p.D && j < 3) __builtin_memcpy(x[i], p.q + y.tok * p.q_nb2 + y.hd * p.q_nb1 + d, 32);
    }
    const uint8_t *kvh = (const uint8_t *)p.kv + hk * p.kv_head, *sch = p.sc + hk * p.sc_head;
    uint8_t *Vs = lds.v[w];
    const uint32_t va = lds_addr(Vs);

    auto load_page = [&](int t) {  // page number of a key of tile t, a lane each
        const Tile tl = tile_at(ps.tl, min(t, t1 - 1), KT);
        return row[3 + paged_div((uint32_t)min(tl.k0 + lane, tl.ke - 1), p.by_page)];
    };
    uint64_t ok = 0, bad = 0;  // the next tile's keys that are there, those on no page
    const int units = (p.D + EL - 1) / EL, uv = min(lane % U, p.D / 16 - 1);
    // A tile is loaded as whole rows, 16 bytes a lane and a row's bytes in neighbouring lanes (loads of the
    // fragments' own places, 64 bytes of a line each, were twice the requests: 64 sequences of
    // 8192 keys in 4 bits: 162 us, 140 so), and goes through LDS to the lanes that need it.
    constexpr int RCH = DP * BITS / 64, RS = 16 * RCH, KPI = 64 / RCH, NLD = KT / KPI;
    uint32_t st[NLD][4], sc[SB / 4];  // (sc: a lane a key)
    const int chunk = 16 * min(lane % RCH, p.D * BITS / 64 - 1);
    auto load_tile = [&]() {
#pragma unroll
        for (int ii = 0; ii < NLD; ii++) {
            load_words(st[ii], kvh + offs[w][0][lane / RCH + KPI * ii] + chunk);
            if (ii & 1) __builtin_amdgcn_sched_barrier(0);
        }
        const uint8_t *at = sch + offs[w][1][lane % KT];
        if constexpr (DP == 64) {
            typedef const __attribute__((address_space(1))) uint16_t *halves;
            sc[0] = *(halves)at | (uint32_t)*(halves)(at + (p.S & 2)) << 16;
        } else {
            load_words(sc, at);
        }
    };
    // (a later load's row differs in bits of its own, and so does its swizzle)
    const int rkey = lane / RCH, rto = rkey * RS + 16 * raw_swz<RCH>(rkey, lane % RCH);
    // the scales go through LDS, from where each lane reads the byte that it needs
    const int vkey = lane / U, vto = 2 * vkey * DP + 16 * v_swz<CH>(vkey, 2 * (lane % U));  // of load 0: a later one's row differs in bits of its own
    const uint8_t *scw = &lds.sc[w][0][0];
    const int vat = p.D * BITS / 8 + uv * 2 * BITS, vfrom = vkey * RS + 16 * raw_swz<RCH>(vkey, vat / 16) + vat % 16;
    const int first = t0 + w;
    int pg = 0;
    if (first < t1) {
        find_keys_mx(p, tile_at(ps.tl, first, KT), KT, load_page(first), offs[w][0], offs[w][1], ok, bad);
        pg = load_page(first + 4);
        load_tile();
    }
#pragma unroll
    for (int i = 0; i < QF; i++) {
        const int f = w + 4 * i, rt = f / (DP / 32), kk = f % (DP / 32);
        if (f >= NF) break;
        Frag<bf16>::v8 terms[NM];
#pragma unroll
        for (int e = 0; e < 4; e++) {
            Frag<bf16>::v2 t[NM];
            group_terms<CG>(v2f{x[i][2 * e], x[i][2 * e + 1]} * (p.scale * kLog2e), j1, j2, t);
#pragma unroll
            for (int m = 0; m < NM; m++) {
                terms[m][2 * e] = t[m][0];
                terms[m][2 * e + 1] = t[m][1];
            }
        }
#pragma unroll
        for (int m = 0; m < NM; m++) *(Frag<bf16>::v8 *)&lds.q[rt][kk][m][16 * lane] = terms[m];
    }
    __syncthreads();
    for (int t = first; t < t1; t += 4) {
        const Tile tile = tile_at(ps.tl, t, KT);
        const uint64_t okc = ok, badc = bad;
#pragma unroll
        for (int ii = 0; ii < NLD; ii++)
            __builtin_memcpy(Vs + (rto ^ (16 * raw_swz<RCH>(KPI * ii, 0))) + KPI * ii * RS, st[ii], 16);
        if (KT == 64 || lane < KT) __builtin_memcpy(lds.sc[w][lane % KT], sc, SB);
        // The next tile's loads, after the last one too (then all of one row): with branches around them the
        // compiler cannot count them and waits for all.
        find_keys_mx(p, tile_at(ps.tl, t + 4, KT), KT, pg, offs[w][0], offs[w][1], ok, bad, t + 4 < t1);
        pg = load_page(t + 8);
        load_tile();
        __builtin_amdgcn_sched_barrier(0);
        const uint8_t *kscale[NU], *kraw[NU], *vscale = scw + vkey * SB + p.S + uv / 2;
#pragma unroll
        for (int u = 0; u < NU; u++) {
            const int un = min(g + 4 * u, units - 1), at = un * (EL * BITS / 8);
            kscale[u] = scw + n * SB + un * EL / 32;
            kraw[u] = Vs + n * RS + 16 * raw_swz<RCH>(n, at / 16) + at % 16;
        }
        // (the reference: in one group)
        v4f start[RW];
#pragma unroll
        for (int rt = 0; rt < RW; rt++) {
            const float ref = CG == 1 || j == 0 ? R.mneg[rt][0] : 0.0f;
            start[rt] = CG == 1 ? R.mneg[rt] : v4f{ref, ref, ref, ref};
        }
        v4f s[NT][RW];
#pragma unroll
        for (int u = 0; u < NU; u++) {
            float f[NT];
            uint32_t kw[NT][WK];
#pragma unroll
            for (int x = 0; x < NT; x++) {
                f[x] = mx_scale(kscale[u][16 * x * SB]);
                __builtin_memcpy(kw[x], kraw[u] + 16 * x * RS, 4 * WK);
            }
#pragma unroll
            for (int e = 0; e < FU; e++) {
                const int kk = u * FU + e;
                Frag<bf16>::v8 q[RW][NM];
#pragma unroll
                for (int rt = 0; rt < RW; rt++)
#pragma unroll
                    for (int m = 0; m < NM; m++) q[rt][m] = *(const Frag<bf16>::v8 *)&lds.q[rt][kk][m][16 * lane];
#pragma unroll
                for (int x = 0; x < NT; x++) {
                    const mx_bf8 a = mx_eight<BITS>(&kw[x][e * (BITS / 4)], f[x]);
#pragma unroll
                    for (int m = NM - 1; m >= 0; m--)
#pragma unroll
                        for (int rt = 0; rt < RW; rt++)
                            s[x][rt] = Frag<bf16>::mfma(a, q[rt][m], kk > 0 || m < NM - 1 ? s[x][rt] : start[rt]);
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
        }
        uint32_t vw[NV][WV];
#pragma unroll
        for (int ii = 0; ii < NV; ii++)
            __builtin_memcpy(vw[ii], Vs + (vfrom ^ (16 * raw_swz<RCH>(64 / U * ii, 0))) + 64 / U * ii * RS, 4 * WV);
        __builtin_amdgcn_sched_barrier(0);
        if constexpr (CG > 1)
#pragma unroll
            for (int x = 0; x < NT; x++)
#pragma unroll
                for (int v = 0; v < 4; v++) s[x][0][v] = all_groups<CG>(s[x][0][v]);
        if (badc || !tile_whole(tile, KT, ps, p.window, p.n_first)) mask_scores<bf16, DP, RW, NT>(R, s, tile.k0, tile.ke, badc, p.window, p.n_first);
        softmax<bf16, DP, RW, NT>(R, s, va, []() {});
        // 32 values at a time through LDS
#pragma unroll
        for (int h = 0; h < KT / 32; h++) {
#pragma unroll
            for (int ii = h * NVH; ii < (h + 1) * NVH; ii++) {
                const float f = mx_scale(vscale[64 / U * ii * SB]);
                mx_bf8 *to = (mx_bf8 *)(Vs + (vto ^ (16 * v_swz<CH>(64 / U * ii, 0))) + 64 / U * (ii - h * NVH) * 2 * DP);
                to[0] = mx_eight<BITS>(&vw[ii][0], f);
                to[1] = mx_eight<BITS>(&vw[ii][WV / 2], f);
            }
            // rows that were not there: no value of theirs may count
            if (const uint32_t miss = ~(uint32_t)(okc >> (32 * h))) {
                int l = lane;
                asm volatile("" : "+v"(l));  // (or what follows is worked out before the loop, into registers that the loop needs)
                for (int c = l; c < 32 * CH; c += 64)
                    if ((miss >> (c / CH)) & 1) *(uint4 *)(Vs + 16 * c) = make_uint4(0, 0, 0, 0);
            }
            __builtin_amdgcn_sched_barrier(0);
            uint32_t at = va;
            asm volatile("" : "+v"(at));  // (the fragments' addresses likewise)
            if constexpr (CG > 1) {
                group_values<DP, CG>(R.o[0], at, s[2 * h][0], s[2 * h + 1][0], j1, j2);
            } else {
                v4f y[2][RW];
#pragma unroll
                for (int rt = 0; rt < RW; rt++) {
                    y[0][rt] = s[2 * h][rt];
                    y[1][rt] = s[2 * h + 1][rt];
                }
                values<bf16, DP, RW, 2>(R, at, y);
            }
        }
    }
    if constexpr (CG > 1) {
#pragma unroll
        for (int dt = 0; dt < DP / 16; dt++)
#pragma unroll
            for (int v = 0; v < 4; v++) R.o[0][dt][v] = all_groups<CG>(CG == 4 && j == 3 ? 0.0f : R.o[0][dt][v]);
    }
    static_assert(sizeof(lds.v) >= ((3 * 16 + 16 / CG - 1) * (DP + 4) + DP) * 4, "the wavefronts' rows fit their values");
#pragma unroll
    for (int rt = 0; rt < RW; rt++) {
        const Row y = row_of(rt);
        if (rt) __syncthreads();  // (the sums of the row tile before have been read)
        few_join<Alone<BITS>, bf16, DP, RW>(p, R, rt, (float *)lds.v, lds.ws, sq.nq * G - 16 * rt, y.valid, table, y.tok, y.hd, y.pi, row + 3);
    }
}

// How a tile comes into LDS: its codes go into registers, 16 elements a lane (load ii of wavefront
// w: unit idx % U of key 16 w + idx / U, idx = 64 ii + lane), and from there as bfloat16 into LDS.
template <int BITS, typename E>
struct Decoded {
    typedef Alone<BITS> Again;
    typedef MxHalf<BITS> Half;
    static constexpr bool NARROW = Frag<E>::SCALED, LATE = true;
    static constexpr int HOME_K = NARROW ? Half::HOME : 0;
    struct Lds {
        int64_t offs[4][2][64];
        // Of the tiles in this place so far: the largest scale's byte of keys, or more where float16 will not do; the largest
        // and 255 less the smallest of values.  And 127 less k of the rows.
        alignas(16) int seen[2][4];
        int news[2]; // the last one's number, and one, where `seen` of it holds more than what was known
    };
    static DEV_M void start(Lds &l) {
        if (threadIdx.x < 8) l.seen[threadIdx.x / 4][threadIdx.x % 4] = 0;
        if (threadIdx.x < 2) l.news[threadIdx.x] = 0;
    }
    typedef typename Frag<E>::v8 v8;
    template <int DP>
    struct Loads {
        static constexpr int KT = 64, CH = DP / 8, U = DP / 16, NL = 16 * U / 64, W = BITS / 2;
        const FapMxParams &p;
        Lds &lds;
        uint8_t (&kvs)[2][2][64 * DP * 2];
        const int32_t *row;
        int w, t1;
        const PagedTiles &tl;
        const uint8_t *kvh, *sch;
        uint64_t ok = 0, bad = 0, ok2 = 0, bad2 = 0;
        int pg[2];                        // page numbers of the tiles to be found next, a lane a key
        // keys, then values, of the tile on its way
        uint32_t x[NL][W], sc[NL];
        // What tiles up to this one have had, in one scalar register, a byte each: keys' scales from Half::KEYS on, values' least
        // scale and how many there are from it on.
        uint32_t known = 0;
        DEV_M Loads(const FapMxParams &p_, Lds &lds_, uint8_t (&kvs_)[2][2][64 * DP * 2], int hk, const int32_t *row_, int w_,
                    const PagedTiles &tl_, int t1_)
            : p(p_), lds(lds_), kvs(kvs_), row(row_), w(w_), t1(t1_), tl(tl_), kvh((const uint8_t *)p_.kv + hk * p_.kv_head),
              sch(p_.sc + hk * p_.sc_head) {}
        DEV_M void rows_at(int k) {
            const int x = lane_max(127 - k), i = threadIdx.x & 63;
            if (i < 2) atomicMax(&lds.seen[i][3], x);
        }
        // (said before the last barrier; the next to say it in this place do so behind the next barrier)
        DEV_M bool beyond(int t) {
            if (__builtin_expect(__builtin_amdgcn_readfirstlane(lds.news[t & 1]) != t + 1, 1)) return false;
            const int4 s = *(const int4 *)lds.seen[t & 1];
            const int keys = max((int)(known & 255) + Half::KEYS - 1, __builtin_amdgcn_readfirstlane(s.x)), n = known >> 16,
                      from = min(n ? (int)(known >> 8) & 255 : 255, 255 - __builtin_amdgcn_readfirstlane(s.z)),
                      to = max(n ? ((int)(known >> 8) & 255) + n - 1 : 0, __builtin_amdgcn_readfirstlane(s.y));
            known = max(to - from + 1, 0) << 16 | from << 8 | (keys + 1 - Half::KEYS);
            return keys > Half::largest_scale(127 - __builtin_amdgcn_readfirstlane(s.w), p.D) || to - from > Half::APART;
        }
        // Is one of the codes of a unit's block, whose other half lane ^ 1 has, STRONG or more?
        static DEV_M bool strong(const uint32_t (&x)[W]) {
            const int y = (int)Half::strong(x);
            return (y | __builtin_amdgcn_mov_dpp(y, 0xB1, 0xf, 0xf, true)) != 0;
        }
        // What decides about float16 of a tile's keys (values), a lane's units.  Hardly ever more than the comparisons with
        // what is known; then those of rows that are there.
        DEV_M void look(int t, int kv, uint64_t ok, const uint32_t (&x)[NL][W], const uint32_t (&sc)[NL]) {
            const uint32_t least = kv ? (known >> 8) & 255 : Half::KEYS, n = kv ? known >> 16 : known & 255;
            uint32_t most = 0;
            bool news = false;
#pragma unroll
            for (int ii = 0; ii < NL; ii++) {
                most = max(most, sc[ii] - least);
                if (kv) news |= !strong(x[ii]);
            }
            if (__builtin_expect(!__ballot(news || most >= n), 1)) return;
            const int l = lane();
            auto there = [&](int ii) { return ((ok >> (16 * w + (64 * ii + l) / U)) & 1) != 0; };
            int to = 0, from = 0, no = 0;
#pragma unroll
            for (int ii = 0; ii < NL; ii++) {
                const int b = (int)sc[ii];
                const bool weak = kv && !strong(x[ii]), counts = there(ii) && (kv || Half::any(x[ii]) || b == 255);
                to = max(to, counts ? b : 0);
                from = max(from, counts ? 255 - b : 0);
                no = counts && (weak || b < (kv ? Half::VALUES : Half::KEYS) || b > Half::TO) ? 256 : no;
            }
            // (one lane for all: 64 atomics on one place take their turns)
            no = lane_max(kv ? no : max(no, to));
            if (kv) {
                to = lane_max(to);
                from = lane_max(from);
            }
            if (l == 0) {
                int *seen = lds.seen[t & 1];
                lds.news[t & 1] = t + 1;
                if (no) atomicMax(&seen[0], no);
                if (kv) {
                    atomicMax(&seen[1], to);
                    atomicMax(&seen[2], from);
                }
            }
        }
        // (the lane as if it were another each time: or the addresses in LDS are worked out before the loop, into
        // registers that the loop needs; 9 would spill)
        static DEV_M int lane() {
            int l = threadIdx.x & 63;
            asm volatile("" : "+v"(l));
            return l;
        }
        DEV_M void load_pages(int t) {
            const Tile tile = tile_at(tl, min(t, t1 - 1), KT);
            const int j = min(tile.k0 + (int)(threadIdx.x & 63), tile.ke - 1);
            pg[0] = pg[1];
            pg[1] = row[3 + paged_div((uint32_t)j, p.by_page)];
        }
        DEV_M void find_tile(int t) {
            // (the pages loaded last are those of the tile after t)
            find_keys_mx(p, tile_at(tl, t, KT), KT, pg[0], lds.offs[w][0], lds.offs[w][1], ok2, bad2);
        }
        DEV_M void load_unit(int kv, int ii, uint32_t (&to)[W], uint32_t &scale) {
            const int l = threadIdx.x & 63, key = 16 * w + (64 * ii + l) / U, unit = min(l % U, p.D / 16 - 1);
            load_words(to, kvh + lds.offs[w][0][key] + unit * (2 * BITS) + (kv ? p.D * BITS / 8 : 0));
            scale = load_byte(sch + lds.offs[w][1][key] + unit / 2 + (kv ? p.S : 0));
        }
        DEV_M void load_part(int, int) {}
        // (before a half's products: among them they cost more, 1702 rows over 4000 .. 8192 keys 415 and 403 us)
        DEV_M void load_half(int, int kv) {
#pragma unroll
            for (int ii = 0; ii < NL; ii++) load_unit(kv, ii, x[ii], sc[ii]);
        }
        DEV_M void load_first(int t) {
            uint32_t y[NL][W], ysc[NL];
#pragma unroll
            for (int ii = 0; ii < NL; ii++) load_unit(0, ii, y[ii], ysc[ii]);
            load_half(t, 1);
            decode(t, 0, ok2, y, ysc);
        }
        DEV_M void middle(int t) { decode(t, 0, ok2, x, sc); }
        DEV_M void loaded(int t) { decode(t, 1, ok, x, sc); }
        DEV_M void decode(int t, int kv, uint64_t ok, const uint32_t (&x)[NL][W], const uint32_t (&sc)[NL]) {
            const int l = lane(), u = l % U;
            if constexpr (NARROW) {
                look(t, kv, ok, x, sc);
                __builtin_amdgcn_sched_barrier(0);
            }
#pragma unroll
            for (int ii = 0; ii < NL; ii++) {
                const int r = 16 * w + (64 * ii + l) / U;
                const bool there = (ok >> r) & 1;
                // (past float16's range 0 is to stay 0)
                const float f = mx_scale(NARROW ? min(sc[ii] + HOME_K, 254u) : sc[ii]);
                v8 lo = mx_eight<BITS>(&x[ii][0], f, v8{}), hi = mx_eight<BITS>(&x[ii][W / 2], f, v8{});
                // rows that were not there: no value of theirs may count
                if (!there) lo = hi = v8{};
                uint8_t *to = kvs[t & 1][kv] + 2 * r * DP;
                *(v8 *)(to + 16 * (kv ? v_swz<CH>(r, 2 * u) : k_swz<CH>(r, 2 * u))) = lo;
                *(v8 *)(to + 16 * (kv ? v_swz<CH>(r, 2 * u + 1) : k_swz<CH>(r, 2 * u + 1))) = hi;
            }
        }
    };
};

// Tiles of 64 BW rows: as float16, two terms of q and p, and where that does not do for the keys and values so
// far (MxHalf) once more as bfloat16, three terms: the workgroup stops at such a tile and starts again.
// (1702 rows over 4000 .. 8192 keys, 8 bits: 568 us as bfloat16 alone, 535 as float16 with 64 rows, 400 with 128,
// whose fragments each serve four products.  All blocks out of range: 625, the two halves of 128 rows one after the
// other as bfloat16; one block, of a late key of each sequence: 957, which is both passes.)
template <int BITS, int DP, int BW>
union FapqTileLds {
    TileLds<Decoded<BITS, f16>, DP, BW> half;
    TileLds<Decoded<BITS, bf16>, DP, BW> wide;
};
template <int BITS, int DP, int BW>
DEV void fapq_tile(const FapMxParams &p, FapqTileLds<BITS, DP, BW> &lds) {
    Decoded<BITS, f16>::start(lds.half.ld);
    if (!fap_tile<Decoded<BITS, f16>, f16, DP, BW>(p, lds.half)) return;
    for (int half = 0; half < BW; half++) {  // (what the registers hold of three terms)
        __syncthreads();
        fap_tile<Decoded<BITS, bf16>, bf16, DP, 1, BW>(p, lds.wide, half);
    }
}

extern "C" __global__ void __launch_bounds__(256) ghip_fapq_join_8(FapMxParams p) { fap_join<Alone<8>>(p); }
extern "C" __global__ void __launch_bounds__(256) ghip_fapq_join_4(FapMxParams p) { fap_join<Alone<4>>(p); }

template <int BITS, int DP, int RW>
union FapqLds {
    FewqLds<BITS, DP, 1, 1> few;
    FapqTileLds<BITS, DP, RW> tile;
};
// (ROWS: up to how many, 16 RW / CG; WG: workgroups a CU)
#define FAPQ_FEW(B, DP, CG, RW, ROWS, WG)                                                                          \
    extern "C" __global__ void __launch_bounds__(256, WG) ghip_fapq_few##ROWS##_##B##_##DP(FapMxParams p) {        \
        __shared__ __attribute__((aligned(1024))) uint8_t lds[sizeof(FewqLds<B, DP, CG, RW>)];                       \
        fapq_few<B, DP, CG, RW>(p, *(FewqLds<B, DP, CG, RW> *)lds);                                              \
    }
#define FAPQ_FEWS(B, DP, WG) FAPQ_FEW(B, DP, 4, 1, 4, WG) FAPQ_FEW(B, DP, 2, 1, 8, WG) FAPQ_FEW(B, DP, 1, 1, 16, WG)
// (R: rows of a workgroup, 64 RW)
#define FAPQ_TILE(B, DP, RW, R)                                                                                    \
    extern "C" __global__ void __launch_bounds__(256, DP == 64 ? 3 : 2) ghip_fapq_tile##R##_##B##_##DP(FapMxParams p) {            \
        __shared__ __attribute__((aligned(1024))) uint8_t lds[sizeof(FapqTileLds<B, DP, RW>)];                      \
        fapq_tile<B, DP, RW>(p, *(FapqTileLds<B, DP, RW> *)lds);                                                    \
    }                                                                                                              \
    extern "C" __global__ void __launch_bounds__(256, DP == 64 ? 3 : 2) ghip_fapq_both##R##_##B##_##DP(FapMxParams p) {            \
        __shared__ __attribute__((aligned(1024))) uint8_t lds[sizeof(FapqLds<B, DP, RW>)];                          \
        if ((int)blockIdx.x < p.wg_sh) fapq_tile<B, DP, RW>(p, *(FapqTileLds<B, DP, RW> *)lds);                     \
        else fapq_few<B, DP, 1, 1>(p, *(FewqLds<B, DP, 1, 1> *)lds);                                                      \
    }
#define FAPQ_B(B)                                                                                                  \
    FAPQ_FEWS(B, 64, 3) FAPQ_FEW(B, 64, 1, 2, 32, 2) FAPQ_FEWS(B, 128, 3) FAPQ_FEW(B, 128, 1, 2, 32, 2) FAPQ_FEWS(B, 256, 1)                                                  \
    FAPQ_TILE(B, 64, 1, 64) FAPQ_TILE(B, 128, 1, 64) FAPQ_TILE(B, 256, 1, 64) FAPQ_TILE(B, 64, 2, 128) FAPQ_TILE(B, 128, 2, 128)
FAPQ_B(8) FAPQ_B(4)
