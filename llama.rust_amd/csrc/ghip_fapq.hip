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

// A wavefront a row (token, head): number b max_q + i names sequence b's row i.
template <int BITS>
DEV void fapq_rows(const FapMxParams &p) {
    const int lane = threadIdx.x & 63;
    const int64_t rows = (int64_t)p.B * p.max_q * p.H;
    for (int64_t id = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); id < rows; id += (int64_t)gridDim.x * 4) {
        const int h = (int)(id % p.H);
        const int64_t x = id / p.H;
        const int b = (int)(x / p.max_q), i = (int)(x - (int64_t)b * p.max_q);
        const PagedSeq sq = seq_of(p, b);
        if (i >= sq.nq) continue;
        const int64_t tok = sq.q0 + i, pos = sq.pos0 + i;
        const float nan = __builtin_nanf("");
        v4f o = {nan, nan, nan, nan};  // it sees a key past its table
        if (pos < (int64_t)p.per * p.page) o = row_alone<BITS>(p, p.seqs + (int64_t)b * p.seq_nb1 + 3, tok, h, pos);
        if (4 * lane < p.D) __builtin_memcpy(p.dst + tok * p.d_nb2 + (int64_t)h * p.d_nb1 + 4 * lane, &o, 16);
    }
}
extern "C" __global__ void __launch_bounds__(256) ghip_fapq_rows_8(FapMxParams p) { fapq_rows<8>(p); }
extern "C" __global__ void __launch_bounds__(256) ghip_fapq_rows_4(FapMxParams p) { fapq_rows<4>(p); }
