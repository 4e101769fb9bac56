// ghip_fap_core.h -- what attention over a paged KV cache is made of, whatever the
// cache's elements are held as: the rows of a wavefront with their running reference and
// sum, scores, masks, softmax and values on the matrix cores, the blocks of rows and
// the join of splits.  ghip_fap.hip has the formula and the reasons for the numbers.
#pragma once
#include "ghip_common.h"
#include "ghip_paged.h"

typedef _Float16 f16;
typedef __bf16 bf16;
typedef float v4f __attribute__((ext_vector_type(4)));
typedef float v2f __attribute__((ext_vector_type(2)));

template <typename E> struct Frag;
template <> struct Frag<f16> {
    typedef _Float16 v8 __attribute__((ext_vector_type(8)));
    typedef _Float16 v4 __attribute__((ext_vector_type(4)));
    typedef _Float16 v2 __attribute__((ext_vector_type(2)));
    typedef __fp16 tr __attribute__((__vector_size__(8)));
    static constexpr int NQ = 2, NP = 2;         // terms of q and of p
    // Where p is held: 2^HOME at a tile's largest key when the reference moves, below
    // 2^TOP from then on (8 apart: with 3 the rescaling of o makes 1702 rows over 2048
    // keys 132 us instead of 125).  Terms of f16 end at 2^-24 however many they are, so a p
    // of 2^-5 has 20 bits and smaller ones have less: the reference follows tiles down
    // whose largest p is below 2^LOW, and where it moves, a tile's keys from 2^REST on take
    // a pass before those below (one: behind two such gaps in one tile bits are lost).
    static constexpr float HOME = 8.0f, TOP = 15.9f, LOW = -2.0f, REST = -5.0f;
    static constexpr bool FOLLOW = true;
    // A row's q is held 2^k times, its largest from 2^14 to 2^15, and the scores lose that
    // again: small elements against large keys keep their bits, and none overflows (q of
    // 1e-2 against keys of 100: error 1.0e-5 without, 2.2e-7; one more operation a score,
    // 1702 rows over 2048 keys 122 us without, 125).
    static constexpr bool SCALED = true;
    typedef float ref;
    static __device__ __forceinline__ v4f mfma(v8 a, v8 b, v4f c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
    static __device__ __forceinline__ v4 read_tr(uint32_t at) {
        return __builtin_bit_cast(v4, __builtin_amdgcn_ds_read_tr16_b64_v4f16((__attribute__((address_space(3))) tr *)at));
    }
};
template <> struct Frag<bf16> {
    typedef __bf16 v8 __attribute__((ext_vector_type(8)));
    typedef __bf16 v4 __attribute__((ext_vector_type(4)));
    typedef __bf16 v2 __attribute__((ext_vector_type(2)));
    static constexpr int NQ = 3, NP = 3;
    static constexpr float HOME = 0.0f, TOP = 8.0f, LOW = 0.0f, REST = 0.0f;  // (32 bits' range: no need to follow)
    static constexpr bool FOLLOW = false, SCALED = false;
    typedef v4f ref;
    static __device__ __forceinline__ v4f mfma(v8 a, v8 b, v4f c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
    static __device__ __forceinline__ v4 read_tr(uint32_t at) {
        return __builtin_bit_cast(v4, __builtin_amdgcn_ds_read_tr16_b64_v4bf16((__attribute__((address_space(3))) v4 *)at));
    }
};

// x as N terms of E: each the rest of the ones before, rounded to nearest
template <typename E, int N>
DEV void split_pair(float x0, float x1, typename Frag<E>::v2 (&t)[N]) {
    v2f x = {x0, x1};
#pragma unroll
    for (int i = 0; i < N; i++) {
        t[i] = __builtin_convertvector(x, typename Frag<E>::v2);
        if (i + 1 < N) {
            x[0] = fmaf((float)t[i][0], -1.0f, x[0]);
            x[1] = fmaf((float)t[i][1], -1.0f, x[1]);
        }
    }
}

struct FapParams {
    const float *q;
    int64_t q_nb1, q_nb2;  // floats: head, token
    const uint16_t *kv;
    int64_t kv_head, kv_row, kv_page;  // elements
    int n_pages, page;
    const int32_t *seqs;  // [B][3 + per]: q0, nq, nkv, pages
    int64_t seq_nb1;      // ints
    int per, B;
    const float *sinks;  // [H] or null
    float *dst;
    int64_t d_nb1, d_nb2;  // floats: head, token
    int T, H, H_kv, D;
    float scale;  // times log2 e: scores are kept in log2 units
    int window, n_first, n_shared, max_q;
    PagedDiv by_page;
    // launch: the first wg_sh workgroups take the shared prefix (nb_sh blocks of
    // rows, zs_sh splits), the others each sequence's own keys (nb_own, zs_own)
    int nb_sh, zs_sh, nb_own, zs_own, wg_sh;
    int join_ragged;  // the join's workgroups go by all sequences' rows in a line, not by sequence and max_q
    // partials of row (token, head), split z (shared prefix first): part[.. + z][D]
    // and stat[.. + z][2] = (maximum, sum); null where zs_sh + zs_own == 1
    float *part, *stat;
};

#define DEV_M __device__ __forceinline__
constexpr float kLog2e = 1.4426950408889634f;

// LDS chunk (16 bytes) of a row of CH chunks that holds chunk c of row r.  Reads of
// K take one chunk of 16 rows; reads of V 32 bytes of 8 rows at a time: both
// touch each of the 64 banks once.
template <int CH>
DEV int k_swz(int r, int c) {
    return CH == 8 ? c ^ ((r >> 1) & 7) : CH == 12 ? c ^ ((r >> 2) & 3) : c ^ (r & 15);
}
template <int CH>
DEV int v_swz(int r, int c) {
    return CH == 8 ? c ^ (((r >> 1) & 3) << 1) : CH == 12 ? c ^ (((r >> 2) & 1) << 1) : c ^ ((r & 7) << 1);
}

DEV uint32_t lds_addr(const void *p) { return (uint32_t)(uintptr_t)(lds_void *)p; }
// 16 / 4 bytes a lane from memory to LDS at `to` (wave-uniform) + lane's place
DEV void load16(const void *from, uint32_t to) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(to), "v"(from) : "memory", "m0");
}
DEV void load4(const void *from, uint32_t to) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off" ::"s"(to), "v"(from) : "memory", "m0");
}
template <int N>
DEV void wait_loads() {
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
DEV void wait_lds() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

// maximum / sum over the 4 lanes of a query row
DEV float row_max(float x) {
    auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
}
DEV float row_sum(float x) {
    auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(a[0]) + __uint_as_float(a[1]);
}

// The wavefront's rows and what they hold: RW tiles of 16 rows.
template <typename E, int DP, int RW>
struct Rows {
    typedef Frag<E> F;
    typename F::v8 q[RW][DP / 32][F::NQ];
    v4f o[RW][DP / 16];
    // minus the reference (log2 units), 0 while unset; where q is not scaled four times,
    // as the products start with it
    typename F::ref mneg[RW];
    float unit[RW]; // what a score counts, 2^-k
    // four registers of 0, where they are to spare: a constant is written out for every
    // product (3 of 43 us, 3 prompts of 16 heads of 64; 128 rows of 128 dims would spill one
    // register for it, 3 of 127 us)
    v4f zero;
    DEV_M v4f start(int rt) const {
        if constexpr (!F::SCALED) return mneg[rt];
        else if constexpr (RW * DP < 256) return zero;
        else return v4f{0, 0, 0, 0};
    }
    float l[RW];    // this lane's share of the sum
    int pos[RW];    // position of this lane's row; -1: there is none, or it sees nothing
    float from[RW]; // scores below this move the reference: infinity until a key has been seen
};

// A row's q: this lane's share as it lies (dims 32 kk + 8 (lane >> 4) ..), loaded
// early; then, once it is in, as the terms of the fragments.
// (row_ref: the reference itself)
DEV float row_ref(float mneg) { return -mneg; }
DEV float row_ref(v4f mneg) { return -mneg[0]; }
template <int DP>
struct RawRow {
    float x[DP / 32][8];
};
template <int DP>
DEV void raw_load(RawRow<DP> &r, const float *qr, int D, bool valid) {
#pragma unroll
    for (int kk = 0; kk < DP / 32; kk++) {
        const int d = 32 * kk + 8 * ((threadIdx.x & 63) >> 4);
#pragma unroll
        for (int e = 0; e < 8; e++) r.x[kk][e] = 0.0f;
        if (valid && d < D) __builtin_memcpy(r.x[kk], qr + d, 32);
    }
}
// (the compiler does not know of wait_loads: it waits here, where nothing else is in flight)
template <int DP>
DEV void raw_wait(RawRow<DP> &r) {
#pragma unroll
    for (int kk = 0; kk < DP / 32; kk++)
#pragma unroll
        for (int e = 0; e < 8; e++) asm volatile("" : "+v"(r.x[kk][e]));
}
// Returns k of a scaled row's 2^k, 127 where that says nothing (all 0, infinite).
template <typename E, int DP, int RW>
DEV int rows_start(Rows<E, DP, RW> &R, int rt, const RawRow<DP> &r, float scale) {
    int k = 0;
    bool sized = false;
    if constexpr (Frag<E>::SCALED) {
        float mx = 0.0f;
#pragma unroll
        for (int kk = 0; kk < DP / 32; kk++)
#pragma unroll
            for (int e = 0; e < 8; e++) mx = fmaxf(mx, fabsf(r.x[kk][e] * scale));
        mx = row_max(mx);
        sized = mx > 0.0f && mx < __builtin_inff();
        if (sized) k = min(15 - __builtin_amdgcn_frexp_expf(mx), 100);
    }
    R.unit[rt] = __builtin_amdgcn_ldexpf(1.0f, -k);
    R.zero = v4f{0, 0, 0, 0};
    asm volatile("" : "+v"(R.zero));
#pragma unroll
    for (int kk = 0; kk < DP / 32; kk++)
#pragma unroll
        for (int e = 0; e < 4; e++) {
            typename Frag<E>::v2 t[Frag<E>::NQ];
            float x0 = r.x[kk][2 * e] * scale, x1 = r.x[kk][2 * e + 1] * scale;
            if constexpr (Frag<E>::SCALED) {
                x0 = __builtin_amdgcn_ldexpf(x0, k);
                x1 = __builtin_amdgcn_ldexpf(x1, k);
            }
            split_pair<E, Frag<E>::NQ>(x0, x1, t);
#pragma unroll
            for (int i = 0; i < Frag<E>::NQ; i++) {
                R.q[rt][kk][i][2 * e] = t[i][0];
                R.q[rt][kk][i][2 * e + 1] = t[i][1];
            }
        }
#pragma unroll
    for (int dt = 0; dt < DP / 16; dt++) R.o[rt][dt] = v4f{0, 0, 0, 0};
    R.mneg[rt] = typename Frag<E>::ref{};
    R.l[rt] = 0.0f;
    R.from[rt] = R.pos[rt] < 0 ? -__builtin_inff() : __builtin_inff();
    return sized ? k : 127;
}

// Fragment reads.  The swizzles touch the low bits of a chunk's number alone, so
// a fragment's address is one lane's constant with the bits of kk (dt) flipped in,
// the rest added: k_at / v_at give the constant, frag_at the address.
template <int DP>
DEV uint32_t k_at(uint32_t Ks) {
    constexpr int CH = DP / 8;
    const int lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
    return Ks + 2 * n * DP + 16 * (CH == 8 ? g ^ ((n >> 1) & 7) : CH == 12 ? g ^ ((n >> 2) & 3) : g ^ n);
}
template <int DP>
DEV uint32_t v_at(uint32_t Vs) {
    constexpr int CH = DP / 8;
    const int lane = threadIdx.x & 63, lj = lane & 15, r = 4 * (lane >> 4) + (lj >> 2), c = (lj & 3) >> 1;
    return Vs + 2 * r * DP + 16 * v_swz<CH>(r, c) + 8 * (lj & 1);
}
template <int STEP, int MASK>
DEV uint32_t frag_at(uint32_t at, int i) {
    return (at ^ (STEP * (i & MASK))) + STEP * (i & ~MASK);
}
// K fragment of the MFMA: keys 16 t + (lane & 15), dims 32 kk + 8 (lane >> 4) ..
template <typename E, int DP>
DEV typename Frag<E>::v8 key_frag(uint32_t kat, int t, int kk) {
    constexpr int CH = DP / 8;
    const uint32_t at = frag_at<64, CH == 8 ? 1 : CH == 12 ? 0 : 3>(kat, kk) + 32 * t * DP;
    return *(const __attribute__((address_space(3))) typename Frag<E>::v8 *)at;
}
// V^T: dims 16 dt + (lane & 15), in slot e key 32 u + 4 g + e, from slot 4 on 16
// further (as the scores lie)
template <typename E, int DP>
DEV typename Frag<E>::v8 value_frag(uint32_t vat, int u, int dt) {
    constexpr int CH = DP / 8;
    const uint32_t at = frag_at<32, CH == 8 ? 3 : CH == 12 ? 1 : 7>(vat, dt) + 64 * u * DP;
    const typename Frag<E>::v4 lo = Frag<E>::read_tr(at), hi = Frag<E>::read_tr(at + 32 * DP);
    return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
}
// Scores of the NT 16-key tiles at Ks, less the reference (where q is scaled: as they
// are, in its units; softmax() takes both off).  between(f) is called after the products of
// fragment f, for what is to go out under them.
template <typename E, int DP, int RW, int NT, typename F>
DEV void scores(const Rows<E, DP, RW> &R, uint32_t Ks, v4f (&s)[NT][RW], F between) {
    constexpr int KK = DP / 32, N = NT * KK;
    const uint32_t kat = k_at<DP>(Ks);
    // fragments are read two ahead of the products that use them
    typename Frag<E>::v8 a[3];
    a[0] = key_frag<E, DP>(kat, 0, 0);
    a[1] = key_frag<E, DP>(kat, 1 / KK, 1 % KK);
#pragma unroll
    for (int f = 0; f < N; f++) {
        const int t = f / KK, kk = f % KK;
        if (f + 2 < N) a[(f + 2) % 3] = key_frag<E, DP>(kat, (f + 2) / KK, (f + 2) % KK);
#pragma unroll
        for (int i = Frag<E>::NQ - 1; i >= 0; i--)
#pragma unroll
            for (int rt = 0; rt < RW; rt++)
                s[t][rt] = Frag<E>::mfma(a[f % 3], R.q[rt][kk][i], kk > 0 || i < Frag<E>::NQ - 1 ? s[t][rt] : R.start(rt));
        between(f);
        __builtin_amdgcn_sched_barrier(0);
    }
}

// What of a tile is to be masked: keys k0 .. , of which [k0, ke) are the pass's,
// `bad` of them on no page.  Key r = 16 t + 4 g + v of the tile is compared as
// 16 t + v with limits less k0 + 4 g.
template <typename E, int DP, int RW, int NT>
DEV void mask_scores(const Rows<E, DP, RW> &R, v4f (&s)[NT][RW], int k0, int ke, uint64_t bad, int window, int n_first) {
    // (first: what a key on no page was scored with may be minus infinity too)
    if (bad) {
        int g4 = 4 * ((threadIdx.x & 63) >> 4);
        asm volatile("" : "+v"(g4));
#pragma unroll
        for (int t = 0; t < NT; t++) {
            const uint32_t mine = (uint32_t)(bad >> (16 * t)) >> g4;
#pragma unroll
            for (int v = 0; v < 4; v++)
                if ((mine >> v) & 1) {
#pragma unroll
                    for (int rt = 0; rt < RW; rt++) s[t][rt][v] = __builtin_nanf("");
                }
        }
    }
    const int at = k0 + 4 * ((threadIdx.x & 63) >> 4);
    // seen(c, lo, hi): is this lane's key c in sight of a row?
    auto cut = [&](auto seen) {
#pragma unroll
        for (int rt = 0; rt < RW; rt++) {
            const int hi = min(R.pos[rt], ke - 1) - at, lo = R.pos[rt] - window - at;
#pragma unroll
            for (int t = 0; t < NT; t++)
#pragma unroll
                for (int v = 0; v < 4; v++)
                    if (!seen(16 * t + v, lo, hi)) s[t][rt][v] = -__builtin_inff();
        }
    };
    if (!window || ke <= n_first) {
        cut([](int c, int, int hi) { return c <= hi; });
    } else if (k0 >= n_first) {  // lo < c <= hi in one comparison
        cut([](int c, int lo, int hi) { return (uint32_t)(c - 1 - lo) < (uint32_t)(max(hi, lo) - lo); });
    } else {
        const int first = n_first - at;
        cut([=](int c, int lo, int hi) { return c <= hi && (c > lo || c < first); });
    }
}

// Row tile rt's keys from 2^REST on: their part of O^T += V^T P^T and of the row's
// sum, after which they are gone from the scores.  (Called hardly ever, and straight
// through: in a loop the compiler copies all of o.)
template <typename E, int DP, int RW, int NT>
DEV void top_keys(Rows<E, DP, RW> &R, int rt, uint32_t Vs, v4f (&s)[NT][RW]) {
    constexpr int NP = Frag<E>::NP;
    const uint32_t vat = v_at<DP>(Vs);
#pragma unroll
    for (int u = 0; u < NT / 2; u++) {
        typename Frag<E>::v8 p[NP];
#pragma unroll
        for (int e = 0; e < 4; e++) {
            float x[2];
#pragma unroll
            for (int k = 0; k < 2; k++) {
                const int v = 2 * (e & 1) + k;
                const float y = s[2 * u + e / 2][rt][v];
                const bool top = !(y < Frag<E>::REST);
                x[k] = top ? __builtin_amdgcn_exp2f(y) : 0.0f;
                s[2 * u + e / 2][rt][v] = top ? -__builtin_inff() : y;
                R.l[rt] += x[k];
            }
            typename Frag<E>::v2 t[NP];
            split_pair<E, NP>(x[0], x[1], t);
#pragma unroll
            for (int i = 0; i < NP; i++) {
                p[i][2 * e] = t[i][0];
                p[i][2 * e + 1] = t[i][1];
            }
        }
#pragma unroll
        for (int dt = 0; dt < DP / 16; dt++) {
            const typename Frag<E>::v8 a = value_frag<E, DP>(vat, u, dt);
#pragma unroll
            for (int i = NP - 1; i >= 0; i--) R.o[rt][dt] = Frag<E>::mfma(a, p[i], R.o[rt][dt]);
            __builtin_amdgcn_sched_barrier(0);
        }
    }
}

// Row tile rt's largest score against its reference.  That moves on the row's first
// key, when a p would pass 2^TOP, and, where it follows, when all of a row's p in the
// tile are below 2^LOW; the tile's largest is then 2^HOME, and o and l are rescaled
// (followed: by powers of two, as it may come often).  Followed down, o and l stay below
// 2^107: the reference is at most 2^90 below what l has.  Returns whether it moved and
// left keys below 2^REST.
template <typename E, int DP, int RW, int NT>
DEV bool find_reference(Rows<E, DP, RW> &R, int rt, v4f (&s)[NT][RW]) {
    typedef Frag<E> F;
    constexpr float INF = __builtin_inff();
    float mx = -INF;
#pragma unroll
    for (int t = 0; t < NT; t++)
#pragma unroll
        for (int v = 0; v < 4; v++) mx = fmaxf(mx, s[t][rt][v]);
    if (!__ballot(mx < R.from[rt] || mx > F::TOP)) return false;
    mx = row_max(mx);
    const bool set = R.from[rt] < INF;
    float shift = mx - F::HOME;
    bool move = mx > F::TOP || (!set && mx > -INF), low = false;
    if constexpr (F::FOLLOW) {
        const bool down = set && mx < F::LOW && mx > -INF;
        if (__builtin_expect(__ballot(down) != 0, 0)) {
            const float least = (float)__builtin_amdgcn_frexp_expf(row_max(R.l[rt])) - 90.0f;
            if (down) shift = fmaxf(shift, least);
        }
        shift = __builtin_rintf(shift);
        move = move || down;
    }
    if (__ballot(move && set)) {  // (o and l are 0 before a row's first key)
        const float alpha = move && set ? __builtin_amdgcn_exp2f(-shift) : 1.0f;
        R.l[rt] *= alpha;
#pragma unroll
        for (int dt = 0; dt < DP / 16; dt++) R.o[rt][dt] *= alpha;
    }
    if (move) {
        R.from[rt] = F::FOLLOW ? F::LOW : -INF;
        R.mneg[rt] -= shift;
#pragma unroll
        for (int t = 0; t < NT; t++) s[t][rt] -= shift;
        if constexpr (F::FOLLOW) {
            // a score in (-inf, 2^REST): bits past those of REST, before those of -inf
            constexpr uint32_t REST = __builtin_bit_cast(uint32_t, F::REST) + 1;
            uint32_t mn = ~0u;
#pragma unroll
            for (int t = 0; t < NT; t++)
#pragma unroll
                for (int v = 0; v < 4; v++) mn = min(mn, __float_as_uint(s[t][rt][v]) - REST);
            low = mn < 0xff800000u - REST && mx - shift > F::LOW;  // (else the reference went as far as it may)
        }
    }
    return F::FOLLOW && __ballot(low);
}

// Scores -> probabilities, 2^(s - reference).  values_in() waits for the tile's V.  (f16, a first key whose own value is 0,
// 299 others of e^-12 its weight: 2.2e-4 of the output in error with p of 1 at the
// largest key and no following, at e^-18 8.6e-2; as it is 9e-7 and 1.6e-6; without the
// pass for the top keys 1.5e-5 at e^-18.)
template <typename E, int DP, int RW, int NT, typename F>
DEV void softmax(Rows<E, DP, RW> &R, v4f (&s)[NT][RW], uint32_t Vs, F values_in) {
    // (one row tile after the other: the next one's products end under this one's work; all
    // references first measured 39.7 for 38.6 us, 3 prompts of 16 heads of 64)
#pragma unroll
    for (int rt = 0; rt < RW; rt++) {
        if constexpr (Frag<E>::SCALED)
#pragma unroll
            for (int t = 0; t < NT; t++)
#pragma unroll
                for (int v = 0; v < 4; v++) s[t][rt][v] = fmaf(s[t][rt][v], R.unit[rt], R.mneg[rt]);
        const bool low = find_reference<E, DP, RW, NT>(R, rt, s);
        if constexpr (Frag<E>::FOLLOW)
            if (__builtin_expect(low, 0)) {
                values_in();
                top_keys<E, DP, RW, NT>(R, rt, Vs, s);
                find_reference<E, DP, RW, NT>(R, rt, s);
            }
        float sum = 0.0f;
#pragma unroll
        for (int t = 0; t < NT; t++)
#pragma unroll
            for (int v = 0; v < 4; v++) {
                s[t][rt][v] = __builtin_amdgcn_exp2f(s[t][rt][v]);
                sum += s[t][rt][v];
            }
        R.l[rt] += sum;
    }
}

// O^T += V^T P^T over NT 16-key tiles at Vs
template <typename E, int DP, int RW, int NT>
DEV void values(Rows<E, DP, RW> &R, uint32_t Vs, const v4f (&s)[NT][RW]) {
    constexpr int NP = Frag<E>::NP;
    const uint32_t vat = v_at<DP>(Vs);
    typename Frag<E>::v8 p[RW][NP];
#pragma unroll
    for (int u = 0; u < NT / 2; u++) {
#pragma unroll
        for (int rt = 0; rt < RW; rt++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                typename Frag<E>::v2 t[NP];
                split_pair<E, NP>(s[2 * u + e / 2][rt][2 * (e & 1)], s[2 * u + e / 2][rt][2 * (e & 1) + 1], t);
#pragma unroll
                for (int i = 0; i < NP; i++) {
                    p[rt][i][2 * e] = t[i][0];
                    p[rt][i][2 * e + 1] = t[i][1];
                }
            }
        typename Frag<E>::v8 a[3];
        a[0] = value_frag<E, DP>(vat, u, 0);
        a[1] = value_frag<E, DP>(vat, u, 1);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int dt = 0; dt < DP / 16; dt++) {
            if (dt + 2 < DP / 16) a[(dt + 2) % 3] = value_frag<E, DP>(vat, u, dt + 2);
#pragma unroll
            for (int i = NP - 1; i >= 0; i--)
#pragma unroll
                for (int rt = 0; rt < RW; rt++) R.o[rt][dt] = Frag<E>::mfma(a[dt % 3], p[rt][i], R.o[rt][dt]);
            __builtin_amdgcn_sched_barrier(0);
        }
    }
}

// A workgroup's keys.
struct Pass {
    int p0, p1;  // least and largest position of its rows
    PagedTiles tl;
};
DEV int clip_pos(int64_t p, int64_t table) { return (int)(p < -1 ? -1 : p > table ? table : p); }

struct Tile {
    int k0, ke;
};
DEV Tile tile_at(const PagedTiles &tl, int t, int kt) {
    const int a0 = tl.a0, a1 = tl.a1, b0 = tl.b0, b1 = tl.b1, na = tl.na;  // (or the choice is between their addresses, in memory)
    Tile r;
    r.k0 = t < na ? a0 + t * kt : b0 + (t - na) * kt;
    r.ke = t < na ? a1 : b1;
    return r;
}
DEV bool tile_whole(const Tile &tile, int kt, const Pass &ps, int window, int n_first) {
    return tile.k0 + kt <= tile.ke && tile.k0 + kt - 1 <= ps.p0 &&
           (!window || tile.k0 > ps.p1 - window || tile.k0 + kt <= n_first);
}

// Rows' results to dst, or to this split's partials.  m, l: of this lane's row.
DEV void finish_stat(const FapParams &p, int h, float &m, float &l, float &f) {
    f = 1.0f;
    if (p.sinks) {
        const float sk = p.sinks[h] * kLog2e;
        const float M = fmaxf(m, sk);
        if (M > -__builtin_inff()) {
            f = __builtin_amdgcn_exp2f(m - M);
            l = l * f + __builtin_amdgcn_exp2f(sk - M);
        }
    }
    f = l == 0.0f ? 0.0f : f / l;
}

// the statistics of a split that holds none of a row's keys (NaN: it has keys
// past its table); its sums are not read
DEV void stat_none(const FapParams &p, int64_t pi, bool nan) {
    p.stat[2 * pi] = -__builtin_inff();
    p.stat[2 * pi + 1] = nan ? __builtin_nanf("") : 0.0f;
}

// infinite or NaN?
DEV bool odd(v4f x) {
    const float y = x[0] * 0.0f + x[1] * 0.0f + x[2] * 0.0f + x[3] * 0.0f;
    return y != y;
}
// The rows of a row tile (lanes n, n + 16, .. hold row n) that have to be computed
// again; mine(d): are dims d .. d + 3 this wavefront's to store?
template <typename A, typename F>
DEV void rows_again(const FapParams &p, const int32_t *table, bool again, int64_t tok, int h, int pos, F mine) {
    const int lane = threadIdx.x & 63;
    uint64_t b = __ballot(again);
    b |= b >> 32;
    b |= b >> 16;
    for (uint32_t rows = b & 0xffff; rows; rows &= rows - 1) {
        const int n = __builtin_ctz(rows);
        const int64_t t = __builtin_amdgcn_readlane((int)tok, n);
        const int hd = __builtin_amdgcn_readlane(h, n);
        const v4f o = A::row(p, table, t, hd, __builtin_amdgcn_readlane(pos, n));
        if (4 * lane < p.D && mine(4 * lane)) __builtin_memcpy(p.dst + t * p.d_nb2 + hd * p.d_nb1 + 4 * lane, &o, 16);
    }
}

// ---- up to 16 rows a KV head, each wavefront over keys of its own

// The 4 wavefronts' rows of row tile rt: everyone takes the common maximum, then thread (dims, row)
// adds the four.  os: [4][16][DP + 4]; rows: how many there are; of this lane's row n = lane & 15:
// is there one, its token, head and place among the partials.
template <typename A, typename E, int DP, int RW>
DEV void few_join(const FapParams &p, Rows<E, DP, RW> &R, int rt, float *os, float (&ws)[4][2][16], int rows, bool valid, int64_t table, int64_t tok,
                  int hd, int64_t pi, const int32_t *pages) {
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n = lane & 15, g = lane >> 4;
    const float l = row_sum(R.l[rt]), m = R.from[rt] < __builtin_inff() ? row_ref(R.mneg[rt]) : -__builtin_inff();
    if (g == 0) {
        ws[w][0][n] = m;
        ws[w][1][n] = l;
    }
    __syncthreads();
    float M = -__builtin_inff(), L = 0.0f;
#pragma unroll
    for (int u = 0; u < 4; u++) M = fmaxf(M, ws[u][0][n]);
#pragma unroll
    for (int u = 0; u < 4; u++) L += M > -__builtin_inff() ? ws[u][1][n] * __builtin_amdgcn_exp2f(ws[u][0][n] - M) : ws[u][1][n];
    if (valid && R.pos[rt] >= table) L = __builtin_nanf("");
    const float f = M > -__builtin_inff() ? __builtin_amdgcn_exp2f(m - M) : 1.0f;
    if (n < rows) {
#pragma unroll
        for (int dt = 0; dt < DP / 16; dt++) *(v4f *)&os[(w * 16 + n) * (DP + 4) + 16 * dt + 4 * g] = R.o[rt][dt] * f;
    }
    __syncthreads();
    const bool direct = !p.part;
    float fin = 1.0f, Mf = M, Lf = L;
    if (direct) finish_stat(p, hd, Mf, Lf, fin);
    // lanes of row n: wavefront w and lane group g take dims 16 w + 4 g + 64 k
    bool again = false;
    if (valid) {
        float *out = direct ? p.dst + tok * p.d_nb2 + hd * p.d_nb1 : p.part + pi * p.D;
        for (int d = 16 * w + 4 * g; d < p.D; d += 64) {
            v4f a = {0, 0, 0, 0};
#pragma unroll
            for (int u = 0; u < 4; u++) a += *(v4f *)&os[(u * 16 + n) * (DP + 4) + d];
            a *= fin;
            __builtin_memcpy(out + d, &a, 16);
            again = again || odd(a);
        }
        if (!direct && w == 0 && g == 0) {
            p.stat[2 * pi] = M;
            p.stat[2 * pi + 1] = L;
        }
    }
    // (each wavefront the dims that it stores)
    if (direct) rows_again<A>(p, pages, again && R.pos[rt] < table, tok, hd, R.pos[rt], [&](int d) { return (d >> 4 & 3) == w; });
}

// ---- up to 64 RW rows: 4 wavefronts of 16 RW rows, 64-key tiles for all

// The rows of a workgroup: for each of its tokens the row of q (-1: none) and
// its position.
template <int R>
struct RowList {
    int tok[R + 1], pos[R + 1];
    int sums[4], found[2];
};
// exclusive sum of v over the 256 threads; total: that of all
template <int R>
DEV int scan256(RowList<R> &ls, int v, int &total) {
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    int x = v;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int y = __shfl_up(x, o, 64);
        if (lane >= o) x += y;
    }
    __syncthreads();
    if (lane == 63) ls.sums[w] = x;
    __syncthreads();
    int before = 0;
    total = 0;
#pragma unroll
    for (int u = 0; u < 4; u++) {
        if (u < w) before += ls.sums[u];
        total += ls.sums[u];
    }
    return before + x - v;
}
DEV PagedSeq seq_of(const FapParams &p, int b) {
    const int32_t *row = p.seqs + (int64_t)b * p.seq_nb1;
    return paged_seq(row[0], row[1], row[2], p.T, p.max_q);
}
// The sequence whose pages hold the shared prefix: the first one with rows (idle ones
// may hold anything) and all of its keys, else the one with the most of them.
DEV int prefix_of(const FapParams &p) {
    if (seq_of(p, 0).nq && p.seqs[2] >= p.n_shared) return 0;
    const int lane = threadIdx.x & 63;
    int best = 0, most = -1;
    for (int b0 = 0; b0 < p.B && most < p.n_shared; b0 += 64) {
        int n = -1;
        if (b0 + lane < p.B && seq_of(p, b0 + lane).nq) n = min(p.seqs[(b0 + lane) * p.seq_nb1 + 2], p.n_shared);
        int mx = n;
#pragma unroll
        for (int o = 32; o; o >>= 1) mx = max(mx, __shfl_xor(mx, o, 64));
        mx = __builtin_amdgcn_readfirstlane(mx);
        if (mx > most) {
            most = mx;
            best = b0 + __builtin_ctzll(__ballot(n == mx));
        }
    }
    return best;
}

// L: how a tile comes into LDS.  L::Loads<DP> has
//   ld.load_pages(t)     the page numbers of tile t's keys are on their way
//   ld.find_tile(t)      where its rows are; ld.ok2, ld.bad2: its keys that are there, those on no page
//   ld.load_part(t, f)   under fragment f of DP / 16 of the tile before's first half: a load of it goes out
//   ld.load_half(t, u)   at the start of that tile's half u (not L::LATE: in place of all load_part): loads go out
//   ld.load_first(t)     the first tile's loads, all of them (in after wait_loads and loaded())
//   ld.middle(t)         between the halves
//   ld.loaded(t)         this wavefront's loads of it are in: LDS holds its rows, 0 for values of keys not in ok
//   L::LATE              both halves have loads, and past the last tile they do no harm (those of the tile found last)
//   L::HOME_K            keys and values are in LDS 2^HOME_K times what they are
//   L::NARROW            E does not do for every tile:
//   ld.rows_at(k)        this lane's rows' least k (rows_start)
//   ld.beyond(t)         does it not do for tile t, or one before?  The same for all wavefronts
// BW: a block's rows, 64 each; RW of them are this pass's, from `half` on.  Returns whether
// a tile was met that E does not do for; then nothing has been stored.
template <typename L, int DP, int BW>
struct TileLds {
    uint8_t kvs[2][2][64 * DP * 2];  // this tile's K and V, the next one's
    typename L::Lds ld;
    RowList<64 * BW> ls;
};
template <typename L, typename E, int DP, int RW, int BW = RW, typename PARAMS>
DEV bool fap_tile(const PARAMS &p, TileLds<L, DP, BW> &lds, int half = 0) {
    constexpr int KT = 64, R = 64 * BW;
    constexpr float LESS = 1.0f / (1 << L::HOME_K);
    auto &kvs = lds.kvs;
    auto &ls = lds.ls;
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6), n = lane & 15, g = lane >> 4;
    const int G = p.H / p.H_kv;
    const int64_t table = (int64_t)p.per * p.page;
    const bool shared = (int)blockIdx.x < p.wg_sh;
    const int id = shared ? blockIdx.x : blockIdx.x - p.wg_sh, nz = shared ? p.zs_sh : p.zs_own;
    const int hk = id % p.H_kv, z = (id / p.H_kv) % nz, blk = id / (p.H_kv * nz);
    const int32_t *row;  // the pages: for the shared prefix those of the sequence that prefix_of finds
    int x0, r0;  // first token of the list, first row of the block (rows of token x0 + k: G (x0 + k) ..)
    if (shared) {
        // tokens x0 .. of all sequences in order
        row = p.seqs + prefix_of(p) * p.seq_nb1;
        r0 = blk * R;
        x0 = r0 / G;
        const int nx = (r0 + R - 1) / G - x0 + 1;
        for (int k = tid; k < nx; k += 256) ls.tok[k] = -1;
        __syncthreads();
        if (p.max_q == 1 && p.B <= p.T) {  // at most one row a sequence, and blocks for all of them: sequence x0 + k
            for (int k = tid; k < nx && x0 + k < p.B; k += 256) {
                const PagedSeq sq = seq_of(p, x0 + k);
                ls.tok[k] = sq.nq ? sq.q0 : -1;
                ls.pos[k] = clip_pos(sq.pos0, table);
            }
        } else {
            int base = 0;
            for (int b0 = 0; b0 < p.B && base < x0 + nx; b0 += 256) {
                PagedSeq sq;
                sq.nq = 0;
                if (b0 + tid < p.B) sq = seq_of(p, b0 + tid);
                int total;
                const int at = base + scan256<R>(ls, sq.nq, total);
                for (int k = max(at, x0); k < min(at + sq.nq, x0 + nx); k++) {
                    ls.tok[k - x0] = sq.q0 + (k - at);
                    ls.pos[k - x0] = clip_pos(sq.pos0 + (k - at), table);
                }
                base += total;
            }
        }
    } else {
        // block blk of the sequences' blocks of R rows
        int b = blk, bb = 0;
        if ((int64_t)p.max_q * G > R) {
            if (tid == 0) ls.found[0] = -1;
            int base = 0;
            for (int b0 = 0; b0 < p.B && base <= blk; b0 += 256) {
                int nb = 0;
                if (b0 + tid < p.B) nb = (int)(((int64_t)seq_of(p, b0 + tid).nq * G + R - 1) / R);
                int total;
                const int at = base + scan256<R>(ls, nb, total);
                if (at <= blk && blk < at + nb) {
                    ls.found[0] = b0 + tid;
                    ls.found[1] = at + nb - 1 - blk;  // the last rows, which see most keys, come first
                }
                base += total;
            }
            __syncthreads();
            b = ls.found[0];
            bb = ls.found[1];
            if (b < 0) return false;
        }
        r0 = bb * R;
        x0 = r0 / G;
        const PagedSeq sq = seq_of(p, b);
        const int nx = (r0 + R - 1) / G - x0 + 1;
        for (int k = tid; k < nx; k += 256) {
            ls.tok[k] = x0 + k < sq.nq ? sq.q0 + x0 + k : -1;
            ls.pos[k] = clip_pos(sq.pos0 + x0 + k, table);
        }
        row = p.seqs + (int64_t)b * p.seq_nb1;
    }
    __syncthreads();
    Pass ps;
    ps.p0 = 0x7fffffff;
    ps.p1 = -1;
    bool any = false;
    for (int k = lane; k <= (r0 + R - 1) / G - x0; k += 64)
        if (ls.tok[k] >= 0) {
            ps.p0 = min(ps.p0, ls.pos[k]);
            ps.p1 = max(ps.p1, ls.pos[k]);
            any = true;
        }
    if (!__ballot(any)) return false;
#pragma unroll
    for (int o = 32; o; o >>= 1) {
        ps.p0 = min(ps.p0, __shfl_xor(ps.p0, o, 64));
        ps.p1 = max(ps.p1, __shfl_xor(ps.p1, o, 64));
    }
    ps.p0 = __builtin_amdgcn_readfirstlane(ps.p0);
    ps.p1 = __builtin_amdgcn_readfirstlane(ps.p1);
    ps.tl = paged_tiles(ps.p0, ps.p1, p.window, p.n_first, shared ? 0 : p.n_shared, shared ? p.n_shared : (int)table, KT);
    const int share = paged_share(ps.tl.n, nz);
    const int t0 = (int)min((int64_t)z * share, (int64_t)ps.tl.n), t1 = min(ps.tl.n, t0 + share);
    // this lane's rows
    struct Row {
        int hd, pos;
        bool valid;
        int64_t tok, pi;
    };
    auto row_of = [&](int rt) {
        Row y;
        const int r = r0 + 64 * half + 16 * (RW * w + rt) + n, k = r / G - x0;
        y.hd = hk * G + r % G;
        y.valid = ls.tok[k] >= 0;
        y.tok = y.valid ? ls.tok[k] : 0;
        y.pos = y.valid ? ls.pos[k] : -1;
        y.pi = (y.tok * p.H + y.hd) * (p.zs_sh + p.zs_own) + (shared ? 0 : p.zs_sh) + z;
        return y;
    };
    if (t0 >= t1 && p.part) {  // nothing in this split
#pragma unroll
        for (int rt = 0; rt < RW; rt++) {
            const Row y = row_of(rt);
            if (y.valid && g == 0) stat_none(p, y.pi, y.pos >= table);
        }
        return false;
    }
    Rows<E, DP, RW> Q;
    RawRow<DP> raw[RW];
    bool mine = false;
#pragma unroll
    for (int rt = 0; rt < RW; rt++) {
        const Row y = row_of(rt);
        raw_load<DP>(raw[rt], p.q + y.tok * p.q_nb2 + y.hd * p.q_nb1, p.D, y.valid);
        Q.pos[rt] = y.pos;
        mine = mine || y.valid;
    }
    const bool work = __ballot(mine) != 0;  // a wavefront without rows only loads
    int w0 = 0x7fffffff, w1 = -1;           // least and largest position of the wavefront's rows
#pragma unroll
    for (int rt = 0; rt < RW; rt++) {
        if (Q.pos[rt] >= 0) w0 = min(w0, Q.pos[rt]);
        w1 = max(w1, Q.pos[rt]);
    }
#pragma unroll
    for (int o = 8; o; o >>= 1) {
        w0 = min(w0, __shfl_xor(w0, o, 64));
        w1 = max(w1, __shfl_xor(w1, o, 64));
    }
    w0 = __builtin_amdgcn_readfirstlane(w0);
    w1 = __builtin_amdgcn_readfirstlane(w1);
    typename L::template Loads<DP> ld(p, lds.ld, kvs, hk, row, w, ps.tl, t1);
    if (t0 < t1) {
        ld.load_pages(t0);
        ld.load_pages(t0 + 1);
    }
    wait_loads<0>();
#pragma unroll
    for (int rt = 0; rt < RW; rt++) raw_wait<DP>(raw[rt]);
    if (t0 < t1) {
        ld.find_tile(t0);
        wait_lds();
        ld.load_pages(t0 + 2);
        ld.load_first(t0);
        ld.ok = ld.ok2;
        ld.bad = ld.bad2;
        if (t0 + 1 < t1) ld.find_tile(t0 + 1);
    }
    int k = 127;
#pragma unroll
    for (int rt = 0; rt < RW; rt++) {
        k = min(k, rows_start<E, DP, RW>(Q, rt, raw[rt], p.scale * kLog2e));
        if constexpr (L::HOME_K != 0) Q.unit[rt] *= LESS;
    }
    if constexpr (L::NARROW) ld.rows_at(k);
    if (t0 < t1) {
        wait_loads<0>();
        ld.loaded(t0);
    }
    __syncthreads();
    for (int t = t0; t < t1; t++) {
        if constexpr (L::NARROW)
            if (ld.beyond(t)) return true;
        const Tile tile = tile_at(ps.tl, t, KT);
        const uint64_t badc = ld.bad;
        const bool part = !tile_whole(tile, KT, ps, p.window, p.n_first);
        const uint32_t Ks = lds_addr(kvs[t & 1][0]), Vs = lds_addr(kvs[t & 1][1]);
        const bool more = t + 1 < t1;
        if (more) ld.load_pages(t + 3);
        // 32 keys at a time: the scores of 64 are 16 registers more, which then spill
#pragma unroll
        for (int u = 0; u < 2; u++) {
            const uint32_t Kh = Ks + 64 * u * DP, Vh = Vs + 64 * u * DP;
            // what none of this wavefront's rows sees of an edge tile is passed over
            const int h0 = tile.k0 + 32 * u, h1 = min(h0 + 32, tile.ke);
            const bool need = work && (!part || (h0 < h1 && h0 <= w1 && (!p.window || h1 - 1 > w0 - p.window || h0 < p.n_first)));
            v4f s[2][RW];
            if (u == 1 && more) ld.middle(t + 1);
            if (L::LATE) ld.load_half(t + 1, u);
            const bool loads = !L::LATE && u == 0 && more;
            if (need) {
                __builtin_amdgcn_s_setprio(1);
                if (loads) scores<E, DP, RW, 2>(Q, Kh, s, [&](int f) { ld.load_part(t + 1, f); });
                else scores<E, DP, RW, 2>(Q, Kh, s, [](int) {});
                __builtin_amdgcn_s_setprio(0);
            } else if (loads) {
                ld.load_half(t + 1, 0);
            }
            if (need) {
                if (part || badc) mask_scores<E, DP, RW, 2>(Q, s, tile.k0 + 32 * u, tile.ke, badc >> (32 * u), p.window, p.n_first);
                softmax<E, DP, RW, 2>(Q, s, Vh, []() {});
            }
            if (need) {
                __builtin_amdgcn_s_setprio(1);
                values<E, DP, RW, 2>(Q, Vh, s);
                __builtin_amdgcn_s_setprio(0);
            }
        }
        if (more) {
            ld.ok = ld.ok2;
            ld.bad = ld.bad2;
            if (t + 2 < t1) ld.find_tile(t + 2);
            wait_loads<0>();
            ld.loaded(t + 1);
        }
        __syncthreads();
    }
#pragma unroll
    for (int rt = 0; rt < RW; rt++) {
        const Row y = row_of(rt);
        bool again = false;
        float l = row_sum(Q.l[rt]), m = Q.from[rt] < __builtin_inff() ? row_ref(Q.mneg[rt]) : -__builtin_inff(), f = 1.0f;
        if (y.pos >= table) l = __builtin_nanf("");
        if (y.valid) {
            if (!p.part) finish_stat(p, y.hd, m, l, f);
            if constexpr (L::HOME_K != 0) f *= LESS;
            float *out = p.part ? p.part + y.pi * p.D : p.dst + y.tok * p.d_nb2 + y.hd * p.d_nb1;
#pragma unroll
            for (int dt = 0; dt < DP / 16; dt++) {
                const int d = 16 * dt + 4 * g;
                const v4f a = Q.o[rt][dt] * f;
                if (d < p.D) __builtin_memcpy(out + d, &a, 16);
                again = again || (d < p.D && odd(a));
            }
            if (p.part && g == 0) {
                p.stat[2 * y.pi] = m;
                p.stat[2 * y.pi + 1] = l;
            }
        }
        if (!p.part) rows_again<typename L::Again>(p, row + 3, again && y.pos < table, y.tok, y.hd, y.pos, [](int) { return true; });
    }
    return false;
}

// ---- the splits' partials of a row -> dst, in the order of the splits

// One wavefront a row (token, head): lane z holds split z's statistics; then NG
// groups of D / 4 lanes take 4 dims a lane of splits group, group + NG, .. (8 of
// them in flight), and the groups are added in order.
template <typename A>
DEV void fap_join(const FapParams &p) {
    const int lane = threadIdx.x & 63;
    const int64_t id = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int h = (int)(id % p.H);
    const int64_t x = id / p.H;  // sequence b, row i as b max_q + i, or the row's number among all sequences' rows
    int b, i;
    if (!p.join_ragged) {
        b = (int)(x / p.max_q);
        i = (int)(x - (int64_t)b * p.max_q);
        if (b >= p.B) return;
    } else {
        int64_t base = 0;
        b = -1;
        for (int b0 = 0; b0 < p.B && base <= x; b0 += 64) {
            const int n = b0 + lane < p.B ? seq_of(p, b0 + lane).nq : 0;
            int to = n;  // rows up to and with this lane's sequence
#pragma unroll
            for (int o = 1; o < 64; o <<= 1) {
                const int y = __shfl_up(to, o, 64);
                if (lane >= o) to += y;
            }
            const uint64_t here = __ballot(base + to - n <= x && x < base + to);
            if (here) {
                const int at = __builtin_ctzll(here);
                b = b0 + at;
                i = (int)(x - base - __builtin_amdgcn_readlane(to - n, at));
                break;
            }
            base += __builtin_amdgcn_readlane(to, 63);
        }
        if (b < 0) return;
    }
    const PagedSeq sq = seq_of(p, b);
    if (i >= sq.nq) return;
    const int64_t tok = sq.q0 + i, row = tok * p.H + h;
    const int nz = p.zs_sh + p.zs_own, LD = p.D / 4, NG = 64 / LD, grp = lane / LD;
    float m = -__builtin_inff(), l = 0.0f;
    if (lane < nz) {
        m = p.stat[2 * (row * nz + lane)];
        l = p.stat[2 * (row * nz + lane) + 1];
    }
    float M = m;
#pragma unroll
    for (int o = 32; o; o >>= 1) M = fmaxf(M, __shfl_xor(M, o, 64));
    const float wt = m > -__builtin_inff() ? __builtin_amdgcn_exp2f(m - M) : 0.0f;
    float L = wave_sum(m > -__builtin_inff() ? l * wt : l), Mf = M, fin;  // l of a split without keys: 0, or NaN
    finish_stat(p, h, Mf, L, fin);
    const float f = wt * fin;
    const float *part = p.part + row * nz * p.D + 4 * (lane - grp * LD);
    v4f a = {0, 0, 0, 0};
    for (int z0 = 0; z0 < nz; z0 += 8 * NG) {
        v4f x[8];
        float w[8];
#pragma unroll
        for (int k = 0; k < 8; k++) {
            const int z = z0 + grp + k * NG;
            w[k] = __shfl(f, min(z, 63), 64);
            if (z >= nz || grp >= NG) w[k] = 0.0f;
            x[k] = v4f{0, 0, 0, 0};
            if (w[k] != 0.0f) __builtin_memcpy(&x[k], part + (int64_t)z * p.D, 16);
        }
#pragma unroll
        for (int k = 0; k < 8; k++) a += x[k] * w[k];
    }
    v4f sum = a;
    for (int k = 1; k < NG; k++)
#pragma unroll
        for (int e = 0; e < 4; e++) sum[e] += __shfl(a[e], (lane + k * LD) & 63, 64);
    if (lane < LD && L != L) sum = v4f{L, L, L, L};
    const int64_t pos = sq.pos0 + i;
    if (__ballot(lane < LD && odd(sum)) && pos >= 0 && pos < (int64_t)p.per * p.page)
        sum = A::row(p, p.seqs + (int64_t)b * p.seq_nb1 + 3, tok, h, pos);
    if (lane < LD) __builtin_memcpy(p.dst + tok * p.d_nb2 + (int64_t)h * p.d_nb1 + 4 * lane, &sum, 16);
}
