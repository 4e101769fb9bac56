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
template <typename E, int DP, int RW>
DEV void rows_start(Rows<E, DP, RW> &R, int rt, const RawRow<DP> &r, float scale) {
    int k = 0;
    if constexpr (Frag<E>::SCALED) {
        float mx = 0.0f;
#pragma unroll
        for (int kk = 0; kk < DP / 32; kk++)
#pragma unroll
            for (int e = 0; e < 8; e++) mx = fmaxf(mx, fabsf(r.x[kk][e] * scale));
        mx = row_max(mx);
        if (mx > 0.0f && mx < __builtin_inff()) k = min(15 - __builtin_amdgcn_frexp_expf(mx), 100);
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
    if (bad) {
        const uint64_t mine = bad >> (4 * ((threadIdx.x & 63) >> 4));
#pragma unroll
        for (int t = 0; t < NT; t++)
#pragma unroll
            for (int v = 0; v < 4; v++)
                if ((mine >> (16 * t + v)) & 1) {
#pragma unroll
                    for (int rt = 0; rt < RW; rt++)
                        if (s[t][rt][v] > -__builtin_inff()) s[t][rt][v] = __builtin_nanf("");
                }
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
    Tile r;
    r.k0 = t < tl.na ? tl.a0 + t * kt : tl.b0 + (t - tl.na) * kt;
    r.ke = t < tl.na ? tl.a1 : tl.b1;
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
// infinite or NaN?
DEV bool odd(v4f x) {
    const float y = x[0] * 0.0f + x[1] * 0.0f + x[2] * 0.0f + x[3] * 0.0f;
    return y != y;
}
// The rows of a row tile (lanes n, n + 16, .. hold row n) that have to be computed
// again; mine(d): are dims d .. d + 3 this wavefront's to store?
template <typename E, typename F>
DEV void rows_again(const FapParams &p, const int32_t *table, bool again, int64_t tok, int h, int pos, F mine) {
    const int lane = threadIdx.x & 63;
    uint64_t b = __ballot(again);
    b |= b >> 32;
    b |= b >> 16;
    for (uint32_t rows = b & 0xffff; rows; rows &= rows - 1) {
        const int n = __builtin_ctz(rows);
        const int64_t t = __builtin_amdgcn_readlane((int)tok, n);
        const int hd = __builtin_amdgcn_readlane(h, n);
        const v4f o = row_again<E>(p, table, t, hd, __builtin_amdgcn_readlane(pos, n));
        if (4 * lane < p.D && mine(4 * lane)) __builtin_memcpy(p.dst + t * p.d_nb2 + hd * p.d_nb1 + 4 * lane, &o, 16);
    }
}

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
    // the 4 wavefronts' rows: everyone takes the common maximum, then thread
    // (dims, row) adds the four
    const float l = row_sum(R.l[0]), m = R.from[0] < __builtin_inff() ? row_ref(R.mneg[0]) : -__builtin_inff();
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
    if (valid && R.pos[0] >= table) L = __builtin_nanf("");
    const float f = M > -__builtin_inff() ? __builtin_amdgcn_exp2f(m - M) : 1.0f;
    float *os = (float *)&kvs[0][0][0];  // [4][16][DP + 4]
    static_assert(sizeof(kvs) >= 4 * 16 * (DP + 4) * 4, "the wavefronts' rows fit the tiles");
    if (n < sq.nq * G) {
#pragma unroll
        for (int dt = 0; dt < DP / 16; dt++) *(v4f *)&os[(w * 16 + n) * (DP + 4) + 16 * dt + 4 * g] = R.o[0][dt] * f;
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
    if (direct) rows_again<E>(p, row + 3, again && R.pos[0] < table, tok, hd, R.pos[0], [&](int d) { return (d >> 4 & 3) == w; });
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

template <int DP, int RW>
struct TileLds {
    uint8_t kvs[2][2][64 * DP * 2];  // this tile's K and V, the next one's
    int64_t offs[4][64];
    int32_t te[4][2][64];
    RowList<64 * RW> ls;
};
template <typename E, int DP, int RW>
DEV void fap_tile(const FapParams &p, TileLds<DP, RW> &lds) {
    constexpr int KT = 64, R = 64 * RW, CH = DP / 8, NI = KT * CH / 256;  // loads of a K tile by each wavefront
    static_assert(KT * CH % 256 == 0 && 2 * NI == DP / 16, "the wavefronts load alike, one load under each of a half's fragments");
    auto &kvs = lds.kvs;
    auto &offs = lds.offs;
    auto &te = lds.te;
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
            if (b < 0) return;
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
    if (!__ballot(any)) return;
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
        const int r = r0 + 16 * (RW * w + rt) + n, k = r / G - x0;
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
        return;
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
    const uint8_t *kvh = (const uint8_t *)(p.kv + hk * p.kv_head);

    auto load_pages = [&](int t) {
        const Tile tl = tile_at(ps.tl, min(t, t1 - 1), KT);
        const int j = min(tl.k0 + lane, tl.ke - 1);
        load4(row + 3 + paged_div((uint32_t)j, p.by_page), lds_addr(te[w][t & 1]));
    };
    // Three tiles are under way: t is computed, t + 1 loaded, and at the step's end,
    // where it would wait for those loads, the rows of t + 2 are found (from pages
    // that were loaded a step before).
    uint64_t ok = 0, bad = 0, ok2 = 0, bad2 = 0;  // keys of tiles t + 1, t + 2 that are there, those on no page
    const uint8_t *at[NI];                        // this lane's rows of the tile found last
    const RowLoads<DP> rl(p.D, NI * w);
    auto find_tile = [&](int t) {
        find_keys(p, tile_at(ps.tl, t, KT), KT, te[w][t & 1], offs[w], ok2, bad2);
#pragma unroll
        for (int ii = 0; ii < NI; ii++) at[ii] = kvh + offs[w][rl.row(ii)];
    };
    // load f of 2 NI of tile t: one goes out under each fragment's products (bf16, 12
    // turns under 4001 keys, 128 rows: 125 us, and 130 with all of them at the step's
    // start; f16 the same)
    auto load_part = [&](int t, int f) {
        const int ii = f >> 1, kv = f & 1;
        load16(at[ii] + (kv ? 2 * p.D + rl.v_chunk(ii) : rl.k_chunk(ii)), lds_addr(kvs[t & 1][kv]) + 1024 * (NI * w + ii));
    };
    auto load_tile = [&](int t) {
#pragma unroll
        for (int f = 0; f < 2 * NI; f++) load_part(t, f);
    };
    // What this wavefront loaded of tile t is in: rows that were not there hold
    // nothing that counts.
    auto loaded = [&](int t) {
        uint8_t *Vs = kvs[t & 1][1];
        if (ok != ~0ull) {
#pragma unroll
            for (int ii = 0; ii < NI; ii++) {
                const int c = 64 * (NI * w + ii) + lane;
                if (!((ok >> (c / CH)) & 1)) *(uint4 *)(Vs + 16 * c) = make_uint4(0, 0, 0, 0);
            }
        }
    };
    if (t0 < t1) {
        load_pages(t0);
        load_pages(t0 + 1);
    }
    wait_loads<0>();
#pragma unroll
    for (int rt = 0; rt < RW; rt++) raw_wait<DP>(raw[rt]);
    if (t0 < t1) {
        find_tile(t0);
        wait_lds();
        load_pages(t0 + 2);
        load_tile(t0);
        ok = ok2;
        bad = bad2;
        if (t0 + 1 < t1) find_tile(t0 + 1);
    }
#pragma unroll
    for (int rt = 0; rt < RW; rt++) rows_start<E, DP, RW>(Q, rt, raw[rt], p.scale * kLog2e);
    if (t0 < t1) {
        wait_loads<0>();
        loaded(t0);
    }
    __syncthreads();
    for (int t = t0; t < t1; t++) {
        const Tile tile = tile_at(ps.tl, t, KT);
        const uint64_t badc = bad;
        const bool part = !tile_whole(tile, KT, ps, p.window, p.n_first);
        const uint32_t Ks = lds_addr(kvs[t & 1][0]), Vs = lds_addr(kvs[t & 1][1]);
        const bool more = t + 1 < t1;
        if (more) load_pages(t + 3);
        // 32 keys at a time: the scores of 64 are 16 registers more, which then spill
#pragma unroll
        for (int u = 0; u < 2; u++) {
            const uint32_t Kh = Ks + 64 * u * DP, Vh = Vs + 64 * u * DP;
            // what none of this wavefront's rows sees of an edge tile is passed over
            const int h0 = tile.k0 + 32 * u, h1 = min(h0 + 32, tile.ke);
            const bool need = work && (!part || (h0 < h1 && h0 <= w1 && (!p.window || h1 - 1 > w0 - p.window || h0 < p.n_first)));
            v4f s[2][RW];
            if (need) {
                __builtin_amdgcn_s_setprio(1);
                if (u == 0 && more) scores<E, DP, RW, 2>(Q, Kh, s, [&](int f) { load_part(t + 1, f); });
                else scores<E, DP, RW, 2>(Q, Kh, s, [](int) {});
                __builtin_amdgcn_s_setprio(0);
            } else if (u == 0 && more) {
                load_tile(t + 1);
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
            ok = ok2;
            bad = bad2;
            if (t + 2 < t1) find_tile(t + 2);
            wait_loads<0>();
            loaded(t + 1);
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
        if (!p.part) rows_again<E>(p, row + 3, again && y.pos < table, y.tok, y.hd, y.pos, [](int) { return true; });
    }
}

// ---- the splits' partials of a row -> dst, in the order of the splits

// One wavefront a row (token, head): lane z holds split z's statistics; then NG
// groups of D / 4 lanes take 4 dims a lane of splits group, group + NG, .. (8 of
// them in flight), and the groups are added in order.
template <typename E>
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
        sum = row_again<E>(p, p.seqs + (int64_t)b * p.seq_nb1 + 3, tok, h, pos);
    if (lane < LD) __builtin_memcpy(p.dst + tok * p.d_nb2 + (int64_t)h * p.d_nb1 + 4 * lane, &sum, 16);
}

extern "C" __global__ void __launch_bounds__(256) ghip_fap_join_f16(FapParams p) { fap_join<f16>(p); }
extern "C" __global__ void __launch_bounds__(256) ghip_fap_join_bf16(FapParams p) { fap_join<bf16>(p); }

// ghip_fap_both: the shared prefix on tiles and each sequence's own keys, for few
// rows each, in one launch, so that the one's loads run under the other's products.
template <int DP, int RW>
union FapLds {
    FewLds<DP> few;
    TileLds<DP, RW> tile;
};
#define FAP_FEW(E, DP)                                                                                   \
    extern "C" __global__ void __launch_bounds__(256, 2) ghip_fap_few_##E##_##DP(FapParams p) {          \
        __shared__ __attribute__((aligned(1024))) uint8_t lds[sizeof(FewLds<DP>)];                       \
        fap_few<E, DP>(p, *(FewLds<DP> *)lds);                                                           \
    }
// (R: rows of a workgroup, 64 RW)
#define FAP_TILE(E, DP, RW, R)                                                                           \
    extern "C" __global__ void __launch_bounds__(256, 2) ghip_fap_tile##R##_##E##_##DP(FapParams p) {    \
        __shared__ __attribute__((aligned(1024))) uint8_t lds[sizeof(TileLds<DP, RW>)];                  \
        fap_tile<E, DP, RW>(p, *(TileLds<DP, RW> *)lds);                                                 \
    }                                                                                                    \
    extern "C" __global__ void __launch_bounds__(256, 2) ghip_fap_both##R##_##E##_##DP(FapParams p) {    \
        __shared__ __attribute__((aligned(1024))) uint8_t lds[sizeof(FapLds<DP, RW>)];                   \
        if ((int)blockIdx.x < p.wg_sh) fap_tile<E, DP, RW>(p, *(TileLds<DP, RW> *)lds);                  \
        else fap_few<E, DP>(p, *(FewLds<DP> *)lds);                                                      \
    }
#define FAP_E(E)                                                                                         \
    FAP_FEW(E, 64) FAP_FEW(E, 96) FAP_FEW(E, 128) FAP_FEW(E, 256)                                        \
    FAP_TILE(E, 64, 1, 64) FAP_TILE(E, 96, 1, 64) FAP_TILE(E, 128, 1, 64) FAP_TILE(E, 256, 1, 64)        \
    FAP_TILE(E, 64, 2, 128) FAP_TILE(E, 96, 2, 128)
FAP_E(f16) FAP_E(bf16)
FAP_TILE(f16, 128, 2, 128)
