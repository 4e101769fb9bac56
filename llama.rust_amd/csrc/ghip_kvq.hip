// ghip_kvq.hip -- writing a quantized KV cache (the keys rotated on the way) and
// reading its rows back; the codes are those of ghip_mx.h.
//
// A code is a rounding to 4 (or 2) significant bits of the rotated key, and how a value
// next to a border falls is to be the formula's doing, not that of a rotation in 32 bits:
// angles, sin, cos and the rotation are formed in 64 bits, the result goes to 32 bits
// with what is cut off left in the last bit (so that the second rounding is as one), and
// the rest is exact.  Long prefills do not feel it, as memory bounds them (8192 tokens below); short ones do: each lane
// works out the 8 (4) angles of its elements, which lanes of other heads work out too (32 tokens: 7.0 us the
// kernel, 4.5 with a rotation in 32 bits).
//
// Work layout.  Append: a thread takes 8 elements of a token's key row and the same of
// its value row, for HN heads that share the angles; 4 neighbouring lanes hold a block and
// find its largest element by two exchanges.  A rotated element needs the other one of its
// pair: with halves as pairs a lane loads those 8 too (from the cache: the row's
// other lanes load them as well).  8192 tokens, 8 heads of 128, F32, E4M3: 19.5 us for
// 84.4 MB, 4.3 TB/s (a large copy: 5.1, at which they are 16.6 us; launch and ramp are 2 .. 3).
// 32 tokens: 8.8 us a call; the kernel waits for its loads and then for the angles' sums.
#include "ghip_mx.h"
#include "ghip_paged.h"

typedef _Float16 f16;
typedef __bf16 bf16;
typedef float f32;

struct alignas(16) RopeTab {
    uint64_t turn[128]; // turns per position of each pair: 64 bits after the point; with factors, a double's bits
    uint8_t axis[128];  // the pair's row of positions
    float mscale;       // factor of cos and sin
    int axes;           // rows of positions
};

// A cache's rows: where slot s of head h has its codes and its scales (bytes).
struct MxRows {
    uint8_t *kv, *sc;
    int64_t kv_head, kv_row, kv_page, sc_head, sc_row, sc_page;
    int64_t n_slots;  // page * pages: other slots there are none
    uint32_t page;    // rows of a page; 0: in both tensors page p's rows follow page p - 1's
    int small;        // slots fit 32 bits
    PagedDiv by_page;
};
DEV void mx_row(const MxRows &m, int64_t slot, int64_t &kv, int64_t &sc) {
    if (!m.page) {
        kv = slot * m.kv_row;
        sc = slot * m.sc_row;
        return;
    }
    const int64_t pg = m.small ? (int64_t)paged_div((uint32_t)slot, m.by_page) : (int64_t)((uint64_t)slot / m.page);
    const int64_t r = slot - pg * m.page;
    kv = pg * m.kv_page + r * m.kv_row;
    sc = pg * m.sc_page + r * m.sc_row;
}

struct AppendMxParams {
    const void *k, *v;
    int64_t k_nb1, k_nb2, v_nb1, v_nb2;  // elements: head, token
    MxRows to;
    const int64_t *slots;
    const int32_t *pos;
    int64_t pos_nb1;
    const float *factors;
    int T, H, D, P;  // P rotated pairs
    int S, HG;       // scale bytes of a key; groups of HN heads
    RopeTab tab;
};

// 8 elements at any multiple of the element's size (gfx950 loads 16 bytes from any address)
template <typename E>
DEV void load8(const E *p, float (&x)[8]) {
    typedef E v8 __attribute__((ext_vector_type(8), aligned(sizeof(E))));
    const v8 y = *(const v8 *)p;
#pragma unroll
    for (int i = 0; i < 8; i++) x[i] = (float)y[i];
}

// sin and cos of u / 2^64 turns: the nearest quarter comes off exactly, the rest, |t|
// <= pi / 4, goes through Taylor sums that end where the next term is below 2^-49.
DEV void sincos_turns(uint64_t u, double &s, double &c) {
    const uint32_t k = (uint32_t)((u + (1ull << 61)) >> 62);
    const double t = 3.4061215800865545e-19 * (double)(int64_t)(u - ((uint64_t)k << 62));
    const double t2 = t * t;
    double ps = fma(t2, -7.6471637318198164e-13, 1.6059043836821613e-10);
    ps = fma(t2, ps, -2.5052108385441720e-08);
    ps = fma(t2, ps, 2.7557319223985893e-06);
    ps = fma(t2, ps, -1.9841269841269841e-04);
    ps = fma(t2, ps, 8.3333333333333332e-03);
    ps = fma(t2, ps, -1.6666666666666666e-01);
    const double sn = fma(t * t2, ps, t);
    double pc = fma(t2, -1.1470745597729725e-11, 2.0876756987868100e-09);
    pc = fma(t2, pc, -2.7557319223985888e-07);
    pc = fma(t2, pc, 2.4801587301587302e-05);
    pc = fma(t2, pc, -1.3888888888888889e-03);
    pc = fma(t2, pc, 4.1666666666666664e-02);
    pc = fma(t2, pc, -0.5);
    const double cn = fma(t2, pc, 1.0);
    const double a = k & 1 ? cn : sn, b = k & 1 ? sn : cn;
    s = k & 2 ? -a : a;
    c = (k + 1) & 2 ? -b : b;
}
// cos and sin of pair i's angle at the token's positions
DEV void pair_angle(const AppendMxParams &p, int i, const int32_t (&at)[4], double &c, double &s) {
    uint64_t f = p.tab.turn[i];
    if (p.factors) {
        const double x = __builtin_bit_cast(double, f) / (double)p.factors[i], y = (x - floor(x)) * 0x1p32, hi = floor(y);
        f = (uint64_t)(uint32_t)hi << 32 | (uint32_t)((y - hi) * 0x1p32);
    }
    const int ax = p.tab.axis[i];
    const int32_t q = ax == 0 ? at[0] : ax == 1 ? at[1] : ax == 2 ? at[2] : at[3];
    sincos_turns((uint64_t)(int64_t)q * f, s, c);
    c *= (double)p.tab.mscale;
    s *= (double)p.tab.mscale;
}
// x in 32 bits, cut, its last bit 1 where anything was cut off: rounded again to fewer
// bits it falls as x would
DEV float to_odd(double x) {
    const float f = (float)x;
    uint32_t b = __float_as_uint(f);
    if (fabs((double)f) > fabs(x)) b--;  // (infinity too, of a finite x)
    if ((double)f != x && x == x) b |= 1;
    return __uint_as_float(b);
}

// The block's scale and this lane's 8 codes, stored at kv; lane 0 of the block's 4 stores the scale.
template <int BITS>
DEV void store_block(const float (&x)[8], int c, int D, uint8_t *kv, uint8_t *sc) {
    uint32_t big = 0;
#pragma unroll
    for (int i = 0; i < 8; i++) big = max(big, __float_as_uint(x[i]) & 0x7fffffffu);
    big = max(big, (uint32_t)__builtin_amdgcn_mov_dpp((int)big, 0xB1, 0xf, 0xf, true));  // lane ^ 1
    big = max(big, (uint32_t)__builtin_amdgcn_mov_dpp((int)big, 0x4E, 0xf, 0xf, true));  // lane ^ 2
    const uint32_t byte = mx_scale_of<BITS>(big);
    const MxCodes<BITS> w = mx_encode<BITS>(x, byte);
    if (8 * c < D) __builtin_memcpy(kv + BITS * c, &w, BITS);
    if ((c & 3) == 0) sc[c >> 2] = (uint8_t)byte;
}

enum { NORM, HALF, ODD };  // pairs (2 i, 2 i + 1); (i, i + P), P a multiple of 8; any P
template <typename E, int BITS, int MODE, int HN>
DEV void append_mx(const AppendMxParams &p) {
    const uint32_t L = 4u * p.S;  // lanes of a head's row: a power of two
    const uint32_t id = blockIdx.x * 256u + threadIdx.x, c = id & (L - 1), r = id >> (31 - __builtin_clz(L));
    const int64_t t = r / (uint32_t)p.HG;
    const int h0 = (int)(r - (uint32_t)t * (uint32_t)p.HG) * HN;
    if (t >= p.T) return;  // (all lanes of a row)
    const int64_t slot = p.slots[t];
    const int e0 = 8 * c;
    const bool in = e0 < p.D;
    const E *k = (const E *)p.k + t * p.k_nb2 + (in ? e0 : 0), *v = (const E *)p.v + t * p.v_nb2 + (in ? e0 : 0);
    // the partners of 8 elements of a half: as many elements on, or back
    const bool turned = in && e0 < 2 * p.P;
    const int to = MODE == HALF && turned ? (e0 < p.P ? p.P : -p.P) : 0;
    float x[HN][8], y[HN][8], z[HN][8];
#pragma unroll
    for (int i = 0; i < HN; i++) {
        const int64_t h = min(h0 + i, p.H - 1);
        load8<E>(k + h * p.k_nb1, x[i]);
        if (MODE == HALF) load8<E>(k + h * p.k_nb1 + to, y[i]);
        load8<E>(v + h * p.v_nb1, z[i]);
    }
    int32_t at[4] = {0, 0, 0, 0};
#pragma unroll
    for (int a = 0; a < 4; a++)
        if (a < p.tab.axes) at[a] = p.pos[a * p.pos_nb1 + t];
    if (slot < 0 || slot >= p.to.n_slots) return;  // padding, or a slot outside the cache
    if (turned) {
        double cs, sn;
        if (MODE == NORM) {
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const int q = e0 / 2 + j;
                if (q >= p.P) break;
                pair_angle(p, q, at, cs, sn);
#pragma unroll
                for (int i = 0; i < HN; i++) {
                    const double a = x[i][2 * j], b = x[i][2 * j + 1];
                    x[i][2 * j] = to_odd(fma(a, cs, -(b * sn)));
                    x[i][2 * j + 1] = to_odd(fma(a, sn, b * cs));
                }
            }
        } else {
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const int e = e0 + j;
                if (MODE == ODD && e >= 2 * p.P) break;
                const bool first = e < p.P;
                pair_angle(p, first ? e : e - p.P, at, cs, sn);
#pragma unroll
                for (int i = 0; i < HN; i++) {
                    if (MODE == ODD) y[i][j] = (float)k[min(h0 + i, p.H - 1) * p.k_nb1 + j + (first ? p.P : -p.P)];
                    const double a = x[i][j], b = y[i][j];
                    x[i][j] = to_odd(first ? fma(a, cs, -(b * sn)) : fma(b, sn, a * cs));
                }
            }
        }
    }
    int64_t kv, sc;
    mx_row(p.to, slot, kv, sc);
#pragma unroll
    for (int i = 0; i < HN; i++) {
        if (h0 + i >= p.H) break;
        uint8_t *o = p.to.kv + kv + (h0 + i) * p.to.kv_head, *so = p.to.sc + sc + (h0 + i) * p.to.sc_head;
        if (!in)
#pragma unroll
            for (int j = 0; j < 8; j++) x[i][j] = z[i][j] = 0.0f;
        store_block<BITS>(x[i], c, p.D, o, so);
        store_block<BITS>(z[i], c, p.D, o + p.D * BITS / 8, so + p.S);
    }
}

// ---- reading rows back: a thread takes CH codes of a row's key or value (16 bytes of what it writes) of RN
// rows, whose loads are all in flight before the first store.  16000 rows of 8 heads of 128, 8 bits to BF16:
// 23.8 us for 98.8 MB, 4.2 TB/s (at a large copy's rate 19.4).
struct ReadMxParams {
    MxRows from;
    const int64_t *slots;
    void *dst;
    int64_t d_nb1, d_nb2;  // elements: head, token
    int T, H, D, S;
    int U;                 // threads of a row
    uint32_t step;         // rows between a thread's rows
};
template <typename O, int BITS, int RN>
DEV void read_mx(const ReadMxParams &p) {
    constexpr int CH = 16 / sizeof(O), W = CH * BITS / 8;  // codes, their bytes
    const uint32_t id = blockIdx.x * 256u + threadIdx.x, r0 = id / (uint32_t)p.U, u = id - r0 * (uint32_t)p.U;
    if (r0 >= p.step) return;
    const uint32_t rows = (uint32_t)p.T * (uint32_t)p.H;
    const int e = CH * u;                                    // element of the row
    const int b = e < p.D ? e / 32 : p.S + (e - p.D) / 32;  // its scale
    uint32_t w[RN][2], sb[RN];
    O *to[RN];
#pragma unroll
    for (int i = 0; i < RN; i++) {
        const uint32_t r = r0 + i * p.step;
        const uint32_t t = min(r, rows - 1) / (uint32_t)p.H, h = min(r, rows - 1) - t * (uint32_t)p.H;
        const int64_t slot = p.slots[t];
        const bool there = r < rows && slot >= 0 && slot < p.from.n_slots;
        to[i] = there ? (O *)p.dst + (int64_t)t * p.d_nb2 + (int64_t)h * p.d_nb1 + e : nullptr;
        w[i][0] = w[i][1] = sb[i] = 0;
        if (there) {
            int64_t kv, sc;
            mx_row(p.from, slot, kv, sc);
            __builtin_memcpy(w[i], p.from.kv + kv + h * p.from.kv_head + e * BITS / 8, W);
            sb[i] = p.from.sc[sc + h * p.from.sc_head + b];
        }
    }
#pragma unroll
    for (int i = 0; i < RN; i++) {
        if (!to[i]) continue;
        const float s = mx_scale(sb[i]);
        mx_f2 x[CH / 2];
        x[0] = mx_pair<BITS, 0>(w[i][0], s);
        x[1] = mx_pair<BITS, 1>(w[i][0], s);
        if constexpr (CH == 8) {
            x[2] = mx_pair<BITS, 2>(w[i][BITS == 8], s);
            x[3] = mx_pair<BITS, 3>(w[i][BITS == 8], s);
        }
        typedef O vo __attribute__((ext_vector_type(CH), aligned(sizeof(O))));
        vo y;
#pragma unroll
        for (int j = 0; j < CH; j++) y[j] = (O)x[j / 2][j & 1];  // one rounding to nearest where O is narrower
        *(vo *)to[i] = y;
    }
}

#define APPEND_K(E, BITS, M, MODE, HN)                                                                          \
    extern "C" __global__ void __launch_bounds__(256) ghip_append_mx##BITS##_##E##_##M##_h##HN(AppendMxParams p) { \
        append_mx<E, BITS, MODE, HN>(p);                                                                        \
    }
#define APPEND_E(E, BITS)                                             \
    APPEND_K(E, BITS, norm, NORM, 1) APPEND_K(E, BITS, norm, NORM, 4) \
    APPEND_K(E, BITS, half, HALF, 1) APPEND_K(E, BITS, half, HALF, 4) \
    APPEND_K(E, BITS, odd, ODD, 1) APPEND_K(E, BITS, odd, ODD, 4)
APPEND_E(f32, 8) APPEND_E(f16, 8) APPEND_E(bf16, 8) APPEND_E(f32, 4) APPEND_E(f16, 4) APPEND_E(bf16, 4)
#define READ_K(O, BITS, RN)                                                                               \
    extern "C" __global__ void __launch_bounds__(256) ghip_read_mx##BITS##_##O##_r##RN(ReadMxParams p) {   \
        read_mx<O, BITS, RN>(p);                                                                          \
    }
#define READ_E(O) READ_K(O, 8, 1) READ_K(O, 8, 4) READ_K(O, 4, 1) READ_K(O, 4, 4)
READ_E(f32) READ_E(f16) READ_E(bf16)
