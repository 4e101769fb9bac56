// ghip_rope.hip -- rotary positions with one or several axes, and appending
// keys and values to a paged KV cache with the rotation on the way.
//
// Pair i of a token is turned by the angle  a = p[axis(i)] * f_i / factor_i:
//   (x0, x1) -> (x0 cos a - x1 sin a, x0 sin a + x1 cos a)
// with the token's position p on the pair's axis (text: one axis; image and
// video: time, height, width).  f_i, which pairs an axis has and the context
// extension are worked out on the host (RopeTab), in turns per position: of
// p * f_i turns only the fraction counts, and as p is whole, f_i's fraction is
// all it takes.  As 64 bits after the point its product with p is two 32-bit
// multiplications and wraps where the turns do: the angle is exact to 2^-32
// turns at any position (a 32-bit float product is off by up to 2^-8 radians at
// position 100000).  sin and cos of the remaining eighth turn are polynomials in
// 32 bits.
//
// Work layout.  Both kernels are bound by memory: every element is read once
// and written once.  A thread takes one unit of a token's head row -- VEC
// pairs, or the 2 VEC elements of a part that is not rotated -- for HN heads:
// the angles are formed once for HN heads, and all HN loads are in flight before
// the first store.  Neighbouring lanes hold neighbouring units of the same row.
#include "ghip_common.h"

typedef _Float16 f16;
typedef __bf16 bf16;

struct alignas(16) RopeTab {
    uint64_t turn[128]; // turns per position of each pair: 64 bits after the point; with factors, a double's bits
    uint8_t axis[128];  // the pair's row of positions
    float mscale;       // factor of cos and sin
    int axes;           // rows of positions
};

template <int N>
using vf = float __attribute__((ext_vector_type(N)));
// N elements as one vector, of the element's alignment (gfx950 loads 16 bytes from
// any address; copied element by element they come one by one)
template <typename E, int N>
struct Vec {
    typedef E type __attribute__((ext_vector_type(N), aligned(sizeof(E))));
};
template <typename E, int N>
DEV vf<N> load_n(const E *p) {
    return __builtin_convertvector(*(const typename Vec<E, N>::type *)p, vf<N>);
}
// one rounding to nearest where E is narrower than 32 bits
template <typename E, int N>
DEV void store_n(E *p, vf<N> v) {
    typedef E ve __attribute__((ext_vector_type(N)));
    *(typename Vec<E, N>::type *)p = __builtin_convertvector(v, ve);
}

// sin and cos of u / 2^32 turns.  The nearest quarter comes off exactly; the rest,
// |t| <= pi / 4, is rounded once (2^-25 radians), and its Taylor sums end where
// the next term is below 2^-29.
DEV void sincos_turns(uint32_t u, float &s, float &c) {
    const uint32_t k = (u + 0x20000000u) >> 30;
    const float t = 1.4629180792671596e-9f * (float)(int32_t)(u - (k << 30));
    const float t2 = t * t;
    float ps = fmaf(t2, 2.7557319e-6f, -1.9841270e-4f);
    ps = fmaf(t2, ps, 8.3333333e-3f);
    ps = fmaf(t2, ps, -1.6666667e-1f);
    const float sn = fmaf(t * t2, ps, t);
    float pc = fmaf(t2, -2.7557319e-7f, 2.4801587e-5f);
    pc = fmaf(t2, pc, -1.3888889e-3f);
    pc = fmaf(t2, pc, 4.1666667e-2f);
    pc = fmaf(t2, pc, -0.5f);
    const float cn = fmaf(t2, pc, 1.0f);
    const float a = k & 1 ? cn : sn, b = k & 1 ? sn : cn;
    s = k & 2 ? -a : a;
    c = (k + 1) & 2 ? -b : b;
}

// cos and sin of VEC pairs from pair i0 on, for token t.  The token's positions on
// all axes are loaded beside the pairs' table and picked by axis afterwards, so
// that no load waits for another.
template <int VEC>
DEV void unit_angles(const RopeTab &tab, const int32_t *pos, int64_t pos_nb1, int axes, const float *factors, int64_t t,
                     int i0, vf<VEC> &c, vf<VEC> &s) {
    typedef uint8_t axis_v __attribute__((ext_vector_type(VEC)));
    typedef uint64_t turn_v __attribute__((ext_vector_type(VEC)));
    turn_v turn;
    axis_v axis;
    __builtin_memcpy(&turn, &tab.turn[i0], sizeof turn);
    __builtin_memcpy(&axis, &tab.axis[i0], sizeof axis);
    int32_t at[4];
#pragma unroll
    for (int a = 0; a < 4; a++) at[a] = a < axes ? pos[a * pos_nb1 + t] : 0;
#pragma unroll
    for (int j = 0; j < VEC; j++) {
        uint64_t f = turn[j];
        if (factors) {
            const double x = __builtin_bit_cast(double, f) / (double)factors[i0 + j], y = (x - floor(x)) * 0x1p32, hi = floor(y);
            f = (uint64_t)(uint32_t)hi << 32 | (uint32_t)((y - hi) * 0x1p32);
        }
        const int ax = axis[j];
        const int32_t p = ax == 0 ? at[0] : ax == 1 ? at[1] : ax == 2 ? at[2] : at[3];
        uint32_t u = (uint32_t)p * (uint32_t)(f >> 32) + __umulhi((uint32_t)p, (uint32_t)f);
        if (p < 0) u -= (uint32_t)f;
        float sj, cj;
        sincos_turns(u, sj, cj);
        s[j] = sj * tab.mscale;
        c[j] = cj * tab.mscale;
    }
}

// one unit of a row: u < UR rotated (pairs VEC u ..), else the elements 2 P + ..
// as they are.  `x` holds the pairs' first elements, `y` the second ones (of a
// part that is not rotated, or of values: the unit's halves).
template <int VEC>
struct Unit {
    vf<VEC> x, y;
};
template <typename E, int VEC>
DEV Unit<VEC> load_plain(const E *row, int e, int D) {
    Unit<VEC> w;
    if constexpr (VEC == 1) {
        w.x[0] = (float)row[e];
        w.y[0] = e + 1 < D ? (float)row[e + 1] : 0.0f;
    } else {
        w.x = load_n<E, VEC>(row + e);
        w.y = load_n<E, VEC>(row + e + VEC);
    }
    return w;
}
template <typename E, int VEC>
DEV void store_plain(E *row, int e, int D, const Unit<VEC> &w) {
    if constexpr (VEC == 1) {
        row[e] = (E)w.x[0];
        if (e + 1 < D) row[e + 1] = (E)w.y[0];
    } else {
        store_n<E, VEC>(row + e, w.x);
        store_n<E, VEC>(row + e + VEC, w.y);
    }
}
template <typename E, int VEC, bool NORM>
DEV Unit<VEC> unit_load(const E *row, int u, int UR, int P, int D) {
    if (NORM || u >= UR) return load_plain<E, VEC>(row, u * 2 * VEC, D);  // 2 P elements before: UR units
    Unit<VEC> w;
    if constexpr (VEC == 1) {
        w.x[0] = (float)row[u];
        w.y[0] = (float)row[P + u];
    } else {
        w.x = load_n<E, VEC>(row + u * VEC);
        w.y = load_n<E, VEC>(row + P + u * VEC);
    }
    return w;
}
template <typename E, int VEC, bool NORM>
DEV void unit_store(E *row, int u, int UR, int P, int D, const Unit<VEC> &w, vf<VEC> c, vf<VEC> s) {
    if (u >= UR) {
        store_plain<E, VEC>(row, u * 2 * VEC, D, w);
        return;
    }
    Unit<VEC> z;
    if constexpr (NORM) {
        // neighbours make a pair: x holds elements 0 .. VEC - 1 of the unit, y the rest
#pragma unroll
        for (int j = 0; j < VEC; j++) {
            const int e = 2 * j;
            const float x0 = VEC == 1 || e < VEC ? w.x[e % VEC] : w.y[e % VEC];
            const float x1 = VEC == 1 ? w.y[0] : e < VEC ? w.x[(e + 1) % VEC] : w.y[(e + 1) % VEC];
            const float a = fmaf(x0, c[j], -(x1 * s[j])), b = fmaf(x0, s[j], x1 * c[j]);
            if (VEC == 1) {
                z.x[0] = a;
                z.y[0] = b;
            } else if (e < VEC) {
                z.x[e % VEC] = a;
                z.x[(e + 1) % VEC] = b;
            } else {
                z.y[e % VEC] = a;
                z.y[(e + 1) % VEC] = b;
            }
        }
        store_plain<E, VEC>(row, u * 2 * VEC, D, z);
    } else {
#pragma unroll
        for (int j = 0; j < VEC; j++) {
            z.x[j] = fmaf(w.x[j], c[j], -(w.y[j] * s[j]));
            z.y[j] = fmaf(w.x[j], s[j], w.y[j] * c[j]);
        }
        if constexpr (VEC == 1) {
            row[u] = (E)z.x[0];
            row[P + u] = (E)z.y[0];
        } else {
            store_n<E, VEC>(row + u * VEC, z.x);
            store_n<E, VEC>(row + P + u * VEC, z.y);
        }
    }
}

struct RopeParams {
    const void *x;
    void *y;
    int64_t x_nb1, x_nb2, y_nb1, y_nb2;  // elements: head, token
    const int32_t *pos;
    int64_t pos_nb1;
    const float *factors;  // or null
    int T, H, D, P;        // P rotated pairs
    int U, UR, HG;         // units of a row, rotated ones; groups of HN heads
    RopeTab tab;
};

template <typename E, int VEC, bool NORM, int HN>
DEV void rope_impl(const RopeParams &p) {
    const uint32_t id = blockIdx.x * 256u + threadIdx.x;
    const uint32_t r = id / (uint32_t)p.U;
    const int u = (int)(id - r * (uint32_t)p.U);
    const int64_t t = r / (uint32_t)p.HG;
    const int h0 = (int)(r - (uint32_t)t * (uint32_t)p.HG) * HN;
    if (t >= p.T) return;
    const E *x = (const E *)p.x + t * p.x_nb2;
    E *y = (E *)p.y + t * p.y_nb2;
    Unit<VEC> w[HN];
    vf<VEC> c, s;
#pragma unroll
    for (int i = 0; i < HN; i++) w[i] = unit_load<E, VEC, NORM>(x + (int64_t)min(h0 + i, p.H - 1) * p.x_nb1, u, p.UR, p.P, p.D);
    if (u < p.UR) unit_angles<VEC>(p.tab, p.pos, p.pos_nb1, p.tab.axes, p.factors, t, u * VEC, c, s);
#pragma unroll
    for (int i = 0; i < HN; i++)
        if (h0 + i < p.H) unit_store<E, VEC, NORM>(y + (int64_t)(h0 + i) * p.y_nb1, u, p.UR, p.P, p.D, w[i], c, s);
}

struct AppendParams {
    const void *k, *v;
    int64_t k_nb1, k_nb2, v_nb1, v_nb2;  // elements: head, token
    void *kv;
    int64_t kv_head, kv_row, kv_page;  // elements
    const int64_t *slots;
    int64_t n_slots;   // page * pages: other slots are not written
    int64_t page;      // rows of a page; 0: page p's rows follow page p - 1's
    const int32_t *pos;
    int64_t pos_nb1;
    const float *factors;
    int T, H, D, P, U, UR, HG;
    RopeTab tab;
};

// Row `slot` of head h: K's D elements (rotated), then V's D.  Unit u of K and
// the same elements of V go together, so a thread's stores fill both halves of
// the row and one slot look-up serves 2 HN of them.
template <typename E, typename C, int VEC, bool NORM, int HN>
DEV void append_impl(const AppendParams &p) {
    const uint32_t id = blockIdx.x * 256u + threadIdx.x;
    const uint32_t r = id / (uint32_t)p.U;
    const int u = (int)(id - r * (uint32_t)p.U);
    const int64_t t = r / (uint32_t)p.HG;
    const int h0 = (int)(r - (uint32_t)t * (uint32_t)p.HG) * HN;
    if (t >= p.T) return;
    const int64_t slot = p.slots[t];
    const E *k = (const E *)p.k + t * p.k_nb2, *v = (const E *)p.v + t * p.v_nb2;
    Unit<VEC> w[HN], z[HN];
    vf<VEC> c, s;
    const int ve = u * 2 * VEC;
#pragma unroll
    for (int i = 0; i < HN; i++) {
        const int64_t h = min(h0 + i, p.H - 1);
        w[i] = unit_load<E, VEC, NORM>(k + h * p.k_nb1, u, p.UR, p.P, p.D);
        z[i] = load_plain<E, VEC>(v + h * p.v_nb1, ve, p.D);
    }
    if (slot < 0 || slot >= p.n_slots) return;  // padding, or a slot outside the cache
    if (u < p.UR) unit_angles<VEC>(p.tab, p.pos, p.pos_nb1, p.tab.axes, p.factors, t, u * VEC, c, s);
    C *row = (C *)p.kv;
    if (p.page) {
        const int64_t pg = (int64_t)((uint64_t)slot / (uint64_t)p.page);
        row += pg * p.kv_page + (slot - pg * p.page) * p.kv_row;
    } else {
        row += slot * p.kv_row;
    }
#pragma unroll
    for (int i = 0; i < HN; i++) {
        if (h0 + i >= p.H) continue;
        C *o = row + (int64_t)(h0 + i) * p.kv_head;
        unit_store<C, VEC, NORM>(o, u, p.UR, p.P, p.D, w[i], c, s);
        store_plain<C, VEC>(o + p.D, ve, p.D, z[i]);
    }
}

#define ROPE_K(E, N, NORM, VEC, HN)                                                                              \
    extern "C" __global__ void __launch_bounds__(256) ghip_rope_##E##_##N##_v##VEC##_h##HN(RopeParams p) {       \
        rope_impl<E, VEC, NORM, HN>(p);                                                                          \
    }
#define APPEND_K(E, C, N, NORM, VEC, HN)                                                                         \
    extern "C" __global__ void __launch_bounds__(256) ghip_append_##E##_##C##_##N##_v##VEC##_h##HN(AppendParams p) { \
        append_impl<E, C, VEC, NORM, HN>(p);                                                                     \
    }
typedef float f32;
#define ROPE_E(E)                                                                                                \
    ROPE_K(E, norm, true, 4, 1) ROPE_K(E, norm, true, 4, 4) ROPE_K(E, norm, true, 1, 1) ROPE_K(E, norm, true, 1, 4) \
    ROPE_K(E, half, false, 4, 1) ROPE_K(E, half, false, 4, 4) ROPE_K(E, half, false, 1, 1) ROPE_K(E, half, false, 1, 4)
#define APPEND_E(E, C)                                                                                           \
    APPEND_K(E, C, norm, true, 4, 1) APPEND_K(E, C, norm, true, 4, 4)                                            \
    APPEND_K(E, C, norm, true, 1, 1) APPEND_K(E, C, norm, true, 1, 4)                                            \
    APPEND_K(E, C, half, false, 4, 1) APPEND_K(E, C, half, false, 4, 4)                                          \
    APPEND_K(E, C, half, false, 1, 1) APPEND_K(E, C, half, false, 1, 4)
ROPE_E(f32) ROPE_E(f16) ROPE_E(bf16)
APPEND_E(f32, f16) APPEND_E(f32, bf16) APPEND_E(f16, f16) APPEND_E(bf16, bf16)
