// ghip_rope.hip -- rotary positions with one or several axes, and appending
// keys and values to a paged KV cache with the rotation on the way.
//
// Pair i of a token is turned by the angle  a = p[axis(i)] * f_i / factor_i:
//   (x0, x1) -> (x0 cos a - x1 sin a, x0 sin a + x1 cos a)
// with the token's position p on the pair's axis (text: one axis; image and
// video: time, height, width).  f_i, which pairs an axis has and the context
// extension are worked out on the host in 64 bits (RopeTab), in turns per
// position: the angle is  p * f_i  turns, and only its fraction counts.  That
// product and the reduction to a fraction are 64-bit here too -- at position
// 100000 a 32-bit product is off by up to 2^-8 radians -- and sin and cos of
// the remaining eighth turn are polynomials in 32 bits.
//
// Work layout.  Both kernels are bound by memory: every element is read once
// and written once.  A thread takes one unit of a token's head row -- VEC
// pairs, or the 2 VEC elements of a part that is not rotated -- for HN heads:
// the angles are formed once for HN heads (they cost as much as the loads of
// two), and all HN loads are in flight before the first store.  Neighbouring
// lanes hold neighbouring units of the same row.
#include "ghip_common.h"

typedef _Float16 f16;
typedef __bf16 bf16;

struct RopeTab {
    double rev[128];    // turns per position of each pair
    uint8_t axis[128];  // the pair's row of positions
    float mscale;       // factor of cos and sin
};

template <typename E, int N>
DEV void load_n(const E *p, float (&v)[N]) {
    E t[N];
    __builtin_memcpy(t, p, sizeof(E) * N);
#pragma unroll
    for (int i = 0; i < N; i++) v[i] = (float)t[i];
}
// one rounding to nearest where E is narrower than 32 bits
template <typename E, int N>
DEV void store_n(E *p, const float (&v)[N]) {
    E t[N];
#pragma unroll
    for (int i = 0; i < N; i++) t[i] = (E)v[i];
    __builtin_memcpy(p, t, sizeof(E) * N);
}

// sin and cos of a turns.  Whole turns and the nearest quarter come off in 64
// bits, exactly; the rest, |t| <= pi / 4, is rounded once (2^-24 radians), and
// its Taylor sums end where the next term is below 2^-29.
DEV void sincos_turns(double a, float &s, float &c) {
    const double a4 = 4.0 * (a - rint(a)), q = rint(a4);
    const float t = 1.5707963267948966f * (float)(a4 - q);
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
    const int k = (int)q;
    const float u = k & 1 ? cn : sn, v = k & 1 ? sn : cn;
    s = k & 2 ? -u : u;
    c = (k + 1) & 2 ? -v : v;
}

// cos and sin of VEC pairs from pair i0 on, for token t
template <int VEC>
DEV void unit_angles(const RopeTab &tab, const int32_t *pos, int64_t pos_nb1, const float *factors, int64_t t, int i0,
                     float (&c)[VEC], float (&s)[VEC]) {
#pragma unroll
    for (int j = 0; j < VEC; j++) {
        const int i = i0 + j;
        double f = tab.rev[i];
        if (factors) f /= (double)factors[i];
        sincos_turns((double)pos[(int64_t)tab.axis[i] * pos_nb1 + t] * f, s[j], c[j]);
        s[j] *= tab.mscale;
        c[j] *= tab.mscale;
    }
}

// one unit of a row: u < UR rotated (pairs VEC u ..), else the elements 2 P + ..
// as they are.  `w` holds the unit's 2 VEC values.
template <typename E, int VEC, bool NORM>
DEV void unit_load(const E *row, int u, int UR, int P, int D, float (&w)[2 * VEC]) {
    if (u >= UR) {
        const int e = 2 * P + (u - UR) * 2 * VEC;
        if constexpr (VEC == 1) {
            w[0] = (float)row[e];
            w[1] = e + 1 < D ? (float)row[e + 1] : 0.0f;
        } else {
            load_n<E, 2 * VEC>(row + e, w);
        }
    } else if constexpr (NORM) {
        load_n<E, 2 * VEC>(row + u * 2 * VEC, w);
    } else {
        float a[VEC], b[VEC];
        load_n<E, VEC>(row + u * VEC, a);
        load_n<E, VEC>(row + P + u * VEC, b);
#pragma unroll
        for (int j = 0; j < VEC; j++) {
            w[2 * j] = a[j];
            w[2 * j + 1] = b[j];
        }
    }
}
template <typename E, int VEC, bool NORM>
DEV void unit_store(E *row, int u, int UR, int P, int D, const float (&w)[2 * VEC], const float (&c)[VEC],
                    const float (&s)[VEC]) {
    if (u >= UR) {
        const int e = 2 * P + (u - UR) * 2 * VEC;
        if constexpr (VEC == 1) {
            row[e] = (E)w[0];
            if (e + 1 < D) row[e + 1] = (E)w[1];
        } else {
            store_n<E, 2 * VEC>(row + e, w);
        }
        return;
    }
    float a[VEC], b[VEC], y[2 * VEC];
#pragma unroll
    for (int j = 0; j < VEC; j++) {
        const float x0 = w[2 * j], x1 = w[2 * j + 1];
        a[j] = fmaf(x0, c[j], -(x1 * s[j]));
        b[j] = fmaf(x0, s[j], x1 * c[j]);
        y[2 * j] = a[j];
        y[2 * j + 1] = b[j];
    }
    if constexpr (NORM) {
        store_n<E, 2 * VEC>(row + u * 2 * VEC, y);
    } else {
        store_n<E, VEC>(row + u * VEC, a);
        store_n<E, VEC>(row + P + u * VEC, b);
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
    float w[HN][2 * VEC], c[VEC], s[VEC];
#pragma unroll
    for (int i = 0; i < HN; i++) unit_load<E, VEC, NORM>(x + (int64_t)min(h0 + i, p.H - 1) * p.x_nb1, u, p.UR, p.P, p.D, w[i]);
    if (u < p.UR) unit_angles<VEC>(p.tab, p.pos, p.pos_nb1, p.factors, t, u * VEC, c, s);
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
    float w[HN][2 * VEC], z[HN][2 * VEC], c[VEC], s[VEC];
    const int ve = u * 2 * VEC;
#pragma unroll
    for (int i = 0; i < HN; i++) {
        const int64_t h = min(h0 + i, p.H - 1);
        unit_load<E, VEC, NORM>(k + h * p.k_nb1, u, p.UR, p.P, p.D, w[i]);
        if constexpr (VEC == 1) {
            z[i][0] = (float)v[h * p.v_nb1 + ve];
            z[i][1] = ve + 1 < p.D ? (float)v[h * p.v_nb1 + ve + 1] : 0.0f;
        } else {
            load_n<E, 2 * VEC>(v + h * p.v_nb1 + ve, z[i]);
        }
    }
    if (slot < 0 || slot >= p.n_slots) return;  // padding, or a slot outside the cache
    if (u < p.UR) unit_angles<VEC>(p.tab, p.pos, p.pos_nb1, p.factors, t, u * VEC, c, s);
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
        if constexpr (VEC == 1) {
            o[p.D + ve] = (C)z[i][0];
            if (ve + 1 < p.D) o[p.D + ve + 1] = (C)z[i][1];
        } else {
            store_n<C, 2 * VEC>(o + p.D + ve, z[i]);
        }
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
