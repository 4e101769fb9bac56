// ghip_fap.hip -- attention over a paged KV cache: a batch of sequences of any
// length, each with its query rows at the end of its keys.
//
// Row i of a sequence with nq rows and nkv keys is at position p = nkv - nq + i
// and sees the keys j <= p with j > p - window or j < n_first (no window: all
// of them):  o = sum_j e^(s_j - m) v_j / sum_j e^(s_j - m),  s_j = scale q . k_j;
// a sink adds e^(sink - m) below the line.  A row that sees nothing gives 0.
// Key j is row j % page of page table[j / page]; a row that sees a key whose
// page does not exist gives NaN, and no key that no row sees is read.
#include "ghip_common.h"
#include "ghip_paged.h"

typedef _Float16 f16;
typedef __bf16 bf16;

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
    float scale;
    int window, n_first, n_shared, max_q;
};

// One wavefront a row of one head: 64 keys at a time, a lane scoring one key;
// then every lane owns dims lane, lane + 64, .. of the output.
template <typename E>
DEV void fap_rows(const FapParams &p) {
    __shared__ float qs[256];
    const int lane = threadIdx.x;
    const int h = blockIdx.x % p.H;
    const int bi = blockIdx.x / p.H, b = bi / p.max_q, i = bi - b * p.max_q;
    const int32_t *row = p.seqs + (int64_t)b * p.seq_nb1;
    const PagedSeq s = paged_seq(row[0], row[1], row[2], p.T, p.max_q);
    if (i >= s.nq) return;
    const int64_t t = s.q0 + i, pos = s.pos0 + i;
    for (int d = lane; d < p.D; d += 64) qs[d] = p.q[t * p.q_nb2 + h * p.q_nb1 + d] * p.scale;
    __syncthreads();
    const E *kv = (const E *)p.kv + (h / (p.H / p.H_kv)) * p.kv_head;
    const PagedKeys kr = paged_keys(pos, pos, p.window, p.n_first);
    const int64_t table = (int64_t)p.per * p.page;
    float m = -__builtin_inff(), l = 0.0f, o[4] = {0, 0, 0, 0};
    bool bad = kr.hi > table;
    for (int part = 0; part < 2; part++) {
        const int64_t a = part ? kr.lo : 0, e = part ? min(kr.hi, table) : min(kr.first, table);
        for (int64_t k0 = a; k0 < e; k0 += 64) {
            const int64_t j = k0 + lane;
            float x = -__builtin_inff();
            int64_t at = -1;
            if (j < e) {
                const int32_t pg = row[3 + j / p.page];
                if (pg >= 0 && pg < p.n_pages) {
                    at = pg * p.kv_page + (j % p.page) * p.kv_row;
                    x = 0.0f;
                    for (int d = 0; d < p.D; d++) x = fmaf(qs[d], (float)kv[at + d], x);
                } else {
                    bad = true;
                }
            }
            float mx = x;
            for (int w = 32; w; w >>= 1) mx = fmaxf(mx, __shfl_xor(mx, w, 64));
            const float mn = fmaxf(m, mx);
            const float alpha = mn == -__builtin_inff() ? 1.0f : __expf(m - mn);
            const float pr = x == -__builtin_inff() ? 0.0f : __expf(x - mn);
            m = mn;
            l = l * alpha + wave_sum(pr);
            for (int u = 0; u < 4; u++) o[u] *= alpha;
            for (int jj = 0; jj < 64; jj++) {
                const float pj = __shfl(pr, jj, 64);
                const int64_t aj = __shfl(at, jj, 64);
                if (aj < 0) continue;
                for (int u = 0; u < 4; u++)
                    if (lane + 64 * u < p.D) o[u] = fmaf(pj, (float)kv[aj + p.D + lane + 64 * u], o[u]);
            }
        }
    }
    if (p.sinks) {
        const float sk = p.sinks[h], mn = fmaxf(m, sk);
        const float alpha = mn == -__builtin_inff() ? 1.0f : __expf(m - mn);
        l = l * alpha + (mn == -__builtin_inff() ? 0.0f : __expf(sk - mn));
        for (int u = 0; u < 4; u++) o[u] *= alpha;
    }
    const bool nan = __ballot(bad) != 0;
    for (int u = 0; u < 4; u++)
        if (lane + 64 * u < p.D)
            p.dst[t * p.d_nb2 + h * p.d_nb1 + lane + 64 * u] = nan ? __builtin_nanf("") : l > 0.0f ? o[u] / l : 0.0f;
}
extern "C" __global__ void __launch_bounds__(64) ghip_fap_rows_f16(FapParams p) { fap_rows<f16>(p); }
extern "C" __global__ void __launch_bounds__(64) ghip_fap_rows_bf16(FapParams p) { fap_rows<bf16>(p); }
