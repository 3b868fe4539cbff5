// Attention over the cache in 8 bits (kv8.cuh): the newest tokens of every sequence against all that it holds, soft-capped,
// windowed, causal, with several query heads on a kv head.
//
//     z = scale * q . k,   cap tanh(z / cap),   key j visible from position p iff 0 <= p - j < window,
//     out = sum_j softmax_j(z) v_j,   zeros where a token sees no key.
#include "kv8.cuh"

namespace {

using namespace kv8;

struct AttnArgs {
    const void* q;
    void* out;
    int q_stride, out_stride;
    const int32_t *cu_q, *kv_len, *slots, *tables;
    const int8_t *k_pages, *v_pages;
    const float *k_scale, *v_scale;
    int rows, n_kv, group, dim, block, n_blocks, n_slots, width, ring, window;
    float scale, cap;
};

// A warp for every (token, query head).
template <typename T>
__global__ void __launch_bounds__(32) attn_kv8_plain_kernel(AttnArgs a) {
    pdl_trigger();
    pdl_wait();
    const int t = blockIdx.x, head = blockIdx.y, lane = threadIdx.x, g = head / a.group;
    if (t >= a.cu_q[a.rows]) return;
    int lo = 0, hi = a.rows;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (a.cu_q[mid] <= t) lo = mid;
        else hi = mid;
    }
    const int s = a.slots[lo], len = a.kv_len[lo], pos = len - (a.cu_q[lo + 1] - t);
    const T* q = reinterpret_cast<const T*>(a.q) + (size_t)t * a.q_stride + head * a.dim;
    float qv[8], o[8] = {};
#pragma unroll
    for (int i = 0; i < 8; ++i) qv[i] = lane + 32 * i < a.dim ? to_float(q[lane + 32 * i]) : 0.0f;
    float m = -INFINITY, l = 0.0f;
    const int first = a.window > 0 ? max(0, pos - a.window + 1) : 0;
    for (int j = first; j <= pos && s >= 0 && s < a.n_slots; ++j) {
        const int place = a.ring > 0 ? j % a.ring : j;
        const int b = place / a.block < a.width ? a.tables[(size_t)s * a.width + place / a.block] : -1;
        if (b < 0 || b >= a.n_blocks) continue;
        const size_t bh = (size_t)b * a.n_kv + g, at = (bh * a.block + place % a.block) * a.dim;
        float z = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (lane + 32 * i < a.dim) z = fmaf(qv[i], (float)a.k_pages[at + lane + 32 * i], z);
        z = soft_cap(warp_sum(z) * a.k_scale[bh] * a.scale, a.cap);
        const float m_new = z > m ? z : m, keep = m > -INFINITY ? expf(m - m_new) : 0.0f, p = expf(z - m_new);
        m = m_new;
        l = l * keep + p;
        const float ps = p * a.v_scale[bh];
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (lane + 32 * i < a.dim) o[i] = fmaf(ps, (float)a.v_pages[at + lane + 32 * i], o[i] * keep);
    }
    T* out = reinterpret_cast<T*>(a.out) + (size_t)t * a.out_stride + head * a.dim;
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (lane + 32 * i < a.dim) out[lane + 32 * i] = from_float<T>(l != 0.0f ? o[i] / l : 0.0f);
}

}  // namespace

BROLM_API int brolm_attn_kv8(const void* q, int q_stride, void* out, int out_stride, int dtype, const void* cu_q,
                             const void* kv_len, const void* slots, const void* tables, const void* k_pages,
                             const void* v_pages, const void* k_scale, const void* v_scale, int tokens, int rows, int n_kv,
                             int group, int dim, int block, int n_blocks, int n_slots, int width, int ring, int window,
                             float scale, float cap, int max_q_len, int max_kv_len, cudaStream_t stream) {
    if (dtype != BROLM_F32 && dtype != BROLM_BF16) return BROLM_ERR_BAD_DTYPE;
    if (tokens < 0 || rows < 0 || n_kv <= 0 || group <= 0 || dim <= 0 || dim % 16 || block <= 0 || block % 32) return BROLM_ERR_BAD_SIZE;
    if (n_blocks <= 0 || n_slots <= 0 || width <= 0 || ring < 0 || ring % block || window < 0) return BROLM_ERR_BAD_SIZE;
    if (dim > MAX_DIM || block > MAX_BLOCK || n_kv * group > 65535) return BROLM_ERR_TOO_LARGE;
    if (tokens == 0 || rows == 0) return BROLM_OK;
    AttnArgs a{q, out, q_stride, out_stride, (const int32_t*)cu_q, (const int32_t*)kv_len, (const int32_t*)slots,
               (const int32_t*)tables, (const int8_t*)k_pages, (const int8_t*)v_pages, (const float*)k_scale,
               (const float*)v_scale, rows, n_kv, group, dim, block, n_blocks, n_slots, width, ring, window, scale, cap};
    const dim3 grid(tokens, n_kv * group);
    if (dtype == BROLM_F32) return launch_pdl(attn_kv8_plain_kernel<float>, grid, dim3(32), 0, stream, a);
    return launch_pdl(attn_kv8_plain_kernel<bf16>, grid, dim3(32), 0, stream, a);
}
