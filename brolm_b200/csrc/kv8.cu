// The cache in 8 bits: new keys and values into its blocks, and what it holds back out (kv8.cuh for the numbers).
#include "kv8.cuh"

namespace {

using namespace kv8;

struct WriteArgs {
    const void* x[2];                    // keys, values: [tokens][heads][D] with these strides (elements)
    long long token_stride[2], head_stride[2];
    int8_t* pages[2];
    float* scales[2];
    const int32_t *cu_q, *positions, *cache_rows;
    int tokens, rows, n_kv, dim, block, n_blocks, single;
};

// Eight consecutive entries of a row as they lie in memory: one load where the row is aligned, one a number where not.
template <typename T, bool WIDE>
__device__ __forceinline__ void fetch8(const T* p, float (&v)[8]) {
    if constexpr (WIDE) load8(p, v);
    else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = to_float(p[i]);
    }
}

// A block of threads takes the new tokens of one cache block for one head, keys or values (blockIdx.y, .z): those of a
// row of the step whose positions fall into it.  blockIdx.x counts the cache blocks that the rows touch: row i begins at
// cu_q[i] / P + 2 i, which leaves every row at least as many places as blocks it can touch (floor(n / P) + 2); `single`:
// no row brings more than one token, and x is the row.
//
//   1. the largest new number (kept in registers, eight at a time: ITEMS x 8 a thread; what is beyond is read again);
//   2. the scale, from that and, where the block was begun before, from the scale that it had;
//   3. where that grew: the numbers that were there, rounded to it;
//   4. the new numbers.
template <typename T, bool WIDE, int ITEMS>
__global__ void __launch_bounds__(512) kv8_write_kernel(WriteArgs a) {
    __shared__ float scratch[33];
    pdl_trigger();
    pdl_wait();
    const int P = a.block, D8 = a.dim >> 3;
    int i = blockIdx.x, k = 0;
    if (!a.single) {
        int lo = 0, hi = a.rows;
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (a.cu_q[mid] / P + 2 * mid <= (int)blockIdx.x) lo = mid;
            else hi = mid;
        }
        i = lo;
        k = blockIdx.x - (a.cu_q[i] / P + 2 * i);
    }
    // (where every row brings one token, token i is row i's: its position and place are asked for with the sums, not after)
    const int likely = min(i, a.tokens - 1);
    const int likely_pos = a.positions[likely], likely_row = a.cache_rows[likely];
    const int first = max(0, a.cu_q[i]), end = min(a.tokens, a.cu_q[i + 1]);
    if (first >= end) return;
    const int p0 = first == likely ? likely_pos : a.positions[first];
    if (p0 < 0) return;                                        // padding
    const int in_block = p0 % P;
    const long long t0 = first + (k == 0 ? 0ll : (long long)k * P - in_block);
    if (t0 >= end) return;
    const int n = (int)min((long long)end - t0, (long long)(k == 0 ? P - in_block : P));
    const int row = t0 == likely ? likely_row : a.cache_rows[t0];
    if (row < 0 || row / P >= a.n_blocks) return;              // the ring keeps none of these
    const int b = row / P, at = row % P, h = blockIdx.y, which = blockIdx.z;
    if (at + n > P) return;                                    // (not a slot map: nothing is written)
    const T* x = reinterpret_cast<const T*>(a.x[which]) + t0 * a.token_stride[which] + h * a.head_stride[which];
    const long long ts = a.token_stride[which];
    int8_t* page = a.pages[which] + ((size_t)b * a.n_kv + h) * P * a.dim;
    float* scale = a.scales[which] + (size_t)b * a.n_kv + h;
    const float s_old = at > 0 ? *scale : 0.0f;

    const int items = n * D8;
    float v[ITEMS][8];
    float most = 0.0f;
    bool finite = true;
#pragma unroll
    for (int j = 0; j < ITEMS; ++j) {
        const int it = threadIdx.x + j * blockDim.x;
        if (it < items) {
            fetch8<T, WIDE>(x + (it / D8) * ts + (it % D8) * 8, v[j]);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                most = fmaxf(most, fabsf(v[j][e]));
                finite = finite && fabsf(v[j][e]) < INFINITY;  // (false for NaN too, which fmaxf passes over)
            }
        }
    }
    for (int it = threadIdx.x + ITEMS * blockDim.x; it < items; it += blockDim.x) {
        float w[8];
        fetch8<T, WIDE>(x + (it / D8) * ts + (it % D8) * 8, w);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            most = fmaxf(most, fabsf(w[e]));
            finite = finite && fabsf(w[e]) < INFINITY;
        }
    }
    most = block_max(finite ? most : INFINITY, scratch);
    const bool bad = !(most < INFINITY) || s_old != s_old;
    int e = 0;
    if (!bad) {
        e = scale_exponent(most);
        if (at > 0) {
            const int e_old = max(-126, (int)(__float_as_uint(s_old) >> 23 & 255u) - 127);
            if (e > e_old) {
                // rint(q 2^(e_old - e)); half of 127 2^-8 rounds to nothing, and so does all below
                const float factor = power_of_two(max(e_old - e, -16));
                const int vecs = at * a.dim / 16;
                for (int it = threadIdx.x; it < vecs; it += blockDim.x) {
                    int4 w = reinterpret_cast<int4*>(page)[it];
                    int8_t* q = reinterpret_cast<int8_t*>(&w);
#pragma unroll
                    for (int c = 0; c < 16; ++c) q[c] = (int8_t)__float2int_rn((float)q[c] * factor);
                    reinterpret_cast<int4*>(page)[it] = w;
                }
            } else {
                e = e_old;
            }
        }
    }
    if (threadIdx.x == 0) *scale = bad ? __int_as_float(0x7fc00000) : power_of_two(e);
    const float inv = bad ? 0.0f : power_of_two(-e);
    int8_t* dst = page + (size_t)at * a.dim;
    auto put = [&](int it, const float (&w)[8]) {
        int q[8];
#pragma unroll
        for (int c = 0; c < 8; ++c) q[c] = bad ? 0 : __float2int_rn(w[c] * inv);
        uint2 r;
        r.x = __byte_perm(__byte_perm(q[0], q[1], 0x0040), __byte_perm(q[2], q[3], 0x0040), 0x5410);
        r.y = __byte_perm(__byte_perm(q[4], q[5], 0x0040), __byte_perm(q[6], q[7], 0x0040), 0x5410);
        reinterpret_cast<uint2*>(dst)[it] = r;
    };
#pragma unroll
    for (int j = 0; j < ITEMS; ++j) {
        const int it = threadIdx.x + j * blockDim.x;
        if (it < items) put(it, v[j]);
    }
    for (int it = threadIdx.x + ITEMS * blockDim.x; it < items; it += blockDim.x) {
        float w[8];
        fetch8<T, WIDE>(x + (it / D8) * ts + (it % D8) * 8, w);
        put(it, w);
    }
}

struct ReadArgs {
    const int8_t* pages[2];
    const float* scales[2];
    void* out[2];
    long long token_stride[2], head_stride[2];
    const int32_t *cu_r, *kv_len, *slots, *tables;
    int tokens, rows, n_kv, dim, block, n_blocks, n_slots, width, ring;
};

constexpr int READ_TOKENS = 8;

// The last n_i = cu_r[i + 1] - cu_r[i] tokens of row i, back to back; what the ring no longer holds reads as zero.
template <typename T>
__global__ void __launch_bounds__(256) kv8_read_kernel(ReadArgs a) {
    __shared__ int block_s[READ_TOKENS], place_s[READ_TOKENS];
    pdl_trigger();
    pdl_wait();
    const int t0 = blockIdx.x * READ_TOKENS, P = a.block;
    if (threadIdx.x < READ_TOKENS) {
        const int t = t0 + threadIdx.x;
        int b = -1, at = 0;
        if (t < a.tokens && t < a.cu_r[a.rows]) {
            int lo = 0, hi = a.rows;
            while (hi - lo > 1) {
                const int mid = (lo + hi) >> 1;
                if (a.cu_r[mid] <= t) lo = mid;
                else hi = mid;
            }
            const int len = a.kv_len[lo], s = a.slots[lo];
            const int pos = len - (a.cu_r[lo + 1] - t);
            if (pos >= 0 && s >= 0 && s < a.n_slots && (a.ring == 0 || pos / P + a.ring / P > (len - 1) / P)) {
                at = a.ring > 0 ? pos % a.ring : pos;
                if (at / P < a.width) b = a.tables[(size_t)s * a.width + at / P];
                at %= P;
            }
        }
        block_s[threadIdx.x] = b;
        place_s[threadIdx.x] = at;
    }
    __syncthreads();
    const int D16 = a.dim >> 4, per = a.n_kv * D16, all = READ_TOKENS * per;
    const int which = blockIdx.y;
    for (int it = threadIdx.x; it < all; it += blockDim.x) {
        const int j = it / per, h = (it - j * per) / D16, c = it % D16;
        const int t = t0 + j;
        if (t >= a.tokens) break;
        const int b = block_s[j];
        int4 w = make_int4(0, 0, 0, 0);
        float s = 0.0f;
        if (b >= 0 && b < a.n_blocks) {
            const size_t bh = (size_t)b * a.n_kv + h;
            w = __ldg(reinterpret_cast<const int4*>(a.pages[which] + (bh * P + place_s[j]) * a.dim) + c);
            s = a.scales[which][bh];
        }
        const int8_t* q = reinterpret_cast<const int8_t*>(&w);
        T* dst = reinterpret_cast<T*>(a.out[which]) + t * a.token_stride[which] + h * a.head_stride[which] + c * 16;
        alignas(16) T v[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) v[e] = from_float<T>((float)q[e] * s);
#pragma unroll
        for (int e = 0; e < (int)sizeof(T); ++e) reinterpret_cast<int4*>(dst)[e] = reinterpret_cast<int4*>(v)[e];
    }
}

bool aligned(const void* p, long long token_stride, long long head_stride, int size) {
    return ((uintptr_t)p & 15) == 0 && token_stride * size % 16 == 0 && head_stride * size % 16 == 0;
}

int check_cache(const void* k_pages, const void* v_pages, int n_kv, int dim, int block, int n_blocks) {
    if (n_kv <= 0 || dim <= 0 || dim % 16 || block <= 0 || block % 32 || n_blocks <= 0) return BROLM_ERR_BAD_SIZE;
    if (dim > MAX_DIM || block > MAX_BLOCK || n_kv > 65535 || (long long)n_blocks * block > 0x7fffffffll) return BROLM_ERR_TOO_LARGE;
    if (((uintptr_t)k_pages | (uintptr_t)v_pages) & 15) return BROLM_ERR_ALIGNMENT;
    return BROLM_OK;
}

template <typename T>
int launch_write(const WriteArgs& a, dim3 grid, int threads, bool wide, cudaStream_t stream) {
    if (wide) return launch_pdl(kv8_write_kernel<T, true, 8>, grid, dim3(threads), 0, stream, a);
    return launch_pdl(kv8_write_kernel<T, false, 8>, grid, dim3(threads), 0, stream, a);
}

}  // namespace

struct WriteCall {
    const void *k, *v, *cu_q, *positions, *cache_rows;
    void *k_pages, *v_pages, *k_scale, *v_scale;
    cudaStream_t stream;
    long long k_token, v_token, k_head, v_head;
    int dtype, tokens, rows, n_kv, dim, block, n_blocks, max_q_len;
};
struct ReadCall {
    const void *cu_r, *kv_len, *slots, *tables, *k_pages, *v_pages, *k_scale, *v_scale;
    void *k, *v;
    cudaStream_t stream;
    long long k_token, v_token, k_head, v_head;
    int dtype, tokens, rows, n_kv, dim, block, n_blocks, n_slots, width, ring;
};

BROLM_API int brolm_kv8_write(const WriteCall* c) {
    if (c->dtype != BROLM_F32 && c->dtype != BROLM_BF16) return BROLM_ERR_BAD_DTYPE;
    if (c->tokens < 0 || c->rows < 0) return BROLM_ERR_BAD_SIZE;
    const int st = check_cache(c->k_pages, c->v_pages, c->n_kv, c->dim, c->block, c->n_blocks);
    if (st) return st;
    if (c->tokens == 0 || c->rows == 0) return BROLM_OK;
    const bool single = c->max_q_len <= 1;
    const long long places = single ? c->rows : (long long)c->tokens / c->block + 2ll * c->rows;
    if (places > 0x7fffffffll) return BROLM_ERR_TOO_LARGE;
    WriteArgs a{{c->k, c->v}, {c->k_token, c->v_token}, {c->k_head, c->v_head}, {(int8_t*)c->k_pages, (int8_t*)c->v_pages},
                {(float*)c->k_scale, (float*)c->v_scale}, (const int32_t*)c->cu_q, (const int32_t*)c->positions,
                (const int32_t*)c->cache_rows, c->tokens, c->rows, c->n_kv, c->dim, c->block, c->n_blocks, single};
    const int size = c->dtype == BROLM_F32 ? 4 : 2;
    const bool wide = aligned(c->k, c->k_token, c->k_head, size) && aligned(c->v, c->v_token, c->v_head, size);
    const int threads = single ? 128 : max(128, min(512, (c->block * c->dim / 64 + 31) / 32 * 32));
    const dim3 grid((unsigned)places, c->n_kv, 2);
    return c->dtype == BROLM_F32 ? launch_write<float>(a, grid, threads, wide, c->stream) : launch_write<bf16>(a, grid, threads, wide, c->stream);
}

BROLM_API int brolm_kv8_read(const ReadCall* c) {
    if (c->dtype != BROLM_F32 && c->dtype != BROLM_BF16) return BROLM_ERR_BAD_DTYPE;
    if (c->tokens < 0 || c->rows < 0 || c->n_slots <= 0 || c->width <= 0 || c->ring < 0 || (c->block > 0 && c->ring % c->block)) return BROLM_ERR_BAD_SIZE;
    const int st = check_cache(c->k_pages, c->v_pages, c->n_kv, c->dim, c->block, c->n_blocks);
    if (st) return st;
    const int size = c->dtype == BROLM_F32 ? 4 : 2;
    if (!aligned(c->k, c->k_token, c->k_head, size) || !aligned(c->v, c->v_token, c->v_head, size)) return BROLM_ERR_ALIGNMENT;
    if (c->tokens == 0 || c->rows == 0) return BROLM_OK;
    ReadArgs a{{(const int8_t*)c->k_pages, (const int8_t*)c->v_pages}, {(const float*)c->k_scale, (const float*)c->v_scale}, {c->k, c->v},
               {c->k_token, c->v_token}, {c->k_head, c->v_head}, (const int32_t*)c->cu_r, (const int32_t*)c->kv_len,
               (const int32_t*)c->slots, (const int32_t*)c->tables, c->tokens, c->rows, c->n_kv, c->dim, c->block, c->n_blocks,
               c->n_slots, c->width, c->ring};
    const dim3 grid((c->tokens + READ_TOKENS - 1) / READ_TOKENS, 2);
    if (c->dtype == BROLM_F32) return launch_pdl(kv8_read_kernel<float>, grid, dim3(256), 0, c->stream, a);
    return launch_pdl(kv8_read_kernel<bf16>, grid, dim3(256), 0, c->stream, a);
}
