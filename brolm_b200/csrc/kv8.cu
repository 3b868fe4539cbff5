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
template <typename T>
struct Eight {
    uint32_t w[2 * sizeof(T)];
    template <bool WIDE>
    __device__ __forceinline__ void fetch(const T* p) {
        if constexpr (WIDE) {
#pragma unroll
            for (int i = 0; i < (int)sizeof(T) / 2; ++i) reinterpret_cast<uint4*>(w)[i] = reinterpret_cast<const uint4*>(p)[i];
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) reinterpret_cast<T*>(w)[i] = p[i];
        }
    }
    // the largest magnitude's bits, as a float's: infinities and NaN are above all else
    __device__ __forceinline__ uint32_t most() const {
        uint32_t m = 0;
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int i = 0; i < 8; ++i) m = max(m, w[i] & 0x7fffffffu);
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) m = __vmaxu2(m, w[i] & 0x7fff7fffu);
            m = max(m << 16, m & 0xffff0000u);
        }
        return m;
    }
    __device__ __forceinline__ float number(int i) const {
        if constexpr (sizeof(T) == 4) return __uint_as_float(w[i]);
        else return __uint_as_float(i & 1 ? w[i >> 1] & 0xffff0000u : w[i >> 1] << 16);
    }
};
// rint(x) in the low byte, for |x| <= 127: the product that x is, is exact, and the sum rounds it to a whole number (a
// conversion instruction takes the special function unit eight cycles).
__device__ __forceinline__ uint32_t whole(float x, float factor) { return __float_as_uint(fmaf(x, factor, 12582912.0f)); }
__device__ __forceinline__ uint32_t pack4(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}
// A byte of w, whose bytes are q + 128, as the float q.
template <int BYTE>
__device__ __forceinline__ float byte_number(uint32_t w) { return __uint_as_float(__byte_perm(w, 0x4b000000u, 0x7440 | BYTE)) - 8388736.0f; }

// A block of threads takes the new tokens of one cache block for one head, keys or values (blockIdx.y, .z): those of a
// row of the step whose positions fall into it.  blockIdx.x counts the cache blocks that the rows touch: row i begins at
// cu_q[i] / P + 2 i, which leaves every row at least as many places as blocks it can touch (floor(n / P) + 2); `single`:
// no row brings more than one token, and x is the row.
//
//   1. the largest new number (kept in registers, eight at a time: ITEMS x 8 a thread; what is beyond is read again);
//   2. the scale, from that and, where the block was begun before, from the scale that it had;
//   3. where that grew: the numbers that were there, rounded to it;
//   4. the new numbers.
//
// A block's numbers are read once and written once; what bounds it is the chain of round trips to memory (whose row, where
// it lies, its numbers, the scale there was), not their bytes: 2,048 bfloat16 tokens of 4 heads of 256 (12.6 MB) take 6.4 us
// in a captured loop, one token each of 64 sequences 3.2.  With a conversion instruction for every number, and a division
// for every eight, the first was 10.1.
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

    // (entry `it` of the block's items is eight entries of row r; the next that this thread takes is blockDim.x items further)
    const int items = n * D8, r0 = threadIdx.x / D8, c0 = threadIdx.x - r0 * D8, dr = blockDim.x / D8, dc = blockDim.x - dr * D8;
    Eight<T> v[ITEMS];
    uint32_t top = 0;
    int r = r0, c = c0;
    auto from = [&]() {
        const T* src = x + r * ts + c * 8;
        c += dc;
        const bool over = c >= D8;
        r += dr + (over ? 1 : 0);
        c -= over ? D8 : 0;
        return src;
    };
#pragma unroll
    for (int j = 0; j < ITEMS; ++j) {
        const T* src = from();
        if (threadIdx.x + j * blockDim.x < items) v[j].template fetch<WIDE>(src);
    }
#pragma unroll
    for (int j = 0; j < ITEMS; ++j)
        if (threadIdx.x + j * blockDim.x < items) top = max(top, v[j].most());
    for (int it = threadIdx.x + ITEMS * blockDim.x; it < items; it += blockDim.x) {
        Eight<T> w;
        w.template fetch<WIDE>(from());
        top = max(top, w.most());
    }
    const float most = block_max(top < 0x7f800000u ? __uint_as_float(top) : INFINITY, scratch);
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
                    uint4 w = reinterpret_cast<uint4*>(page)[it];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const uint32_t q = (&w.x)[i] ^ 0x80808080u;
                        (&w.x)[i] = pack4(whole(byte_number<0>(q), factor), whole(byte_number<1>(q), factor),
                                          whole(byte_number<2>(q), factor), whole(byte_number<3>(q), factor));
                    }
                    reinterpret_cast<uint4*>(page)[it] = w;
                }
            } else {
                e = e_old;
            }
        }
    }
    if (threadIdx.x == 0) *scale = bad ? __int_as_float(0x7fc00000) : power_of_two(e);
    const float inv = bad ? 0.0f : power_of_two(-e);
    int8_t* dst = page + (size_t)at * a.dim;
    auto put = [&](int it, const Eight<T>& w) {
        uint32_t q[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) q[i] = whole(w.number(i), inv);
        reinterpret_cast<uint2*>(dst)[it] = bad ? make_uint2(0u, 0u) : make_uint2(pack4(q[0], q[1], q[2], q[3]), pack4(q[4], q[5], q[6], q[7]));
    };
    r = r0;
    c = c0;
#pragma unroll
    for (int j = 0; j < ITEMS; ++j) {
        const int it = threadIdx.x + j * blockDim.x;
        from();
        if (it < items) put(it, v[j]);
    }
    for (int it = threadIdx.x + ITEMS * blockDim.x; it < items; it += blockDim.x) {
        Eight<T> w;
        w.template fetch<WIDE>(from());
        put(it, w);
    }
}

struct ReadArgs {
    const int8_t* pages[2];
    const float* scales[2];
    void* out[2];
    long long token_stride[2], head_stride[2];
    const int32_t *cu_r, *kv_len, *slots, *tables;
    int tokens, rows, n_kv, dim, block, n_blocks, n_slots, width, ring, most;
};

constexpr int READ_TOKENS = 8;

// The last n_i = cu_r[i + 1] - cu_r[i] tokens of row i, back to back; what the ring no longer holds reads as zero, and so does
// what comes before the last `most`.  A thread
// makes sixteen numbers from sixteen bytes.  Bounded by the memory: 26,575 bfloat16 tokens of 8 heads of 256 (327 MB) in 57.1
// us, 5.7 TB/s, 0.87 of a copy's rate.  Eight bytes a thread, so that its store fills half a sector by itself, took 97 us, and
// two threads that swap halves, so that each store of theirs fills one, 69.
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
            const int back = a.cu_r[lo + 1] - t, pos = len - back;
            if (pos >= 0 && back <= a.most && s >= 0 && s < a.n_slots && (a.ring == 0 || pos / P + a.ring / P > (len - 1) / P)) {
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
            w = reinterpret_cast<const int4*>(a.pages[which] + (bh * P + place_s[j]) * a.dim)[c];
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
    if (wide && a.single) return launch_pdl(kv8_write_kernel<T, true, 1>, grid, dim3(threads), 0, stream, a);
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
    int dtype, tokens, rows, n_kv, dim, block, n_blocks, n_slots, width, ring, max_q_len;
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
               c->n_slots, c->width, c->ring, c->max_q_len};
    const dim3 grid((c->tokens + READ_TOKENS - 1) / READ_TOKENS, 2);
    if (c->dtype == BROLM_F32) return launch_pdl(kv8_read_kernel<float>, grid, dim3(256), 0, c->stream, a);
    return launch_pdl(kv8_read_kernel<bf16>, grid, dim3(256), 0, c->stream, a);
}
