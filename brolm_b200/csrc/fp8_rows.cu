// Rows to 8 bits and back (the format is in fp8.cuh).
//
//   fp8_quantize   rows of float or bfloat16 numbers -> e4m3 numbers and a scale byte for every 128 of them
//   fp8_read       the values that they stand for
//   norm           a residual sum with the norms around it whose result is rows of 8 bits
#include "fp8_round.cuh"

namespace {

using namespace fp8;

constexpr int THREADS = 256, WARPS = THREADS / 32;

struct RowsArgs {
    const void* x; long ldx;        // elements
    uint8_t* values; long ldv;      // bytes
    uint8_t* scales;
    long rows;                      // of all groups
    int cols, quads;
    // rows come in groups of `group` rows; in the matrix a group takes `group_pad` rows (the same for a plain matrix)
    int group, group_pad;
    int early;                      // the next kernel may begin before this one's results are there
};

// The row of the matrix that row r of x is.
__device__ __forceinline__ long place_of(const RowsArgs& g, long r) { return g.group == g.group_pad ? r : r / g.group * g.group_pad + r % g.group; }

// A warp has four blocks of a row at a time.  8,192 x 4,608 bfloat16 numbers take 21.8 us, 5.2 TB/s where a copy of them runs at
// 6.0; two or four rows at a time (26.8, 28.6 us where one took 24.8) or the next one's numbers asked for ahead (24.8 to 26.1) gained
// nothing.
template <typename T, bool WIDE>
__global__ void __launch_bounds__(THREADS) quantize_kernel(RowsArgs g) {
    const int lane = threadIdx.x & 31;
    const long items = g.rows * g.quads;
    pdl_wait();
    // Products read a matrix that is not new before they wait for the kernel before them.  A kernel that writes a matrix lets
    // nothing begin before its blocks have ended, and products wait for it like any reader until one has been launched on its
    // stream (a fence here instead took 4 of 26 us); one that writes rows that a product waits for lets it begin at once.
    if (g.early) pdl_trigger();
    for (long item = (long)blockIdx.x * WARPS + (threadIdx.x >> 5); item < items; item += (long)gridDim.x * WARPS) {
        const long row = items <= 0xffffffffl ? (long)((uint32_t)item / (uint32_t)g.quads) : item / g.quads;    // (a division of 32 bits is much shorter)
        const int quad = (int)(item - row * g.quads), c = quad * 512 + lane * 16;
        const T* x = (const T*)g.x + row * g.ldx;
        Piece<T, WIDE> piece;
        piece.ask(x, c, g.cols, true);
        float v[16];
        piece.get(x, c, g.cols, v);
        uint32_t word;
        const uint4 q = round16(v, word);
        const long at = place_of(g, row);
        if (c < g.ldv) *reinterpret_cast<uint4*>(g.values + at * g.ldv + c) = q;     // ldv is a multiple of 16
        if (lane == 0) *reinterpret_cast<uint32_t*>(g.scales + scale_at(at, quad, g.quads)) = word;
    }
}

// For reading back the lanes' words lie side by side: eight bfloat16 numbers or four floats a word of sixteen bytes.  (With
// sixteen numbers a lane 8,192 x 4,608 floats took 44.7 us for 30.8.)
template <typename T>
struct Lay {
    static constexpr int WORDS = (int)sizeof(T);                 // words of sixteen bytes a lane
    static constexpr int EACH = 16 / (int)sizeof(T);             // numbers of a word
    static constexpr int LANES = BLOCK / EACH;                   // lanes of a block
    // the first column, from the piece's first on, of this lane's word i
    static __device__ __forceinline__ int column(int i, int lane) { return i * 32 * EACH + lane * EACH; }
};
__device__ __forceinline__ void store_wide(float* to, const float (&v)[4]) { *reinterpret_cast<float4*>(to) = make_float4(v[0], v[1], v[2], v[3]); }
__device__ __forceinline__ void store_wide(bf16* to, const float (&v)[8]) {
    uint4 p;
    __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&p);
#pragma unroll
    for (int e = 0; e < 4; ++e) h[e] = __floats2bfloat162_rn(v[2 * e], v[2 * e + 1]);
    *reinterpret_cast<uint4*>(to) = p;
}

template <typename T>
__global__ void __launch_bounds__(THREADS) read_kernel(RowsArgs g, T* __restrict__ y, long ldy, bool wide) {
    using L = Lay<T>;
    const int lane = threadIdx.x & 31, quad = blockIdx.x, c0 = quad * 512;
    pdl_wait();
    for (long row = (long)blockIdx.y * WARPS + (threadIdx.x >> 5); row < g.rows; row += (long)gridDim.y * WARPS) {
        const long at = place_of(g, row);
        const uint32_t scales = *reinterpret_cast<const uint32_t*>(g.scales + scale_at(at, quad, g.quads));
        uint32_t q[L::WORDS][L::EACH / 4];
#pragma unroll
        for (int i = 0; i < L::WORDS; ++i) {
            const int c = c0 + L::column(i, lane);
#pragma unroll
            for (int j = 0; j < L::EACH / 4; ++j) q[i][j] = c < g.ldv ? *reinterpret_cast<const uint32_t*>(g.values + at * g.ldv + c + 4 * j) : 0u;
        }
#pragma unroll
        for (int i = 0; i < L::WORDS; ++i) {
            const int c = c0 + L::column(i, lane);
            const float s = scale_value((scales >> (8 * (i * (32 / L::LANES) + lane / L::LANES))) & 255u);
            float v[L::EACH];
#pragma unroll
            for (int j = 0; j < L::EACH / 4; ++j) {
                uint32_t lo, hi;                     // e4m3 numbers are f16 numbers
                asm("{\n.reg .b16 a, b;\nmov.b32 {a, b}, %2;\ncvt.rn.f16x2.e4m3x2 %0, a;\ncvt.rn.f16x2.e4m3x2 %1, b;\n}" : "=r"(lo), "=r"(hi) : "r"(q[i][j]));
                const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&lo)), h = __half22float2(*reinterpret_cast<const __half2*>(&hi));
                v[4 * j] = f.x * s; v[4 * j + 1] = f.y * s; v[4 * j + 2] = h.x * s; v[4 * j + 3] = h.y * s;
            }
            if (wide && c + L::EACH <= g.cols) {
                store_wide(y + row * ldy + c, v);
            } else {
#pragma unroll
                for (int j = 0; j < L::EACH; ++j) if (c + j < g.cols) y[row * ldy + c + j] = from_float<T>(v[j]);
            }
        }
    }
    pdl_trigger();
}

struct NormArgs {
    float* h;
    const float* y;
    const void *w_post, *w_next;        // (w_post null: y is added as it is)
    float eps_post, off_post, eps_next, off_next;
    uint8_t* values; long ldv;
    uint8_t* scales;
    int quads, hidden;
};
__device__ __forceinline__ void four(const float* p, float (&v)[4]) {
    const float4 u = *reinterpret_cast<const float4*>(p);
    v[0] = u.x; v[1] = u.y; v[2] = u.z; v[3] = u.w;
}
__device__ __forceinline__ void four(const bf16* p, float (&v)[4]) {
    const uint2 u = *reinterpret_cast<const uint2*>(p);
    v[0] = __uint_as_float(u.x << 16); v[1] = __uint_as_float(u.x & 0xffff0000u);
    v[2] = __uint_as_float(u.y << 16); v[3] = __uint_as_float(u.y & 0xffff0000u);
}
// h += post(y);  values, scales = next(h), both norms being v * rsqrt(mean(v^2) + eps) * (offset + w).  A block has a row and
// thread t of it numbers 4 t + 1,024 c on: a warp's four numbers each are a block of 128, whose scale is the warp's largest.
// Statistics and sums are floats; what is rounded is the norm's float result, once.  Rows are few or many, the row stays in
// registers: memory bounds it, 13 bytes a number (8,192 x 4,608 86.7 us, 5.7 TB/s; the norm and the rounding apart 188; 8,192 x 2,304
// 52.5 and 56.9), and few rows take as long as a launch, against two of them.
template <typename W, int C>
__global__ void __launch_bounds__(256, C <= 3 ? 4 : 1) residual_rmsnorm_fp8_kernel(NormArgs g) {
    __shared__ float scratch[64];
    const long r = blockIdx.x;
    const W *w_post = (const W*)g.w_post, *w_next = (const W*)g.w_next;
    pdl_trigger();
    {
        const size_t line = (size_t)threadIdx.x * 128;      // the gains are weights: brought near while the kernel before this one ends
        if (line < (size_t)g.hidden * sizeof(W)) {
            if (w_post) prefetch_l1(reinterpret_cast<const char*>(w_post) + line);
            prefetch_l1(reinterpret_cast<const char*>(w_next) + line);
        }
    }
    pdl_wait();
    float* h = g.h + r * g.hidden;
    const float* y = g.y + r * g.hidden;
    float v[C][4], res[C][4];
#pragma unroll
    for (int c = 0; c < C; ++c) {
        const int i = (c * 256 + threadIdx.x) * 4;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[c][e] = res[c][e] = 0.0f;
        if (i < g.hidden) { four(h + i, res[c]); four(y + i, v[c]); }
    }
    if (w_post) {
        float ss = 0.0f;
#pragma unroll
        for (int c = 0; c < C; ++c) ss += v[c][0] * v[c][0] + v[c][1] * v[c][1] + v[c][2] * v[c][2] + v[c][3] * v[c][3];
        ss = block_sum_once(ss, scratch, 0);
        const float inv = rsqrtf(ss / (float)g.hidden + g.eps_post);
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const int i = (c * 256 + threadIdx.x) * 4;
            float gain[4] = {0.0f, 0.0f, 0.0f, 0.0f};
            if (i < g.hidden) four(w_post + i, gain);
#pragma unroll
            for (int e = 0; e < 4; ++e) v[c][e] = v[c][e] * inv * (g.off_post + gain[e]);
        }
    }
    float ss = 0.0f;
#pragma unroll
    for (int c = 0; c < C; ++c) {
        const int i = (c * 256 + threadIdx.x) * 4;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if (i < g.hidden) res[c][e] += v[c][e];
            ss += res[c][e] * res[c][e];
        }
        if (i < g.hidden) *reinterpret_cast<float4*>(h + i) = make_float4(res[c][0], res[c][1], res[c][2], res[c][3]);
    }
    ss = block_sum_once(ss, scratch, 1);
    const float inv = rsqrtf(ss / (float)g.hidden + g.eps_next);
#pragma unroll
    for (int c = 0; c < C; ++c) {
        const int i = (c * 256 + threadIdx.x) * 4, b = i >> 7;          // (the same block for the whole warp)
        float gain[4] = {0.0f, 0.0f, 0.0f, 0.0f}, o[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        if (i < g.hidden) {
            four(w_next + i, gain);
#pragma unroll
            for (int e = 0; e < 4; ++e) o[e] = res[c][e] * inv * (g.off_next + gain[e]);
        }
        uint32_t most = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) most = max(most, __float_as_uint(o[e]) & 0x7fffffffu);
        const uint32_t byte = scale_byte(__reduce_max_sync(0xffffffffu, most));
        if (i < g.ldv) *reinterpret_cast<uint32_t*>(g.values + r * g.ldv + i) = byte == 255u ? NAN4 : pack4(o[0], o[1], o[2], o[3], scale_inverse(byte));
        if ((threadIdx.x & 31) == 0 && b < 4 * g.quads) g.scales[scale_at(r, b >> 2, g.quads) + (b & 3)] = (uint8_t)byte;
    }
}

unsigned rows_grid(long long rows) {
    const long long blocks = (rows + WARPS - 1) / WARPS;
    return (unsigned)(blocks < 65535 ? blocks : 65535);
}
}  // namespace

// x [rows, cols] (float or bfloat16, ldx elements between rows) -> values (ldv bytes between rows, a multiple of 16, at least
// cols) and scales.  Rows come in groups of `group`, which lie `group_pad` rows (a multiple of 128 if not `group`) apart.
BROLM_API int brolm_fp8_quantize(const fp8::RowsCall* c) {
    if (c->rows <= 0 || c->cols <= 0) return BROLM_OK;
    if (c->ldv % 16 != 0 || c->ldv < c->cols || ((uintptr_t)c->values & 15) || ((uintptr_t)c->scales & 15)) return BROLM_ERR_ALIGNMENT;
    if (c->group <= 0 || c->group_pad < c->group) return BROLM_ERR_BAD_SIZE;
    RowsArgs g = {c->x, (long)c->ldx, (uint8_t*)c->values, (long)c->ldv, (uint8_t*)c->scales, (long)c->rows, c->cols, fp8::quads_of(c->cols),
                  c->group, c->group_pad, c->early};
    const long long blocks = (c->rows * g.quads + WARPS - 1) / WARPS, most = 16LL * tc::device_sms();
    const dim3 grid((unsigned)(blocks < most ? blocks : most)), block(THREADS);
    const bool base = ((uintptr_t)c->x & 15) == 0;
    if (c->dtype == BROLM_BF16) {
        if (base && c->ldx % 8 == 0) return launch_pdl(quantize_kernel<bf16, true>, grid, block, 0, c->stream, g);
        return launch_pdl(quantize_kernel<bf16, false>, grid, block, 0, c->stream, g);
    }
    if (c->dtype != BROLM_F32) return BROLM_ERR_BAD_DTYPE;
    if (base && c->ldx % 4 == 0) return launch_pdl(quantize_kernel<float, true>, grid, block, 0, c->stream, g);
    return launch_pdl(quantize_kernel<float, false>, grid, block, 0, c->stream, g);
}

// The same the other way: x the result.
BROLM_API int brolm_fp8_read(const fp8::RowsCall* c) {
    if (c->rows <= 0 || c->cols <= 0) return BROLM_OK;
    if (c->ldv % 16 != 0 || c->ldv < c->cols || ((uintptr_t)c->values & 15)) return BROLM_ERR_ALIGNMENT;
    if (c->group <= 0 || c->group_pad < c->group) return BROLM_ERR_BAD_SIZE;
    RowsArgs g = {nullptr, 0, (uint8_t*)c->values, (long)c->ldv, (uint8_t*)c->scales, (long)c->rows, c->cols, fp8::quads_of(c->cols), c->group, c->group_pad, 1};
    const dim3 grid(g.quads, rows_grid(c->rows)), block(THREADS);
    const bool base = ((uintptr_t)c->x & 15) == 0;
    if (c->dtype == BROLM_BF16)
        return launch_pdl(read_kernel<bf16>, grid, block, 0, c->stream, g, (bf16*)c->x, (long)c->ldx, base && c->ldx % 8 == 0);
    if (c->dtype != BROLM_F32) return BROLM_ERR_BAD_DTYPE;
    return launch_pdl(read_kernel<float>, grid, block, 0, c->stream, g, (float*)c->x, (long)c->ldx, base && c->ldx % 4 == 0);
}

// h [rows, hidden] float += post(y), y float alike; values and scales as brolm_fp8_quantize has them (group = rows) = next(h).  Both
// gains have one element type.  hidden is a multiple of 4, 8,192 at most; all pointers lie on borders of 16 bytes.
struct NormCall {
    void *h;
    const void *y, *w_post, *w_next;
    void *values, *scales;
    cudaStream_t stream;
    long long ldv;
    int rows, hidden, w_dtype;
    float eps_post, off_post, eps_next, off_next;
};
template <typename W>
static int norm_launch(const NormArgs& g, int rows, cudaStream_t stream) {
    const dim3 grid(rows), block(256);
    const int c = (g.hidden + 1023) / 1024;
    if (c <= 1) return launch_pdl(residual_rmsnorm_fp8_kernel<W, 1>, grid, block, 0, stream, g);
    if (c == 2) return launch_pdl(residual_rmsnorm_fp8_kernel<W, 2>, grid, block, 0, stream, g);
    if (c == 3) return launch_pdl(residual_rmsnorm_fp8_kernel<W, 3>, grid, block, 0, stream, g);
    if (c <= 5) return launch_pdl(residual_rmsnorm_fp8_kernel<W, 5>, grid, block, 0, stream, g);
    return launch_pdl(residual_rmsnorm_fp8_kernel<W, 8>, grid, block, 0, stream, g);
}
BROLM_API int brolm_residual_rmsnorm_fp8(const NormCall* c) {
    if (c->rows <= 0) return BROLM_OK;
    if (c->hidden <= 0 || c->hidden > 8192 || c->hidden % 4 || !c->w_next) return BROLM_ERR_BAD_SIZE;
    if ((((uintptr_t)c->h | (uintptr_t)c->y | (uintptr_t)c->w_post | (uintptr_t)c->w_next | (uintptr_t)c->values | (uintptr_t)c->scales) & 15) ||
        c->ldv % 16 || c->ldv < c->hidden || c->ldv >= c->hidden + 16)
        return BROLM_ERR_ALIGNMENT;
    const NormArgs g = {(float*)c->h, (const float*)c->y, c->w_post, c->w_next, c->eps_post, c->off_post, c->eps_next, c->off_next,
                        (uint8_t*)c->values, (long)c->ldv, (uint8_t*)c->scales, fp8::quads_of(c->hidden), c->hidden};
    if (c->w_dtype == BROLM_F32) return norm_launch<float>(g, c->rows, c->stream);
    if (c->w_dtype == BROLM_BF16) return norm_launch<bf16>(g, c->rows, c->stream);
    return BROLM_ERR_BAD_DTYPE;
}

// Two products one after the other, from one call of the host.
BROLM_API int brolm_fp8_two(const fp8::ProductCall* a, int (*first)(const fp8::ProductCall*), const fp8::ProductCall* b,
                            int (*second)(const fp8::ProductCall*)) {
    const int st = first(a);
    return st ? st : second(b);
}
