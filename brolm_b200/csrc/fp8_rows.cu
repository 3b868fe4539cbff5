// Rows to 8 bits and back (the format is in fp8.cuh).
//
//   fp8_quantize   rows of float or bfloat16 numbers -> e4m3 numbers and a scale byte for every 128 of them
//   fp8_read       the values that they stand for
//   fp8_group      (token, choice) pairs sorted by expert, and the list of the experts' tiles of rows
//   fp8_gather     the pairs' rows in that order in 8 bits
//   fp8_combine    a token's results, multiplied by their weights and added
//
// The first two are one pass over the data: a warp takes four blocks of a row at a time (512 numbers, one word of scales), eight
// lanes a block and sixteen numbers a lane; the block's largest magnitude goes round its eight lanes in three shuffles.
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

template <typename T, bool WIDE>
__global__ void __launch_bounds__(THREADS) quantize_kernel(RowsArgs g) {
    const int lane = threadIdx.x & 31;
    const long items = g.rows * g.quads;
    pdl_wait();
    for (long item = (long)blockIdx.x * WARPS + (threadIdx.x >> 5); item < items; item += (long)gridDim.x * WARPS) {
        const long row = item / g.quads;
        const int quad = (int)(item - row * g.quads), c = quad * 512 + lane * 16;
        const long at = g.group == g.group_pad ? row : row / g.group * g.group_pad + row % g.group;
        float v[16];
        load16<WIDE>((const T*)g.x + row * g.ldx, c, g.cols, v);
        uint32_t word;
        const uint4 q = round16(v, word);
        if (c < g.ldv) *reinterpret_cast<uint4*>(g.values + at * g.ldv + c) = q;     // ldv is a multiple of 16
        if (lane == 0) *reinterpret_cast<uint32_t*>(g.scales + scale_at(at, quad, g.quads)) = word;
    }
    // The products read their matrix before they wait for the kernel before them, so a kernel that writes a matrix lets
    // nothing begin before it has ended; one that writes rows that a product waits for may.
    if (g.early) pdl_trigger();
}

template <typename T> __device__ __forceinline__ void store16(T* row, int c, int cols, const float (&v)[16], bool wide);
template <> __device__ __forceinline__ void store16<float>(float* row, int c, int cols, const float (&v)[16], bool wide) {
    if (wide && c + 16 <= cols) {
#pragma unroll
        for (int i = 0; i < 16; i += 4) *reinterpret_cast<float4*>(row + c + i) = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
        return;
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) if (c + i < cols) row[c + i] = v[i];
}
template <> __device__ __forceinline__ void store16<bf16>(bf16* row, int c, int cols, const float (&v)[16], bool wide) {
    if (wide && c + 16 <= cols) {
#pragma unroll
        for (int i = 0; i < 16; i += 8) {
            uint4 p;
            __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&p);
#pragma unroll
            for (int e = 0; e < 4; ++e) h[e] = __floats2bfloat162_rn(v[i + 2 * e], v[i + 2 * e + 1]);
            *reinterpret_cast<uint4*>(row + c + i) = p;
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) if (c + i < cols) row[c + i] = __float2bfloat16_rn(v[i]);
}

template <typename T>
__global__ void __launch_bounds__(THREADS) read_kernel(RowsArgs g, T* __restrict__ y, long ldy, bool wide) {
    const int lane = threadIdx.x & 31;
    const long items = g.rows * g.quads;
    pdl_wait();
    for (long item = (long)blockIdx.x * WARPS + (threadIdx.x >> 5); item < items; item += (long)gridDim.x * WARPS) {
        const long row = item / g.quads;
        const int quad = (int)(item - row * g.quads), c = quad * 512 + lane * 16;
        const long at = g.group == g.group_pad ? row : row / g.group * g.group_pad + row % g.group;
        if (c >= g.cols) continue;
        const uint4 q = *reinterpret_cast<const uint4*>(g.values + at * g.ldv + c);
        const float s = scale_value(g.scales[scale_at(at, quad, g.quads) + (lane >> 3)]);
        const uint32_t words[4] = {q.x, q.y, q.z, q.w};
        float v[16];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            uint32_t lo, hi;                     // e4m3 numbers are f16 numbers
            asm("{\n.reg .b16 a, b;\nmov.b32 {a, b}, %2;\ncvt.rn.f16x2.e4m3x2 %0, a;\ncvt.rn.f16x2.e4m3x2 %1, b;\n}" : "=r"(lo), "=r"(hi) : "r"(words[i]));
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&lo)), h = __half22float2(*reinterpret_cast<const __half2*>(&hi));
            v[4 * i] = f.x * s; v[4 * i + 1] = f.y * s; v[4 * i + 2] = h.x * s; v[4 * i + 3] = h.y * s;
        }
        store16<T>(y + row * ldy, c, g.cols, v, wide);
    }
    pdl_trigger();
}

// The pairs sorted by expert, by one block: counts of the experts, their first rows by a scan, every pair's place by a counter in
// shared memory (which of an expert's pairs comes first is left open: a pair's result hangs on its own row alone).  A choice
// that is no expert's is in no group.  scale_row: of row s of the order, where its scales lie (row r of tile t of the list:
// `pad` t + r, pad being the tile's rows rounded up to 128); -1 behind the last row.
__global__ void __launch_bounds__(1024) group_kernel(const int32_t* __restrict__ ids, int P, int E, int tile_rows, int pad,
                                                     int32_t* __restrict__ perm, int32_t* __restrict__ scale_row,
                                                     int32_t* __restrict__ offsets, int32_t* __restrict__ tile_group,
                                                     int32_t* __restrict__ tile_row0, int max_tiles) {
    extern __shared__ int sh[];                        // counts (then places) [E], first rows [E + 1], first tiles [E + 1]
    int *counts = sh, *starts = sh + E, *tiles = starts + E + 1;
    __shared__ int carry[2][33];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    for (int e = threadIdx.x; e < E; e += 1024) counts[e] = 0;
    __syncthreads();
    pdl_wait();
    for (int p = threadIdx.x; p < P; p += 1024) {
        const int e = ids[p];
        if (e >= 0 && e < E) atomicAdd(&counts[e], 1);
    }
    __syncthreads();
    int rows_before = 0, tiles_before = 0;
    for (int e0 = 0; e0 < E; e0 += 1024) {
        const int e = e0 + threadIdx.x, n = e < E ? counts[e] : 0, t = (n + tile_rows - 1) / tile_rows;
        int a = n, b = t;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int x = __shfl_up_sync(0xffffffffu, a, o), y = __shfl_up_sync(0xffffffffu, b, o);
            if (lane >= o) { a += x; b += y; }
        }
        if (lane == 31) { carry[0][warp] = a; carry[1][warp] = b; }
        __syncthreads();
        if (warp == 0) {
            int x = carry[0][lane], y = carry[1][lane];
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int u = __shfl_up_sync(0xffffffffu, x, o), v = __shfl_up_sync(0xffffffffu, y, o);
                if (lane >= o) { x += u; y += v; }
            }
            carry[0][lane] = x; carry[1][lane] = y;
        }
        __syncthreads();
        if (e < E) {
            starts[e] = rows_before + a - n + (warp ? carry[0][warp - 1] : 0);
            tiles[e] = tiles_before + b - t + (warp ? carry[1][warp - 1] : 0);
            offsets[e] = starts[e];
        }
        rows_before += carry[0][31];
        tiles_before += carry[1][31];
        __syncthreads();
    }
    if (threadIdx.x == 0) {
        starts[E] = offsets[E] = rows_before;
        tiles[E] = tiles_before;
    }
    __syncthreads();
    for (int t = threadIdx.x; t < max_tiles; t += 1024) {
        int group = -1, row0 = 0;
        if (t < tiles_before) {
            int lo = 0, hi = E;                        // the last expert whose first tile is not behind t and that has one
            while (hi - lo > 1) {
                const int mid = (lo + hi) / 2;
                if (tiles[mid] <= t) lo = mid; else hi = mid;
            }
            group = lo;
            row0 = starts[lo] + (t - tiles[lo]) * tile_rows;
        }
        tile_group[t] = group;
        tile_row0[t] = row0;
    }
    for (int e = threadIdx.x; e < E; e += 1024) counts[e] = 0;
    __syncthreads();
    for (int p = threadIdx.x; p < P; p += 1024) {
        const int e = ids[p];
        if (e >= 0 && e < E) {
            const int r = atomicAdd(&counts[e], 1), s = starts[e] + r;
            perm[s] = p;
            scale_row[s] = (tiles[e] + r / tile_rows) * pad + r % tile_rows;
        }
    }
    for (int s = rows_before + threadIdx.x; s < P; s += 1024) {
        perm[s] = 0;
        scale_row[s] = -1;
    }
    pdl_trigger();
}

// Row s of the order: the row perm[s] / top of x (top 0: row s itself) in 8 bits.
template <typename T, bool WIDE>
__global__ void __launch_bounds__(THREADS) gather_kernel(RowsArgs g, const int32_t* __restrict__ perm, const int32_t* __restrict__ scale_row, int top) {
    const int lane = threadIdx.x & 31;
    const long items = g.rows * g.quads;
    pdl_wait();
    for (long item = (long)blockIdx.x * WARPS + (threadIdx.x >> 5); item < items; item += (long)gridDim.x * WARPS) {
        const long s = item / g.quads;
        const int quad = (int)(item - s * g.quads), c = quad * 512 + lane * 16;
        const int place = scale_row[s];
        if (place < 0) continue;
        const long row = top ? perm[s] / top : s;
        float v[16];
        load16<WIDE>((const T*)g.x + row * g.ldx, c, g.cols, v);
        uint32_t word;
        const uint4 q = round16(v, word);
        if (c < g.ldv) *reinterpret_cast<uint4*>(g.values + s * g.ldv + c) = q;
        if (lane == 0) *reinterpret_cast<uint32_t*>(g.scales + scale_at(place, quad, g.quads)) = word;
    }
    pdl_trigger();
}

__device__ __forceinline__ void store4(float* p, const float (&v)[4]) { *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]); }
__device__ __forceinline__ void store4(bf16* p, const float (&v)[4]) {
    uint2 u;
    __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&u);
    h[0] = __floats2bfloat162_rn(v[0], v[1]);
    h[1] = __floats2bfloat162_rn(v[2], v[3]);
    *reinterpret_cast<uint2*>(p) = u;
}

// out[t] = sum over t's choices, in their order, of weight * y[choice][t]; those that are no expert's give nothing.
template <typename T>
__global__ void __launch_bounds__(THREADS) combine_kernel(const float* __restrict__ y, const int32_t* __restrict__ ids, const float* __restrict__ weights,
                                                          int top, int experts, int tokens, int cols, T* __restrict__ out, long ldo, int wide, int out_wide) {
    pdl_wait();
    const int t = blockIdx.x, c = (blockIdx.y * THREADS + threadIdx.x) * 4;
    if (c < cols) {
        float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        for (int k0 = 0; k0 < top; k0 += 4) {                  // four choices' numbers on their way at a time
            float4 v[4];
            float w[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int k = k0 + j, e = k < top ? ids[(long)t * top + k] : -1;
                v[j] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                w[j] = 0.0f;
                if (e < 0 || e >= experts) continue;
                w[j] = weights ? weights[(long)t * top + k] : 1.0f;
                const float* row = y + ((long)k * tokens + t) * cols + c;
                if (wide) {
                    v[j] = *reinterpret_cast<const float4*>(row);
                } else {
                    v[j].x = row[0];
                    if (c + 1 < cols) v[j].y = row[1];
                    if (c + 2 < cols) v[j].z = row[2];
                    if (c + 3 < cols) v[j].w = row[3];
                }
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                acc[0] = fmaf(w[j], v[j].x, acc[0]); acc[1] = fmaf(w[j], v[j].y, acc[1]);
                acc[2] = fmaf(w[j], v[j].z, acc[2]); acc[3] = fmaf(w[j], v[j].w, acc[3]);
            }
        }
        if (out_wide) {
            store4(out + (long)t * ldo + c, acc);
            pdl_trigger();
            return;
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) if (c + i < cols) out[(long)t * ldo + c + i] = from_float<T>(acc[i]);
    }
    pdl_trigger();
}

int grid_for(long items) {
    const long blocks = (items + WARPS - 1) / WARPS, most = 16L * tc::device_sms();
    return (int)(blocks < most ? blocks : most);
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
    const dim3 grid(grid_for(c->rows * g.quads)), block(THREADS);
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
    const dim3 grid(grid_for(c->rows * g.quads)), block(THREADS);
    const bool base = ((uintptr_t)c->x & 15) == 0;
    if (c->dtype == BROLM_BF16)
        return launch_pdl(read_kernel<bf16>, grid, block, 0, c->stream, g, (bf16*)c->x, (long)c->ldx, base && c->ldx % 8 == 0);
    if (c->dtype != BROLM_F32) return BROLM_ERR_BAD_DTYPE;
    return launch_pdl(read_kernel<float>, grid, block, 0, c->stream, g, (float*)c->x, (long)c->ldx, base && c->ldx % 4 == 0);
}

// ids [pairs] -> perm, scale_row [pairs], offsets [experts + 1], the list [max_tiles] (expert -1 behind its end).
struct GroupCall {
    const void* ids;
    void *perm, *scale_row, *offsets, *tile_group, *tile_row0;
    cudaStream_t stream;
    int pairs, experts, tile_rows, max_tiles;
};
BROLM_API int brolm_fp8_group(const GroupCall* c) {
    if (c->pairs <= 0) return BROLM_OK;
    const int E = c->experts;
    if (E <= 0 || E > 4096) return BROLM_ERR_TOO_LARGE;
    if (c->tile_rows < 16 || c->max_tiles < (c->pairs + c->tile_rows - 1) / c->tile_rows + (E < c->pairs ? E : c->pairs)) return BROLM_ERR_BAD_SIZE;
    static OncePerDevice done;
    const int st = allow_shared_memory(group_kernel, (3 * 4096 + 2) * sizeof(int), done);
    if (st) return st;
    return launch_pdl(group_kernel, dim3(1), dim3(1024), (3 * (size_t)E + 2) * sizeof(int), c->stream, (const int32_t*)c->ids, c->pairs, E, c->tile_rows,
                      (c->tile_rows + 127) / 128 * 128, (int32_t*)c->perm, (int32_t*)c->scale_row, (int32_t*)c->offsets, (int32_t*)c->tile_group,
                      (int32_t*)c->tile_row0, c->max_tiles);
}

// The rows of the order in 8 bits: row perm[s] / top of x, or with top 0 row s of it.
struct GatherCall {
    const void *x, *perm, *scale_row;
    void *values, *scales;
    cudaStream_t stream;
    long long ldx, ldv;
    int dtype, top, pairs, cols;
};
BROLM_API int brolm_fp8_gather(const GatherCall* c) {
    if (c->pairs <= 0 || c->cols <= 0) return BROLM_OK;
    if (c->ldv % 16 != 0 || c->ldv < c->cols || ((uintptr_t)c->values & 15) || ((uintptr_t)c->scales & 15)) return BROLM_ERR_ALIGNMENT;
    RowsArgs g = {c->x, (long)c->ldx, (uint8_t*)c->values, (long)c->ldv, (uint8_t*)c->scales, c->pairs, c->cols, fp8::quads_of(c->cols), 1, 1, 1};
    const dim3 grid(grid_for((long)c->pairs * g.quads)), block(THREADS);
    const int32_t *pm = (const int32_t*)c->perm, *sr = (const int32_t*)c->scale_row;
    const bool base = ((uintptr_t)c->x & 15) == 0;
    if (c->dtype == BROLM_BF16) {
        if (base && c->ldx % 8 == 0) return launch_pdl(gather_kernel<bf16, true>, grid, block, 0, c->stream, g, pm, sr, c->top);
        return launch_pdl(gather_kernel<bf16, false>, grid, block, 0, c->stream, g, pm, sr, c->top);
    }
    if (c->dtype != BROLM_F32) return BROLM_ERR_BAD_DTYPE;
    if (base && c->ldx % 4 == 0) return launch_pdl(gather_kernel<float, true>, grid, block, 0, c->stream, g, pm, sr, c->top);
    return launch_pdl(gather_kernel<float, false>, grid, block, 0, c->stream, g, pm, sr, c->top);
}

// y float [top, tokens, cols]; weights [tokens, top], or null for ones; out float or bfloat16.
struct CombineCall {
    const void *y, *ids, *weights;
    void* out;
    cudaStream_t stream;
    long long ldo;
    int top, experts, tokens, cols, out_f32;
};
BROLM_API int brolm_fp8_combine(const CombineCall* c) {
    if (c->tokens <= 0 || c->cols <= 0) return BROLM_OK;
    const dim3 grid(c->tokens, (c->cols + 4 * THREADS - 1) / (4 * THREADS)), block(THREADS);
    if (grid.y > 65535) return BROLM_ERR_TOO_LARGE;
    const int wide = c->cols % 4 == 0 && ((uintptr_t)c->y & 15) == 0;
    const int out_wide = c->cols % 4 == 0 && c->ldo % 4 == 0 && ((uintptr_t)c->out & 15) == 0;
    const float *y = (const float*)c->y, *w = (const float*)c->weights;
    const int32_t* ids = (const int32_t*)c->ids;
    if (c->out_f32)
        return launch_pdl(combine_kernel<float>, grid, block, 0, c->stream, y, ids, w, c->top, c->experts, c->tokens, c->cols, (float*)c->out, (long)c->ldo, wide, out_wide);
    return launch_pdl(combine_kernel<bf16>, grid, block, 0, c->stream, y, ids, w, c->top, c->experts, c->tokens, c->cols, (bf16*)c->out, (long)c->ldo, wide, out_wide);
}
