// Routed experts with matrices in 8-bit floating point: what happens to the rows around the products (the format is in fp8.cuh).
//
//   group          (token, choice) pairs sorted by expert, and the list of the experts' tiles of rows
//   gather         the tokens' rows in 8 bits, each at its pairs' places of that order
//   combine        a token's results, multiplied by their weights and added
//
// and the launches of a whole pass, from one call of the host: group and gather, the first product with its activation, which
// leaves 8 bits, the second product, combine.
#include "fp8_round.cuh"

namespace {

using namespace fp8;

constexpr int THREADS = 256, WARPS = THREADS / 32;

struct RowsArgs {
    const void* x; long ldx;        // elements
    uint8_t* values; long ldv;      // bytes
    uint8_t* scales;
    long rows;
    int cols, quads;
};

// Where this lane's pair lies among the warp's pairs of its expert, and how many those are; the first of them is the leader.
struct Match { int before, all; bool leader; };
__device__ __forceinline__ Match match(int e, int lane) {
    const uint32_t same = __match_any_sync(0xffffffffu, e);
    return {__popc(same & ((1u << lane) - 1)), __popc(same), (same & ((1u << lane) - 1)) == 0};
}

// Of a table of n counts in shared memory by a block of N threads: the sums of those before each, and of their tiles; the last
// place has all of them.  `carry`: 2 * 33 numbers.
template <int N>
__device__ __forceinline__ void scan(const int* counts, int n, int tile_rows, int* starts, int* tiles, int* carry) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int rows_before = 0, tiles_before = 0;
    for (int e0 = 0; e0 < n; e0 += N) {
        const int e = e0 + threadIdx.x, c = e < n ? counts[e] : 0, t = (c + tile_rows - 1) / tile_rows;
        int a = c, b = t;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int x = __shfl_up_sync(0xffffffffu, a, o), y = __shfl_up_sync(0xffffffffu, b, o);
            if (lane >= o) { a += x; b += y; }
        }
        if (lane == 31) { carry[warp] = a; carry[33 + warp] = b; }
        __syncthreads();
        if (warp == 0) {
            int x = lane < N / 32 ? carry[lane] : 0, y = lane < N / 32 ? carry[33 + lane] : 0;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int u = __shfl_up_sync(0xffffffffu, x, o), v = __shfl_up_sync(0xffffffffu, y, o);
                if (lane >= o) { x += u; y += v; }
            }
            carry[lane] = x; carry[33 + lane] = y;
        }
        __syncthreads();
        if (e < n) {
            starts[e] = rows_before + a - c + (warp ? carry[warp - 1] : 0);
            tiles[e] = tiles_before + b - t + (warp ? carry[33 + warp - 1] : 0);
        }
        rows_before += carry[31];
        tiles_before += carry[33 + 31];
        __syncthreads();
    }
    if (threadIdx.x == 0) {
        starts[n] = rows_before;
        tiles[n] = tiles_before;
    }
    __syncthreads();
}

// The list of the experts' tiles, written by a block of N threads.
template <int N>
__device__ __forceinline__ void write_list(const int* starts, const int* tiles, int E, int tile_rows, int32_t* offsets, int32_t* tile_group,
                                           int32_t* tile_row0, int max_tiles) {
    for (int e = threadIdx.x; e <= E; e += N) offsets[e] = starts[e];
    if (threadIdx.x == 0) offsets[E + 1] = tiles[E];
    for (int t = threadIdx.x; t < max_tiles; t += N) {
        int group = -1, row0 = 0;
        if (t < tiles[E]) {
            int lo = 0, hi = E;                            // the last expert whose first tile is not behind t (those without any lie before it)
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
}

struct Lists {
    int32_t *perm, *place, *scale_row, *offsets, *tile_group, *tile_row0;      // offsets[E + 1]: how many tiles there are
    int max_tiles, tile_rows, pad;
};

// The pairs sorted by expert, by the eight blocks of a cluster.  Counters in shared memory give every pair its number among those
// of its expert in its block; the blocks read one another's counters, and a scan gives the experts' first rows and tiles; then
// every pair's place is known.  Which of an expert's pairs come first within a block is left open: a pair's result hangs on its
// own row alone.  A choice that is no expert's is in no group.  perm: the pair of a row of the order; place: the row of a pair;
// scale_row: of row s of the order, where its scales lie (row r of tile t of the list: `pad` t + r, pad being the tile's rows
// rounded up to 128); -1 behind the last row.  What it takes is the scattered words that are written, two a pair: one block of
// 1,024 threads took 8.8 us for 8,192 pairs and 37 for 32,768.
constexpr int BLOCKS = 8;
__device__ __forceinline__ int peer_int(const int* p, int rank) {
    const uint32_t at = (uint32_t)__cvta_generic_to_shared(p);
    int v;
    asm volatile("{\n.reg .b32 r;\nmapa.shared::cluster.u32 r, %1, %2;\nld.shared::cluster.s32 %0, [r];\n}" : "=r"(v) : "r"(at), "r"(rank));
    return v;
}
__device__ __forceinline__ void cluster_sync_all() {
    asm volatile("barrier.cluster.arrive.aligned;\nbarrier.cluster.wait.aligned;" ::: "memory");
}
__global__ void __cluster_dims__(BLOCKS, 1, 1) __launch_bounds__(1024) group_kernel(const int32_t* __restrict__ ids, int P, int E, Lists g) {
    extern __shared__ int sh[];                        // this block's counters [E], all blocks' [E], first rows [E + 1], first tiles [E + 1]
    int *mine = sh, *counts = sh + E, *starts = counts + E, *tiles = starts + E + 1;
    __shared__ int carry[66];
    const int rank = blockIdx.x;
    for (int e = threadIdx.x; e < E; e += 1024) mine[e] = 0;
    __syncthreads();
    pdl_wait();
    pdl_trigger();                                      // (what follows waits for this kernel's end)
    auto id = [&](int p) {
        const int e = p < P ? ids[p] : -1;
        return e >= 0 && e < E ? e : -1;
    };
    constexpr int DEEP = 4, STEP = BLOCKS * 1024;
    const int first = rank * 1024 + threadIdx.x;
    for (int p0 = first; p0 < P; p0 += STEP * DEEP) {
        int e[DEEP];
#pragma unroll
        for (int j = 0; j < DEEP; ++j) e[j] = id(p0 + j * STEP);
#pragma unroll
        for (int j = 0; j < DEEP; ++j) if (e[j] >= 0) g.place[p0 + j * STEP] = atomicAdd(&mine[e[j]], 1);
    }
    __syncthreads();
    cluster_sync_all();
    int before[4];                                      // (E is 4,096 at most)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int e = i * 1024 + threadIdx.x;
        before[i] = 0;
        if (e < E) {
            int sum = 0;
#pragma unroll
            for (int k = 0; k < BLOCKS; ++k) {
                const int n = peer_int(&mine[e], k);
                if (k < rank) before[i] += n;
                sum += n;
            }
            counts[e] = sum;
        }
    }
    cluster_sync_all();                                 // nobody reads them any more: they become the first places of this block's
#pragma unroll
    for (int i = 0; i < 4; ++i) if (i * 1024 + threadIdx.x < E) mine[i * 1024 + threadIdx.x] = before[i];
    __syncthreads();
    scan<1024>(counts, E, g.tile_rows, starts, tiles, carry);
    if (rank == 0) write_list<1024>(starts, tiles, E, g.tile_rows, g.offsets, g.tile_group, g.tile_row0, g.max_tiles);
    for (int p0 = first; p0 < P; p0 += STEP * DEEP) {
        int e[DEEP], r[DEEP];
#pragma unroll
        for (int j = 0; j < DEEP; ++j) {
            e[j] = id(p0 + j * STEP);
            r[j] = e[j] >= 0 ? g.place[p0 + j * STEP] : 0;     // (this thread's own)
        }
#pragma unroll
        for (int j = 0; j < DEEP; ++j) {
            const int p = p0 + j * STEP;
            if (p >= P) break;
            if (e[j] < 0) { g.place[p] = -1; continue; }
            const int n = mine[e[j]] + r[j], s = starts[e[j]] + n;
            g.perm[s] = p;
            g.place[p] = s;
            g.scale_row[s] = (tiles[e[j]] + n / g.tile_rows) * g.pad + n % g.tile_rows;
        }
    }
    for (int s = starts[E] + first; s < P; s += STEP) {
        g.perm[s] = 0;
        g.scale_row[s] = -1;
    }
}

// One piece of a row of x in 8 bits to each of its pairs' places: place[p] is pair p's row of the order, -1 if it is in no group.
template <typename T, bool WIDE>
__device__ __forceinline__ void gather_row(const RowsArgs& g, long row, int quad, int c, int lane, const int32_t* place, const int32_t* scale_row, int top) {
    const T* x = (const T*)g.x + row * g.ldx;
    Piece<T, WIDE> piece;
    piece.ask(x, c, g.cols, true);
    float v[16];
    piece.get(x, c, g.cols, v);
    uint32_t word;
    const uint4 q = round16(v, word);
    for (int k = 0; k < top; ++k) {
        const long s = place[row * top + k];
        const int at = s < 0 ? -1 : scale_row[s];
        if (at < 0) continue;
        if (c < g.ldv) *reinterpret_cast<uint4*>(g.values + s * g.ldv + c) = q;
        if (lane == 0) *reinterpret_cast<uint32_t*>(g.scales + scale_at(at, quad, g.quads)) = word;
    }
}
template <typename T, bool WIDE>
__global__ void __launch_bounds__(THREADS) gather_kernel(RowsArgs g, const int32_t* __restrict__ place, const int32_t* __restrict__ scale_row, int top) {
    const int lane = threadIdx.x & 31, quad = blockIdx.x, c = quad * 512 + lane * 16;
    pdl_wait();
    pdl_trigger();                                      // (a product fetches its matrices meanwhile)
    for (long row = (long)blockIdx.y * WARPS + (threadIdx.x >> 5); row < g.rows; row += (long)gridDim.y * WARPS)
        gather_row<T, WIDE>(g, row, quad, c, lane, place, scale_row, top);
}

// Both at once for up to 256 pairs of up to 256 experts (a step of decoding): every block sorts them for itself, one pair a
// thread, in an order that is the same everywhere (that of the pairs), the first block writes it down, each rounds its part of
// the rows.  A launch less: 8 tokens, 4 of 32 experts 6.5 -> 4.0 us.
constexpr int FEW = 256;
template <typename T, bool WIDE>
__global__ void __launch_bounds__(FEW) group_gather_kernel(RowsArgs x, const int32_t* __restrict__ ids, int P, int E, int top, Lists g) {
    __shared__ int by_warp[FEW / 32][FEW], counts[FEW], starts[FEW + 1], tiles[FEW + 1], carry[66], place[FEW], scale_row[FEW];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    for (int w = 0; w < FEW / 32; ++w) by_warp[w][tid] = 0;
    place[tid] = scale_row[tid] = -1;
    __syncthreads();
    pdl_wait();
    pdl_trigger();
    int e = tid < P ? ids[tid] : -1;
    e = e >= 0 && e < E ? e : -1;
    const Match m = match(e, lane);
    if (e >= 0 && m.leader) by_warp[warp][e] = m.all;
    __syncthreads();
    int sum = 0;
    for (int w = 0; w < FEW / 32; ++w) {
        const int n = by_warp[w][tid];
        by_warp[w][tid] = sum;
        sum += n;
    }
    counts[tid] = sum;
    __syncthreads();
    scan<FEW>(counts, E, g.tile_rows, starts, tiles, carry);
    if (e >= 0) {
        const int r = by_warp[warp][e] + m.before, s = starts[e] + r;
        place[tid] = s;
        scale_row[s] = (tiles[e] + r / g.tile_rows) * g.pad + r % g.tile_rows;
        if (blockIdx.x == 0 && blockIdx.y == 0) g.perm[s] = tid;
    }
    __syncthreads();
    if (blockIdx.x == 0 && blockIdx.y == 0) {
        write_list<FEW>(starts, tiles, E, g.tile_rows, g.offsets, g.tile_group, g.tile_row0, g.max_tiles);
        if (tid < P) {
            g.place[tid] = place[tid];
            g.scale_row[tid] = scale_row[tid];
            if (tid >= starts[E]) g.perm[tid] = 0;
        }
    }
    const int quad = blockIdx.x, c = quad * 512 + lane * 16;
    for (long row = (long)blockIdx.y * WARPS + warp; row < x.rows; row += (long)gridDim.y * WARPS)
        gather_row<T, WIDE>(x, row, quad, c, lane, place, scale_row, top);
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
    pdl_trigger();
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
            return;
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) if (c + i < cols) out[(long)t * ldo + c + i] = from_float<T>(acc[i]);
    }
}

unsigned rows_grid(long long rows) {
    const long long blocks = (rows + WARPS - 1) / WARPS;
    return (unsigned)(blocks < 65535 ? blocks : 65535);
}

template <typename T>
int gather(const RowsArgs& g, const int32_t* place, const int32_t* scale_row, int top, cudaStream_t stream) {
    const dim3 grid(g.quads, rows_grid(g.rows)), block(THREADS);
    if (((uintptr_t)g.x & 15) == 0 && g.ldx % (16 / (int)sizeof(T)) == 0)
        return launch_pdl(gather_kernel<T, true>, grid, block, 0, stream, g, place, scale_row, top);
    return launch_pdl(gather_kernel<T, false>, grid, block, 0, stream, g, place, scale_row, top);
}
template <typename T>
int group_gather(const RowsArgs& x, const int32_t* ids, int P, int E, int top, const Lists& g, cudaStream_t stream) {
    if (P <= FEW && E <= FEW) {
        const dim3 grid(x.quads, rows_grid(x.rows)), block(FEW);
        if (((uintptr_t)x.x & 15) == 0 && x.ldx % (16 / (int)sizeof(T)) == 0)
            return launch_pdl(group_gather_kernel<T, true>, grid, block, 0, stream, x, ids, P, E, top, g);
        return launch_pdl(group_gather_kernel<T, false>, grid, block, 0, stream, x, ids, P, E, top, g);
    }
    static OncePerDevice done;
    int st = allow_shared_memory(group_kernel, (4 * 4096 + 2) * sizeof(int), done);
    if (!st) st = launch_pdl(group_kernel, dim3(BLOCKS), dim3(1024), (4 * (size_t)E + 2) * sizeof(int), stream, ids, P, E, g);
    return st ? st : gather<T>(x, g.place, g.scale_row, top, stream);
}

}  // namespace

// A pass.  x [tokens, K] (float or bfloat16, ldx elements between rows), ids [tokens, top]; up [experts] matrices of up_rows rows
// (gated: 2 inter; a multiple of 128 rows apart), down of N.  Tiles have `rows` rows: of 16 or 32 the experts'
// matrices are streamed, of 256 they go to the pairs of SMs; `product` is the launcher of the one or the other.  pairs [top, tokens, N] float; out (or null) the combined rows.
// scale (or null) [tokens, top] multiplies a pair's first sums, weights (or null, for ones) its result.  `work` holds
// `work_bytes`: the order and the list, then both products' rows in 8 bits.
struct ExpertsCall {
    const void *x, *ids, *scale, *weights, *up, *up_scales, *down, *down_scales;
    void *pairs, *out, *work;
    cudaStream_t stream;
    int (*product)(const fp8::ProductCall*);
    long long ldx, up_ld, down_ld, ldo, work_bytes;
    int dtype, tokens, top, experts, K, inter, N, up_rows, down_rows, gated, act, rows, piece, out_f32;
    float limit;
};
BROLM_API int brolm_fp8_experts(const ExpertsCall* c) {
    const int T = c->tokens, top = c->top, E = c->experts, rows = c->rows;
    if (T <= 0 || top <= 0 || E <= 0 || c->N <= 0) return BROLM_OK;
    if (E > 4096 || (long long)T * top > 0x7fffffff / 2) return BROLM_ERR_TOO_LARGE;
    if (c->dtype != BROLM_BF16 && c->dtype != BROLM_F32) return BROLM_ERR_BAD_DTYPE;
    if (rows != 16 && rows != 32 && rows != 256) return BROLM_ERR_BAD_SIZE;
    const int P = T * top, pad = (rows + 127) / 128 * 128, most = (P + rows - 1) / rows + (E < P ? E : P);
    uint8_t* at = (uint8_t*)c->work;
    auto take = [&](long long bytes) {
        uint8_t* p = at;
        at += (bytes + 511) / 512 * 512;
        return p;
    };
    Lists g;
    g.perm = (int32_t*)take(4LL * P); g.place = (int32_t*)take(4LL * P); g.scale_row = (int32_t*)take(4LL * P);
    g.offsets = (int32_t*)take(4LL * (E + 2)); g.tile_group = (int32_t*)take(4LL * most); g.tile_row0 = (int32_t*)take(4LL * most);
    g.max_tiles = most; g.tile_rows = rows; g.pad = pad;
    auto matrix = [&](int cols) {
        RowsArgs m = {};
        m.cols = cols; m.quads = quads_of(cols); m.ldv = (cols + 15) / 16 * 16; m.rows = P;
        m.values = take((long long)P * m.ldv);
        m.scales = take((long long)(pad / 128) * most * m.quads * SF_TILE);
        return m;
    };
    RowsArgs a = matrix(c->K), h = matrix(c->inter);
    if (((uintptr_t)c->work & 511) || at - (uint8_t*)c->work > c->work_bytes) return BROLM_ERR_BAD_SIZE;
    a.x = c->x; a.ldx = (long)c->ldx; a.rows = T;
    const int32_t* ids = (const int32_t*)c->ids;
    int st = c->dtype == BROLM_BF16 ? group_gather<bf16>(a, ids, P, E, top, g, c->stream) : group_gather<float>(a, ids, P, E, top, g, c->stream);
    if (st) return st;
    ProductCall p = {};
    p.x = a.values; p.x_scales = a.scales; p.ldx = a.ldv; p.w = c->up; p.w_scales = c->up_scales; p.ldw = c->up_ld; p.stream = c->stream;
    p.M = P; p.N = c->inter; p.K = c->K; p.epilogue = c->gated; p.act = c->act; p.limit = c->limit; p.cut = c->piece;
    p.y = h.values; p.y_scales = h.scales; p.ldy = h.ldv; p.out = 2;
    p.experts = E; p.tile_group = g.tile_group; p.tile_row0 = g.tile_row0; p.offsets = g.offsets; p.perm = g.perm; p.scale = c->scale;
    p.group_rows = c->up_rows; p.top = top; p.tokens = T; p.rows = rows; p.max_tiles = most;
    st = c->product(&p);
    if (st) return st;
    p.x = h.values; p.x_scales = h.scales; p.ldx = h.ldv; p.w = c->down; p.w_scales = c->down_scales; p.ldw = c->down_ld;
    p.y = c->pairs; p.y_scales = nullptr; p.ldy = c->N; p.out = 1; p.N = c->N; p.K = c->inter; p.epilogue = 0; p.act = 0; p.limit = 0.0f;
    // (the first product has waited before it lets this one begin, and so has the list been written)
    p.scale = nullptr; p.group_rows = c->down_rows; p.down = 1; p.listed = 1; p.piece = c->piece;
    st = c->product(&p);
    if (st || !c->out) return st;
    const dim3 grid(T, (c->N + 4 * THREADS - 1) / (4 * THREADS)), block(THREADS);
    if (grid.y > 65535) return BROLM_ERR_TOO_LARGE;
    const int wide = c->N % 4 == 0 && ((uintptr_t)c->pairs & 15) == 0;
    const int out_wide = c->N % 4 == 0 && c->ldo % 4 == 0 && ((uintptr_t)c->out & 15) == 0;
    const float *y = (const float*)c->pairs, *w = (const float*)c->weights;
    if (c->out_f32) return launch_pdl(combine_kernel<float>, grid, block, 0, c->stream, y, ids, w, top, E, T, c->N, (float*)c->out, (long)c->ldo, wide, out_wide);
    return launch_pdl(combine_kernel<bf16>, grid, block, 0, c->stream, y, ids, w, top, E, T, c->N, (bf16*)c->out, (long)c->ldo, wide, out_wide);
}
