// Products with a matrix in 8-bit floating point for few rows (the format is in fp8.cuh), on tcgen05:
//     Y[m,n] = sum over blocks b of 2^(sx[m,b] + sw[n,b]) * (sum over the block's k of X[m,k] W[n,k]),  float sums.
//
// With few rows the product is a stream of W from memory.  The roles of the operands are swapped: 128 rows of W are the M side
// of tcgen05.mma.kind::mxf8f6f4, the rows of X (16, 32, 64 or 128 of them) the N side, and the tensor core multiplies by the
// scales itself.  A stage of the ring is one block of K: 16 KB of W, the rows of X beside it and, for the first block of every
// four, the 512 bytes of scales of each side, which tcgen05.cp carries into tensor memory ahead of the products that need
// them (copies and products of one thread are executed in order).
//
//   warp 0    one thread: TMA loads, and untiled copies of the scales' tiles
//   warp 1    one thread: copies of scales and products into one of two accumulators, commits
//   warps 2-5 an accumulator's lane is a row of W, its column a row of X: epilogue, Y[row of X][row of W]
//
// Dense: X has up to 128 rows.  Where W has fewer tiles of 128 rows than the device has SMs, K is cut into slices that are the
// blocks of a cluster; their float sums are added in the order of the slices through the cluster's shared memory.
// Experts: a list made on the device names for every tile of rows of X the expert whose matrix it meets, its first row and
// so its last one; an item of work is one such tile and 128 rows of its expert's matrix.
//
// Epilogues: store (float or bfloat16; with the square of relu), or a gated activation of neighbouring rows of W, row 2 j being
// the gate of output j and row 2 j + 1 its partner: the two lie in neighbouring lanes.
//
// Every mbarrier wait is bounded (tcgen05.cuh).
#include "fp8.cuh"

namespace {

using namespace tc;
using namespace fp8;

constexpr int BR = 128, BK = 128;
constexpr int THREADS = 192;
constexpr int W_BYTES = BR * BK;
constexpr int MAX_STAGES = 12;

enum : int { EPI_STORE = 0, EPI_GATED = 1 };
enum : int { ACT_NONE = 0, ACT_RELU2 = 1 };

__device__ int g_fp8_stream_error;

struct StreamArgs {
    void* y;
    long ldy;
    int M, N;                // rows of X (dense); output columns
    int out_f32, act;
    float limit;
    int nkb, quads;          // blocks of K, words of scales
    int row_tiles, items, stages;
    int per;                 // blocks of K of a slice (dense; the cluster's rank is the slice)
    const uint8_t* w_scales;
    const uint8_t* x_scales;
    // experts
    const int32_t* tile_group;      // null: dense
    const int32_t* tile_row0;
    const int32_t* offsets;
    const int32_t* perm;
    const float* scale;      // of a pair, before the activation
    int down, top, tokens, group_rows;
};

__device__ __forceinline__ bool wait_on(uint32_t bar, uint32_t parity, volatile int* give_up, int code) {
    return mbar_wait(bar, parity, give_up, &g_fp8_stream_error, code);
}
__device__ __forceinline__ bool drain_on(uint32_t bar, uint32_t parity, volatile int* give_up, int code) {
    return mbar_wait(bar, parity, give_up, &g_fp8_stream_error, code, true);
}
__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ uint32_t cluster_size() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_sync_all() {
    asm volatile("barrier.cluster.arrive.aligned;\nbarrier.cluster.wait.aligned;" ::: "memory");
}
__device__ __forceinline__ float peer_float(uint32_t addr, uint32_t rank) {
    float v;
    asm volatile("{\n.reg .b32 r;\nmapa.shared::cluster.u32 r, %1, %2;\nld.shared::cluster.f32 %0, [r];\n}" : "=f"(v) : "r"(addr), "r"(rank) : "memory");
    return v;
}
__device__ __forceinline__ float act_of(float v, int act) {
    if (act == ACT_RELU2) {
        v = fmaxf(v, 0.0f);
        return v * v;
    }
    return v;
}
__device__ __forceinline__ void put(const StreamArgs& g, long at, float v) {
    if (g.out_f32) reinterpret_cast<float*>(g.y)[at] = v;
    else reinterpret_cast<bf16*>(g.y)[at] = __float2bfloat16_rn(v);
}

template <int BT>
struct Shape {
    static constexpr int X_BYTES = BT * BK;
    static constexpr int STAGE_BYTES = W_BYTES + X_BYTES;              // multiples of 1024
    static constexpr int COLS = 2 * BT + 16;                            // two accumulators, two pairs of scales
    static constexpr int TMEM_COLS = COLS <= 64 ? 64 : COLS <= 128 ? 128 : COLS <= 256 ? 256 : 512;
    static constexpr int SCALES = 2 * SF_TILE;                          // of a stage
    static size_t smem(int stages, bool split) {
        return (size_t)stages * (STAGE_BYTES + SCALES) + (2 * MAX_STAGES + 4) * 8 + 16 + (split ? (size_t)BT * BR * 4 : 0);
    }
};

template <int BT, int EPI, bool EXPERTS>
__global__ void __launch_bounds__(THREADS) fp8_stream_kernel(const __grid_constant__ CUtensorMap map_w,
                                                             const __grid_constant__ CUtensorMap map_x, StreamArgs g) {
    using S = Shape<BT>;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t* base = smem_raw;
    const int stages = g.stages;
    uint8_t* scale_slots = base + stages * S::STAGE_BYTES;
    uint64_t* bars = reinterpret_cast<uint64_t*>(scale_slots + stages * S::SCALES);
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 2 * MAX_STAGES + 4);
    volatile int* give_up = reinterpret_cast<volatile int*>(tmem_slot + 1);
    float* sums = reinterpret_cast<float*>(tmem_slot + 4);             // slices: this one's [rows of X][128]
    const uint32_t stage0 = smem_u32(base), scale0 = smem_u32(scale_slots);
    const uint32_t full0 = smem_u32(bars), empty0 = full0 + 8 * MAX_STAGES, acc_full0 = empty0 + 8 * MAX_STAGES,
                   acc_empty0 = acc_full0 + 16;
    const bool aligned = (stage0 & 1023u) == 0;
    const int slices = EXPERTS ? 1 : (int)cluster_size(), slice = EXPERTS ? 0 : (int)cluster_rank();
    const int first = EXPERTS ? blockIdx.x : blockIdx.x / slices, step = EXPERTS ? gridDim.x : gridDim.x / slices;
    const int lo = slice * g.per, hi = min(g.nkb, lo + g.per);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int s = 0; s < stages; ++s) {
            mbar_init(full0 + 8 * s, 1);
            mbar_init(empty0 + 8 * s, 1);
        }
        for (int s = 0; s < 2; ++s) {
            mbar_init(acc_full0 + 8 * s, 1);
            mbar_init(acc_empty0 + 8 * s, 4);
        }
        give_up[0] = aligned ? 0 : 1;
        give_up[1] = 0;
        give_up[2] = tc::g_stall_code;
        if (!aligned) atomicCAS(&g_fp8_stream_error, 0, 13);
        mbar_init_fence();
    }
    if (warp == 1) tmem_alloc(smem_u32(tmem_slot), S::TMEM_COLS);
    fence_before_sync();
    __syncthreads();
    fence_after_sync();
    const uint32_t tmem = *tmem_slot;

    // the tile of rows of X and the tile of rows of W of an item; false behind the experts' last tile
    auto find = [&](int item, int& rt, int& group, int& row0, int& tile) {
        if (!EXPERTS) {
            rt = item; group = 0; row0 = 0; tile = 0;
            return true;
        }
        tile = item / g.row_tiles;
        rt = item - tile * g.row_tiles;
        group = g.tile_group[tile];
        if (group < 0) return false;
        row0 = g.tile_row0[tile];
        return true;
    };

    if (warp == 0) {
        if (lane == 0 && !*give_up) {
            auto bytes_of = [&](int kb) { return (uint32_t)(S::STAGE_BYTES + ((kb & 3) == 0 || kb == lo ? S::SCALES : 0)); };
            auto load_w = [&](int s, int rt, int group, int kb) {
                const uint32_t full = full0 + 8 * s;
                const int row = group * g.group_rows + rt * BR;
                mbar_expect_tx(full, bytes_of(kb));
                tma_load_2d(stage0 + s * S::STAGE_BYTES, &map_w, kb * BK, row, full);
                if ((kb & 3) == 0 || kb == lo)
                    bulk_load(scale0 + s * S::SCALES, g.w_scales + ((size_t)(row >> 7) * g.quads + (kb >> 2)) * SF_TILE, SF_TILE, full);
            };
            auto load_x = [&](int s, int row0, int tile, int kb) {
                const uint32_t full = full0 + 8 * s;
                tma_load_2d(stage0 + s * S::STAGE_BYTES + W_BYTES, &map_x, kb * BK, row0, full);
                if ((kb & 3) == 0 || kb == lo)
                    bulk_load(scale0 + s * S::SCALES + SF_TILE, g.x_scales + ((size_t)tile * g.quads + (kb >> 2)) * SF_TILE, SF_TILE, full);
            };
            int item = first, kb = lo, it = 0, rt = 0, group = 0, row0 = 0, tile = 0;
            bool more;
            if (EXPERTS) pdl_wait();                     // the list of tiles is an earlier kernel's
            more = item < g.items && lo < hi && find(item, rt, group, row0, tile);
            if (!EXPERTS) {
                // the ring fills with weights before the kernel before this one has finished
                const int rt0 = rt;
                int n = 0;
                for (; n < stages && lo + n < hi && more; ++n) load_w(n, rt0, 0, lo + n);
                pdl_wait();
                for (int i = 0; i < n; ++i) load_x(i, 0, 0, lo + i);
                it = n;
                kb = lo + n;
                if (more && kb >= hi) {
                    item += step;
                    kb = lo;
                    more = item < g.items && find(item, rt, group, row0, tile);
                }
            }
            int s = it % stages, phase = (it / stages) & 1;
            while (more) {
                if (!wait_on(empty0 + 8 * s, phase ^ 1, give_up, 1)) break;
                load_w(s, rt, group, kb);
                load_x(s, row0, tile, kb);
                ++it;
                if (++s == stages) { s = 0; phase ^= 1; }
                if (++kb >= hi) {
                    item += step;
                    kb = lo;
                    more = item < g.items && find(item, rt, group, row0, tile);
                }
            }
            pdl_trigger();                               // the stream is asked for: the next kernel may move in
            if (*give_up) {
                for (int j = max(0, it - stages); j < it; ++j) drain_on(full0 + 8 * (j % stages), (j / stages) & 1, give_up, 4);
            }
        }
    } else if (warp == 1) {
        if (lane == 0 && !*give_up) {
            const uint32_t id = idesc_mx(BR, BT);
            if (EXPERTS) pdl_wait();
            int s = 0, phase = 0, local = 0, set = 0;
            bool ok = true;
            int rt, group, row0, tile;
            for (int item = first; item < g.items && lo < hi && ok; item += step, ++local) {
                if (!find(item, rt, group, row0, tile)) break;
                const int as = local & 1;
                ok = wait_on(acc_empty0 + 8 * as, ((local >> 1) & 1) ^ 1, give_up, 5);
                if (!ok) break;
                fence_after_sync();
                const uint32_t acc = tmem + as * BT;
                uint32_t sfw = 0, sfx = 0;
                for (int kb = lo; kb < hi; ++kb) {
                    ok = wait_on(full0 + 8 * s, phase, give_up, 2);
                    if (!ok) break;
                    fence_after_sync();
                    if ((kb & 3) == 0 || kb == lo) {
                        sfw = tmem + 2 * BT + 8 * set;
                        sfx = sfw + 4;
                        set ^= 1;
                        scales_to_tmem(sfw, desc_scales(scale0 + s * S::SCALES));
                        scales_to_tmem(sfx, desc_scales(scale0 + s * S::SCALES + SF_TILE));
                    }
                    const uint32_t idk = with_block(id, kb & 3, kb & 3);
                    const uint64_t a = desc_kmajor(stage0 + s * S::STAGE_BYTES), b = desc_kmajor(stage0 + s * S::STAGE_BYTES + W_BYTES);
#pragma unroll
                    for (int k = 0; k < BK / 32; ++k) umma_mx(acc, a + 2 * k, b + 2 * k, idk, sfw, sfx, (kb > lo) | (k > 0));
                    umma_commit(empty0 + 8 * s);
                    if (++s == stages) { s = 0; phase ^= 1; }
                }
                if (ok) umma_commit(acc_full0 + 8 * as);
            }
        }
    } else {
        const int quarter = warp & 3;
        const int lrow = quarter * 32 + lane;                   // row of the tile of W = lane of tensor memory
        if (EXPERTS) pdl_wait();
        int local = 0, rt, group, row0, tile;
        for (int item = first; item < g.items && lo < hi; item += step, ++local) {
            if (!find(item, rt, group, row0, tile)) break;
            const int as = local & 1;
            const bool ready = !*give_up && wait_on(acc_full0 + 8 * as, (local >> 1) & 1, give_up, 3);
            if (!__all_sync(0xffffffffu, ready)) break;
            fence_after_sync();
            const uint32_t acc = tmem + as * BT + ((uint32_t)(quarter * 32) << 16);
            const int rows = EXPERTS ? min(BT, g.offsets[group + 1] - row0) : g.M;
            const int wide = (rows + 15) & ~15;
            for (int c = 0; c < wide; c += 16) {
                uint32_t v[16];
                tmem_ld16(acc + c, v);
                tmem_wait_ld();
                if (c + 16 >= wide) {                           // all of this accumulator that is wanted is in registers
                    fence_before_sync();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(acc_empty0 + 8 * as);
                }
                float o[16];
#pragma unroll
                for (int i = 0; i < 16; ++i) o[i] = __uint_as_float(v[i]);
                if (slices > 1) {
#pragma unroll
                    for (int i = 0; i < 16; ++i) sums[(c + i) * BR + lrow] = o[i];
                    continue;
                }
                if (EXPERTS && g.scale) {
#pragma unroll
                    for (int i = 0; i < 16; ++i) if (c + i < rows) o[i] *= g.scale[g.perm[row0 + c + i]];
                }
                int first_row = 0, row_step = 1, col = rt * BR + lrow;
                if (EPI == EPI_GATED) {
                    // lane 2 j has output j's gate and lane 2 j + 1 its partner: of every two rows each makes one
                    const bool odd = lane & 1;
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const float got = __shfl_xor_sync(0xffffffffu, odd ? o[2 * i] : o[2 * i + 1], 1);
                        o[i] = fast_gate_pair(odd ? got : o[2 * i], odd ? o[2 * i + 1] : got, g.act, g.limit);
                    }
                    first_row = odd; row_step = 2; col >>= 1;
                } else {
#pragma unroll
                    for (int i = 0; i < 16; ++i) o[i] = act_of(o[i], g.act);
                }
                if (col < g.N) {
#pragma unroll
                    for (int i = 0; i < (EPI == EPI_GATED ? 8 : 16); ++i) {
                        const int r = c + first_row + i * row_step;
                        if (r < rows) {
                            long at = EXPERTS ? row0 + r : r;
                            if (EXPERTS && g.down) {
                                const int p = g.perm[row0 + r], tok = p / g.top;
                                at = (long)(p - tok * g.top) * g.tokens + tok;
                            }
                            put(g, at * g.ldy + col, o[i]);
                        }
                    }
                }
            }
        }
    }
    pdl_trigger();
    fence_before_sync();
    if (!EXPERTS && slices > 1) {
        // one tile a cluster: the slices' sums are added in their order, every block takes some of the rows
        __syncwarp();
        cluster_sync_all();
        if (warp >= 2 && !*give_up) {
            const uint32_t mine = smem_u32(sums);
            const int t = threadIdx.x - 64, rt = first;
            for (int r = slice; r < g.M; r += slices) {
                float v = 0.0f;
                for (int k = 0; k < slices; ++k) v += peer_float(mine + (r * BR + t) * 4, k);
                int col = rt * BR + t;
                if (EPI == EPI_GATED) {
                    const float up = __shfl_down_sync(0xffffffffu, v, 1);
                    v = fast_gate_pair(v, up, g.act, g.limit);
                    col = (col & 1) ? g.N : col >> 1;
                } else {
                    v = act_of(v, g.act);
                }
                if (col < g.N) put(g, (long)r * g.ldy + col, v);
            }
        }
        __syncwarp();
        cluster_sync_all();                                     // no block leaves while another reads its sums
    }
    __syncthreads();
    if (warp == 1) tmem_dealloc(tmem, S::TMEM_COLS);
}

template <int BT, int EPI, bool EXPERTS>
int launch(const CUtensorMap& mw, const CUtensorMap& mx, StreamArgs g, int slices, cudaStream_t stream) {
    using S = Shape<BT>;
    const int sms = device_sms();
    const bool split = slices > 1;
    // two blocks an SM where there are more items than SMs (and tensor memory holds both)
    const int per_sm = S::TMEM_COLS <= 256 && g.items * slices > sms ? 2 : 1;
    const size_t room = per_sm == 2 ? 112 * 1024 : 220 * 1024;
    int stages = MAX_STAGES;
    while (stages > 2 && S::smem(stages, split) > room) --stages;
    g.stages = stages;
    const size_t smem = S::smem(stages, split);
    static OncePerDevice done;
    const int st = allow_shared_memory(fp8_stream_kernel<BT, EPI, EXPERTS>, 225 * 1024, done);
    if (st) return st;
    const int places = per_sm * sms;
    const int grid = split ? g.items * slices : g.items < places ? g.items : places;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(THREADS);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = pdl_enabled() ? 1 : 0;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = slices;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = EXPERTS ? 1 : 2;
    return (int)cudaLaunchKernelEx(&cfg, fp8_stream_kernel<BT, EPI, EXPERTS>, mw, mx, g);
}

template <int EPI, bool EXPERTS>
int dispatch(const CUtensorMap& mw, const CUtensorMap& mx, const StreamArgs& g, int bt, int slices, cudaStream_t stream) {
    if (bt == 16) return launch<16, EPI, EXPERTS>(mw, mx, g, slices, stream);
    if (bt == 32) return launch<32, EPI, EXPERTS>(mw, mx, g, slices, stream);
    if (bt == 64) return launch<64, EPI, EXPERTS>(mw, mx, g, slices, stream);
    return launch<128, EPI, EXPERTS>(mw, mx, g, slices, stream);
}

}  // namespace

// Y [M, N] = X W^T (epilogue 0) or the gated activation of W's neighbouring rows (epilogue 1: W has 2 N rows).  X and W as
// brolm_fp8_quantize leaves them; K is cut into `slices` (1 to 8), none of which is empty.  M <= 128.
BROLM_API int brolm_fp8_stream(const void* x, long long ldx, const void* x_scales, const void* w, long long ldw, const void* w_scales,
                               void* y, long long ldy, int out_f32, int M, int N, int K, int epilogue, int act, float limit, int slices,
                               cudaStream_t stream) {
    if (M <= 0 || N <= 0) return BROLM_OK;
    if (M > 128) return BROLM_ERR_TOO_LARGE;
    if (K <= 0 || ldx % 16 || ldw % 16 || (((uintptr_t)x | (uintptr_t)w | (uintptr_t)x_scales | (uintptr_t)w_scales) & 15)) return BROLM_ERR_ALIGNMENT;
    if (epilogue < 0 || epilogue > 1 || act < 0 || act > 2 || (epilogue == EPI_STORE && act > ACT_RELU2)) return BROLM_ERR_BAD_SIZE;
    const int nkb = blocks_of(K), w_rows = epilogue == EPI_GATED ? 2 * N : N;
    if (slices < 1 || slices > 8 || slices > nkb) return BROLM_ERR_BAD_SIZE;
    StreamArgs g = {};
    g.per = (nkb + slices - 1) / slices;
    if ((slices - 1) * g.per >= nkb) return BROLM_ERR_BAD_SIZE;
    const int bt = M <= 16 ? 16 : M <= 32 ? 32 : M <= 64 ? 64 : 128;
    CUtensorMap mw, mx;
    int st = make_map_u8(&mw, w, w_rows, K, ldw, BR);
    if (!st) st = make_map_u8(&mx, x, M, K, ldx, bt);
    if (st) return st;
    g.y = y; g.ldy = (long)ldy; g.M = M; g.N = N; g.out_f32 = out_f32; g.act = act; g.limit = limit;
    g.nkb = nkb; g.quads = quads_of(K);
    g.row_tiles = (w_rows + BR - 1) / BR; g.items = g.row_tiles;
    g.w_scales = (const uint8_t*)w_scales; g.x_scales = (const uint8_t*)x_scales;
    if (epilogue == EPI_GATED) return dispatch<EPI_GATED, false>(mw, mx, g, bt, slices, stream);
    return dispatch<EPI_STORE, false>(mw, mx, g, bt, slices, stream);
}

// The products of experts: rows [pairs] in the order of their experts, w the experts' matrices of w_rows rows, group_rows apart (a
// multiple of 128).  The list (expert, first row) of tiles of `rows` (16, 32, 64 or 128) rows and what it stands on come from
// brolm_fp8_group; x_scales has a tile of 128 rows for every tile of the list.  Y [pairs, N], or with `down` the float
// [top, tokens, N]; `scale` (or null): a number for every pair that multiplies its sums before the activation.
BROLM_API int brolm_fp8_experts_stream(const void* x, long long ldx, const void* x_scales, const void* w, long long ldw, const void* w_scales,
                                       void* y, long long ldy, int out_f32, int pairs, int N, int K, int experts, int group_rows, int epilogue,
                                       int act, float limit, const void* tile_group, const void* tile_row0, const void* offsets,
                                       const void* perm, const void* scale, int down, int top, int tokens, int rows, int max_tiles,
                                       cudaStream_t stream) {
    if (pairs <= 0 || N <= 0 || experts <= 0) return BROLM_OK;
    if (K <= 0 || ldx % 16 || ldw % 16 || (((uintptr_t)x | (uintptr_t)w | (uintptr_t)x_scales | (uintptr_t)w_scales) & 15)) return BROLM_ERR_ALIGNMENT;
    if (epilogue < 0 || epilogue > 1 || act < 0 || act > 2 || (epilogue == EPI_STORE && act > ACT_RELU2)) return BROLM_ERR_BAD_SIZE;
    if (group_rows % BR || (rows != 16 && rows != 32 && rows != 64 && rows != 128) || (down && !out_f32)) return BROLM_ERR_BAD_SIZE;
    const int w_rows = epilogue == EPI_GATED ? 2 * N : N;
    const long long all = (long long)experts * group_rows;
    if (all > 0x7fffffff || (long long)max_tiles * ((w_rows + BR - 1) / BR) > 0x7fffffff) return BROLM_ERR_TOO_LARGE;
    StreamArgs g = {};
    CUtensorMap mw, mx;
    int st = make_map_u8(&mw, w, all, K, ldw, BR);
    if (!st) st = make_map_u8(&mx, x, pairs, K, ldx, rows);
    if (st) return st;
    g.y = y; g.ldy = (long)ldy; g.N = N; g.out_f32 = out_f32; g.act = act; g.limit = limit;
    g.nkb = blocks_of(K); g.quads = quads_of(K); g.per = g.nkb;
    g.row_tiles = (w_rows + BR - 1) / BR; g.items = g.row_tiles * max_tiles;
    g.w_scales = (const uint8_t*)w_scales; g.x_scales = (const uint8_t*)x_scales;
    g.tile_group = (const int32_t*)tile_group; g.tile_row0 = (const int32_t*)tile_row0; g.offsets = (const int32_t*)offsets;
    g.perm = (const int32_t*)perm; g.scale = (const float*)scale;
    g.down = down; g.top = top; g.tokens = tokens; g.group_rows = group_rows;
    if (epilogue == EPI_GATED) return dispatch<EPI_GATED, true>(mw, mx, g, rows, 1, stream);
    return dispatch<EPI_STORE, true>(mw, mx, g, rows, 1, stream);
}

BROLM_API int brolm_fp8_stream_status(int reset) {
    int v = 0;
    if (cudaMemcpyFromSymbol(&v, g_fp8_stream_error, sizeof(int)) != cudaSuccess) return -1;
    if (reset && v) {
        const int zero = 0;
        cudaMemcpyToSymbol(g_fp8_stream_error, &zero, sizeof(int));
    }
    return v;
}

BROLM_WAIT_CONTROL(fp8_stream)
