// Products with a matrix in 8-bit floating point for few rows (the format is in fp8.cuh), on tcgen05:
//     Y[m,n] = sum over blocks b of 2^(sx[m,b] + sw[n,b]) * (sum over the block's k of X[m,k] W[n,k]),  float sums.
//
// With few rows the product is a stream of W from memory.  The roles of the operands are swapped: 128 rows of W are the M side
// of tcgen05.mma.kind::mxf8f6f4, the rows of X (16, 32, 64 or 128 of them) the N side, and the tensor core multiplies by the
// scales itself.  A stage of the ring is one block of K: 16 KB of W, the rows of X beside it and, for the first block of every
// four, the 512 bytes of scales of each side, which tcgen05.cp carries into tensor memory ahead of the products that need
// them (copies and products of one thread are executed in order).
//
//   warp 0    one thread: TMA loads, and untiled copies of the scales' tiles; those of W begin before the kernel before this one
//             has ended
//   warp 1    one thread: copies of scales and products into one of two accumulators (128 rows of X: the one there is room for),
//             commits
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
#include "fp8_round.cuh"

#include <type_traits>

namespace {

using namespace tc;
using namespace fp8;

constexpr int BR = 128, BK = 128;
constexpr int W_BYTES = BR * BK;
constexpr int MAX_STAGES = 12;
constexpr int FUSED_BLOCKS = 24;       // 48 KB of the rows, five stages beside them

enum : int { EPI_STORE = 0, EPI_GATED = 1 };

__device__ int g_fp8_stream_error;

struct StreamArgs {
    void* y;
    long ldy;
    int M, N;                // rows of X (dense); output columns
    int out_f32, act, y_wide;
    float limit;
    int nkb, quads;          // blocks of K, words of scales
    int row_tiles, items, stages;
    int per;                 // blocks of K of a slice (dense; the cluster's rank is the slice)
    const void* x;           // rows that are no 8-bit numbers yet (FUSED), elements apart
    long ldx;
    int x_wide, K;
    const uint8_t* w_scales;
    const uint8_t* x_scales;
    // experts
    const int32_t* tile_group;      // null: dense
    const int32_t* tile_row0;
    const int32_t* offsets;
    const int32_t* perm;
    const float* scale;      // of a pair, before the activation
    int down, top, tokens, group_rows;
    int listed;
};

__device__ __forceinline__ bool wait_on(uint32_t bar, uint32_t parity, volatile int* give_up, int code) {
    return mbar_wait<4>(bar, parity, give_up, &g_fp8_stream_error, code);      // (others begin to wait when a stalled one does)
}
// a wait that is mostly over when it begins: the flags are looked at only if it is not
__device__ __forceinline__ bool wait_one(uint32_t bar, uint32_t parity, volatile int* give_up, int code) {
    return mbar_try(bar, parity) || wait_on(bar, parity, give_up, code);
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
__device__ __forceinline__ float4 peer_floats(uint32_t addr, uint32_t rank) {
    float4 v;
    asm volatile("{\n.reg .b32 r;\nmapa.shared::cluster.u32 r, %4, %5;\nld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [r];\n}"
                 : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr), "r"(rank));
    return v;
}
__device__ __forceinline__ void put(const StreamArgs& g, long at, float v) {
    if (g.out_f32) reinterpret_cast<float*>(g.y)[at] = v;
    else reinterpret_cast<bf16*>(g.y)[at] = __float2bfloat16_rn(v);
}

// The rows of X of this block's slice of K, in 8 bits as the products want them: row r of block kb at r * 128 bytes of its
// X_BYTES, its sixteen-byte pieces swapped as a TMA load with the 128-byte swizzle would leave them; scales in tiles of four
// blocks.  A warp takes four blocks of a row at a time and asks for four such pieces before it rounds the first.
template <typename T, int BT, bool WIDE>
__device__ __forceinline__ void round_rows(const StreamArgs& g, uint8_t* x_blocks, uint8_t* x_scales, int lo, int hi, int w, int lane) {
    constexpr int DEEP = 4;
    const int q0 = lo >> 2, n = ((hi + 3) >> 2) - q0, tasks = n * g.M;
    const T* x = (const T*)g.x;
    for (int t0 = w; t0 < tasks; t0 += 8 * DEEP) {
        Piece<T, WIDE> piece[DEEP];
        int row[DEEP], quad[DEEP];
#pragma unroll
        for (int d = 0; d < DEEP; ++d) {
            const int t = t0 + 8 * d;
            row[d] = t / n;
            quad[d] = t - row[d] * n;
            piece[d].ask(x + row[d] * g.ldx, (q0 + quad[d]) * 512 + lane * 16, g.K, t < tasks);
        }
#pragma unroll
        for (int d = 0; d < DEEP; ++d) {
            if (t0 + 8 * d >= tasks) break;                     // (the same for the whole warp)
            const int kb = (q0 + quad[d]) * 4 + (lane >> 3);
            float v[16];
            piece[d].get(x + row[d] * g.ldx, (q0 + quad[d]) * 512 + lane * 16, g.K, v);
            uint32_t word;
            const uint4 u = round16(v, word);
            if (kb >= lo && kb < hi)
                *reinterpret_cast<uint4*>(x_blocks + (kb - lo) * (BT * BK) + row[d] * BK + (((lane & 7) ^ (row[d] & 7)) << 4)) = u;
            if (lane == 0) *reinterpret_cast<uint32_t*>(x_scales + quad[d] * SF_TILE + row[d] * 16) = word;
        }
    }
}

// FUSED: 0 the rows are 8-bit numbers in memory; 1, 2: they are bfloat16, float numbers, and every block rounds what it needs.
template <int BT, int FUSED>
struct Shape {
    static constexpr int THREADS = FUSED ? 320 : 192;                   // (eight warps that round, of which four have an epilogue)
    static constexpr int X_BYTES = BT * BK;
    static constexpr int STAGE_BYTES = FUSED ? W_BYTES : W_BYTES + X_BYTES;      // multiples of 1024
    // accumulators and two pairs of scales in at most half of tensor memory, so that an SM holds two blocks
    static constexpr int ACCS = BT == 128 ? 1 : 2;
    static constexpr int COLS = ACCS * BT + 16;
    static constexpr int TMEM_COLS = COLS <= 64 ? 64 : COLS <= 128 ? 128 : 256;
    static constexpr int SCALES = FUSED ? SF_TILE : 2 * SF_TILE;        // of a stage
    static size_t x_room(int per) { return FUSED ? (size_t)per * X_BYTES + (size_t)((per + 3) / 4 + 1) * SF_TILE : 0; }
    static size_t smem(int stages, int per) {
        return x_room(per) + (size_t)stages * (STAGE_BYTES + SCALES) + (2 * MAX_STAGES + 6) * 8 + 16;
    }
};

template <int BT, int EPI, bool EXPERTS, int FUSED>
__global__ void __launch_bounds__(Shape<BT, FUSED>::THREADS, 2) fp8_stream_kernel(const __grid_constant__ CUtensorMap map_w,
                                                             const __grid_constant__ CUtensorMap map_x, StreamArgs g) {
    using S = Shape<BT, FUSED>;
    constexpr int ACCS = S::ACCS;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t* base = smem_raw;
    const int stages = g.stages;
    // the ring, (FUSED) the slice's rows in 8 bits, the scales of the ring, (FUSED) those of the rows, barriers
    uint8_t* x_blocks = base + stages * S::STAGE_BYTES;
    uint8_t* scale_slots = x_blocks + (FUSED ? g.per * S::X_BYTES : 0);
    uint8_t* x_scales = scale_slots + stages * S::SCALES;
    uint64_t* bars = reinterpret_cast<uint64_t*>(x_scales + (FUSED ? ((g.per + 3) / 4 + 1) * SF_TILE : 0));
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 2 * MAX_STAGES + 6);
    volatile int* give_up = reinterpret_cast<volatile int*>(tmem_slot + 1);
    // slices: this one's sums [rows of X][128], in the ring, which is read to its end by then
    float* sums = reinterpret_cast<float*>(base);
    const uint32_t stage0 = smem_u32(base), scale0 = smem_u32(scale_slots);
    const uint32_t full0 = smem_u32(bars), empty0 = full0 + 8 * MAX_STAGES, acc_full0 = empty0 + 8 * MAX_STAGES,
                   acc_empty0 = acc_full0 + 16, x_ready = acc_empty0 + 16, ended = x_ready + 8;
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
        mbar_init(x_ready, 8);
        mbar_init(ended, 1);
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
        group = __ldcg(&g.tile_group[tile]);             // (perhaps read before this kernel's wait)
        if (group < 0) return false;
        row0 = __ldcg(&g.tile_row0[tile]);
        return true;
    };

    if (warp == 0) {
        if (elect_one() && !*give_up) {
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
                if (FUSED) return;
                const uint32_t full = full0 + 8 * s;
                tma_load_2d(stage0 + s * S::STAGE_BYTES + W_BYTES, &map_x, kb * BK, row0, full);
                if ((kb & 3) == 0 || kb == lo)
                    bulk_load(scale0 + s * S::SCALES + SF_TILE, g.x_scales + ((size_t)tile * g.quads + (kb >> 2)) * SF_TILE, SF_TILE, full);
            };
            int item = first, kb = lo, it = 0, rt = 0, group = 0, row0 = 0, tile = 0;
            bool more;
            // The ring fills with weights before the kernel before this one has ended; experts' where their list is known by then.
            const bool ahead = !EXPERTS || g.listed;
            if (!ahead) pdl_wait();
            more = item < g.items && lo < hi && find(item, rt, group, row0, tile);
            if (ahead) {
                int n = 0;
                for (; n < stages && lo + n < hi && more; ++n) load_w(n, rt, group, lo + n);
                pdl_wait();
                for (int i = 0; i < n; ++i) load_x(i, row0, tile, lo + i);
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
                if (!(kb > lo ? wait_one(empty0 + 8 * s, phase ^ 1, give_up, 1) : wait_on(empty0 + 8 * s, phase ^ 1, give_up, 1))) break;
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
        if (elect_one() && !*give_up) {
            const uint32_t id = idesc_mx(BR, BT);
            if (EXPERTS) pdl_wait();
            int s = 0, phase = 0, local = 0, set = 0;
            bool ok = true;
            int rt, group, row0, tile;
            for (int item = first; item < g.items && lo < hi && ok; item += step, ++local) {
                if (!find(item, rt, group, row0, tile)) break;
                const int as = local % ACCS;
                ok = wait_on(acc_empty0 + 8 * as, ((local / ACCS) & 1) ^ 1, give_up, 5);
                if (FUSED && ok && local == 0) ok = wait_on(x_ready, 0, give_up, 6);
                if (!ok) break;
                fence_after_sync();
                const uint32_t acc = tmem + as * BT;
                uint32_t sfw = 0, sfx = 0;
                for (int kb = lo; kb < hi; ++kb) {
                    ok = kb > lo ? wait_one(full0 + 8 * s, phase, give_up, 2) : wait_on(full0 + 8 * s, phase, give_up, 2);
                    if (!ok) break;
                    fence_after_sync();
                    if ((kb & 3) == 0 || kb == lo) {
                        sfw = tmem + ACCS * BT + 8 * set;
                        sfx = sfw + 4;
                        set ^= 1;
                        scales_to_tmem(sfw, desc_scales(scale0 + s * S::SCALES));
                        scales_to_tmem(sfx, desc_scales(FUSED ? smem_u32(x_scales) + ((kb >> 2) - (lo >> 2)) * SF_TILE : scale0 + s * S::SCALES + SF_TILE));
                    }
                    const uint32_t idk = with_block(id, kb & 3, kb & 3);
                    const uint64_t a = desc_kmajor(stage0 + s * S::STAGE_BYTES);
                    const uint64_t b = desc_kmajor(FUSED ? smem_u32(x_blocks) + (kb - lo) * S::X_BYTES : stage0 + s * S::STAGE_BYTES + W_BYTES);
#pragma unroll
                    for (int k = 0; k < BK / 32; ++k) umma_mx(acc, a + 2 * k, b + 2 * k, idk, sfw, sfx, (kb > lo) | (k > 0));
                    umma_commit(empty0 + 8 * s);
                    if (++s == stages) { s = 0; phase ^= 1; }
                }
                if (ok) umma_commit(acc_full0 + 8 * as);
            }
            if (!ok) {                                      // products in flight end before their operands go
                umma_commit(ended);
                drain_on(ended, 0, give_up, 8);
            }
        }
    } else {
        const int quarter = warp & 3;
        const int lrow = quarter * 32 + lane;                   // row of the tile of W = lane of tensor memory
        if (EXPERTS || FUSED) pdl_wait();
        if (FUSED) {
            using T = typename std::conditional<FUSED == 1, bf16, float>::type;
            if (g.x_wide) round_rows<T, BT, true>(g, x_blocks, x_scales, lo, hi, warp - 2, lane);
            else round_rows<T, BT, false>(g, x_blocks, x_scales, lo, hi, warp - 2, lane);
            fence_proxy_async();
            __syncwarp();
            if (lane == 0) mbar_arrive(x_ready);
        }
        int local = 0, rt, group, row0, tile;
        for (int item = first; item < g.items && lo < hi && warp < 6; item += step, ++local) {
            if (!find(item, rt, group, row0, tile)) break;
            const int as = local % ACCS;
            const bool ready = !*give_up && wait_on(acc_full0 + 8 * as, (local / ACCS) & 1, give_up, 3);
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
                        o[i] = gate_of(odd ? got : o[2 * i], odd ? o[2 * i + 1] : got, g.act, g.limit);
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
        if (warp >= 2 && warp < 6 && !*give_up) {
            // four neighbouring columns a thread, four rows at a time; the slices' numbers are asked for together
            const int t = threadIdx.x - 64, at = (t & 31) * 4;
            const uint32_t mine = smem_u32(sums) + at * 4;
            for (int r = slice + (t >> 5) * slices; r < g.M; r += 4 * slices) {
                float4 part[8];
                float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int k = 0; k < 8; ++k) if (k < slices) part[k] = peer_floats(mine + r * BR * 4, k);
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    if (k < slices) { v[0] += part[k].x; v[1] += part[k].y; v[2] += part[k].z; v[3] += part[k].w; }
                }
                if (EPI == EPI_GATED) {
                    const int col = (first * BR + at) >> 1;
#pragma unroll
                    for (int i = 0; i < 2; ++i) if (col + i < g.N) put(g, (long)r * g.ldy + col + i, gate_of(v[2 * i], v[2 * i + 1], g.act, g.limit));
                } else {
                    const int col = first * BR + at;
#pragma unroll
                    for (int i = 0; i < 4; ++i) v[i] = act_of(v[i], g.act);
                    if (g.y_wide && col + 4 <= g.N) {
                        if (g.out_f32) {
                            *reinterpret_cast<float4*>((float*)g.y + (long)r * g.ldy + col) = make_float4(v[0], v[1], v[2], v[3]);
                        } else {
                            uint2 u;
                            __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&u);
                            h[0] = __floats2bfloat162_rn(v[0], v[1]);
                            h[1] = __floats2bfloat162_rn(v[2], v[3]);
                            *reinterpret_cast<uint2*>((bf16*)g.y + (long)r * g.ldy + col) = u;
                        }
                    } else {
#pragma unroll
                        for (int i = 0; i < 4; ++i) if (col + i < g.N) put(g, (long)r * g.ldy + col + i, v[i]);
                    }
                }
            }
        }
        __syncwarp();
        cluster_sync_all();                                     // no block leaves while another reads its sums
    }
    __syncthreads();
    if (warp == 1) tmem_dealloc(tmem, S::TMEM_COLS);
}

template <int BT, int EPI, bool EXPERTS, int FUSED>
int launch(const CUtensorMap& mw, const CUtensorMap& mx, StreamArgs g, int slices, cudaStream_t stream) {
    using S = Shape<BT, FUSED>;
    const int sms = device_sms();
    const bool split = slices > 1;
    // Two blocks an SM: one streams while the other starts or ends, and clusters of up to eight find room.  (Three with 74 KB,
    // where experts' items fill their rounds better, gained nothing.)
    constexpr size_t ROOM = 112 * 1024;
    int stages = MAX_STAGES;
    while (stages > 2 && S::smem(stages, g.per) > ROOM) --stages;
    const size_t smem = S::smem(stages, g.per);
    if (smem > ROOM || (split && (size_t)stages * S::STAGE_BYTES < (size_t)BT * BR * 4)) return BROLM_ERR_TOO_LARGE;
    g.stages = stages;
    static OncePerDevice done;
    const int st = allow_shared_memory(fp8_stream_kernel<BT, EPI, EXPERTS, FUSED>, ROOM, done);
    if (st) return st;
    const int places = 2 * sms;
    const int grid = split ? g.items * slices : g.items < places ? g.items : places;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(S::THREADS);
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
    return (int)cudaLaunchKernelEx(&cfg, fp8_stream_kernel<BT, EPI, EXPERTS, FUSED>, mw, mx, g);
}

template <int EPI, bool EXPERTS>
int dispatch(const CUtensorMap& mw, const CUtensorMap& mx, const StreamArgs& g, int bt, int slices, int fused, cudaStream_t stream) {
    if constexpr (!EXPERTS) {
        if (fused == 1) return launch<16, EPI, false, 1>(mw, mx, g, slices, stream);
        if (fused == 2) return launch<16, EPI, false, 2>(mw, mx, g, slices, stream);
    }
    if (bt == 16) return launch<16, EPI, EXPERTS, 0>(mw, mx, g, slices, stream);
    if (bt == 32) return launch<32, EPI, EXPERTS, 0>(mw, mx, g, slices, stream);
    if constexpr (!EXPERTS) {
        if (bt == 64) return launch<64, EPI, false, 0>(mw, mx, g, slices, stream);
        return launch<128, EPI, false, 0>(mw, mx, g, slices, stream);
    }
    return BROLM_ERR_BAD_SIZE;
}

}  // namespace

// Y [M, N] = X W^T (epilogue 0, act 0 or the square of relu) or the gated activation of W's neighbouring rows (epilogue 1: W
// has 2 N rows); out 0: bfloat16, 1: float.  X and W as brolm_fp8_quantize leaves them.
// Dense (experts 0): M <= 128; K is cut into `cut` slices (1 to 8), none of which is empty.  fused 1, 2: X are bfloat16, float
// numbers (ldx elements between rows, x_scales unused), M <= 16, and a slice has at most FUSED_BLOCKS blocks of 128 of K.
// Experts: M pairs' rows in the order of their experts, W the experts' matrices, group_rows (a multiple of 128) rows each.  The
// list (expert, first row) of tiles of `rows` (16 or 32) rows and what it stands on come from brolm_fp8_group; x_scales
// has a tile of 128 rows for every tile of the list.  Y [M, N], or with `down` float [top, tokens, N]; `scale` (or null): a
// number for every pair that multiplies its sums before the activation.
BROLM_API int brolm_fp8_stream(const fp8::ProductCall* c) {
    const int M = c->M, N = c->N, K = c->K;
    if (M <= 0 || N <= 0) return BROLM_OK;
    if (K <= 0 || c->ldw % 16 || (((uintptr_t)c->w | (uintptr_t)c->w_scales) & 15)) return BROLM_ERR_ALIGNMENT;
    if (!c->fused && (c->ldx % 16 || (((uintptr_t)c->x | (uintptr_t)c->x_scales) & 15))) return BROLM_ERR_ALIGNMENT;
    if (c->fused < 0 || c->fused > 2 || (c->fused && (M > 16 || c->experts))) return BROLM_ERR_BAD_SIZE;
    if (c->epilogue < 0 || c->epilogue > 1 || c->act < 0 || c->act > 2 || (c->epilogue == EPI_STORE && c->act > ACT_RELU2)) return BROLM_ERR_BAD_SIZE;
    if (c->out < 0 || c->out > 1) return BROLM_ERR_BAD_SIZE;
    const long long w_rows = c->epilogue == EPI_GATED ? 2LL * N : N;
    StreamArgs g = {};
    g.y = c->y; g.ldy = (long)c->ldy; g.M = M; g.N = N; g.out_f32 = c->out; g.act = c->act; g.limit = c->limit;
    g.y_wide = ((uintptr_t)c->y & 15) == 0 && c->ldy % 4 == 0;
    g.nkb = blocks_of(K); g.quads = quads_of(K);
    g.w_scales = (const uint8_t*)c->w_scales; g.x_scales = (const uint8_t*)c->x_scales;
    const long long row_tiles = (w_rows + BR - 1) / BR;
    CUtensorMap mw, mx;
    if (c->experts) {
        const int rows = c->rows;
        if (c->group_rows % BR || (rows != 16 && rows != 32) || (c->down && !c->out)) return BROLM_ERR_BAD_SIZE;
        const long long all = (long long)c->experts * c->group_rows;
        if (all > 0x7fffffff || c->max_tiles * row_tiles > 0x7fffffff) return BROLM_ERR_TOO_LARGE;
        int st = make_map_u8(&mw, c->w, all, K, c->ldw, BR);
        if (!st) st = make_map_u8(&mx, c->x, M, K, c->ldx, rows);
        if (st) return st;
        g.per = g.nkb; g.row_tiles = (int)row_tiles; g.items = (int)(row_tiles * c->max_tiles);
        g.tile_group = (const int32_t*)c->tile_group; g.tile_row0 = (const int32_t*)c->tile_row0; g.offsets = (const int32_t*)c->offsets;
        g.perm = (const int32_t*)c->perm; g.scale = (const float*)c->scale;
        g.down = c->down; g.top = c->top; g.tokens = c->tokens; g.group_rows = c->group_rows; g.listed = c->listed;
        if (c->epilogue == EPI_GATED) return dispatch<EPI_GATED, true>(mw, mx, g, rows, 1, 0, c->stream);
        return dispatch<EPI_STORE, true>(mw, mx, g, rows, 1, 0, c->stream);
    }
    const int slices = c->cut;
    if (M > 128 || w_rows > 0x7fffffff - BR) return BROLM_ERR_TOO_LARGE;
    if (slices < 1 || slices > 8 || slices > g.nkb) return BROLM_ERR_BAD_SIZE;
    g.per = (g.nkb + slices - 1) / slices;
    if ((slices - 1) * g.per >= g.nkb) return BROLM_ERR_BAD_SIZE;
    const int bt = M <= 16 ? 16 : M <= 32 ? 32 : M <= 64 ? 64 : 128;
    int st = make_map_u8(&mw, c->w, w_rows, K, c->ldw, BR);
    if (!st && !c->fused) st = make_map_u8(&mx, c->x, M, K, c->ldx, bt);
    if (st) return st;
    if (c->fused) {
        if (g.per > FUSED_BLOCKS) return BROLM_ERR_TOO_LARGE;
        g.x = c->x; g.ldx = (long)c->ldx; g.K = K;
        g.x_wide = ((uintptr_t)c->x & 15) == 0 && c->ldx % (c->fused == 1 ? 8 : 4) == 0;
        mx = mw;
    }
    g.row_tiles = g.items = (int)row_tiles;
    st = round_first(c);
    if (st) return st;
    if (c->epilogue == EPI_GATED) return dispatch<EPI_GATED, false>(mw, mx, g, bt, slices, c->fused, c->stream);
    return dispatch<EPI_STORE, false>(mw, mx, g, bt, slices, c->fused, c->stream);
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
