// Products with a matrix in 8-bit floating point for many rows (the format is in fp8.cuh), on pairs of SMs:
//     Y[m,n] = sum over blocks b of 2^(sx[m,b] + sw[n,b]) * (sum over the block's k of X[m,k] W[n,k]),  float sums.
//
// Two blocks of a cluster make a tile of 256 x 256 (tcgen05.mma.cta_group::2.kind::mxf8f6f4, which multiplies by the scales
// itself): each loads its 128 rows of X and its half of the 256 rows of W.  A stage is one block of 128 along K, 32 KB a block
// of the pair; with the first block of every four come their scales, 512 bytes for the block's rows of X and 1,024 for all 256
// rows of W, which tcgen05.cp carries into both blocks' tensor memory.
//
//   warp 0 (both blocks)   one thread: TMA loads, their bytes counted on the first block's barrier; the first stages' part of W
//                          before the kernel before this one has ended
//   warp 1 (first block)   one thread: copies of scales, products, commits to both blocks
//   warps 4-11 (both)      epilogue: a thread has a row of the tile and half of its columns, in up to 224 registers, which the first
//                          four warps leave them (two of those are there for that alone: registers go by four warps)
//
// Tensor memory has 512 columns: two accumulators of 256 leave no room for the scales.  So the second accumulator begins 32
// columns before the first ends.  A tile's products begin when the epilogue has taken those 32 columns of the tile before
// (its first loads), and when the accumulator's own tile, two before, has been taken whole.
//
// The tensor core cuts off where an fma rounds, so float results are summed in pieces of `piece` blocks of K, which the
// epilogue adds in registers; results that are rounded to fewer bits are one piece.
//
// Epilogues: the product (with the square of relu, or a gated activation of neighbouring rows of W) as bfloat16, as float, or
// rounded to 8 bits as rows for the next product: a block of 128 results of a row is within a tile.  Experts: a list made on
// the device names for every tile of 256 rows its expert and its first row.
//
// Every mbarrier wait is bounded (tcgen05.cuh).
#include "fp8.cuh"

#include <type_traits>

namespace {

using namespace tc;
using namespace fp8;

constexpr int BM = 128, PM = 256, BN = 256, HN = 128, BK = 128, STAGES = 5;
constexpr int A_BYTES = BM * BK, B_BYTES = HN * BK, STAGE_BYTES = A_BYTES + B_BYTES, SCALES = 3 * SF_TILE;
constexpr int THREADS = 384;
constexpr int FIRST = 4;             // the epilogue's first warp
constexpr int TMEM_COLS = 512, ACC1 = 224, SF_COL = 480;
constexpr int ROOM_BYTES = 8 * 4096;        // of the epilogue's warps, for results on their way out
constexpr int ROWS_BYTES = 4 * BM * 4;      // largest magnitudes of a row's two halves

enum : int { EPI_STORE = 0, EPI_GATED = 1 };
enum : int { OUT_BF16 = 0, OUT_F32 = 1, OUT_FP8 = 2 };

__device__ int g_fp8_gemm_error;

struct GemmArgs {
    void* y;
    long ldy;                // elements (OUT_FP8: bytes)
    uint8_t* y_scales;
    int y_quads, y_wide;
    int M, N;                // rows; output columns
    int act;
    float limit;
    int nkb, piece;
    int quads;               // words of scales of a row of X and W
    int m_tiles, n_tiles;
    // experts
    const int32_t* tile_group;      // null: dense
    const int32_t* tile_row0;
    const int32_t* offsets;
    const int32_t* perm;
    const float* scale;
    int down, top, tokens, group_rows, experts, listed;
};

__device__ __forceinline__ bool wait_on(uint32_t bar, uint32_t parity, volatile int* give_up, int code) {
    return mbar_wait<4>(bar, parity, give_up, &g_fp8_gemm_error, code);      // (others begin to wait when a stalled one does)
}
// a wait that is mostly over when it begins
__device__ __forceinline__ bool wait_one(uint32_t bar, uint32_t parity, volatile int* give_up, int code) {
    return mbar_try(bar, parity) || wait_on(bar, parity, give_up, code);
}
__device__ __forceinline__ bool drain_on(uint32_t bar, uint32_t parity, volatile int* give_up, int code) {
    return mbar_wait(bar, parity, give_up, &g_fp8_gemm_error, code, true);
}
__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_sync_all() {
    asm volatile("barrier.cluster.arrive.aligned;\nbarrier.cluster.wait.aligned;" ::: "memory");
}
// The cta_group::2 forms.  A shared-memory address with bit 24 cleared names the same place in the first block of the pair.
constexpr uint32_t PEER_MASK = 0xFEFFFFFFu;
__device__ __forceinline__ void tma_load_pair(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
                 ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(bar & PEER_MASK) : "memory");
}
__device__ __forceinline__ void umma_mx_pair(uint32_t d, uint64_t a, uint64_t b, uint32_t id, uint32_t sfa, uint32_t sfb, uint32_t accumulate) {
    asm volatile("{\n.reg .pred p;\nsetp.ne.b32 p, %6, 0;\n"
                 "tcgen05.mma.cta_group::2.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [%5], p;\n}"
                 ::"r"(d), "l"(a), "l"(b), "r"(id), "r"(sfa), "r"(sfb), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void scales_to_tmem_pair(uint32_t taddr, uint64_t desc) {
    asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
}
__device__ __forceinline__ void umma_commit_pair(uint32_t bar) {      // arrives on the barrier in both blocks
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
                 ::"r"(bar), "h"((uint16_t)3) : "memory");
}
__device__ __forceinline__ void tmem_alloc_pair(uint32_t slot_smem, uint32_t cols) {     // whole warp, in both blocks
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(slot_smem), "r"(cols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_dealloc_pair(uint32_t taddr, uint32_t cols) {
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(cols) : "memory");
}
__device__ __forceinline__ void arrive_first_block(uint32_t bar) {                       // from either block
    asm volatile("{\n.reg .b32 remote;\nmapa.shared::cluster.u32 remote, %0, 0;\nmbarrier.arrive.shared::cluster.b64 _, [remote];\n}"
                 ::"r"(bar) : "memory");
}

// N / 2 gated pairs of neighbouring numbers, to the front.  Code for two kinds of gates and not for three: the shorter the epilogue,
// the less the issue of products waits for instructions (512 tokens through experts 73 -> 70 us).
template <int N>
__device__ __forceinline__ void gate_pairs(float (&o)[N], int act, float limit) {
    if (act == 2) {
#pragma unroll
        for (int i = 0; i < N / 2; ++i) o[i] = gate_of(o[2 * i], o[2 * i + 1], 2, limit);
    } else {
        const int kind = act == 0 ? 0 : 1;
#pragma unroll
        for (int i = 0; i < N / 2; ++i) o[i] = gate_of(o[2 * i], o[2 * i + 1], kind, 0.0f);
    }
}

// Results on their way out.  A thread has a row, and stores of sixteen bytes in 32 rows are half sectors in 32 lines: they took
// longer than the products of a tile (2,304 along K: 18,500 cycles a tile, of which 6,400 were that).  So a warp leaves 128
// bytes of each of its 32 rows in four KB of shared memory of its own, sixteen-byte pieces swapped by the row, and stores whole
// lines from there, eight lanes a row.
__device__ __forceinline__ void stage16(uint8_t* room, int lane, int piece, uint4 v) {
    *reinterpret_cast<uint4*>(room + lane * 128 + ((piece ^ (lane & 7)) << 4)) = v;
}
// Row r of the warp goes to dst + (r or, SCATTER, lane r's `at`) * ld, if r < rows; of its ROW bytes staged `bytes` are wanted,
// in units of `unit` bytes where they do not lie in sixteens (`wide`).
template <int ROW, bool SCATTER>
__device__ __forceinline__ void flush_rows(const uint8_t* room, int lane, uint8_t* dst, long ld, int at, int rows, int bytes, bool wide, int unit) {
    __syncwarp();
    constexpr int PIECES = ROW / 16, ROWS = 32 / PIECES;       // rows a round
    const int piece = lane % PIECES, left = bytes - piece * 16;
    dst += piece * 16;
    if (wide && bytes >= ROW) {
        uint8_t* to = dst + (lane / PIECES) * ld;
#pragma unroll
        for (int r0 = 0; r0 < 32; r0 += ROWS) {
            const int r = r0 + lane / PIECES;
            const uint4 v = *reinterpret_cast<const uint4*>(room + r * 128 + ((piece ^ (r & 7)) << 4));
            if (SCATTER) to = dst + (long)__shfl_sync(0xffffffffu, at, r) * ld;
            if (r < rows) *reinterpret_cast<uint4*>(to) = v;
            if (!SCATTER) to += ROWS * ld;
        }
    } else {
        // few tiles come here: short code, since the products' issue suffers where the epilogue's is long
#pragma unroll 1
        for (int r0 = 0; r0 < 32; r0 += ROWS) {
            const int r = r0 + lane / PIECES;
            const uint8_t* from = room + r * 128 + ((piece ^ (r & 7)) << 4);
            uint8_t* to = dst + (long)(SCATTER ? __shfl_sync(0xffffffffu, at, r) : r) * ld;
            const int n = r < rows ? min(left, 16) : 0;
            if (wide && n == 16) {
                *reinterpret_cast<uint4*>(to) = *reinterpret_cast<const uint4*>(from);
            } else if (unit == 4) {
#pragma unroll 1
                for (int i = 0; i < n; i += 4) *reinterpret_cast<uint32_t*>(to + i) = *reinterpret_cast<const uint32_t*>(from + i);
            } else {
#pragma unroll 1
                for (int i = 0; i < n; i += 2) *reinterpret_cast<uint16_t*>(to + i) = *reinterpret_cast<const uint16_t*>(from + i);
            }
        }
    }
    __syncwarp();
}
__device__ __forceinline__ uint4 pack_bf16(const float* o) {
    uint4 p;
    __nv_bfloat162* p2 = reinterpret_cast<__nv_bfloat162*>(&p);
#pragma unroll
    for (int e = 0; e < 4; ++e) p2[e] = __floats2bfloat162_rn(o[2 * e], o[2 * e + 1]);
    return p;
}

// Numbers that a load from tensor memory brought are not to be touched before the wait for it.
__device__ __forceinline__ void arrived(uint32_t (&v)[32]) {
    tmem_wait_ld();
#pragma unroll
    for (int i = 0; i < 32; ++i) asm volatile("" : "+r"(v[i]));
}
// The 128 columns at `acc` in parts of 32, those from BACK parts before the end on first, the next part's load under way while
// one is used: there(turn) once a part is in registers, use(part, numbers).
template <int BACK, int TURN, typename T, typename F>
__device__ __forceinline__ void walk(uint32_t acc, uint32_t (&now)[32], uint32_t (&next)[32], T&& there, F&& use) {
    arrived(now);
    there(TURN);
    if constexpr (TURN < 3) tmem_ld32(acc + (TURN + 1 + 4 - BACK) % 4 * 32, next);
    use(std::integral_constant<int, (TURN + 4 - BACK) % 4>{}, now);
    if constexpr (TURN < 3) walk<BACK, TURN + 1>(acc, next, now, there, use);
}

template <int EPI, int OUT, bool EXPERTS>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(THREADS, 1)
fp8_gemm_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w,
                const __grid_constant__ CUtensorMap map_xs, const __grid_constant__ CUtensorMap map_ws, GemmArgs g) {
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t* base = smem_raw;
    const uint32_t rank = cluster_rank();
    uint8_t* rooms = base + STAGES * (STAGE_BYTES + SCALES);
    uint64_t* bars = reinterpret_cast<uint64_t*>(rooms + ROOM_BYTES);
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 2 * STAGES + 10);
    volatile int* give_up = reinterpret_cast<volatile int*>(tmem_slot + 1);
    uint32_t* most_of = tmem_slot + 4;                        // [2][2][128]
    const uint32_t stage0 = smem_u32(base), scale0 = stage0 + STAGES * STAGE_BYTES;
    const uint32_t full0 = smem_u32(bars), empty0 = full0 + 8 * STAGES, acc_full0 = empty0 + 8 * STAGES,
                   acc_free0 = acc_full0 + 16, lap_free = acc_free0 + 16, halves0 = lap_free + 16, ended = lap_free + 8;
    const bool aligned = (stage0 & 1023u) == 0;               // both blocks have the same layout

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int pair = blockIdx.x >> 1, n_pairs = gridDim.x >> 1;
    constexpr int OUT_COLS = EPI == EPI_GATED ? BN / 2 : BN;
    // where the tiles end in a round that keeps half of the pairs or less, those are two items of half the columns each (a
    // gated row's block of 128 results in 8 bits is a whole tile)
    constexpr bool HALVES = !(OUT == OUT_FP8 && EPI == EPI_GATED);
    auto items_of = [&](int tiles, int& whole) {
        const int rest = tiles % n_pairs;
        whole = HALVES && 2 * rest <= n_pairs ? tiles - rest : tiles;
        return tiles + (tiles - whole);
    };

    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) {
            mbar_init(full0 + 8 * s, 1);
            mbar_init(empty0 + 8 * s, 1);
        }
        for (int s = 0; s < 2; ++s) {
            mbar_init(acc_full0 + 8 * s, 1);
            mbar_init(acc_free0 + 8 * s, 16);     // eight epilogue warps of each block
        }
        for (int q = 0; q < 4; ++q) mbar_init(halves0 + 8 * q, 2);      // the two warps that share rows
        mbar_init(ended, 1);
        mbar_init(lap_free, 8);                   // the four of each whose columns lie in both accumulators
        give_up[0] = aligned ? 0 : 1;
        give_up[1] = 0;
        give_up[2] = tc::g_stall_code;
        if (!aligned) atomicCAS(&g_fp8_gemm_error, 0, 13);
        mbar_init_fence();
    }
    if (warp == 1) tmem_alloc_pair(smem_u32(tmem_slot), TMEM_COLS);
    fence_before_sync();
    cluster_sync_all();
    fence_after_sync();
    const uint32_t tmem = *tmem_slot;

    // what an item is: its tile, and -1 or which half of its columns
    auto find = [&](int item, int whole, int& mt, int& nt, int& half_of, int& group, int& row0) {
        const int tile = item < whole ? item : whole + (item - whole) / 2;
        half_of = item < whole ? -1 : (item - whole) & 1;
        if (!EXPERTS) {
            nt = tile / g.m_tiles;
            mt = tile - nt * g.m_tiles;
            group = 0;
            row0 = mt * PM;
            return;
        }
        mt = tile / g.n_tiles;
        nt = tile - mt * g.n_tiles;
        group = __ldcg(&g.tile_group[mt]);               // (perhaps read before this kernel's wait)
        row0 = __ldcg(&g.tile_row0[mt]);
    };
    // (experts: how many tiles of rows there are stands behind the list's first rows)
    auto tiles_of = [&]() { return (EXPERTS ? __ldcg(&g.offsets[g.experts + 1]) : g.m_tiles) * g.n_tiles; };

    // a stage's part of W and its scales; all of the stage's bytes, of both blocks, are counted here
    auto load_w = [&](int s, int kb, int w_row, int each) {
        const uint32_t full = full0 + 8 * s, s_dst = scale0 + s * SCALES;
        const bool with_scales = (kb & 3) == 0;
        if (rank == 0) mbar_expect_tx(full, 2 * (STAGE_BYTES + (with_scales ? SCALES : 0)));
        tma_load_pair(stage0 + s * STAGE_BYTES + A_BYTES, &map_w, kb * BK, w_row + (int)rank * each, full);
        if (with_scales) {
            const int ws_row = w_row >> 7, q = kb >> 2;
            tma_load_pair(s_dst + SF_TILE, &map_ws, 0, ws_row * g.quads + q, full);
            tma_load_pair(s_dst + 2 * SF_TILE, &map_ws, 0, (ws_row + 1) * g.quads + q, full);
        }
    };
    if (warp < FIRST) {
    // 128 x 56 + 256 x 224 = 384 x 168, what a block is launched with
    asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
    if (warp == 0) {
        if (elect_one()) {
            int it = 0, s = 0, phase = 0;
            bool ok = !*give_up;
            // Launched with programmatic stream serialization: nothing of this kernel touches memory before its first
            // operands have arrived, so (but for the experts' lists) the loader's wait is the kernel's.  W depends on no
            // kernel, once it is not new: the first stages' part of it is asked for before (experts': where their list is
            // known by then).
            int early = 0;
            if (g.listed && ok) {
                int whole, mt, nt, half_of, group, row0;
                if (pair < items_of(tiles_of(), whole)) {
                    find(pair, whole, mt, nt, half_of, group, row0);
                    early = min(STAGES, g.nkb);
                    for (int kb = 0; kb < early; ++kb) load_w(kb, kb, group * g.group_rows + nt * BN + (half_of > 0 ? BN / 2 : 0), half_of < 0 ? HN : HN / 2);
                }
            }
            pdl_wait();
            int mt, nt, half_of, group, row0, whole;
            const int total = items_of(tiles_of(), whole);
            for (int item = pair; item < total && ok; item += n_pairs) {
                find(item, whole, mt, nt, half_of, group, row0);
                // half the columns: a block of the pair needs 64 rows of W (it is brought 128), the scales are one tile
                const int w_row = group * g.group_rows + nt * BN + (half_of > 0 ? BN / 2 : 0), each = half_of < 0 ? HN : HN / 2;
                const int xs_row = (EXPERTS ? mt * (PM / 128) : row0 >> 7) + (int)rank;
                for (int kb = 0; kb < g.nkb; ++kb, ++it) {
                    if (!(kb > 0 ? wait_one(empty0 + 8 * s, phase ^ 1, give_up, 1) : wait_on(empty0 + 8 * s, phase ^ 1, give_up, 1))) { ok = false; break; }
                    const uint32_t full = full0 + 8 * s;
                    if (it >= early) load_w(s, kb, w_row, each);
                    tma_load_pair(stage0 + s * STAGE_BYTES, &map_x, kb * BK, row0 + (int)rank * BM, full);
                    if ((kb & 3) == 0) tma_load_pair(scale0 + s * SCALES, &map_xs, 0, xs_row * g.quads + (kb >> 2), full);
                    if (++s == STAGES) { s = 0; phase ^= 1; }
                }
            }
            pdl_trigger();                                  // the operands are asked for: the next kernel may move in
            if (*give_up && rank == 0) {
                // (a stage that has its part of W alone is never full: the wait for it is as long as the limit)
                for (int asked = max(it, early), j = max(0, asked - STAGES); j < asked; ++j)
                    drain_on(full0 + 8 * (j % STAGES), (j / STAGES) & 1, give_up, 4);
            }
        }
    } else if (warp == 1) {
        if (rank == 0 && elect_one()) {
            int s = 0, phase = 0, local = 0, set = 0;
            bool ok = !*give_up;
            if (EXPERTS) pdl_wait();
            int whole;
            const int total = items_of(tiles_of(), whole);
            for (int item = pair; item < total && ok; item += n_pairs) {
                const uint32_t id = idesc_mx(PM, item < whole ? BN : BN / 2);
                uint32_t sfw = 0, sfx = 0;
                for (int lo = 0; lo < g.nkb && ok; lo += g.piece, ++local) {
                    const int as = local & 1, hi = min(g.nkb, lo + g.piece);
                    // The wait that ends last is the one for the columns that this piece's accumulator shares with the piece
                    // before; all else that the first block needs comes ahead of it (2,048 x 9,216 x 2,304 gated 80.9 -> 78.8 us).
                    ok = wait_on(acc_free0 + 8 * as, ((local >> 1) & 1) ^ 1, give_up, 5);
                    if (!ok) break;
                    const uint32_t acc = tmem + as * ACC1;
                    for (int kb = lo; kb < hi; ++kb) {
                        // (the flags are looked at where a piece begins and where the stage is not there yet)
                        ok = kb > lo ? wait_one(full0 + 8 * s, phase, give_up, 2) : wait_on(full0 + 8 * s, phase, give_up, 2);
                        if (!ok) break;
                        fence_after_sync();
                        if ((kb & 3) == 0) {
                            sfw = tmem + SF_COL + 16 * set;
                            sfx = sfw + 8;
                            set ^= 1;
                            const uint32_t src = scale0 + s * SCALES;
                            scales_to_tmem_pair(sfx, desc_scales(src));
                            scales_to_tmem_pair(sfw, desc_scales(src + SF_TILE));
                            scales_to_tmem_pair(sfw + 4, desc_scales(src + 2 * SF_TILE));
                        }
                        if (kb == lo) {
                            ok = wait_on(lap_free, (local & 1) ^ 1, give_up, 6);
                            if (!ok) break;
                            fence_after_sync();
                        }
                        const uint32_t idk = with_block(id, kb & 3, kb & 3);
                        const uint64_t a = desc_kmajor(stage0 + s * STAGE_BYTES), b = desc_kmajor(stage0 + s * STAGE_BYTES + A_BYTES);
#pragma unroll
                        for (int k = 0; k < BK / 32; ++k) umma_mx_pair(acc, a + 2 * k, b + 2 * k, idk, sfx, sfw, (kb > lo) | (k > 0));
                        umma_commit_pair(empty0 + 8 * s);
                        if (++s == STAGES) { s = 0; phase ^= 1; }
                    }
                    if (ok) umma_commit_pair(acc_full0 + 8 * as);
                }
            }
            if (!ok) {                                      // products in flight end before their operands go
                umma_commit_pair(ended);
                drain_on(ended, 0, give_up, 8);
            }
        }
    }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 224;");
        const int quarter = warp & 3, half = (warp - FIRST) >> 2;
        uint8_t* room = rooms + (warp - FIRST) * 4096;
        int local = 0;
        if (EXPERTS) pdl_wait();
        int whole;
        bool ok = true;
        const int total = items_of(tiles_of(), whole);
        // An expert's item is known by three loads one after the other (its tile's first row and expert, that expert's end, this
        // row's pair): each is asked for while an item before is at work, or they cost as much as the item's results.
        struct Item { int mt, nt, half_of, group, row0; };
        Item now, next;
        auto look = [&](int item, Item& t) { if (item < total) find(item, whole, t.mt, t.nt, t.half_of, t.group, t.row0); };
        auto end_of = [&](int item, const Item& t) { return item < total ? (EXPERTS ? g.offsets[t.group + 1] : g.M) : 0; };
        auto pair_of = [&](int item, const Item& t, int end) {
            const int row = t.row0 + (int)rank * BM + quarter * 32 + lane;
            return EXPERTS && item < total && row < end && (g.down || g.scale) ? g.perm[row] : 0;
        };
        look(pair, now);
        look(pair + n_pairs, next);
        int end = end_of(pair, now), p = pair_of(pair, now, end);
        for (int item = pair; item < total && ok; item += n_pairs) {
            const int mt = now.mt, nt = now.nt, half_of = now.half_of;
            const int first = now.row0 + (int)rank * BM + quarter * 32;         // the warp's first row
            // how many of its rows there are (more than 32: all); none where half the columns are the other half's warps'
            const int rows = half_of >= 0 && half ? 0 : end - first;
            int at = first + lane;
            float mul = 1.0f;
            if (EXPERTS) {
                if (g.down) {
                    const int tok = p / g.top;
                    at = (p - tok * g.top) * g.tokens + tok;
                }
                if (g.scale && lane < rows) mul = g.scale[p];
            }
            const int next_end = end_of(item + n_pairs, next);
            constexpr int W = EPI == EPI_GATED ? 64 : 128;      // this thread's results
            const int col = nt * OUT_COLS + (half_of > 0 || half ? W : 0);
            // results of `unit` bytes from the thread's result c on, staged as ROW bytes a row
            auto flush = [&](auto row_bytes, int c, int unit, bool wide) {
                constexpr int ROW = decltype(row_bytes)::value;
                uint8_t* dst = (uint8_t*)g.y + (EXPERTS ? 0 : first * (g.ldy * unit)) + (long)(col + c) * unit;
                flush_rows<ROW, EXPERTS>(room, lane, dst, g.ldy * unit, at, rows, (OUT == OUT_FP8 ? (int)g.ldy - col - c : (g.N - col - c) * unit), wide, unit);
            };
            float sum[OUT == OUT_BF16 ? 1 : W == 64 && OUT == OUT_FP8 ? 64 : 128];      // OUT_F32: the pieces' sum; OUT_FP8: the row's results
            uint4 packed[8];                                    // OUT_BF16: 64 results on their way out
            for (int lo = 0; lo < g.nkb; lo += g.piece, ++local) {
                const int as = local & 1;
                const bool ready = wait_on(acc_full0 + 8 * as, (local >> 1) & 1, give_up, 3);
                if (!__all_sync(0xffffffffu, ready)) { ok = false; break; }
                fence_after_sync();
                if (lo == 0) {
                    p = pair_of(item + n_pairs, next, next_end);
                    now = next;
                    end = next_end;
                    look(item + 2 * n_pairs, next);
                }
                const uint32_t acc = tmem + as * ACC1 + half * 128 + ((uint32_t)(quarter * 32) << 16);
                // the first 32 columns read are those that the other accumulator wants
                auto there = [&](int turn) {
                    if (turn != 3 && (turn != 0 || half == as)) return;
                    fence_before_sync();
                    __syncwarp();
                    if (lane == 0) arrive_first_block(turn == 0 ? lap_free : acc_free0 + 8 * as);
                };
                auto use = [&](auto part, uint32_t (&v)[32]) {
                    constexpr int P = decltype(part)::value;
                    if constexpr (OUT == OUT_F32) {
#pragma unroll
                        for (int i = 0; i < 32; ++i) sum[P * 32 + i] = lo == 0 ? __uint_as_float(v[i]) : sum[P * 32 + i] + __uint_as_float(v[i]);
                    } else {
                        float o[32];
#pragma unroll
                        for (int i = 0; i < 32; ++i) o[i] = EXPERTS ? __uint_as_float(v[i]) * mul : __uint_as_float(v[i]);
                        if constexpr (EPI == EPI_GATED) {
                            gate_pairs<32>(o, g.act, g.limit);
                        } else if (g.act == ACT_RELU2) {
#pragma unroll
                            for (int i = 0; i < 32; ++i) o[i] = act_of(o[i], ACT_RELU2);
                        }
                        constexpr int R = EPI == EPI_GATED ? 16 : 32;
                        if constexpr (OUT == OUT_FP8) {
#pragma unroll
                            for (int i = 0; i < R; ++i) sum[P * R + i] = o[i];
                        } else {
                            constexpr int S = EPI == EPI_GATED ? P * 2 : P % 2 * 4;
#pragma unroll
                            for (int i = 0; i < R / 8; ++i) packed[S + i] = pack_bf16(o + 8 * i);
                        }
                    }
                    // plain results in bfloat16 go out 32 at a time where they are read back to front, else 64
                    if constexpr (OUT == OUT_BF16 && EPI == EPI_STORE) {
                        if (P % 2 == 1 || as == 0) {
                            if (as == 0) {
#pragma unroll
                                for (int i = 0; i < 4; ++i) stage16(room, lane, i, packed[P % 2 * 4 + i]);
                                flush(std::integral_constant<int, 64>{}, P * 32, 2, g.y_wide);
                            } else {
#pragma unroll
                                for (int i = 0; i < 8; ++i) stage16(room, lane, i, packed[i]);
                                flush(std::integral_constant<int, 128>{}, P * 32 - 32, 2, g.y_wide);
                            }
                        }
                    }
                };
                uint32_t u[32], v[32];
                if (as == 0) {
                    tmem_ld32(acc + 96, u);
                    walk<1, 0>(acc, u, v, there, use);
                } else {
                    tmem_ld32(acc, u);
                    walk<0, 0>(acc, u, v, there, use);
                }
            }
            if (!ok) break;
            if constexpr (OUT == OUT_BF16 && EPI == EPI_GATED) {
#pragma unroll
                for (int i = 0; i < 8; ++i) stage16(room, lane, i, packed[i]);
                flush(std::integral_constant<int, 128>{}, 0, 2, g.y_wide);
            }
            if constexpr (OUT == OUT_F32) {
#pragma unroll
                for (int c = 0; c < 128; c += 32) {
                    float o[32];
#pragma unroll
                    for (int i = 0; i < 32; ++i) o[i] = EXPERTS ? sum[c + i] * mul : sum[c + i];
                    if constexpr (EPI == EPI_GATED) {
                        gate_pairs<32>(o, g.act, g.limit);
                    } else if (g.act == ACT_RELU2) {
#pragma unroll
                        for (int i = 0; i < 32; ++i) o[i] = act_of(o[i], ACT_RELU2);
                    }
                    constexpr int R = EPI == EPI_GATED ? 16 : 32;
#pragma unroll
                    for (int i = 0; i < R / 4; ++i)
                        stage16(room, lane, i, make_uint4(__float_as_uint(o[4 * i]), __float_as_uint(o[4 * i + 1]), __float_as_uint(o[4 * i + 2]), __float_as_uint(o[4 * i + 3])));
                    flush(std::integral_constant<int, 4 * R>{}, c * R / 32, 4, g.y_wide);
                }
            }
            if constexpr (OUT == OUT_FP8) {
                uint32_t most = 0;
#pragma unroll
                for (int i = 0; i < W; ++i) {
                    if (col + i >= g.N) sum[i] = 0.0f;          // columns of no output are no part of the block
                    most = max(most, __float_as_uint(sum[i]) & 0x7fffffffu);
                }
                if constexpr (EPI == EPI_GATED) {               // the block's other half is another warp's
                    // (two rooms in turn; a wait with a limit like all others: the other warp may have given up)
                    uint32_t* here = most_of + (local & 1) * 256 + quarter * 32 + lane;
                    here[half * 128] = most;
                    __syncwarp();
                    if (lane == 0) mbar_arrive(halves0 + 8 * quarter);
                    const bool both = wait_on(halves0 + 8 * quarter, (local & 1) ^ 1, give_up, 7);
                    if (!__all_sync(0xffffffffu, both)) { ok = false; break; }
                    most = max(most, here[(half ^ 1) * 128]);
                }
                const uint32_t byte = scale_byte(most);
                const float inv = byte == 255u ? 1.0f : scale_inverse(byte);
#pragma unroll
                for (int i = 0; i < W; i += 16) {
                    uint4 q = make_uint4(NAN4, NAN4, NAN4, NAN4);
                    if (byte != 255u)
                        q = make_uint4(pack4(sum[i], sum[i + 1], sum[i + 2], sum[i + 3], inv), pack4(sum[i + 4], sum[i + 5], sum[i + 6], sum[i + 7], inv),
                                       pack4(sum[i + 8], sum[i + 9], sum[i + 10], sum[i + 11], inv), pack4(sum[i + 12], sum[i + 13], sum[i + 14], sum[i + 15], inv));
                    stage16(room, lane, i / 16, q);
                }
                // (a row's bytes are a multiple of 16)
                flush(std::integral_constant<int, W>{}, 0, 1, true);
                if (lane < rows && col < g.N && (EPI != EPI_GATED || half == 0)) {
                    const int b = col >> 7;
                    // scales by the row's tile: rows of the matrix (dense), rows of the list's tile (experts)
                    const long s_row = EXPERTS ? (long)mt * PM + rank * BM + quarter * 32 + lane : first + lane;
                    g.y_scales[scale_at(s_row, b >> 2, g.y_quads) + (b & 3)] = (uint8_t)byte;
                }
            }
        }
    }
    fence_before_sync();
    __syncwarp();
    cluster_sync_all();                 // neither block frees memory the other may still signal
    if (warp == 1) tmem_dealloc_pair(tmem, TMEM_COLS);
}

constexpr size_t SMEM_BYTES = (size_t)STAGES * (STAGE_BYTES + SCALES) + ROOM_BYTES + (2 * STAGES + 10) * 8 + 16 + ROWS_BYTES;

// a matrix of scale tiles: rows of 512 bytes
int make_map_scales(CUtensorMap* map, const void* ptr, long long tiles) {
    EncodeTiled enc = encoder();
    if (!enc) return BROLM_ERR_BAD_SIZE;
    const cuuint64_t dims[2] = {128, (cuuint64_t)tiles}, strides[1] = {SF_TILE};
    const cuuint32_t box[2] = {128, 1}, elem[2] = {1, 1};
    const CUresult r = enc(map, CU_TENSOR_MAP_DATA_TYPE_INT32, 2, const_cast<void*>(ptr), dims, strides, box, elem,
                           CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
                           CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? BROLM_OK : BROLM_ERR_ALIGNMENT;
}

struct Maps { CUtensorMap x, w, xs, ws; };

template <int EPI, int OUT, bool EXPERTS>
int launch(const Maps& m, const GemmArgs& g, cudaStream_t stream) {
    static OncePerDevice done;
    const int st = allow_shared_memory(fp8_gemm_kernel<EPI, OUT, EXPERTS>, SMEM_BYTES, done);
    if (st) return st;
    const int most = device_sms() / 2;
    int pairs = g.m_tiles * g.n_tiles;
    if (!(OUT == OUT_FP8 && EPI == EPI_GATED) && 2LL * pairs <= most) pairs *= 2;       // all tiles in halves
    if (pairs > most) pairs = most;
    return launch_pdl(fp8_gemm_kernel<EPI, OUT, EXPERTS>, dim3(2 * pairs), dim3(THREADS), SMEM_BYTES, stream, m.x, m.w, m.xs, m.ws, g);
}
template <bool EXPERTS>
int dispatch(const Maps& m, const GemmArgs& g, int epilogue, int out, cudaStream_t stream) {
    if (epilogue == EPI_GATED) {
        if (out == OUT_BF16) return launch<EPI_GATED, OUT_BF16, EXPERTS>(m, g, stream);
        if (out == OUT_F32) return launch<EPI_GATED, OUT_F32, EXPERTS>(m, g, stream);
        return launch<EPI_GATED, OUT_FP8, EXPERTS>(m, g, stream);
    }
    if (out == OUT_BF16) return launch<EPI_STORE, OUT_BF16, EXPERTS>(m, g, stream);
    if (out == OUT_F32) return launch<EPI_STORE, OUT_F32, EXPERTS>(m, g, stream);
    return launch<EPI_STORE, OUT_FP8, EXPERTS>(m, g, stream);
}

}  // namespace

// As brolm_fp8_stream, for any M and, for experts, tiles of 256 rows: x_scales then has two tiles of 128 rows for every tile of the
// list.  out 1: float, summed in pieces of `cut` blocks of K; 2: 8 bits (ldy bytes between rows, a multiple of 16; for experts
// scales as x_scales has them).
BROLM_API int brolm_fp8_gemm(const fp8::ProductCall* c) {
    const int M = c->M, N = c->N, K = c->K;
    if (M <= 0 || N <= 0) return BROLM_OK;
    if (K <= 0 || c->ldx % 16 || c->ldw % 16 || (((uintptr_t)c->x | (uintptr_t)c->w | (uintptr_t)c->x_scales | (uintptr_t)c->w_scales) & 15)) return BROLM_ERR_ALIGNMENT;
    if (c->out == OUT_FP8 && (c->ldy % 16 || c->ldy < N || !c->y_scales || ((uintptr_t)c->y & 15))) return BROLM_ERR_ALIGNMENT;
    if (c->epilogue < 0 || c->epilogue > 1 || c->out < 0 || c->out > 2 || c->act < 0 || c->act > 2 || (c->epilogue == EPI_STORE && c->act > ACT_RELU2)) return BROLM_ERR_BAD_SIZE;
    const long long w_rows = c->epilogue == EPI_GATED ? 2LL * N : N;
    const long long all = c->experts ? (long long)c->experts * c->group_rows : w_rows;
    Maps m;
    GemmArgs g = {};
    g.quads = quads_of(K);
    const long long m_tiles = c->experts ? c->max_tiles : ((long long)M + PM - 1) / PM;
    const int out_cols = c->epilogue == EPI_GATED ? BN / 2 : BN;
    const long long n_tiles = ((long long)N + out_cols - 1) / out_cols;
    if (all > 0x7fffffff - BN || m_tiles * n_tiles > 0x7fffffff - 1024) return BROLM_ERR_TOO_LARGE;
    if (c->experts && (c->group_rows % 128 || (c->down && c->out != OUT_F32))) return BROLM_ERR_BAD_SIZE;
    int st = make_map_u8(&m.x, c->x, M, K, c->ldx, BM);
    if (!st) st = make_map_u8(&m.w, c->w, all, K, c->ldw, HN);
    if (!st) st = make_map_scales(&m.xs, c->x_scales, (c->experts ? 2 * m_tiles : ((long long)M + 127) / 128) * g.quads);
    if (!st) st = make_map_scales(&m.ws, c->w_scales, (all + 127) / 128 * g.quads);
    if (st) return st;
    g.y = c->y; g.ldy = (long)c->ldy; g.y_scales = (uint8_t*)c->y_scales; g.y_quads = quads_of(N);
    g.y_wide = ((uintptr_t)c->y & 15) == 0 && c->ldy % (c->out == OUT_F32 ? 4 : 8) == 0;
    g.M = M; g.N = N; g.act = c->act; g.limit = c->limit; g.nkb = blocks_of(K);
    g.piece = c->out == OUT_F32 && c->cut > 0 && c->cut < g.nkb ? c->cut : g.nkb;
    g.m_tiles = (int)m_tiles; g.n_tiles = (int)n_tiles;
    if (!c->experts) {
        g.listed = !c->fresh;
        st = round_first(c);
        return st ? st : dispatch<false>(m, g, c->epilogue, c->out, c->stream);
    }
    g.tile_group = (const int32_t*)c->tile_group; g.tile_row0 = (const int32_t*)c->tile_row0; g.offsets = (const int32_t*)c->offsets;
    g.perm = (const int32_t*)c->perm; g.scale = (const float*)c->scale;
    g.down = c->down; g.top = c->top; g.tokens = c->tokens; g.group_rows = c->group_rows; g.experts = c->experts; g.listed = c->listed;
    return dispatch<true>(m, g, c->epilogue, c->out, c->stream);
}

BROLM_API int brolm_fp8_gemm_status(int reset) {
    int v = 0;
    if (cudaMemcpyFromSymbol(&v, g_fp8_gemm_error, sizeof(int)) != cudaSuccess) return -1;
    if (reset && v) {
        const int zero = 0;
        cudaMemcpyToSymbol(g_fp8_gemm_error, &zero, sizeof(int));
    }
    return v;
}

BROLM_WAIT_CONTROL(fp8_gemm)
