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
// The tensor core cuts off where an fma rounds, so the sums of long slices drift (all terms positive, 18,432 along K: 1.1e-5 of the
// result).  Float results of more than `piece` blocks of K are summed in pieces of that many, which the epilogue adds in registers, as
// in tiles (PIECES; kernels of their own, for the registers): 1.3e-6.  Results in fewer bits are one piece.
//
// Dense: X has up to 128 rows.  Where W has fewer tiles of 128 rows than the device has SMs, K is cut into slices that are the
// blocks of a cluster; their float sums are added in the order of the slices through the cluster's shared memory.
// Experts: a list made on the device names for every tile of rows of X the expert whose matrix it meets, its first row and
// so its last one; an item of work is one such tile and 128 rows of its expert's matrix.
//
// Epilogues: store (float or bfloat16; with the square of relu), or a gated activation of neighbouring rows of W, row 2 j being
// the gate of output j and row 2 j + 1 its partner: the two lie in neighbouring lanes.  Or (K in one piece) 8 bits, as rows for
// the next product: a block of 128 results of a row is a tile of W, gated two of them, which the two blocks of a cluster make
// side by side; they tell one another the rows' largest magnitudes.
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
constexpr int FUSED_BLOCKS = 16;       // 32 KB of the rows, four stages beside them (six where no more than half of the SMs get a block)

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
    uint8_t* y_scales;       // (ROUND)
    int y_quads, last;       // last: the last tile of W, of which row_tiles counts pairs where two blocks are a team
    int per;                 // blocks of K of a slice (dense; the cluster's rank is the slice)
    int piece;               // (PIECES) blocks of K that go into an accumulator
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
    int listed;              // what names W is there, and W itself, before this kernel's wait
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
__device__ __forceinline__ void peer_store(const uint32_t* p, uint32_t rank, uint32_t v) {
    asm volatile("{\n.reg .b32 r;\nmapa.shared::cluster.u32 r, %0, %1;\nst.shared::cluster.b32 [r], %2;\n}"
                 ::"r"(smem_u32(p)), "r"(rank), "r"(v) : "memory");
}
// The largest of four warps' words for a row, which they leave in this block's shared memory with the highest bit telling that they
// are there; bounded as all waits are (code 7).  No fence goes with them: the words are all there is to read.
__device__ __forceinline__ bool words_wait(const uint32_t* p, uint32_t tag, uint32_t& most, volatile int* give_up) {
    volatile const uint32_t* w = p;
    const bool stalled = give_up[2] == 7;
    long long t0 = 0;
    for (uint32_t turn = 1;; ++turn) {
        const uint32_t a = w[0], b = w[32], c = w[64], d = w[96];
        most = max(max(a, b), max(c, d)) & 0x7fffffffu;
        if (!stalled && (tag ? a & b & c & d : ~(a | b | c | d)) >> 31) return true;
        if (*give_up) return false;
        if (turn % 1024) continue;                          // (some 30 us; the limit lies in memory, a miss is a microsecond)
        if (!t0) t0 = clock64();
        if (clock64() - t0 > (stalled ? g_wait_cycles / 4 : g_wait_cycles)) {
            *give_up = 1;
            atomicCAS(&g_fp8_stream_error, 0, 7);
            return false;
        }
    }
}
__device__ __forceinline__ void peer_arrive(uint32_t bar, uint32_t rank) {
    asm volatile("{\n.reg .b32 r;\nmapa.shared::cluster.u32 r, %0, %1;\nmbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [r];\n}"
                 ::"r"(bar), "r"(rank) : "memory");
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

constexpr int MOST = 2 * 8 * 32;         // rows' largest magnitudes: two rooms in turn, eight warps, 32 rows

// FUSED: 0 the rows are 8-bit numbers in memory; 1, 2: they are bfloat16, float numbers, and every block rounds what it needs.
// ROUND: results are 8-bit rows (a kernel of its own: as a branch it cost the others 0.4 to 0.8 us a launch).
// PIECES: a float result of many blocks of K is summed in pieces, which the epilogue adds: no slower (64 rows 18,432 x 18,432 61.1 us
// for 61.4, 100 rows 4,608 x 36,864 in slices of 42 blocks 34.4 for 34.9) as long as its code is short: with each of a thread's sums
// stored by the other forms' code 100 rows took 94 us for 68.
template <int BT, int FUSED, bool PIECES>
struct Shape {
    // warps with an epilogue: 128 sums a thread are more registers than two blocks an SM leave it, so there eight warps have 64 each
    static constexpr int LEAVING = PIECES && BT == 128 ? 8 : 4;
    static constexpr int THREADS = FUSED || LEAVING == 8 ? 320 : 192;   // (FUSED: eight warps that round, of which four have an epilogue)
    static constexpr int X_BYTES = BT * BK;
    static constexpr int STAGE_BYTES = FUSED ? W_BYTES : W_BYTES + X_BYTES;      // multiples of 1024
    // accumulators and two pairs of scales in at most half of tensor memory, so that an SM holds two blocks
    static constexpr int ACCS = BT == 128 ? 1 : 2;
    static constexpr int COLS = ACCS * BT + 16;
    static constexpr int TMEM_COLS = COLS <= 64 ? 64 : COLS <= 128 ? 128 : 256;
    static constexpr int SCALES = FUSED ? SF_TILE : 2 * SF_TILE;        // of a stage
    static size_t x_room(int per) { return FUSED ? (size_t)per * X_BYTES + (size_t)((per + 3) / 4 + 1) * SF_TILE : 0; }
    static size_t smem(int stages, int per) {
        return x_room(per) + (size_t)stages * (STAGE_BYTES + SCALES) + (2 * MAX_STAGES + 8) * 8 + 16 + MOST * 4;
    }
};

// Two numbers of a lane become one: of numbers i and i + HALF the lanes without bit `BIT` keep the first, the others the second,
// each with the other lane's in it.
template <int HALF>
__device__ __forceinline__ void fold(uint32_t* m, int lane, int bit) {
#pragma unroll
    for (int i = 0; i < HALF; ++i) {
        const bool up = lane & bit;
        const uint32_t got = __shfl_xor_sync(0xffffffffu, up ? m[i] : m[i + HALF], bit);
        m[i] = max(up ? m[i + HALF] : m[i], got);
    }
}

// An accumulator's results as rows of 8-bit numbers: 16 or 32 rows of X at a time, since each time costs a wait for the other
// warps of the block of 128 results (a microsecond at the end of a launch).  False: that wait ran out.  A launch less: a feed-forward
// of 8 rows, 2,304 and 9,216, 24.0 -> 21.0 us, 64 rows 23.8 -> 22.5; 8 tokens, 4 of 32 experts, 41.2 -> 38.9, 64 tokens 50.3 -> 46.9.
template <int EPI, bool EXPERTS, int BT>
__device__ __forceinline__ bool rounded_results(const StreamArgs& g, uint32_t acc, uint32_t acc_empty, int rows, int row0, int tile, int rt, int side, int quarter,
                                                int lane, uint32_t* most_of, uint32_t joined, int& turn, volatile int* give_up) {
    constexpr int ROWS = BT < 32 ? BT : 32, LANES = EPI == EPI_GATED ? 2 : 1, V = ROWS / LANES;      // gated: lanes with an odd number have the odd rows
    constexpr bool team = EPI == EPI_GATED;
    const int odd = EPI == EPI_GATED ? lane & 1 : 0;
    const int col = (rt * BR + quarter * 32 + lane) / LANES;
    for (int c = 0; c < rows; c += ROWS) {
        float o[V];
#pragma unroll
        for (int c16 = 0; c16 < ROWS; c16 += 16) {
            uint32_t v[16];
            tmem_ld16(acc + c + c16, v);
            tmem_wait_ld();
            float z[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) z[i] = __uint_as_float(v[i]);
            if (EXPERTS && g.scale) {
#pragma unroll
                for (int i = 0; i < 16; ++i) if (c + c16 + i < rows) z[i] *= g.scale[g.perm[row0 + c + c16 + i]];
            }
            if (EPI == EPI_GATED) {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float got = __shfl_xor_sync(0xffffffffu, odd ? z[2 * i] : z[2 * i + 1], 1);
                    o[c16 / 2 + i] = gate_of(odd ? got : z[2 * i], odd ? z[2 * i + 1] : got, g.act, g.limit);
                }
            } else {
#pragma unroll
                for (int i = 0; i < 16; ++i) o[c16 / LANES + i / LANES] = act_of(z[i], g.act);
            }
        }
        if (c + ROWS >= rows) {                                 // all of this accumulator that is wanted is in registers
            fence_before_sync();
            __syncwarp();
            if (lane == 0) mbar_arrive(acc_empty);
        }
        // a row's largest magnitude goes round the warp's columns (a lane is left with row `place`'s), then to all of the team's warps
        uint32_t m[V];
#pragma unroll
        for (int i = 0; i < V; ++i) {
            if (col >= g.N) o[i] = 0.0f;                        // columns of no output are no part of the block
            m[i] = __float_as_uint(o[i]) & 0x7fffffffu;
        }
        int place = odd;
        if constexpr (V == 32) { fold<16>(m, lane, 16); fold<8>(m, lane, 8); fold<4>(m, lane, 4); fold<2>(m, lane, 2); fold<1>(m, lane, 1); place = lane; }
        if constexpr (V == 16) { fold<8>(m, lane, 16); fold<4>(m, lane, 8); fold<2>(m, lane, 4); fold<1>(m, lane, 2); place += (lane >> 1) * LANES; }
        if constexpr (V == 8) { fold<4>(m, lane, 16); fold<2>(m, lane, 8); fold<1>(m, lane, 4); place += (lane >> 2) * LANES; }
        if constexpr (V < 32) {
            constexpr int ANY = V == 8 ? 2 : LANES == 1 ? 1 : 0;          // the lanes that have the same row
            if constexpr (ANY > 0) m[0] = max(m[0], __shfl_xor_sync(0xffffffffu, m[0], ANY));
        }
        // (two rooms in turn: a warp writes into one again when it has read the other, and so has every warp left the first.  The
        // barrier is where the warps wait; its arrivals are ordered with nothing, for a fence across the cluster cost 0.5 to 1 us a
        // turn, and the words' tags tell what is there.  Polling the words alone kept the SM from its other work: 1 to 2 us.)
        uint32_t* room = most_of + (turn & 1) * (MOST / 2);
        uint32_t* mine = room + (side * 4 + quarter) * 32 + place;
        const uint32_t tag = (turn >> 1 & 1) ^ 1, word = m[0] | tag << 31;
        *(volatile uint32_t*)mine = word;                       // (lanes of the same row: the same number)
        if (team) peer_store(mine, side ^ 1, word);
        __syncwarp();
        if (lane == 0) {
            mbar_arrive(joined);
            if (team) peer_arrive(joined, side ^ 1);
        }
        if (!__all_sync(0xffffffffu, wait_on(joined, turn & 1, give_up, 7))) return false;
        ++turn;
        // lane l: of row l (16 rows: l % 16, half of the lanes for each of the team's sides)
        uint32_t most;
        bool there = words_wait(room + (ROWS == 16 ? (team ? lane >> 4 : 0) * 128 + (lane & 15) : lane), tag, most, give_up);
        if (ROWS == 32 && team) {
            uint32_t other;
            there = there && words_wait(room + 128 + lane, tag, other, give_up);
            most = max(most, other);
        }
        if (ROWS == 16) most = max(most, __shfl_xor_sync(0xffffffffu, most, 16));
        if (!__all_sync(0xffffffffu, there)) return false;
        const uint32_t byte = scale_byte(most);                 // of row c + lane
        if (quarter == 0 && side == 0 && lane < ROWS && c + lane < rows) {
            const int b = EPI == EPI_GATED ? rt >> 1 : rt;
            g.y_scales[scale_at((EXPERTS ? (long)tile * 128 : 0) + c + lane, b >> 2, g.y_quads) + (b & 3)] = (uint8_t)byte;
        }
        // four rows at a time: a lane's word is its column's numbers in them; four lanes exchange, and each has four columns of a row
        const int a = lane / LANES & 3;
#pragma unroll
        for (int i = 0; i < V; i += 4) {
            float u[4];
            uint32_t nan = 0;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint32_t s = __shfl_sync(0xffffffffu, byte, (i + j) * LANES + odd);
                u[j] = s == 255u ? 0.0f : o[i + j] * scale_inverse(s);
                if (s == 255u) nan |= (NAN4 & 255u) << (8 * j);
            }
            uint32_t q = pack4(u[0], u[1], u[2], u[3], 1.0f) | nan;
            uint32_t got = __shfl_xor_sync(0xffffffffu, q, LANES);
            q = __byte_perm(q, got, a & 1 ? 0x3715 : 0x6240);
            got = __shfl_xor_sync(0xffffffffu, q, 2 * LANES);
            q = __byte_perm(q, got, a & 2 ? 0x3276 : 0x5410);
            const int r = c + (i + a) * LANES + odd, at = col & ~3;
            if (r < rows && at < g.ldy) *reinterpret_cast<uint32_t*>((uint8_t*)g.y + (EXPERTS ? row0 + r : r) * g.ldy + at) = q;
        }
    }
    return true;
}

template <int BT, int EPI, bool EXPERTS, int FUSED, bool ROUND, bool PIECES>
__global__ void __launch_bounds__(Shape<BT, FUSED, PIECES>::THREADS, 2) fp8_stream_kernel(const __grid_constant__ CUtensorMap map_w,
                                                             const __grid_constant__ CUtensorMap map_x, StreamArgs g) {
    using S = Shape<BT, FUSED, PIECES>;
    constexpr int ACCS = S::ACCS;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t* base = smem_raw;
    const int stages = g.stages;
    // the ring, (FUSED) the slice's rows in 8 bits, the scales of the ring, (FUSED) those of the rows, barriers
    uint8_t* x_blocks = base + stages * S::STAGE_BYTES;
    uint8_t* scale_slots = x_blocks + (FUSED ? g.per * S::X_BYTES : 0);
    uint8_t* x_scales = scale_slots + stages * S::SCALES;
    uint64_t* bars = reinterpret_cast<uint64_t*>(x_scales + (FUSED ? ((g.per + 3) / 4 + 1) * SF_TILE : 0));
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 2 * MAX_STAGES + 8);
    volatile int* give_up = reinterpret_cast<volatile int*>(tmem_slot + 1);
    uint32_t* most_of = tmem_slot + 4;                         // [2][8][32]
    // slices: this one's sums [rows of X][128], in the ring, which is read to its end by then
    float* sums = reinterpret_cast<float*>(base);
    const uint32_t stage0 = smem_u32(base), scale0 = smem_u32(scale_slots);
    const uint32_t full0 = smem_u32(bars), empty0 = full0 + 8 * MAX_STAGES, acc_full0 = empty0 + 8 * MAX_STAGES,
                   acc_empty0 = acc_full0 + 16, x_ready = acc_empty0 + 16, ended = x_ready + 8, joined = ended + 8;
    const bool aligned = (stage0 & 1023u) == 0;
    // the blocks of a cluster are the slices of K or the sides of a team
    constexpr bool team = ROUND && EPI == EPI_GATED;
    constexpr int TEAM = team ? 2 : 1;
    const int members = EXPERTS && !team ? 1 : (int)cluster_size(), member = EXPERTS && !team ? 0 : (int)cluster_rank();
    const int slices = EXPERTS || team ? 1 : members, slice = EXPERTS || team ? 0 : member, side = team ? member : 0;
    const int first = blockIdx.x / members, step = gridDim.x / members;
    const int lo = slice * g.per, hi = min(g.nkb, lo + g.per);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int s = 0; s < stages; ++s) {
            mbar_init(full0 + 8 * s, 1);
            mbar_init(empty0 + 8 * s, 1);
        }
        for (int s = 0; s < 2; ++s) {
            mbar_init(acc_full0 + 8 * s, 1);
            mbar_init(acc_empty0 + 8 * s, S::LEAVING);
        }
        mbar_init(x_ready, 8);
        mbar_init(ended, 1);
        if (ROUND) mbar_init(joined, 4 * TEAM);
        give_up[0] = aligned ? 0 : 1;
        give_up[1] = 0;
        give_up[2] = tc::g_stall_code;
        if (!aligned) {
            atomicCAS(&g_fp8_stream_error, 0, 13);
            pdl_wait();                                        // (no loader will: a block does not end ahead of the kernel before)
        }
        mbar_init_fence();
    }
    if (ROUND) for (int i = threadIdx.x; i < MOST; i += S::THREADS) most_of[i] = 0;
    if (warp == 1) tmem_alloc(smem_u32(tmem_slot), S::TMEM_COLS);
    fence_before_sync();
    __syncthreads();
    fence_after_sync();
    if (team) asm volatile("barrier.cluster.arrive.aligned;" ::: "memory");      // (waited for where the other block is first spoken to)
    const uint32_t tmem = *tmem_slot;

    // the tile of rows of X and the tile of rows of W of an item; false behind the experts' last tile
    auto find = [&](int item, int& rt, int& group, int& row0, int& tile) {
        if (!EXPERTS) {
            rt = item * TEAM + side; group = 0; row0 = 0; tile = 0;
            return true;
        }
        tile = item / g.row_tiles;
        rt = (item - tile * g.row_tiles) * TEAM + side;
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
                const int row = group * g.group_rows + min(rt, g.last) * BR;      // (a team's second tile may lie behind the last)
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
            // The ring fills with weights before the kernel before this one has ended, if they are not what it writes; experts'
            // where their list is known by then.
            const bool ahead = g.listed;
            // One thread's word stands for the block's, so none lets the next kernel move in that has not waited, as this one has:
            // what that kernel reads ahead of its own wait (an experts' list, a matrix that is not new) is there by then.  At once
            // for experts and few rows, else once the stream is asked for: experts of 8 tokens 38.5 -> 35.6 us, 8 rows in 8 bits on
            // 2,304 x 9,216 7.1 -> 6.3, a decode step of 8 sequences at the 2B sizes 1.460 -> 1.449 ms; but at once everywhere a
            // feed-forward of 32 rows takes 21.8 us for 21.2, the step of 32 sequences 2.11 ms for 2.085, 8 rows rounded here 8.5 us
            // for 8.1.
            constexpr bool AT_ONCE = EXPERTS || (BT == 16 && !ROUND && !FUSED);
            auto wait = [&]() {
                pdl_wait();
                if (AT_ONCE) pdl_trigger();
            };
            if (!ahead) wait();
            more = item < g.items && lo < hi && find(item, rt, group, row0, tile);
            if (ahead) {
                int n = 0;
                for (; n < stages && lo + n < hi && more; ++n) load_w(n, rt, group, lo + n);
                wait();
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
            if (!AT_ONCE) pdl_trigger();
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
            for (int item = first; item < g.items && lo < hi && ok; item += step) {
                if (!find(item, rt, group, row0, tile)) break;
                uint32_t sfw = 0, sfx = 0;
                for (int from = lo, to; from < hi && ok; from = to, ++local) {
                    to = PIECES ? min(hi, from + g.piece) : hi;
                    const int as = local % ACCS;
                    ok = wait_on(acc_empty0 + 8 * as, ((local / ACCS) & 1) ^ 1, give_up, 5);
                    if (FUSED && ok && local == 0) ok = wait_on(x_ready, 0, give_up, 6);
                    if (!ok) break;
                    fence_after_sync();
                    const uint32_t acc = tmem + as * BT;
                    for (int kb = from; kb < to; ++kb) {
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
                        for (int k = 0; k < BK / 32; ++k) umma_mx(acc, a + 2 * k, b + 2 * k, idk, sfw, sfx, (kb > from) | (k > 0));
                        umma_commit(empty0 + 8 * s);
                        if (++s == stages) { s = 0; phase ^= 1; }
                    }
                    if (ok) umma_commit(acc_full0 + 8 * as);
                }
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
            // (these four warps have waited, too, and have nothing else to do: the next kernel's stream begins sooner.  A product of
            // one row, 2,304 x 9,216, 7.9 -> 7.15 us, of eight 8.6 -> 8.1.)
            if (warp >= 6) pdl_trigger();
        }
        __syncwarp();
        if (team && warp < 6) asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
        int local = 0, turn = 0, rt, group, row0, tile;
        for (int item = first; item < g.items && lo < hi && warp < 2 + S::LEAVING; item += step) {
            if (!find(item, rt, group, row0, tile)) break;
            const int rows = EXPERTS ? min(BT, g.offsets[group + 1] - row0) : g.M;
            const int wide = (rows + 15) & ~15;
            // sixteen rows of X, from row c on, of this lane's row of W: the epilogue
            auto leave = [&](int c, float (&o)[16]) {
                if (slices > 1) {
#pragma unroll
                    for (int i = 0; i < 16; ++i) sums[(c + i) * BR + lrow] = o[i];
                    return;
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
                if (PIECES && !EXPERTS) {                       // (floats; short code, of which there are up to eight copies)
                    float* to = reinterpret_cast<float*>(g.y) + (c + first_row) * g.ldy + col;
                    const int left = col < g.N ? rows - c - first_row : 0;
#pragma unroll
                    for (int i = 0; i < (EPI == EPI_GATED ? 8 : 16); ++i, to += row_step * g.ldy) if (i * row_step < left) *to = o[i];
                } else if (col < g.N) {
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
            };
            constexpr int EACH = BT * 4 / S::LEAVING;           // rows of X of a warp (PIECES)
            const int c0 = S::LEAVING == 8 && warp >= 6 ? EACH : 0;
            float sum[PIECES ? EACH : 16];                      // PIECES: of the accumulators that have been, in their order
#pragma unroll
            for (int i = 0; i < (PIECES ? EACH : 0); ++i) sum[i] = 0.0f;
            bool there = true;
            for (int from = lo; from < hi; from = PIECES ? from + g.piece : hi, ++local) {
                const int as = local % ACCS;
                const bool ready = !*give_up && wait_on(acc_full0 + 8 * as, (local / ACCS) & 1, give_up, 3);
                there = __all_sync(0xffffffffu, ready);
                if (!there) break;
                fence_after_sync();
                const uint32_t acc = tmem + as * BT + ((uint32_t)(quarter * 32) << 16);
                if constexpr (ROUND) {
                    there = rounded_results<EPI, EXPERTS, BT>(g, acc, acc_empty0 + 8 * as, rows, row0, tile, rt, side, quarter, lane, most_of, joined, turn, give_up);
                    continue;
                }
                auto take = [&](int c, float* o) {
                    uint32_t v[16];
                    tmem_ld16(acc + c, v);
                    tmem_wait_ld();
#pragma unroll
                    for (int i = 0; i < 16; ++i) o[i] = PIECES ? o[i] + __uint_as_float(v[i]) : __uint_as_float(v[i]);
                };
                auto taken = [&]() {                            // all of this accumulator that is wanted is in registers
                    fence_before_sync();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(acc_empty0 + 8 * as);
                };
                if constexpr (PIECES) {
#pragma unroll
                    for (int c = 0; c < EACH; c += 16) if (c0 + c < wide) take(c0 + c, sum + c);
                    taken();
                } else {
                    for (int c = 0; c < wide; c += 16) {
                        take(c, sum);
                        if (c + 16 >= wide) taken();
                        leave(c, sum);
                    }
                }
            }
            if (!there) break;
            if constexpr (PIECES) {
#pragma unroll
                for (int c = 0; c < EACH; c += 16) {
                    float o[16];
#pragma unroll
                    for (int i = 0; i < 16; ++i) o[i] = sum[c + i];
                    if (c0 + c < wide) leave(c0 + c, o);
                }
            }
        }
    }
    fence_before_sync();
    if (team) {
        __syncwarp();
        if (warp < 2 || warp >= 6) asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
        cluster_sync_all();                                     // neither block leaves while the other may speak to it
    }
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

template <int BT, int EPI, bool EXPERTS, int FUSED, bool ROUND, bool PIECES>
int launch(const CUtensorMap& mw, const CUtensorMap& mx, StreamArgs g, int slices, cudaStream_t stream) {
    using S = Shape<BT, FUSED, PIECES>;
    const int sms = device_sms();
    const bool split = slices > 1;
    const int members = split ? slices : ROUND && EPI == EPI_GATED ? 2 : 1;
    // Two blocks an SM: one streams while the other starts or ends, and clusters of up to eight find room.  (Three with 74 KB,
    // where experts' items fill their rounds better, gained nothing.)  Where no more than half of the SMs get a block, its ring
    // is longer: a layer of 1,152 and 6,912 with 48 rows 25.2 -> 24.2 us.  (With more blocks the kernel behind
    // finds no room to begin beside them: 98 of 148 SMs 20.1 -> 21.7, all of them 26.9 -> 28.2.)
    constexpr size_t HALF = 112 * 1024, MORE = 150 * 1024;
    const int places = 2 * sms / members;
    const int grid = members * (split || g.items < places ? g.items : places);
    const size_t room = 2 * grid <= sms ? MORE : HALF;
    int stages = MAX_STAGES;
    while (stages > 2 && S::smem(stages, g.per) > room) --stages;
    const size_t smem = S::smem(stages, g.per);
    if (smem > room || (split && (size_t)stages * S::STAGE_BYTES < (size_t)BT * BR * 4)) return BROLM_ERR_TOO_LARGE;
    g.stages = stages;
    static OncePerDevice done;
    const int st = allow_shared_memory(fp8_stream_kernel<BT, EPI, EXPERTS, FUSED, ROUND, PIECES>, MORE, done);
    if (st) return st;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(S::THREADS);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = pdl_enabled() ? 1 : 0;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = members;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = EXPERTS && members == 1 ? 1 : 2;
    return (int)cudaLaunchKernelEx(&cfg, fp8_stream_kernel<BT, EPI, EXPERTS, FUSED, ROUND, PIECES>, mw, mx, g);
}

template <int EPI, bool EXPERTS, bool ROUND, bool PIECES>
int dispatch(const CUtensorMap& mw, const CUtensorMap& mx, const StreamArgs& g, int bt, int slices, int fused, cudaStream_t stream) {
    if constexpr (!EXPERTS && !PIECES) {
        if (fused == 1) return launch<16, EPI, false, 1, ROUND, false>(mw, mx, g, slices, stream);
        if (fused == 2) return launch<16, EPI, false, 2, ROUND, false>(mw, mx, g, slices, stream);
    }
    if (bt == 16) return launch<16, EPI, EXPERTS, 0, ROUND, PIECES>(mw, mx, g, slices, stream);
    if (bt == 32) return launch<32, EPI, EXPERTS, 0, ROUND, PIECES>(mw, mx, g, slices, stream);
    if constexpr (!EXPERTS) {
        if (bt == 64) return launch<64, EPI, false, 0, ROUND, PIECES>(mw, mx, g, slices, stream);
        if constexpr (!ROUND) return launch<128, EPI, false, 0, false, PIECES>(mw, mx, g, slices, stream);
    }
    return BROLM_ERR_BAD_SIZE;
}
template <int EPI, bool EXPERTS>
int dispatch(const CUtensorMap& mw, const CUtensorMap& mx, const StreamArgs& g, int bt, int slices, int fused, int out, cudaStream_t stream) {
    if (out == 2) return dispatch<EPI, EXPERTS, true, false>(mw, mx, g, bt, slices, fused, stream);
    if (out == 1 && g.piece > 0 && g.per > g.piece) return dispatch<EPI, EXPERTS, false, true>(mw, mx, g, bt, slices, fused, stream);
    return dispatch<EPI, EXPERTS, false, false>(mw, mx, g, bt, slices, fused, stream);
}
template <bool EXPERTS>
int dispatch(const CUtensorMap& mw, const CUtensorMap& mx, const StreamArgs& g, int bt, int slices, int fused, int epilogue, int out, cudaStream_t stream) {
    if (epilogue == EPI_GATED) return dispatch<EPI_GATED, EXPERTS>(mw, mx, g, bt, slices, fused, out, stream);
    return dispatch<EPI_STORE, EXPERTS>(mw, mx, g, bt, slices, fused, out, stream);
}

}  // namespace

// Y [M, N] = X W^T (epilogue 0, act 0 or the square of relu) or the gated activation of W's neighbouring rows (epilogue 1: W
// has 2 N rows); out 0: bfloat16, 1: float, summed in pieces of `piece` blocks of K (0: in one), 2 (cut 1, M <= 64): 8 bits, ldy bytes between rows, a multiple of 16, for experts scales as
// x_scales has them.  X and W as brolm_fp8_quantize leaves them.
// Dense (experts 0): M <= 128; K is cut into `cut` slices (1 to 8), none of which is empty.  fused 1, 2: X are bfloat16, float
// numbers (ldx elements between rows, x_scales unused), M <= 16, and a slice has at most FUSED_BLOCKS blocks of 128 of K.
// Experts: M pairs' rows in the order of their experts, W the experts' matrices, group_rows (a multiple of 128) rows each.  The
// list (expert, first row) of tiles of `rows` (16 or 32) rows and what it stands on come from brolm_fp8_experts; x_scales
// has a tile of 128 rows for every tile of the list.  Y [M, N], or with `down` float [top, tokens, N]; `scale` (or null): a
// number for every pair that multiplies its sums before the activation.
BROLM_API int brolm_fp8_stream(const fp8::ProductCall* c) {
    const int M = c->M, N = c->N, K = c->K;
    if (M <= 0 || N <= 0) return BROLM_OK;
    if (K <= 0 || c->ldw % 16 || (((uintptr_t)c->w | (uintptr_t)c->w_scales) & 15)) return BROLM_ERR_ALIGNMENT;
    if (!c->fused && (c->ldx % 16 || (((uintptr_t)c->x | (uintptr_t)c->x_scales) & 15))) return BROLM_ERR_ALIGNMENT;
    if (c->fused < 0 || c->fused > 2 || (c->fused && (M > 16 || c->experts))) return BROLM_ERR_BAD_SIZE;
    if (c->epilogue < 0 || c->epilogue > 1 || c->act < 0 || c->act > 2 || (c->epilogue == EPI_STORE && c->act > ACT_RELU2)) return BROLM_ERR_BAD_SIZE;
    if (c->out < 0 || c->out > 2 || (c->out == 2 && !c->experts && (c->cut != 1 || M > 64))) return BROLM_ERR_BAD_SIZE;
    if (c->out == 2 && (c->ldy % 16 || c->ldy < N || !c->y_scales || ((uintptr_t)c->y & 15))) return BROLM_ERR_ALIGNMENT;
    const long long w_rows = c->epilogue == EPI_GATED ? 2LL * N : N;
    StreamArgs g = {};
    g.y = c->y; g.ldy = (long)c->ldy; g.M = M; g.N = N; g.out_f32 = c->out == 1; g.act = c->act; g.limit = c->limit;
    g.y_wide = ((uintptr_t)c->y & 15) == 0 && c->ldy % 4 == 0;
    g.nkb = blocks_of(K); g.quads = quads_of(K); g.piece = c->fused ? 0 : c->piece;
    g.w_scales = (const uint8_t*)c->w_scales; g.x_scales = (const uint8_t*)c->x_scales;
    g.last = (int)((w_rows + BR - 1) / BR - 1);
    if (c->out == 2) { g.y_scales = (uint8_t*)c->y_scales; g.y_quads = quads_of(N); }
    const int team = c->out == 2 && c->epilogue == EPI_GATED ? 2 : 1;
    const long long row_tiles = (g.last + team) / team;          // a team's tiles of W count once
    CUtensorMap mw, mx;
    if (c->experts) {
        const int rows = c->rows;
        if (c->group_rows % BR || (rows != 16 && rows != 32) || (c->down && c->out != 1)) return BROLM_ERR_BAD_SIZE;
        const long long all = (long long)c->experts * c->group_rows;
        if (all > 0x7fffffff || c->max_tiles * row_tiles > 0x7fffffff - 65536) return BROLM_ERR_TOO_LARGE;
        int st = make_map_u8(&mw, c->w, all, K, c->ldw, BR);
        if (!st) st = make_map_u8(&mx, c->x, M, K, c->ldx, rows);
        if (st) return st;
        g.per = g.nkb; g.row_tiles = (int)row_tiles; g.items = (int)(row_tiles * c->max_tiles);
        g.tile_group = (const int32_t*)c->tile_group; g.tile_row0 = (const int32_t*)c->tile_row0; g.offsets = (const int32_t*)c->offsets;
        g.perm = (const int32_t*)c->perm; g.scale = (const float*)c->scale;
        g.down = c->down; g.top = c->top; g.tokens = c->tokens; g.group_rows = c->group_rows; g.listed = c->listed;
        return dispatch<true>(mw, mx, g, rows, 1, 0, c->epilogue, c->out, c->stream);
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
    g.listed = !c->fresh;
    st = round_first(c);
    if (st) return st;
    return dispatch<false>(mw, mx, g, bt, slices, c->fused, c->epilogue, c->out, c->stream);
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
