// Attention of many new tokens over the cache in 8 bits (kv8.cuh) on the 5th-generation tensor cores (tcgen05), bfloat16,
// sm_100a: pieces of prompts whose keys and values are in the cache already.
//
//     z = scale * q . k,   cap tanh(z / cap),   key j visible from position p iff 0 <= p - j < window,
//     out = sum_j softmax_j(z) v_j,   zeros where a token sees no key.
//
// One block owns 128 rows of one (sequence, kv head); a row is a (token, query head of the group) pair.  The cache's
// numbers become f16 in shared memory, exactly, and both products are f16 with float sums:
//
//   warps 0-15  softmax: four threads own each row, 32 of a tile's 128 scores each (a group of keys with one scale).  Scores
//               come out of tensor memory, the weights go back over them as f16 pairs, and at the end the thread scales and
//               stores its quarter of the row.  (Eight warps with 64 scores a thread took 5,600 cycles a tile: two warps on a
//               scheduler do not cover what each waits for.)
//   warps 16-23 turn keys and values into f16 (1024 + 128 + q has the bits 0x6400 | (q + 128): one byte permutation makes
//               two, one subtraction takes 1152 away) and store them as the tensor core reads them: keys in units of 64
//               entries of a head, values in units of as many bytes, all in one ring of slots in the order of their use (the
//               keys of tile 0; then the keys of tile j + 1 and the values of tile j; the values of the last tile), four
//               warps every other unit (with four warps for all of them a tile took 8,600 cycles: a unit is 260 of
//               arithmetic and 500 of waiting for shared memory and barriers);
//   warp 24     one thread (of elect.sync) issues tcgen05.mma: S = Q K^T (128 x 128) into one of two buffers in tensor memory, O += P V
//               (128 x head size, P from tensor memory, the values as they lie, keys x entries);
//   warp 25     looks up where the keys lie and what their scales are, 32 groups of 32 keys at a time, for all the others;
//   warp 26, 27 issue the TMA loads of the units' bytes, of keys and of values, each into a ring of its own.  (Loads into the
//               converting threads' registers were as many, but what tells the tensor core of a thread's stores waits for its
//               loads too: 6.4 us a tile of 128 keys and 256 entries.  One thread for all loads needs 1,000 cycles a unit.)
//
// Scales.  A key block's scale multiplies the scores.  A value block's scale 2^e goes into the weights: a weight is
// 2^(z - m) 2^(e - e0), e0 the largest exponent of the keys this block of threads sees, and m the row's running maximum of
// z + e - e0, so that what is rounded to f16 is at most 2^8 and exact to 11 bits for all that matters to the sum, however
// the blocks' scales differ; the sum of 2^(z - m) is kept in 32 bits, without the values' scales.  (m is raised only when it
// would be passed by more than 8: the accumulator in tensor memory is then scaled anew.)  Beside a block whose scale is 2^60
// above a key's, 2^(z - m) may be beyond a float (a block of zeros has the least scale there is): such keys' weights go into
// a sum of their own, relative to the largest of their own z, and the two are added up at the end.  A query row is scaled by a power
// of two to below 2^14 and held in f16, exactly but for numbers 2^-38 of the row's largest.
//
// What bounds it: of a tile of 128 keys and 256 entries, about 5,300 cycles, a block's start and end in them (2,048 tokens on
// 14,336 keys, 8 kv heads of 256, two query heads each: 569 to 581 us, 770 to 786 TFLOP/s of 1,700), the tensor core takes
// 2,050, shared memory 3,500 (bytes in, f16 out, f16 to the tensor core: 448 KB), the softmax of a row's scores and then of its
// weights, which wait for each other and for the products, 1,700 to 2,000 (fma units) and 1,200 to 1,400 (special function
// units), and the instructions of all roles 61 % of the issue slots; the tensor core waits for what is turned into f16 (1,400
// cycles a tile for keys, 1,300 for values).  That is with scores below 0.4 of the cap.  A tile of which a warp finds one beyond
// that takes its scores twice, the second time by exponentials: 775 us with queries of 20 times the size (without a cap 504).
// The sum of far values' weights put 1.5 % on heads of 256 and nothing on smaller ones (561.7 us without it, and wrong).
// Four groups of two converting warps instead of two of four were slower (609 us).  To put scores and weights side by side
// was slower too, both as two sets of softmax warps that take turns on tiles and as rounds that take the next tile's scores
// while they make this one's weights (681 us; with three score buffers for heads of 128 entries 144 us for 158, which is
// another kernel's worth of code): with two score buffers a tile's scores then wait for the values of the tile before the
// last, and a thread has too few registers for both.
//
// Every mbarrier wait is bounded; a wait that runs out records a code that brolm_attn_kv8_tc_status() returns, and the
// launch ends without its results.
#include "tcgen05.cuh"
#include "attn_kv8_join.cuh"

#include <cuda_fp16.h>

#include <type_traits>

namespace {

using namespace tc;
using namespace kv8;

constexpr int BM = 128, BN = 128;
constexpr int SOFTMAX_WARPS = 16, CONVERT_WARPS = 4, CONVERT_GROUPS = 2;      // (warps of a group)
constexpr int ISSUER = SOFTMAX_WARPS + CONVERT_GROUPS * CONVERT_WARPS, LOOKUP = ISSUER + 1, LOADER = LOOKUP + 1;
constexpr int THREADS = 32 * (LOADER + 2);   // seven groups of four warps
// registers of a thread: 72 at launch, 64,512 in all, then 512 x 88 + 256 x 56 + 128 x 40 = 64,512
constexpr int LAUNCH_REGS = 72, SOFTMAX_REGS = 88, CONVERT_REGS = 56, OTHER_REGS = 40;
static_assert(THREADS * LAUNCH_REGS == 512 * SOFTMAX_REGS + 256 * CONVERT_REGS + 128 * OTHER_REGS, "registers of the block");
constexpr int TMEM_COLS = 512;
constexpr int UNIT = 16384;               // bytes of a slot: 128 keys x 64 entries, or the same number of values
constexpr int RAW = UNIT / 2;             // .. as they come from the cache
constexpr int CHUNK = 8;                  // tiles whose places and scales are looked up at a time (32 groups of 32 keys)
constexpr float RESCALE_GAP = 8.0f;

__device__ int g_attn_kv8_tc_error;

struct TcArgs {
    const bf16* q;
    bf16* out;
    int q_stride, out_stride;
    const int32_t *cu_q, *kv_len, *slots, *tables;
    const int8_t *k_pages, *v_pages;
    const float *k_scale, *v_scale;
    int tokens, rows, n_kv, group, dim, block, n_blocks, n_slots, width, ring, window, row_tiles, wide;
    float scale, cap;
    int whole, spans;                     // the first `whole` row tiles have a block each, the others' keys are shared by `spans`,
                                          // whose parts a second launch joins
    float *part_o, *part_ml;
};

template <int HD>
struct Shape {
    static constexpr int PARTS = HD / 64;                    // units of a key tile, and of a value tile
    static constexpr int VK = BN / PARTS;                    // keys of a value unit
    static constexpr int SLOTS = HD == 256 ? 5 : HD == 128 ? 7 : 8;
    static constexpr int Q_BYTES = BM * HD * 2;
};

// Units on their way from the cache: a ring for keys and one for values.  A wait tells a slot's uses apart by their parity
// alone, so whoever waits for one must have waited for, or worked on, the one before: each ring has one loading warp, and an
// even number of slots gives a slot's units to one group of converting warps.
constexpr int KIND_RAWS = 4, RAWS = 2 * KIND_RAWS;
static_assert(KIND_RAWS % CONVERT_GROUPS == 0, "a raw slot's units belong to one group");

// barriers
enum : int { S_FULL = 0, P_FULL = 2, PV_DONE = 4, META_FULL = 6, META_EMPTY = 8, Q_FULL = 10, U_FULL = 11 };

struct Meta {                             // of a group of 32 keys
    int row;                              // the group's first row in the pages
    float k_scale;
    int v_exp;                            // exponent of the value scale; BAD: a scale that is NaN; GONE: no block of the cache
};
constexpr int BAD = 0x7fffffff, GONE = 0x7ffffffe;

__device__ __forceinline__ uint32_t idesc_f16(int m, int n, int b_mn_major) {
    return (1u << 4) | ((uint32_t)b_mn_major << 16) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}
__device__ __forceinline__ bool wait_on(uint32_t bar, uint32_t parity, volatile int* give_up, int code) {
    return mbar_wait(bar, parity, give_up, &g_attn_kv8_tc_error, code);
}
// One lane of a warp that is there as a whole.  The compiler knows of this one that it is alone, and keeps what the products
// are given in uniform registers: a tile of 256 entries is 24 products, and where `lane == 0` issued them the tensor core
// waited for their issue (2,048 tokens on 14,336 keys 626 us for 565).
__device__ __forceinline__ bool elect_one() {
    uint32_t one;
    asm volatile("{\n.reg .pred p;\nelect.sync _|p, 0xffffffff;\nselp.u32 %0, 1, 0, p;\n}" : "=r"(one));
    return one != 0;
}
template <int N> __device__ __forceinline__ void more_registers() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N> __device__ __forceinline__ void fewer_registers() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }
// Waits that are mostly over when they begin: the limit and the flags are looked at only if they are not (which takes 190
// cycles).  Only the softmax warps' waits, codes 8 and 9, and that for the queries,
// 15, can be stalled by brolm_attn_kv8_tc_wait_control at any time.
__device__ __forceinline__ bool wait_one(uint32_t bar, uint32_t parity, volatile int* give_up, int code) {
    return mbar_try(bar, parity) || wait_on(bar, parity, give_up, code);
}
__device__ __forceinline__ bool wait_soon(uint32_t bar, uint32_t parity, volatile int* give_up, int code) {
    bool ok = mbar_try(bar, parity);
    if (__all_sync(0xffffffffu, ok)) return true;
    ok = wait_on(bar, parity, give_up, code);
    return __all_sync(0xffffffffu, ok);
}
__device__ __forceinline__ bool wait_warp(uint32_t bar, uint32_t parity, volatile int* give_up, int code) {
    const bool ok = wait_on(bar, parity, give_up, code);
    return __all_sync(0xffffffffu, ok);
}
__device__ __forceinline__ void st_shared16(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
__device__ __forceinline__ uint4 ld_shared16(uint32_t p) {
    uint4 v;
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(p) : "memory");
    return v;
}
// Two floats in one instruction, and the largest of three.
__device__ __forceinline__ uint64_t pair_of(float a, float b) {
    uint64_t v;
    asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(a), "f"(b));
    return v;
}
__device__ __forceinline__ float2 halves(uint64_t v) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
    return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t v;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(v) : "l"(a), "l"(b));
    return v;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t v;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(v) : "l"(a), "l"(b));
    return v;
}
__device__ __forceinline__ uint64_t mad2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t v;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(v) : "l"(a), "l"(b), "l"(c));
    return v;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float v;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(v) : "f"(a), "f"(b), "f"(c));
    return v;
}

// A barrier of the four warps that share 32 rows; tells whether all of them are well.
__device__ __forceinline__ bool all_ok(int id, bool ok) {
    uint32_t all;
    asm volatile("{\n.reg .pred p, q;\nsetp.ne.u32 q, %2, 0;\nbarrier.cta.red.and.aligned.pred p, %1, 128, q;\nselp.u32 %0, 1, 0, p;\n}"
                 : "=r"(all) : "r"(id), "r"((uint32_t)ok) : "memory");
    return all != 0;
}
template <int SELECT>
__device__ __forceinline__ uint32_t bytes_to_f16(uint32_t w) {
    const uint32_t x = __byte_perm(w, 0x64646464u, SELECT);
    const __half2 y = __hsub2(*reinterpret_cast<const __half2*>(&x), __half2half2(__ushort_as_half(0x6480)));
    return *reinterpret_cast<const uint32_t*>(&y);
}

// 16 bytes of the cache as 16 f16 numbers: the pieces of 16 bytes `piece` and `piece ^ 1` of a 128-byte row.
__device__ __forceinline__ void put_f16(uint32_t row_at, int piece, const uint4& raw) {
    uint32_t h[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t w = (&raw.x)[i] ^ 0x80808080u;
        h[2 * i] = bytes_to_f16<0x4140>(w);
        h[2 * i + 1] = bytes_to_f16<0x4342>(w);
    }
    st_shared16(row_at + piece * 16, h[0], h[1], h[2], h[3]);
    st_shared16(row_at + (piece ^ 1) * 16, h[4], h[5], h[6], h[7]);
}

template <int HD>
__global__ void __launch_bounds__(THREADS, 1) attn_kv8_tc_kernel(const __grid_constant__ CUtensorMap map_k,
                                                                 const __grid_constant__ CUtensorMap map_v, TcArgs a) {
    using SH = Shape<HD>;
    constexpr int PARTS = SH::PARTS, VK = SH::VK, SLOTS = SH::SLOTS;
    constexpr uint32_t S_COL = 0, O_COL = 2 * BN;            // tensor-memory columns: two score buffers, then the output
    static_assert(O_COL + HD <= TMEM_COLS, "tensor memory");
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    if ((smem_u32(smem_raw) & 1023u) != 0) {                 // never seen; refuse rather than compute wrongly
        if (threadIdx.x == 0) atomicCAS(&g_attn_kv8_tc_error, 0, 13);
        return;
    }
    const uint32_t q_s = smem_u32(smem_raw), ring = q_s + SH::Q_BYTES;
    const uint32_t raw_s = ring + SLOTS * UNIT;
    uint8_t* rest = smem_raw + SH::Q_BYTES + SLOTS * UNIT + RAWS * RAW;
    Meta* meta = reinterpret_cast<Meta*>(rest);              // [2][CHUNK][4]
    float* xch = reinterpret_cast<float*>(meta + 2 * CHUNK * 4);     // [2][4][BM]: maxima by tile parity and part; the sums reuse it
    float* q_scale = xch + 8 * BM;                           // [BM]
    float2* far_sums = reinterpret_cast<float2*>(q_scale + BM);   // [4][BM]: sums of weights of values far below the largest, and their reference
    uint64_t* bars = reinterpret_cast<uint64_t*>(far_sums + 4 * BM);
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + U_FULL + 2 * SLOTS + 2 * RAWS);
    volatile int* give_up = reinterpret_cast<volatile int*>(tmem_slot + 1);       // three
    volatile int* top_exp = reinterpret_cast<volatile int*>(tmem_slot + 4);
    const uint32_t bar0 = smem_u32(bars);
    auto bar = [&](int i) { return bar0 + 8u * i; };
    auto u_full = [&](int sl) { return bar0 + 8u * (U_FULL + sl); };
    auto u_empty = [&](int sl) { return bar0 + 8u * (U_FULL + SLOTS + sl); };
    auto r_full = [&](int sl) { return bar0 + 8u * (U_FULL + 2 * SLOTS + sl); };
    auto r_empty = [&](int sl) { return bar0 + 8u * (U_FULL + 2 * SLOTS + RAWS + sl); };

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    pdl_wait();
    // blocks start in the order of their index: the last rows, which see the most keys, of every sequence and head first
    int item = blockIdx.x, span = 0, spans = 1;
    if (item >= a.whole) {
        span = (item - a.whole) % a.spans;
        item = a.whole + (item - a.whole) / a.spans;
        spans = a.spans;
    }
    const int per = a.n_kv * a.rows, xt = a.row_tiles - 1 - item / per, which = item % per;
    const int b = which / a.n_kv, g = which - b * a.n_kv;
    const int first_tok = a.cu_q[b], n_tok = min(a.cu_q[b + 1], a.tokens) - first_tok;
    const int kv_len = a.kv_len[b], slot = a.slots[b];
    const int row0 = xt * BM;
    const int rows_here = first_tok < 0 ? 0 : (int)min((long long)BM, (long long)n_tok * a.group - row0);
    if (rows_here <= 0) return;                              // (the whole block)
    const int window = a.window > 0 ? a.window : ALL_KEYS;
    const int pos0 = kv_len - n_tok, pos_lo = pos0 + row0 / a.group, pos_hi = pos0 + (row0 + rows_here - 1) / a.group;
    int t_first = 0, n_tiles = 0;
    if (pos_hi >= 0 && slot >= 0 && slot < a.n_slots) {
        t_first = max(0, pos_lo - window + 1) / BN;
        n_tiles = pos_hi / BN - t_first + 1;
        const int share = (n_tiles + spans - 1) / spans;
        t_first += span * share;
        n_tiles = max(0, min(share, n_tiles - span * share));
    }
    const int key_hi = min(pos_hi, (t_first + n_tiles) * BN - 1);     // the last key of this block's share
    const int32_t* table = a.tables + (size_t)max(slot, 0) * a.width;

    if (threadIdx.x == 0) {
        for (int s = 0; s < 2; ++s) {
            mbar_init(bar(S_FULL + s), 1);
            mbar_init(bar(P_FULL + s), SOFTMAX_WARPS);
            mbar_init(bar(PV_DONE + s), 1);
            mbar_init(bar(META_FULL + s), 1);
            mbar_init(bar(META_EMPTY + s), SOFTMAX_WARPS + 2);
        }
        mbar_init(bar(Q_FULL), 1);
        for (int s = 0; s < SLOTS; ++s) {
            mbar_init(u_full(s), CONVERT_WARPS);
            mbar_init(u_empty(s), 1);
        }
        for (int s = 0; s < RAWS; ++s) {
            mbar_init(r_full(s), 1);
            mbar_init(r_empty(s), CONVERT_WARPS);
        }
        give_up[0] = 0;
        give_up[1] = 0;
        give_up[2] = tc::g_stall_code;
        *top_exp = -126;
        mbar_init_fence();
    }
    if (warp == ISSUER) tmem_alloc(smem_u32(tmem_slot), TMEM_COLS);
    fence_before_sync();
    __syncthreads();
    fence_after_sync();
    const uint32_t tmem = *tmem_slot;
    // where a key's block is, from its place in units of 32 (a block is a multiple of that)
    const int block32 = a.block >> 5;
    auto block_of = [&](int place32) -> int {
        const int e = place32 / block32;
        const int id = e < a.width ? table[e] : -1;
        return id < a.n_blocks ? id : -1;                    // (below 0: none of the cache's, and nobody sees its keys)
    };

    if (warp >= ISSUER) {
        fewer_registers<OTHER_REGS>();
        if (warp == LOOKUP) {
            for (int m = 0; m * CHUNK < n_tiles; ++m) {
                if (!wait_warp(bar(META_EMPTY + (m & 1)), ((m >> 1) & 1) ^ 1, give_up, 3)) break;
                const int at32 = (t_first + m * CHUNK) * (BN / 32) + lane;
                Meta x{0, 0.0f, 0};
                if (at32 <= key_hi / 32) {
                    const int place32 = a.ring > 0 ? at32 % (a.ring >> 5) : at32;
                    const int id = block_of(place32);
                    x.v_exp = GONE;
                    if (id >= 0) {
                        const size_t bh = (size_t)id * a.n_kv + g;
                        x.row = (int)bh * a.block + (place32 % block32) * 32;
                        x.k_scale = a.k_scale[bh];
                        const float sv = a.v_scale[bh];
                        x.v_exp = max((int)(__float_as_uint(sv) >> 23 & 255u) - 127, -126);
                        if (x.k_scale != x.k_scale || sv != sv) {
                            x.k_scale = 0.0f;
                            x.v_exp = BAD;
                        }
                    }
                }
                meta[(m & 1) * CHUNK * 4 + lane] = x;
                __syncwarp();
                if (lane == 0) mbar_arrive(bar(META_FULL + (m & 1)));
            }
        } else if (warp == ISSUER) {
            if (n_tiles > 0 && elect_one()) {
                const uint32_t id_qk = idesc_f16(BM, BN, 0), id_pv = idesc_f16(BM, HD, 1);
                int u = 0;
                // S(j) goes over the buffer that P(j-2) was read from: the product that read it was issued before
                auto issue_qk = [&](int j) -> bool {
                    const int s = j & 1;
#pragma unroll
                    for (int ku = 0; ku < PARTS; ++ku) {
                        const int sl = u % SLOTS;
                        if (!wait_one(u_full(sl), (u / SLOTS) & 1, give_up, 4)) return false;
                        fence_after_sync();
                        const uint64_t qa = desc_kmajor(q_s + ku * (BM * 128)), kb = desc_kmajor(ring + sl * UNIT);
#pragma unroll
                        for (int k = 0; k < 4; ++k) umma(tmem + S_COL + s * BN, qa + 2 * k, kb + 2 * k, id_qk, (ku | k) != 0);
                        umma_commit(u_empty(sl));
                        ++u;
                    }
                    umma_commit(bar(S_FULL + s));
                    return true;
                };
                const bool begun = wait_on(bar(Q_FULL), 0, give_up, 15);
                bool ok = begun && issue_qk(0);
                for (int j = 0; j < n_tiles && ok; ++j) {
                    if (j + 1 < n_tiles) { ok = issue_qk(j + 1); if (!ok) break; }
                    const int s = j & 1;
                    ok = wait_one(bar(P_FULL + s), (j >> 1) & 1, give_up, 6);
                    if (!ok) break;
#pragma unroll
                    for (int vu = 0; vu < PARTS; ++vu) {
                        const int sl = u % SLOTS;
                        ok = wait_one(u_full(sl), (u / SLOTS) & 1, give_up, 7);
                        if (!ok) break;
                        fence_after_sync();
#pragma unroll
                        for (int k = 0; k < VK / 16; ++k) {
                            // sixteen keys further: eight columns of P, sixteen 128-byte rows down in V
                            const uint64_t vb = desc_mnmajor(ring + sl * UNIT + k * (16 * 128), (VK * 128) >> 4, 1024 >> 4);
                            umma_ts(tmem + O_COL, tmem + S_COL + s * BN + vu * (VK / 2) + k * 8, vb, id_pv, (j | vu | k) != 0);
                        }
                        umma_commit(u_empty(sl));
                        ++u;
                    }
                    if (!ok) break;
                    umma_commit(bar(PV_DONE + s));
                }
                if (begun) {                       // products in flight end before their operands go
                    umma_commit(bar(Q_FULL));
                    mbar_wait(bar(Q_FULL), 1, give_up, &g_attn_kv8_tc_error, 16, true);
                }
            }
        } else {
            // keys or values: a lane for each of a unit's boxes
            const bool keys = warp == LOADER;
            const int boxes = keys ? 4 : VK / 32;
            const uint32_t box_bytes = keys ? RAW / 4 : 32 * HD;
            const int raw0 = keys ? 0 : KIND_RAWS;
            int asked = 0;                         // units of this kind
            bool ok = true;
            for (int tile = 0; tile < n_tiles && ok; ++tile) {
                const int chunk = tile / CHUNK;
                if (tile % CHUNK == 0) ok = wait_soon(bar(META_FULL + (chunk & 1)), (chunk >> 1) & 1, give_up, 2);
                const Meta* m = meta + (chunk & 1) * CHUNK * 4 + (tile % CHUNK) * 4;
#pragma unroll
                for (int part = 0; part < PARTS; ++part) {
                    if (!ok) break;
                    const int sl = raw0 + asked % KIND_RAWS;
                    ok = wait_soon(r_empty(sl), ((asked / KIND_RAWS) & 1) ^ 1, give_up, 1);
                    if (!ok) break;
                    if (lane == 0) mbar_expect_tx(r_full(sl), RAW);
                    __syncwarp();
                    if (lane < boxes)
                        tma_load_2d(raw_s + sl * RAW + lane * box_bytes, keys ? &map_k : &map_v, keys ? part * 64 : 0,
                                    m[keys ? lane : part * (VK / 32) + lane].row, r_full(sl));
                    ++asked;
                }
                __syncwarp();
                if (lane == 0 && tile % CHUNK == CHUNK - 1) mbar_arrive(bar(META_EMPTY + (chunk & 1)));
            }
            if (lane == 0) pdl_trigger();      // every tile is asked for: the next kernel may move in
            if (*give_up)                      // let the loads in flight land before the block goes away
                for (int i = max(0, asked - KIND_RAWS); i < asked; ++i)
                    mbar_wait(r_full(raw0 + i % KIND_RAWS), (i / KIND_RAWS) & 1, give_up, &g_attn_kv8_tc_error, 10, true);
        }
    } else if (warp >= SOFTMAX_WARPS) {
        fewer_registers<CONVERT_REGS>();
        // A thread has four pieces of 16 bytes of a unit: of keys [128][64], rows 32 i + t / 4; of values [VK][HD], rows
        // VK / 4 further each.  Lanes are laid out so that eight of them store to all banks.
        const int group = (warp - SOFTMAX_WARPS) / CONVERT_WARPS, t = threadIdx.x & (32 * CONVERT_WARPS - 1);
        const int k_row = t >> 2, k_c = t & 3;
        // (values: the second four of eight lanes take the other four pieces of 128 bytes in the other of two rows, so that
        // neither the loads nor the stores of the eight meet a bank twice)
        const int v_c = PARTS == 1 ? t & 3 : (t & 3) | ((((t >> 2) ^ (t >> 3)) & 1) << 2) | (PARTS == 4 ? ((t >> 4) & 1) << 3 : 0);
        const int v_row = ((t >> 2) & 1) | (PARTS == 1 ? t >> 3 : PARTS == 2 ? t >> 4 : t >> 5) << 1;
        const uint32_t k_src = k_row * 64 + k_c * 16, v_src = v_row * HD + v_c * 16;
        const uint32_t k_dst = k_row * 128, v_dst = (v_c >> 2) * (VK * 128) + v_row * 128;
        const int k_piece = (2 * k_c) ^ (k_row & 7), v_piece = (2 * (v_c & 3)) ^ (v_row & 7);
        bool ok = true;
        // unit u, the i-th of its kind
        auto convert = [&](auto kind, int u, int i_kind) {
            constexpr bool KEYS = decltype(kind)::value;
            const int sl = u % SLOTS, rs = (KEYS ? 0 : KIND_RAWS) + i_kind % KIND_RAWS;
            ok = ok && wait_soon(r_full(rs), (i_kind / KIND_RAWS) & 1, give_up, 5);
            if (!ok) return;
            uint4 raw[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) raw[i] = ld_shared16(raw_s + rs * RAW + (KEYS ? k_src + i * (32 * 64) : v_src + i * (VK / 4 * HD)));
            ok = wait_soon(u_empty(sl), ((u / SLOTS) & 1) ^ 1, give_up, 14);
            if (!ok) return;
            const uint32_t at = ring + sl * UNIT + (KEYS ? k_dst : v_dst);
#pragma unroll
            for (int i = 0; i < 4; ++i) put_f16(at + i * (KEYS ? 32 * 128 : VK / 4 * 128), KEYS ? k_piece : v_piece, raw[i]);
            fence_proxy_async();
            __syncwarp();
            if (lane == 0) {
                mbar_arrive(r_empty(rs));
                mbar_arrive(u_full(sl));
            }
        };
        // every other unit (where a tile is one unit: one group the keys, one the values), each group's in the ring's order
        const int first = PARTS > 1 ? group : 0, stride = PARTS > 1 ? CONVERT_GROUPS : 1;
        const bool keys = PARTS > 1 || group == 0, values = PARTS > 1 || group == 1;
        for (int j = -1; j < n_tiles && ok; ++j) {
            if (keys && j + 1 < n_tiles)
                for (int p = first; p < PARTS; p += stride) convert(std::true_type(), (j < 0 ? 0 : 2 * j + 1) * PARTS + p, (j + 1) * PARTS + p);
            if (values && j >= 0)
                for (int p = first; p < PARTS; p += stride) convert(std::false_type(), min(2 * j + 2, 2 * n_tiles - 1) * PARTS + p, j * PARTS + p);
        }
    } else {
        more_registers<SOFTMAX_REGS>();
        // While the first tiles are on their way: e0, the largest exponent among the value scales of the keys that this block
        // sees, and the queries, a warp a row, eight entries a lane, rows of 128 bytes per 64 entries, pieces of 16 bytes
        // swizzled.  (Done by all warps before the roles part: 64 tokens on 4,096 keys 30.0 us for 27.0, 2,048 on 2,048 77.1
        // for 74.2.)
        constexpr int Q_ROWS = BM / SOFTMAX_WARPS / 2;
#pragma unroll 1
        for (int r0 = warp; r0 < BM; r0 += BM / 2) {
            uint4 raw[Q_ROWS];
#pragma unroll
            for (int i = 0; i < Q_ROWS; ++i) {
                const int r = r0 + i * SOFTMAX_WARPS, row = row0 + r;
                raw[i] = make_uint4(0u, 0u, 0u, 0u);
                if (r < rows_here && lane * 8 < a.dim) {
                    const bf16* src = a.q + (size_t)(first_tok + row / a.group) * a.q_stride + (g * a.group + row % a.group) * a.dim + lane * 8;
                    if (a.wide) raw[i] = *reinterpret_cast<const uint4*>(src);
                    else {
#pragma unroll
                        for (int e = 0; e < 8; ++e) reinterpret_cast<bf16*>(&raw[i])[e] = src[e];
                    }
                }
            }
            if (n_tiles > 0 && r0 == warp) {
                const int first32 = t_first * (BN / 32), n32 = key_hi / 32 - first32 + 1;
                int top = -126;
                for (int i = threadIdx.x; i * block32 < n32 + block32; i += 32 * SOFTMAX_WARPS) {
                    const int at = min(first32 + i * block32, key_hi / 32);
                    const int id = block_of(a.ring > 0 ? at % (a.ring >> 5) : at);
                    const float s = id >= 0 ? a.v_scale[(size_t)id * a.n_kv + g] : 0.0f;
                    if (s == s) top = max(top, (int)(__float_as_uint(s) >> 23 & 255u) - 127);
                }
                top = __reduce_max_sync(0xffffffffu, top);
                if (lane == 0 && top > -126) atomicMax(const_cast<int*>(top_exp), top);
            }
#pragma unroll
            for (int i = 0; i < Q_ROWS; ++i) {
                const int r = r0 + i * SOFTMAX_WARPS;
                float v[8], most = 0.0f;
                bool finite = true;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    v[e] = to_float(reinterpret_cast<const bf16*>(&raw[i])[e]);
                    most = fmaxf(most, fabsf(v[e]));
                    finite = finite && fabsf(v[e]) < INFINITY;
                }
                most = warp_max(most);
                finite = __all_sync(0xffffffffu, finite);
                const int up = max(min(13 + 127 - (int)(__float_as_uint(most) >> 23), 120), -126);
                const float f = power_of_two(up);
                if (lane == 0) q_scale[r] = finite ? power_of_two(-up) : __int_as_float(0x7fc00000);
                if (lane * 8 < HD) {
                    uint32_t h[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const __half2 t = __floats2half2_rn(finite ? v[2 * e] * f : 0.0f, finite ? v[2 * e + 1] * f : 0.0f);
                        h[e] = *reinterpret_cast<const uint32_t*>(&t);
                    }
                    st_shared16(q_s + (lane >> 3) * (BM * 128) + r * 128 + (((lane & 7) ^ (r & 7)) << 4), h[0], h[1], h[2], h[3]);
                }
            }
        }
        fence_proxy_async();
        asm volatile("bar.sync 5, %0;" ::"n"(32 * SOFTMAX_WARPS) : "memory");
        if (threadIdx.x == 0) mbar_arrive(bar(Q_FULL));
        const int e0 = *top_exp;
        // Four warps share each quarter of the rows (a warp may only touch the 32 lanes of tensor memory of its quarter), 32
        // score columns each.  They agree on the rows' reference maxima through shared memory and a barrier of their own.
        constexpr int W = BN / 4, OUT = HD / 4;
        const int quarter = warp & 3, part = warp >> 2;
        const int r = quarter * 32 + lane;
        const uint32_t lane_addr = tmem + ((uint32_t)(quarter * 32) << 16);
        const bool row_ok = r < rows_here;
        const int pos = pos0 + (row0 + r) / a.group;
        const float qs = q_scale[r];
        const float unit = qs * (a.cap > 0.0f ? a.scale / a.cap : a.scale * LOG2E);
        const float c1 = a.cap * LOG2E, c2 = 2.0f * a.cap * LOG2E;
        // tanh(x) / x up to |x| = 0.4, of the third degree in x^2 with the least largest error (1e-7; an exchange of the points
        // where it is largest gives the four numbers; the series to x^9 has 4e-7)
        const uint64_t t0 = pair_of(c1 * 0.9999999f, c1 * 0.9999999f), t1 = pair_of(c1 * -0.33331362f, c1 * -0.33331362f);
        const uint64_t t2 = pair_of(c1 * 0.13270977f, c1 * 0.13270977f), t3 = pair_of(c1 * -0.047553604f, c1 * -0.047553604f);
        float m_ref = -INFINITY, l = 0.0f;                   // l: the sum over this thread's columns only
        far_sums[part * BM + r] = make_float2(0.0f, -INFINITY);
        bool ok = true, sees_bad = false;
        for (int j = 0; j < n_tiles; ++j) {
            const int s = j & 1;
            if (ok && j % CHUNK == 0) ok = wait_warp(bar(META_FULL + ((j / CHUNK) & 1)), (j / CHUNK >> 1) & 1, give_up, 9);
            const Meta& m = meta[((j / CHUNK) & 1) * CHUNK * 4 + (j % CHUNK) * 4 + part];
            const float f = m.k_scale * unit;
            int ve = m.v_exp >= GONE ? m.v_exp : m.v_exp - e0;
            if (ok) ok = wait_warp(bar(S_FULL + s), (j >> 1) & 1, give_up, 8);
            fence_after_sync();
            const int key_base = (t_first + j) * BN, kp0 = key_base + part * W;
            const bool edge = key_base + BN - 1 > pos_lo || key_base < pos_hi - window + 1;
            // visible: lo <= c <= hi for column c of this thread
            const int hi = row_ok ? pos - kp0 : -1, lo = pos - window + 1 - kp0;
            uint64_t z[W / 2];                               // scores in log2 units, two by two
            auto scores = [&](auto&& to_z) {
                uint32_t sv[W];
                tmem_ld32(lane_addr + S_COL + s * BN + part * W, sv);
                tmem_wait_ld();
#pragma unroll
                for (int c = 0; c < W / 2; ++c)
                    z[c] = to_z(mul2(pair_of(__uint_as_float(sv[2 * c]), __uint_as_float(sv[2 * c + 1])), pair_of(f, f)));
            };
            if (a.cap > 0.0f) {
                // cap log2e tanh(x).  Scores are mostly well below the cap, and there a polynomial is as exact and leaves the
                // special function units to the weights
                float far = 0.0f;
                scores([&](uint64_t x) {
                    const uint64_t y = mul2(x, x);
                    const float2 yy = halves(y);
                    far = max3(far, yy.x, yy.y);
                    return mul2(x, mad2(mad2(mad2(t3, y, t2), y, t1), y, t0));
                });
                if (!__all_sync(0xffffffffu, far <= 0.16f))
                    scores([&](uint64_t x) {
                        const float2 xx = halves(x);
                        return pair_of(fmaf(-c2, fast_rcp(1.0f + fast_exp2(xx.x * (2.0f * LOG2E))), c1),
                                       fmaf(-c2, fast_rcp(1.0f + fast_exp2(xx.y * (2.0f * LOG2E))), c1));
                    });
            } else {
                scores([&](uint64_t x) { return x; });
            }
            if (edge) {
#pragma unroll
                for (int c = 0; c < W / 2; ++c) {
                    float2 x = halves(z[c]);
                    if (2 * c > hi || 2 * c < lo) x.x = -INFINITY;
                    if (2 * c + 1 > hi || 2 * c + 1 < lo) x.y = -INFINITY;
                    z[c] = pair_of(x.x, x.y);
                }
            }
            float m_t = -INFINITY;
#pragma unroll
            for (int c = 0; c < W / 2; ++c) {
                const float2 x = halves(z[c]);
                m_t = max3(m_t, x.x, x.y);
            }
            float e = (float)ve;
            if (ve >= GONE) {                                // a NaN block: whoever sees a key of it gets NaN; none: weights of 0
                if (ve == BAD) sees_bad = sees_bad || (hi >= 0 && lo < W);
                e = ve == BAD ? 0.0f : -INFINITY;
                ve = 0;
            }
            xch[(s * 4 + part) * BM + r] = m_t + e;          // double-buffered by the tile's parity
            // after this barrier all four threads of the row hold their scores in registers, so the weights may go over them
            ok = all_ok(1 + quarter, ok);                    // (a wait that ran out ends all four, or some would wait for the others)
            if (!ok) break;
            m_t = max3(fmaxf(xch[s * 4 * BM + r], xch[(s * 4 + 1) * BM + r]), xch[(s * 4 + 2) * BM + r], xch[(s * 4 + 3) * BM + r]);
            const bool raise = m_t > m_ref + RESCALE_GAP;    // also true for the first visible tile of a row
            if (__any_sync(0xffffffffu, raise && m_ref > -INFINITY)) {
                const float corr = raise && m_ref > -INFINITY ? fast_exp2(m_ref - m_t) : 1.0f;
                l *= corr;
                // rare: the accumulator has to be at rest (the product of the tile before is done), then every row of the
                // warp is scaled anew; each of the four warps takes a quarter of the entries
                ok = wait_warp(bar(PV_DONE + (s ^ 1)), ((j - 1) >> 1) & 1, give_up, 12);
                fence_after_sync();
#pragma unroll 1
                for (int c = part * OUT; c < (part + 1) * OUT; c += 16) {
                    uint32_t ov[16];
                    tmem_ld16(lane_addr + O_COL + c, ov);
                    tmem_wait_ld();
#pragma unroll
                    for (int i = 0; i < 16; ++i) ov[i] = __float_as_uint(__uint_as_float(ov[i]) * corr);
                    tmem_st16(lane_addr + O_COL + c, ov);
                }
            }
            if (raise) m_ref = m_t;
            // weights -> tensor memory, f16 pairs: keys 2c, 2c+1 of this thread in column c of its 16
            const float m_sub = m_ref > -INFINITY ? m_ref : 0.0f;    // a row that has seen nothing: 2^(-inf - 0) = 0
            uint64_t sums = 0ull;
            uint32_t pw[W / 2];
#pragma unroll
            for (int c = 0; c < W / 2; ++c) {
                const float2 x = halves(add2(z[c], pair_of(e - m_sub, e - m_sub)));
                const float p0 = fast_exp2(x.x), p1 = fast_exp2(x.y);
                sums = add2(sums, pair_of(p0, p1));
                const __half2 t = __floats2half2_rn(p0, p1);
                pw[c] = *reinterpret_cast<const uint32_t*>(&t);
            }
            tmem_st16(lane_addr + S_COL + s * BN + part * (W / 2), pw);
            if (ve >= -60) {
                const float2 sum = halves(sums);
                l = fmaf(sum.x + sum.y, power_of_two(-ve), l);
            } else {
                // scales more than 2^60 apart: what a weight is without its scale may be lost with it, or pass a float's range
                // relative to m
                float2 sum = far_sums[part * BM + r];
                float top = sum.y;
#pragma unroll
                for (int c = 0; c < W / 2; ++c) {
                    const float2 x = halves(z[c]);
                    top = max3(top, x.x, x.y);
                }
                if (top > -INFINITY) {
                    sum.x *= fast_exp2(sum.y - top);
#pragma unroll
                    for (int c = 0; c < W / 2; ++c) {
                        const float2 x = halves(z[c]);
                        sum.x += fast_exp2(x.x - top) + fast_exp2(x.y - top);
                    }
                    far_sums[part * BM + r] = make_float2(sum.x, top);
                }
            }
            tmem_wait_st();
            fence_before_sync();
            __syncwarp();
            if (lane == 0) {
                mbar_arrive(bar(P_FULL + s));
                if (j % CHUNK == CHUNK - 1) mbar_arrive(bar(META_EMPTY + ((j / CHUNK) & 1)));
            }
        }
        if (ok && n_tiles > 0) ok = wait_warp(bar(PV_DONE + ((n_tiles - 1) & 1)), ((n_tiles - 1) >> 1) & 1, give_up, 11);
        // the row's sum is that of its four threads (always added in the same order), and so is what they have seen
        float* last = xch + (n_tiles & 1) * 4 * BM;          // the buffer that the next tile would have used
        last[part * BM + r] = sees_bad || (qs != qs && pos >= 0) ? __int_as_float(0x7fc00000) : qs != qs ? 0.0f : l;
        asm volatile("bar.sync %0, 128;" ::"r"(1 + quarter) : "memory");
        float total = (last[r] + last[BM + r]) + (last[2 * BM + r] + last[3 * BM + r]);
        if (ok) {
            fence_after_sync();
            float v0 = power_of_two(e0), ref = m_ref;
            const float far_ref = max3(fmaxf(far_sums[r].y, far_sums[BM + r].y), far_sums[2 * BM + r].y, far_sums[3 * BM + r].y);
            if (far_ref > -INFINITY) {                       // (m is finite, too)
                ref = fmaxf(m_ref, far_ref);
                total *= fast_exp2(m_ref - ref);
#pragma unroll
                for (int p = 0; p < 4; ++p) total = fmaf(far_sums[p * BM + r].x, fast_exp2(far_sums[p * BM + r].y - ref), total);
                v0 = fast_exp2((float)e0 + (m_ref - ref));
            }
            const float inv = total > 0.0f ? 1.0f / total : 0.0f;
            const bool nan = total != total;
            const int row = row0 + r, tok = first_tok + row / a.group, head = g * a.group + row % a.group;
            bf16* dst = a.out + (size_t)tok * a.out_stride + (size_t)head * a.dim;
            const size_t share = ((size_t)(item - a.whole) * spans + span) * BM + r;      // (where there are several)
            if (spans > 1 && row_ok && part == 0) *reinterpret_cast<float2*>(a.part_ml + share * 2) = make_float2(ref, total);
            const bool wide = ((uintptr_t)a.out & 15) == 0 && (a.out_stride & 7) == 0;
#pragma unroll 1
            for (int c = part * OUT; c < min((part + 1) * OUT, a.dim); c += 16) {
                uint32_t ov[16];
                if (n_tiles > 0) {
                    tmem_ld16(lane_addr + O_COL + c, ov);
                    tmem_wait_ld();
                }
                if (row_ok && spans > 1) {
#pragma unroll
                    for (int i = 0; i < 16; i += 4) {
                        float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                        if (n_tiles > 0)
                            x = make_float4(__uint_as_float(ov[i]) * v0, __uint_as_float(ov[i + 1]) * v0, __uint_as_float(ov[i + 2]) * v0,
                                            __uint_as_float(ov[i + 3]) * v0);
                        *reinterpret_cast<float4*>(a.part_o + share * a.dim + c + i) = x;
                    }
                } else if (row_ok) {
#pragma unroll
                    for (int i = 0; i < 16; i += 8) {
                        uint4 pk;
                        __nv_bfloat162* p2 = reinterpret_cast<__nv_bfloat162*>(&pk);
#pragma unroll
                        for (int h = 0; h < 4; ++h) {
                            float x = n_tiles > 0 ? __uint_as_float(ov[i + 2 * h]) * inv * v0 : 0.0f;
                            float y = n_tiles > 0 ? __uint_as_float(ov[i + 2 * h + 1]) * inv * v0 : 0.0f;
                            if (nan) x = y = total;
                            p2[h] = __floats2bfloat162_rn(x, y);
                        }
                        if (wide) *reinterpret_cast<uint4*>(dst + c + i) = pk;
                        else {
#pragma unroll
                            for (int h = 0; h < 8; ++h) dst[c + i + h] = reinterpret_cast<const bf16*>(&pk)[h];
                        }
                    }
                }
            }
        }
    }
    fence_before_sync();
    __syncthreads();
    if (warp == ISSUER) tmem_dealloc(tmem, TMEM_COLS);
}

// The rows of the tiles whose keys were shared: a thread for four entries of a row.
constexpr int JOIN_CHUNK = 256;
__global__ void __launch_bounds__(JOIN_CHUNK) attn_kv8_tc_join_kernel(TcArgs a) {
    pdl_trigger();
    pdl_wait();
    const int per = a.dim >> 2, each = JOIN_CHUNK / per, chunks = (BM + each - 1) / each, mine = threadIdx.x / per;
    const int tile = blockIdx.x / chunks, r = (blockIdx.x - tile * chunks) * each + mine, d = (threadIdx.x - mine * per) * 4;
    const int item = a.whole + tile, xt = a.row_tiles - 1 - item / (a.n_kv * a.rows), which = item % (a.n_kv * a.rows);
    const int b = which / a.n_kv, g = which - b * a.n_kv, row = xt * BM + r;
    const int first_tok = a.cu_q[b], n_tok = min(a.cu_q[b + 1], a.tokens) - first_tok;
    if (mine >= each || r >= BM || first_tok < 0 || row >= (long long)n_tok * a.group) return;
    float sum;
    const float4 acc = join_parts(a.part_o, a.part_ml, (size_t)tile * a.spans * BM + r, BM, a.spans, a.dim, d, sum);
    store_row<bf16>(a.out, a.out_stride, a.dim, first_tok + row / a.group, g * a.group + row % a.group, d, acc, sum);
}

// The rows of the pages [rows][dim] of bytes; box = box_bytes x 32 rows, zeros beyond a row's end.
int make_map(CUtensorMap* map, const void* ptr, long long rows, int dim, int box_bytes) {
    EncodeTiled enc = encoder();
    if (!enc) return BROLM_ERR_BAD_SIZE;
    const cuuint64_t dims[2] = {(cuuint64_t)dim, (cuuint64_t)rows};
    const cuuint64_t strides[1] = {(cuuint64_t)dim};
    const cuuint32_t box[2] = {(cuuint32_t)box_bytes, 32}, elem[2] = {1, 1};
    const CUresult r = enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(ptr), dims, strides, box, elem,
                           CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                           CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? BROLM_OK : BROLM_ERR_ALIGNMENT;
}

template <int HD>
int launch(const TcArgs& a, cudaStream_t stream) {
    using SH = Shape<HD>;
    constexpr size_t smem = (size_t)SH::Q_BYTES + (size_t)SH::SLOTS * UNIT + RAWS * RAW + 2 * CHUNK * 4 * sizeof(Meta) + 9 * BM * 4 + 4 * BM * 8 +
                            (U_FULL + 2 * SH::SLOTS + 2 * RAWS) * 8 + 32;
    static_assert(smem <= 232448, "shared memory of a block");
    static OncePerDevice raised;
    int st = allow_shared_memory(attn_kv8_tc_kernel<HD>, smem, raised);
    if (st) return st;
    const long long blocks = a.whole + ((long long)a.row_tiles * a.n_kv * a.rows - a.whole) * a.spans, rows = (long long)a.n_blocks * a.n_kv * a.block;
    if (blocks > 0x7fffffffll || rows > 0x7fffffffll) return BROLM_ERR_TOO_LARGE;
    CUtensorMap mk, mv;
    st = make_map(&mk, a.k_pages, rows, a.dim, 64);
    if (st) return st;
    st = make_map(&mv, a.v_pages, rows, a.dim, HD);
    if (st) return st;
    st = launch_pdl(attn_kv8_tc_kernel<HD>, dim3((unsigned)blocks), dim3(THREADS), smem, stream, mk, mv, a);
    if (st || a.spans == 1) return st;
    const int each = JOIN_CHUNK / (a.dim >> 2);
    const long long shared = (long long)a.row_tiles * a.n_kv * a.rows - a.whole, joins = shared * ((BM + each - 1) / each);
    if (shared == 0) return st;
    if (joins > 0x7fffffffll) return BROLM_ERR_TOO_LARGE;
    return launch_pdl(attn_kv8_tc_join_kernel, dim3((unsigned)joins), dim3(JOIN_CHUNK), 0, stream, a);
}

}  // namespace

struct AttnTcCall {
    const void* q;
    void* out;
    const void *cu_q, *kv_len, *slots, *tables, *k_pages, *v_pages, *k_scale, *v_scale;
    void *part_o, *part_ml;               // spans > 1: [(tiles of 128 rows - whole) * spans * 128 * dim] and [.. * 2]
    cudaStream_t stream;
    int q_stride, out_stride, tokens, rows, n_kv, group, dim, block, n_blocks, n_slots, width, ring, window, max_q_len, whole, spans;
    float scale, cap;
};

// bfloat16, heads of up to 256 entries; what is between 64, 128 and 256 takes the time of the next, its last columns zeros.
BROLM_API int brolm_attn_kv8_tc(const AttnTcCall* c) {
    const int n_kv = c->n_kv, group = c->group, block = c->block;
    if (c->dim <= 0 || c->dim % 16) return BROLM_ERR_BAD_SIZE;
    if (c->tokens < 0 || c->rows < 0 || n_kv <= 0 || group <= 0 || block <= 0 || block % 32) return BROLM_ERR_BAD_SIZE;
    if (c->n_blocks <= 0 || c->n_slots <= 0 || c->width <= 0 || c->ring < 0 || c->ring % block || c->window < 0 || c->max_q_len <= 0) return BROLM_ERR_BAD_SIZE;
    if (c->dim > MAX_DIM || block > MAX_BLOCK || (long long)n_kv * group > 65535 || (long long)c->max_q_len * group > 0x3fffffff) return BROLM_ERR_TOO_LARGE;
    if ((long long)c->n_blocks * block > 0x7fffffffll || c->tokens > 0x3fffffff) return BROLM_ERR_TOO_LARGE;
    if (c->spans < 1 || (c->spans > 1 && (!c->part_o || !c->part_ml))) return BROLM_ERR_BAD_SIZE;
    if (((uintptr_t)c->k_pages | (uintptr_t)c->v_pages | (uintptr_t)c->part_o) & 15) return BROLM_ERR_ALIGNMENT;
    if (c->tokens == 0 || c->rows == 0) return BROLM_OK;
    const int row_tiles = (c->max_q_len * group + BM - 1) / BM;
    const long long items = (long long)row_tiles * n_kv * c->rows;
    if (items > 0x7fffffffll) return BROLM_ERR_TOO_LARGE;
    if (c->whole < 0 || c->whole > items) return BROLM_ERR_BAD_SIZE;
    const int wide = ((uintptr_t)c->q & 15) == 0 && c->q_stride % 8 == 0;
    TcArgs a{(const bf16*)c->q, (bf16*)c->out, c->q_stride, c->out_stride, (const int32_t*)c->cu_q, (const int32_t*)c->kv_len,
             (const int32_t*)c->slots, (const int32_t*)c->tables, (const int8_t*)c->k_pages, (const int8_t*)c->v_pages,
             (const float*)c->k_scale, (const float*)c->v_scale, c->tokens, c->rows, n_kv, group, c->dim, block, c->n_blocks, c->n_slots,
             c->width, c->ring, min(c->window, ALL_KEYS), row_tiles, wide, c->scale, c->cap, c->whole, c->spans, (float*)c->part_o, (float*)c->part_ml};
    if (c->dim <= 64) return launch<64>(a, c->stream);
    if (c->dim <= 128) return launch<128>(a, c->stream);
    return launch<256>(a, c->stream);
}

BROLM_API int brolm_attn_kv8_tc_status(int reset) {
    int v = 0;
    if (cudaMemcpyFromSymbol(&v, g_attn_kv8_tc_error, sizeof(int)) != cudaSuccess) return -1;
    if (reset && v) {
        const int zero = 0;
        cudaMemcpyToSymbol(g_attn_kv8_tc_error, &zero, sizeof(int));
    }
    return v;
}

BROLM_WAIT_CONTROL(attn_kv8_tc)
