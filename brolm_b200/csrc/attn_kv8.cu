// Attention over the cache in 8 bits (kv8.cuh): the newest tokens of every sequence against all that it holds, soft-capped,
// windowed, causal, with several query heads on a kv head.
//
//     z = scale * q . k,   cap tanh(z / cap),   key j visible from position p iff 0 <= p - j < window,
//     out = sum_j softmax_j(z) v_j,   zeros where a token sees no key.
//
// A row is a (token, query head of the group) pair; a block of threads owns 8 or 16 rows of one (sequence, kv head) and a
// share of its keys, and its four warps take tiles of 32 keys in turn.  A tile lies inside one cache block, so it has one
// scale for its keys and one for its values:
//
//     S^T [32 keys x rows] = K q^T,    m_t = max over the tile,  p = 2^(z - m_t),    O^T += s_v 2^(m_t - m) (V^T p)
//
// Both products run on mma.sync (f16, float sums) with the cache's numbers as the left operand, where the 16 rows of an
// instruction are keys or entries of a head and its 8 columns are query rows, so that two to eight query heads waste
// little.  int8 becomes f16 exactly and without a conversion instruction: 1024 + 128 + q has the bits 0x6400 | (q + 128),
// one byte permutation makes two of them and one subtraction takes 1152 away.  The weights of a tile are relative to the
// tile's own maximum and its sums are scaled in 32 bits when they join the row's, so blocks whose scales differ by any
// factor keep all their bits.  A query row is scaled by a power of two to below 2^14, so that it is held by one f16 a
// number (bfloat16 queries, exactly but for numbers 2^-38 of the row's largest) or two (float32: 22 bits or more).
// Weights are one f16 (bfloat16) or two (float32).
//
// What bounds it is reading the cache: a tile of 32 keys of 256 entries is 16 KB and some 1,200 instructions of a warp,
// 300 cycles of an SM's four schedulers, while an SM's share of the memory's rate brings 16 KB in 700.  Every warp keeps a
// ring of its own of key and value tiles in flight (cp.async, no barrier but its own), two blocks on an SM.
//
// The shares of a row's keys are joined inside the launch: they form a cluster, whose blocks read each other's partial
// results out of shared memory.  Nothing is kept between launches.
#include "kv8.cuh"

#include <cuda_fp16.h>

namespace {

using namespace kv8;

constexpr float LOG2E = 1.4426950408889634f;
constexpr int WARPS = 4, THREADS = 32 * WARPS;
constexpr int KT = 32;                    // keys of a tile: a divisor of every block size

struct AttnArgs {
    const void* q;
    void* out;
    int q_stride, out_stride;
    const int32_t *cu_q, *kv_len, *slots, *tables;
    const int8_t *k_pages, *v_pages;
    const float *k_scale, *v_scale;
    int tokens, rows, n_kv, group, dim, block, n_blocks, n_slots, width, ring, window;
    float scale, cap;
    int shares, spans, row_tiles, wide;   // blocks of a cluster, clusters that share a row's keys, row tiles of a sequence
    float *part_o, *part_ml;              // [token][head][span][dim] and [..][2] where spans > 1
};

__device__ __forceinline__ uint32_t smem_addr(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float rcp(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ void cluster_barrier() {
    asm volatile("barrier.cluster.arrive.aligned;\nbarrier.cluster.wait.aligned;\n" ::: "memory");
}
__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ uint32_t of_rank(uint32_t addr, uint32_t rank) {
    uint32_t r;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}
__device__ __forceinline__ float4 ld_cluster4(uint32_t addr) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ float2 ld_cluster2(uint32_t addr) {
    float2 v;
    asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ uint4 lds128(uint32_t addr) {
    uint4 v;
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ uint2 lds64(uint32_t addr) {
    uint2 v;
    asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
// Two bytes, q + 128 each, as f16 numbers q: bytes LO and HI of `w` under the exponent of 1024, less 1152.
template <int SELECT>
__device__ __forceinline__ uint32_t bytes_to_f16(uint32_t w) {
    const uint32_t x = __byte_perm(w, 0x64646464u, SELECT);
    const __half2 y = __hsub2(*reinterpret_cast<const __half2*>(&x), __half2half2(__ushort_as_half(0x6480)));
    return *reinterpret_cast<const uint32_t*>(&y);
}
constexpr int FIRST = 0x4140, SECOND = 0x4342;       // bytes 0, 1 and bytes 2, 3
constexpr uint32_t FLIP = 0x80808080u;               // int8 to q + 128

__device__ __forceinline__ uint32_t pack_half(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}

// Where a 16-byte piece of a key or value tile lies.  Keys are read a row of 64 bytes by four threads, two rows at a time;
// values eight entries of four keys (2t, 2t + 1, 2t + 8, 2t + 9), 32 bytes of four rows at a time: in both cases what is
// read at once lies in different banks.
template <int DP>
__device__ __forceinline__ int key_offset(int row, int c) {
    if constexpr (DP % 128 == 0) return row * DP + ((c ^ ((row & 1) << 2)) << 4);
    else return row * DP + (c << 4);
}
template <int DP>
__device__ __forceinline__ int value_offset(int row, int c) {
    if constexpr (DP % 128 == 0) return row * DP + ((c ^ (((row >> 1) & 3) << 1)) << 4);
    else {
        const int at = (row & ~7) | ((row >> 1) & 3) | ((row & 1) << 2);
        return at * DP + ((c ^ (((at >> 1) & 1) << 1)) << 4);
    }
}

template <typename T, int DP, int NT>
struct Shape {
    static constexpr int ROWS = 8 * NT;
    static constexpr int PARTS = sizeof(T) == 4 ? 2 : 1;
    static constexpr int SEGS = DP / 64;
    static constexpr int UNIT = KT * DP;                                   // a key or value tile
    static constexpr int SLOTS = DP == 256 ? 3 : DP == 192 ? 4 : DP == 128 ? 6 : 8;
    static constexpr int RING = WARPS * SLOTS * UNIT;
    static constexpr int Q_BYTES = PARTS * NT * SEGS * 1024;
    static constexpr int PITCH = DP + 4;                                   // floats of a row of partial results
    static constexpr int MERGE = (WARPS * ROWS * PITCH + WARPS * ROWS * 2 + ROWS * PITCH + ROWS * 2 + 16) * 4;
    static constexpr int SMEM = Q_BYTES + (RING > MERGE ? RING : MERGE);
};

template <typename T, int DP, int NT>
__global__ void __launch_bounds__(THREADS, 2) attn_kv8_kernel(AttnArgs a) {
    using SH = Shape<T, DP, NT>;
    constexpr int ROWS = SH::ROWS, PARTS = SH::PARTS, SEGS = SH::SEGS, UNIT = SH::UNIT, SLOTS = SH::SLOTS;
    constexpr bool EXACT = sizeof(T) == 4;
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ float q_scale[ROWS];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g8 = lane >> 2, t4 = lane & 3;

    const int share = blockIdx.x % a.shares;
    int rest = blockIdx.x / a.shares;
    const int span = rest % a.spans;
    rest /= a.spans;
    const int tile_of_rows = rest % a.row_tiles, b = rest / a.row_tiles;
    const int g = blockIdx.y;
    pdl_wait();
    const int first_tok = a.cu_q[b], n_tok = min(a.cu_q[b + 1], a.tokens) - first_tok;
    const int row0 = tile_of_rows * ROWS, n_rows = min(ROWS, n_tok * a.group - row0);
    if (n_rows <= 0) return;                                   // (the whole cluster)
    const int kv_len = a.kv_len[b], slot = a.slots[b];
    const int pos0 = kv_len - n_tok;                           // position of the sequence's first new token
    const int pos_lo = pos0 + row0 / a.group, pos_hi = pos0 + (row0 + n_rows - 1) / a.group;
    const int window = a.window > 0 ? a.window : 0x3fffffff;

    // the tiles of this share: [t_begin, t_end), the warps in turn
    int t_begin = 0, t_end = 0;
    if (pos_hi >= 0 && slot >= 0 && slot < a.n_slots) {
        const int t_lo = max(0, pos_lo - window + 1) / KT, t_hi = pos_hi / KT;
        const int parts = a.shares * a.spans, per = (t_hi - t_lo + parts) / parts;
        t_begin = t_lo + (span * a.shares + share) * per;
        t_end = min(t_hi + 1, t_begin + per);
    }
    const int n_tiles = t_begin + warp < t_end ? (t_end - t_begin - warp + WARPS - 1) / WARPS : 0;
    const int32_t* table = a.tables + (size_t)max(slot, 0) * a.width;

    // of this warp's tiles n .. n + 31, lane by lane: where the numbers lie and their scales
    auto look_up = [&](int n, long long& at, float& sk, float& sv) {
        at = 0;
        sk = sv = 0.0f;
        if (n + lane < n_tiles) {
            const long long key = (long long)(t_begin + warp + (n + lane) * WARPS) * KT;
            const int place = a.ring > 0 ? (int)(key % a.ring) : (int)key, e = place / a.block;
            int id = e < a.width ? table[e] : 0;
            if (id < 0 || id >= a.n_blocks) id = 0;            // (never followed out of the cache)
            const size_t bh = (size_t)id * a.n_kv + g;
            at = (long long)bh * a.block + (place - e * a.block);
            sk = a.k_scale[bh];
            sv = a.v_scale[bh];
            if (sk != sk || sv != sv) {                        // a NaN block: scores of zero, values of NaN
                sk = 0.0f;
                sv = __int_as_float(0x7fc00000);
            }
        }
    };
    long long at_l;                                            // of the tiles that are being asked for
    float sk_l, sv_l, sk_c = 0.0f, sv_c = 0.0f;                // .. and the scales of those that are being multiplied
    look_up(0, at_l, sk_l, sv_l);

    const uint32_t ring = smem_addr(smem) + SH::Q_BYTES + warp * SLOTS * UNIT;
    const int n_units = 2 * n_tiles;
    auto load_unit = [&](int u) {                              // key tile u / 2 or value tile u / 2 into slot u % SLOTS
        const int n = u >> 1;
        if (u > 0 && (u & 63) == 0) look_up(n, at_l, sk_l, sv_l);
        const long long at = __shfl_sync(0xffffffffu, at_l, n & 31);
        const int8_t* src = (u & 1 ? a.v_pages : a.k_pages) + at * a.dim;
        const uint32_t dst = ring + (u % SLOTS) * UNIT;
#pragma unroll
        for (int i = 0; i < DP / 16; ++i) {
            const int piece = i * 32 + lane, row = piece / (DP / 16), c = piece % (DP / 16);
            if (c * 16 < a.dim)
                copy16(dst + (u & 1 ? value_offset<DP>(row, c) : key_offset<DP>(row, c)), src + row * a.dim + c * 16, true);
        }
    };
#pragma unroll
    for (int u = 0; u < SLOTS - 1; ++u) {
        if (u < n_units) load_unit(u);
        copy_commit();
    }

    // the query rows, a warp a row: scaled to below 2^14 and laid out as the products read them (entry 16 t + e of a
    // segment of 64 belongs to thread t of the row's four; eight entries are 16 bytes)
    for (int r = warp; r < ROWS; r += WARPS) {
        float v[8] = {};
        if (r < n_rows && lane * 8 < a.dim) {
            const int row = row0 + r;
            const T* src = reinterpret_cast<const T*>(a.q) + (size_t)(first_tok + row / a.group) * a.q_stride +
                           (g * a.group + row % a.group) * a.dim + lane * 8;
            if (a.wide) load8(src, v);
            else {
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] = to_float(src[e]);
            }
        }
        float most = 0.0f;
        bool finite = true;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            most = fmaxf(most, fabsf(v[e]));
            finite = finite && fabsf(v[e]) < INFINITY;
        }
        most = warp_max(most);
        finite = __all_sync(0xffffffffu, finite);
        const int up = min(13 - ((int)(__float_as_uint(most) >> 23) - 127), 120);
        const float f = finite ? power_of_two(max(up, -126)) : 0.0f;
        if (lane == 0) q_scale[r] = finite ? power_of_two(-max(up, -126)) : __int_as_float(0x7fc00000);
        if (lane * 8 < DP) {
            const int s = lane >> 3, t = (lane >> 1) & 3, half = lane & 1;
            uint8_t* dst = smem + ((((r >> 3) * SEGS + s) * 2 + half) * 32 + (r & 7) * 4 + t) * 16;
            uint32_t hi[4], lo[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float x = finite ? v[2 * e] * f : 0.0f, y = finite ? v[2 * e + 1] * f : 0.0f;
                const __half2 h = __floats2half2_rn(x, y);
                hi[e] = *reinterpret_cast<const uint32_t*>(&h);
                if constexpr (PARTS == 2) lo[e] = pack_half(x - __low2float(h), y - __high2float(h));
            }
            *reinterpret_cast<uint4*>(dst) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
            if constexpr (PARTS == 2) *reinterpret_cast<uint4*>(dst + NT * SEGS * 1024) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
        }
    }
    __syncthreads();

    // this thread's query rows: 2 t4 and 2 t4 + 1 of every eight
    float qf[NT][2], m[NT][2], l[NT][2];
    int pos[NT][2];
    const float unit = a.cap > 0.0f ? (EXACT ? a.scale / a.cap : a.scale / a.cap * (2.0f * LOG2E)) : a.scale * LOG2E;
    const float c1 = a.cap * LOG2E, c2 = 2.0f * a.cap * LOG2E;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int r = nt * 8 + t4 * 2 + e;
            qf[nt][e] = q_scale[r] * unit;
            pos[nt][e] = r < n_rows ? pos0 + (row0 + r) / a.group : -1;
            m[nt][e] = -INFINITY;
            l[nt][e] = 0.0f;
        }
    float o[SEGS][4][NT][4];
#pragma unroll
    for (int s = 0; s < SEGS; ++s)
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) o[s][i][nt][0] = o[s][i][nt][1] = o[s][i][nt][2] = o[s][i][nt][3] = 0.0f;

    int unit_no = 0;
    auto next_unit = [&]() -> uint32_t {                       // waits for the next unit and asks for one more; its address
        copy_wait<SLOTS - 2>();
        __syncwarp();                                          // it has landed for all lanes; all are done with the one before
        if (unit_no + SLOTS - 1 < n_units) load_unit(unit_no + SLOTS - 1);
        copy_commit();
        return ring + (unit_no++ % SLOTS) * UNIT;
    };
    const uint32_t q_frag = smem_addr(smem) + lane * 16;

    for (int n = 0; n < n_tiles; ++n) {
        // (the scales of the next 32 tiles have been asked for when the first of them was, one or more tiles ago)
        if ((n & 31) == 0) { sk_c = sk_l; sv_c = sv_l; }
        const float sk = __shfl_sync(0xffffffffu, sk_c, n & 31), sv = __shfl_sync(0xffffffffu, sv_c, n & 31);
        const int key0 = (t_begin + warp + n * WARPS) * KT;
        uint32_t tile = next_unit();

        // S^T: keys 16 mt + g8 (+ 8) by query rows 2 t4 (+ 1)
        float z[2][NT][4];
#pragma unroll
        for (int mt = 0; mt < 2; ++mt)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) z[mt][nt][0] = z[mt][nt][1] = z[mt][nt][2] = z[mt][nt][3] = 0.0f;
#pragma unroll
        for (int s = 0; s < SEGS; ++s) {
            uint4 qb[PARTS][NT][2];
#pragma unroll
            for (int p = 0; p < PARTS; ++p)
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int h = 0; h < 2; ++h) qb[p][nt][h] = lds128(q_frag + (((p * NT + nt) * SEGS + s) * 2 + h) * 512);
#pragma unroll
            for (int mt = 0; mt < 2; ++mt) {
                const uint4 ka = lds128(tile + key_offset<DP>(16 * mt + g8, 4 * s + t4));
                const uint4 kb = lds128(tile + key_offset<DP>(16 * mt + g8 + 8, 4 * s + t4));
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const uint32_t wa = (&ka.x)[j] ^ FLIP, wb = (&kb.x)[j] ^ FLIP;
                    const uint32_t af[4] = {bytes_to_f16<FIRST>(wa), bytes_to_f16<FIRST>(wb), bytes_to_f16<SECOND>(wa), bytes_to_f16<SECOND>(wb)};
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int p = PARTS - 1; p >= 0; --p) {          // (the small parts first)
                            const uint4& q4 = qb[p][nt][j >> 1];
                            mma_f16(z[mt][nt], af, j & 1 ? q4.z : q4.x, j & 1 ? q4.w : q4.y);
                        }
                }
            }
        }

        // scores in log2 units, their maximum over the tile, weights relative to it
        const bool edge = key0 + KT - 1 > pos_lo || key0 < pos_hi - window + 1;
        float alpha[NT][2], coef[NT][2];
        uint32_t pf[PARTS][2][NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            float mt_max[2] = {-INFINITY, -INFINITY};
#pragma unroll
            for (int mt = 0; mt < 2; ++mt)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    float x = z[mt][nt][e] * (qf[nt][e & 1] * sk);
                    if (a.cap > 0.0f) x = EXACT ? c1 * tanhf(x) : fmaf(-c2, rcp(1.0f + ex2(x)), c1);
                    if (edge) {
                        const int back = pos[nt][e & 1] - (key0 + 16 * mt + g8 + (e & 2) * 4);
                        if (back < 0 || back >= window) x = -INFINITY;
                    }
                    z[mt][nt][e] = x;
                    mt_max[e & 1] = fmaxf(mt_max[e & 1], x);
                }
#pragma unroll
            for (int e = 0; e < 2; ++e) {
#pragma unroll
                for (int w = 4; w < 32; w *= 2) mt_max[e] = fmaxf(mt_max[e], __shfl_xor_sync(0xffffffffu, mt_max[e], w));
                const bool seen = mt_max[e] > -INFINITY;
                const float m_new = fmaxf(m[nt][e], mt_max[e]);
                alpha[nt][e] = m[nt][e] == m_new ? 1.0f : ex2(m[nt][e] - m_new);     // (2^(-inf) = 0; both -inf: 1)
                const float f = seen ? ex2(mt_max[e] - m_new) : 0.0f;
                const float base = seen ? mt_max[e] : 0.0f;
                float sum = 0.0f;
#pragma unroll
                for (int mt = 0; mt < 2; ++mt)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const float p = ex2(z[mt][nt][2 * h + e] - base);
                        z[mt][nt][2 * h + e] = p;
                        sum += p;
                    }
                m[nt][e] = m_new;
                l[nt][e] = fmaf(l[nt][e], alpha[nt][e], f * sum);
                coef[nt][e] = seen ? sv * f : 0.0f;
            }
#pragma unroll
            for (int mt = 0; mt < 2; ++mt)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const __half2 hi = __floats2half2_rn(z[mt][nt][2 * h], z[mt][nt][2 * h + 1]);
                    pf[0][mt][nt][h] = transpose8x8(*reinterpret_cast<const uint32_t*>(&hi));
                    if constexpr (PARTS == 2)
                        pf[1][mt][nt][h] = transpose8x8(pack_half(z[mt][nt][2 * h] - __low2float(hi), z[mt][nt][2 * h + 1] - __high2float(hi)));
                }
        }
        bool still = true;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) still = still && alpha[nt][0] == 1.0f && alpha[nt][1] == 1.0f;
        if (!__all_sync(0xffffffffu, still)) {
#pragma unroll
            for (int s = 0; s < SEGS; ++s)
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int e = 0; e < 4; ++e) o[s][i][nt][e] *= alpha[nt][e & 1];
        }

        // O^T: entries 64 s + 8 g8 + 2 i (+ 1) by query rows 2 t4 (+ 1)
        tile = next_unit();
#pragma unroll
        for (int s = 0; s < SEGS; ++s) {
            uint2 v[2][4];
#pragma unroll
            for (int ks = 0; ks < 2; ++ks)
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    const int row = 16 * ks + 2 * t4 + (c & 1) + (c >> 1) * 8;
                    v[ks][c] = lds64(tile + value_offset<DP>(row, 4 * s + (g8 >> 1)) + (g8 & 1) * 8);
                    v[ks][c].x ^= FLIP;
                    v[ks][c].y ^= FLIP;
                }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float add[NT][4];
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) add[nt][0] = add[nt][1] = add[nt][2] = add[nt][3] = 0.0f;
#pragma unroll
                for (int ks = 0; ks < 2; ++ks) {
                    uint32_t w[4];
#pragma unroll
                    for (int c = 0; c < 4; ++c) w[c] = i < 2 ? v[ks][c].x : v[ks][c].y;
                    // bytes 2i, 2i + 1 of two keys side by side
                    const uint32_t u01 = __byte_perm(w[0], w[1], i & 1 ? 0x7362 : 0x5140);
                    const uint32_t u23 = __byte_perm(w[2], w[3], i & 1 ? 0x7362 : 0x5140);
                    const uint32_t af[4] = {bytes_to_f16<FIRST>(u01), bytes_to_f16<SECOND>(u01), bytes_to_f16<FIRST>(u23), bytes_to_f16<SECOND>(u23)};
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int p = PARTS - 1; p >= 0; --p) mma_f16(add[nt], af, pf[p][ks][nt][0], pf[p][ks][nt][1]);
                }
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[s][i][nt][e] = fmaf(add[nt][e], coef[nt][e & 1], o[s][i][nt][e]);
            }
        }
    }
    copy_wait<0>();
    pdl_trigger();
    __syncthreads();

    // the four warps' results, then the cluster's, then (spans > 1) the launch's second kernel
    float* wo = reinterpret_cast<float*>(smem + SH::Q_BYTES);          // [WARPS][ROWS][PITCH]
    float* wml = wo + WARPS * ROWS * SH::PITCH;                        // [WARPS][ROWS][2]
    float* co = wml + WARPS * ROWS * 2;                                // [ROWS][PITCH]
    float* cml = co + ROWS * SH::PITCH;                                // [ROWS][2]
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            float sum = l[nt][e];
#pragma unroll
            for (int w = 4; w < 32; w *= 2) sum += __shfl_xor_sync(0xffffffffu, sum, w);
            const int r = nt * 8 + t4 * 2 + e;
            if (g8 == 0) {
                wml[(warp * ROWS + r) * 2] = m[nt][e];
                wml[(warp * ROWS + r) * 2 + 1] = sum;
            }
            if (r < n_rows) {
                float* dst = wo + (warp * ROWS + r) * SH::PITCH + 8 * g8;
#pragma unroll
                for (int s = 0; s < SEGS; ++s) {
                    *reinterpret_cast<float4*>(dst + 64 * s) = make_float4(o[s][0][nt][e], o[s][0][nt][e + 2], o[s][1][nt][e], o[s][1][nt][e + 2]);
                    *reinterpret_cast<float4*>(dst + 64 * s + 4) = make_float4(o[s][2][nt][e], o[s][2][nt][e + 2], o[s][3][nt][e], o[s][3][nt][e + 2]);
                }
            }
        }
    __syncthreads();
    const int d4 = a.dim >> 2;
    for (int it = threadIdx.x; it < n_rows * d4; it += THREADS) {
        const int r = it / d4, d = (it - r * d4) * 4;
        float most = -INFINITY;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) most = fmaxf(most, wml[(w * ROWS + r) * 2]);
        float sum = 0.0f;
        float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
        for (int w = 0; w < WARPS; ++w) {
            const float f = most > -INFINITY ? ex2(wml[(w * ROWS + r) * 2] - most) : 0.0f;
            const float4 x = *reinterpret_cast<const float4*>(wo + (w * ROWS + r) * SH::PITCH + d);
            sum = fmaf(wml[(w * ROWS + r) * 2 + 1], f, sum);
            acc.x = fmaf(x.x, f, acc.x); acc.y = fmaf(x.y, f, acc.y); acc.z = fmaf(x.z, f, acc.z); acc.w = fmaf(x.w, f, acc.w);
        }
        *reinterpret_cast<float4*>(co + r * SH::PITCH + d) = acc;
        if (d == 0) {
            cml[r * 2] = most;
            cml[r * 2 + 1] = sum;
        }
    }
    if (a.shares > 1) cluster_barrier();
    else __syncthreads();
    for (int it = share * THREADS + threadIdx.x; it < n_rows * d4; it += a.shares * THREADS) {
        const int r = it / d4, d = (it - r * d4) * 4;
        const uint32_t o_at = smem_addr(co + r * SH::PITCH + d), ml_at = smem_addr(cml + r * 2);
        float most = -INFINITY, sum = 0.0f;
        float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (a.shares == 1) {
            most = cml[r * 2];
            sum = cml[r * 2 + 1];
            acc = *reinterpret_cast<const float4*>(co + r * SH::PITCH + d);
        } else {
            for (int s = 0; s < a.shares; ++s) most = fmaxf(most, ld_cluster2(of_rank(ml_at, s)).x);
#pragma unroll 4
            for (int s = 0; s < a.shares; ++s) {
                const float2 ml = ld_cluster2(of_rank(ml_at, s));
                const float4 x = ld_cluster4(of_rank(o_at, s));
                const float f = most > -INFINITY ? ex2(ml.x - most) : 0.0f;
                sum = fmaf(ml.y, f, sum);
                acc.x = fmaf(x.x, f, acc.x); acc.y = fmaf(x.y, f, acc.y); acc.z = fmaf(x.z, f, acc.z); acc.w = fmaf(x.w, f, acc.w);
            }
        }
        const int row = row0 + r, tok = first_tok + row / a.group, head = g * a.group + row % a.group;
        if (q_scale[r] != q_scale[r]) acc.x = acc.y = acc.z = acc.w = pos0 + row / a.group >= 0 ? q_scale[r] : 0.0f;
        if (a.spans > 1) {
            const size_t at = ((size_t)tok * a.n_kv * a.group + head) * a.spans + span;
            *reinterpret_cast<float4*>(a.part_o + at * a.dim + d) = acc;
            if (d == 0) *reinterpret_cast<float2*>(a.part_ml + at * 2) = make_float2(most, sum);
        } else {
            const float inv = sum > 0.0f ? 1.0f / sum : (acc.x != acc.x ? 1.0f : 0.0f);
            T* dst = reinterpret_cast<T*>(a.out) + (size_t)tok * a.out_stride + head * a.dim + d;
            dst[0] = from_float<T>(acc.x * inv);
            dst[1] = from_float<T>(acc.y * inv);
            dst[2] = from_float<T>(acc.z * inv);
            dst[3] = from_float<T>(acc.w * inv);
        }
    }
    if (a.shares > 1) cluster_barrier();                       // nobody leaves while its results are being read
}

// Rows whose keys were shared by several clusters: a block of threads for every (token, head).
template <typename T>
__global__ void __launch_bounds__(64) attn_kv8_join_kernel(AttnArgs a) {
    pdl_trigger();
    pdl_wait();
    const int tok = blockIdx.x, head = blockIdx.y;
    if (tok >= a.cu_q[a.rows]) return;
    const size_t at = ((size_t)tok * a.n_kv * a.group + head) * a.spans;
    float most = -INFINITY, sum = 0.0f;
    for (int s = 0; s < a.spans; ++s) most = fmaxf(most, a.part_ml[(at + s) * 2]);
    const int d = threadIdx.x * 4;
    float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (d >= a.dim) return;
    for (int s = 0; s < a.spans; ++s) {
        const float f = most > -INFINITY ? ex2(a.part_ml[(at + s) * 2] - most) : 0.0f;
        const float4 x = *reinterpret_cast<const float4*>(a.part_o + (at + s) * a.dim + d);
        sum = fmaf(a.part_ml[(at + s) * 2 + 1], f, sum);
        acc.x = fmaf(x.x, f, acc.x); acc.y = fmaf(x.y, f, acc.y); acc.z = fmaf(x.z, f, acc.z); acc.w = fmaf(x.w, f, acc.w);
    }
    const float inv = sum > 0.0f ? 1.0f / sum : (acc.x != acc.x ? 1.0f : 0.0f);
    T* dst = reinterpret_cast<T*>(a.out) + (size_t)tok * a.out_stride + head * a.dim + d;
    dst[0] = from_float<T>(acc.x * inv);
    dst[1] = from_float<T>(acc.y * inv);
    dst[2] = from_float<T>(acc.z * inv);
    dst[3] = from_float<T>(acc.w * inv);
}

template <typename T, int DP, int NT>
int launch(const AttnArgs& a, cudaStream_t stream) {
    using SH = Shape<T, DP, NT>;
    static OncePerDevice raised;
    const int st = allow_shared_memory(attn_kv8_kernel<T, DP, NT>, SH::SMEM, raised);
    if (st) return st;
    cudaLaunchConfig_t cfg = {};
    const long long blocks = (long long)a.rows * a.row_tiles * a.spans * a.shares;
    if (blocks > 0x7fffffffll) return BROLM_ERR_TOO_LARGE;
    cfg.gridDim = dim3((unsigned)blocks, a.n_kv);
    cfg.blockDim = dim3(THREADS);
    cfg.dynamicSmemBytes = SH::SMEM;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = a.shares;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = pdl_enabled() ? 1 : 0;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    const int e = (int)cudaLaunchKernelEx(&cfg, attn_kv8_kernel<T, DP, NT>, a);
    if (e || a.spans == 1) return e;
    return launch_pdl(attn_kv8_join_kernel<T>, dim3(a.tokens, a.n_kv * a.group), dim3(64), 0, stream, a);
}

template <typename T, int NT>
int launch_dim(const AttnArgs& a, cudaStream_t stream) {
    if (a.dim <= 64) return launch<T, 64, NT>(a, stream);
    if (a.dim <= 128) return launch<T, 128, NT>(a, stream);
    if (a.dim <= 192) return launch<T, 192, NT>(a, stream);
    return launch<T, 256, NT>(a, stream);
}

}  // namespace

// shares (1 .. 8): blocks of a cluster that share a row's keys; spans: clusters that do, joined by a second launch through
// part_o [tokens * n_kv * group * spans * dim] and part_ml [.. * 2].
BROLM_API int brolm_attn_kv8(const void* q, int q_stride, void* out, int out_stride, int dtype, const void* cu_q,
                             const void* kv_len, const void* slots, const void* tables, const void* k_pages,
                             const void* v_pages, const void* k_scale, const void* v_scale, int tokens, int rows, int n_kv,
                             int group, int dim, int block, int n_blocks, int n_slots, int width, int ring, int window,
                             float scale, float cap, int max_q_len, int shares, int spans, void* part_o, void* part_ml,
                             cudaStream_t stream) {
    if (dtype != BROLM_F32 && dtype != BROLM_BF16) return BROLM_ERR_BAD_DTYPE;
    if (tokens < 0 || rows < 0 || n_kv <= 0 || group <= 0 || dim <= 0 || dim % 16 || block <= 0 || block % 32) return BROLM_ERR_BAD_SIZE;
    if (n_blocks <= 0 || n_slots <= 0 || width <= 0 || ring < 0 || ring % block || window < 0 || max_q_len <= 0) return BROLM_ERR_BAD_SIZE;
    if (shares < 1 || shares > 8 || spans < 1 || (spans > 1 && (!part_o || !part_ml))) return BROLM_ERR_BAD_SIZE;
    if (dim > MAX_DIM || block > MAX_BLOCK || (long long)n_kv * group > 65535 || (long long)max_q_len * group > 0x3fffffff) return BROLM_ERR_TOO_LARGE;
    if ((long long)n_blocks * block > 0x7fffffffll || tokens > 0x3fffffff) return BROLM_ERR_TOO_LARGE;
    if (((uintptr_t)k_pages | (uintptr_t)v_pages) & 15) return BROLM_ERR_ALIGNMENT;
    if (tokens == 0 || rows == 0) return BROLM_OK;
    const int size = dtype == BROLM_F32 ? 4 : 2, most = max_q_len * group, per = most <= 8 ? 8 : 16;
    const int wide = ((uintptr_t)q & 15) == 0 && (long long)q_stride * size % 16 == 0;
    AttnArgs a{q, out, q_stride, out_stride, (const int32_t*)cu_q, (const int32_t*)kv_len, (const int32_t*)slots,
               (const int32_t*)tables, (const int8_t*)k_pages, (const int8_t*)v_pages, (const float*)k_scale,
               (const float*)v_scale, tokens, rows, n_kv, group, dim, block, n_blocks, n_slots, width, ring, window, scale, cap,
               shares, spans, (most + per - 1) / per, wide, (float*)part_o, (float*)part_ml};
    if (dtype == BROLM_F32) return per == 8 ? launch_dim<float, 1>(a, stream) : launch_dim<float, 2>(a, stream);
    return per == 8 ? launch_dim<bf16, 1>(a, stream) : launch_dim<bf16, 2>(a, stream);
}
