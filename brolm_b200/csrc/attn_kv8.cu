// Attention over the cache in 8 bits (kv8.cuh): the newest tokens of every sequence against all that it holds, soft-capped,
// windowed, causal, with several query heads on a kv head.
//
//     z = scale * q . k,   cap tanh(z / cap),   key j visible from position p iff 0 <= p - j < window,
//     out = sum_j softmax_j(z) v_j,   zeros where a token sees no key.
//
// A row is a (token, query head of the group) pair; a block of threads owns 2 to 16 rows of one (sequence, kv head) and a
// share of its keys, and its four warps take tiles of 32 keys in turn.  A tile lies inside one cache block, so it has one
// scale for its keys and one for its values:
//
//     S^T [32 keys x rows] = K q^T,    m_t = max over the tile,  p = 2^(z - m_t),    O^T += s_v 2^(m_t - m) (V^T p)
//
// The weights of a tile are relative to the tile's own maximum and its sums are scaled in 32 bits when they join the row's,
// so blocks whose scales differ by any factor keep all their bits.  Both products run on mma.sync with the cache's numbers as
// the left operand, where the 16 rows of an instruction are keys or entries of a head and its 8 columns are query rows or
// their digits: whole numbers for up to eight rows, f16 for more (each at its kernel below).
//
// What bounds it is reading the cache, with 16 KB in flight a warp, 128 an SM: every warp keeps a ring of its own of key and
// value tiles on their way (cp.async, no barrier but its own), two blocks on an SM.  A launch takes 7 us more than its bytes:
// three round trips to memory before the first product, the warps' and the cluster's merge behind the last.
//
// The shares of a row's keys are joined inside the launch: they form a cluster, whose blocks read each other's partial
// results out of shared memory.  Where that is not enough, or where clusters are dealt out over sequences of different
// lengths, the clusters' results are joined by a second launch (attn_kv8_join.cuh).  Nothing is kept between launches.
#include "attn_kv8_join.cuh"

#include <cuda_fp16.h>

namespace {

using namespace kv8;

constexpr int WARPS = 4, THREADS = 32 * WARPS;
constexpr int MAX_SHARES = 8;             // blocks of a cluster
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
    int dealt;                            // 0, or: clusters dealt out over the sequences by their lengths (then spans = 1)
    float *part_o, *part_ml;              // [token][head][span][dim] and [..][2] where spans > 1
    int2* plan;                           // dealt: where the parts of a (token, head) begin, and how many there are
};

__device__ __forceinline__ uint32_t smem_addr(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ float rcp(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// cap tanh(x) of float32 scores, in log2 units.  Scores are mostly well below the cap, and there the series to x^13 is as exact
// as a float (|x| up to 0.4: the next term is 2e-9).
__device__ __forceinline__ float near_tanh(float x) {
    const float y = x * x;
    float p = fmaf(21844.0f / 6081075.0f, y, -1382.0f / 155925.0f);
    p = fmaf(p, y, 62.0f / 2835.0f);
    p = fmaf(p, y, -17.0f / 315.0f);
    p = fmaf(p, y, 2.0f / 15.0f);
    p = fmaf(p, y, -1.0f / 3.0f);
    return fmaf(x * y, p, x);
}
template <int N>
__device__ __forceinline__ void cap_exactly(float (&x)[N], float c1) {
    float far = 0.0f;
#pragma unroll
    for (int i = 0; i < N; ++i) far = fmaxf(far, fabsf(x[i]));
    if (__all_sync(0xffffffffu, far <= 0.4f)) {
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] = c1 * near_tanh(x[i]);
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] = c1 * tanhf(x[i]);
    }
}
__device__ __forceinline__ void cluster_barrier() {
    asm volatile("barrier.cluster.arrive.aligned;\nbarrier.cluster.wait.aligned;\n" ::: "memory");
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

__device__ __forceinline__ int ld_now(const int32_t* p) {
    int v;
    asm volatile("ld.global.b32 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
    return v;
}
// Eight entries of a row, asked for now and looked at later; zeros where nothing was asked for.
template <typename T>
struct Eight {
    static constexpr int PIECES = sizeof(T) / 2;               // of 16 bytes
    uint4 raw[PIECES];
    __device__ __forceinline__ Eight() {
#pragma unroll
        for (int i = 0; i < PIECES; ++i) raw[i] = make_uint4(0, 0, 0, 0);
    }
    __device__ __forceinline__ void fetch(const T* p, bool wide) {
        if (wide) {
#pragma unroll
            for (int i = 0; i < PIECES; ++i)
                asm volatile("ld.global.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(raw[i].x), "=r"(raw[i].y), "=r"(raw[i].z), "=r"(raw[i].w)
                             : "l"(reinterpret_cast<const uint4*>(p) + i) : "memory");
        } else {
            alignas(16) T v[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = p[e];
#pragma unroll
            for (int i = 0; i < PIECES; ++i) raw[i] = reinterpret_cast<const uint4*>(v)[i];
        }
    }
    __device__ __forceinline__ void numbers(float (&v)[8]) const {
#pragma unroll
        for (int i = 0; i < 4 * PIECES; ++i) {
            const uint32_t w = (&raw[i / 4].x)[i % 4];
            if constexpr (PIECES == 2) v[i] = __uint_as_float(w);
            else {
                v[2 * i] = __uint_as_float(w << 16);
                v[2 * i + 1] = __uint_as_float(w & 0xffff0000u);
            }
        }
    }
};

// What a block works on: rows of one sequence and kv head, and the tiles [t_begin, t_end) of their keys.
struct Item {
    int share, span, spans, part0, g, first_tok, row0, n_rows, pos0, pos_lo, pos_hi, slot, t_begin, t_end;
};
// Sequences of different lengths: the launch's clusters are dealt out over them, so that no cluster has more than w rounds of
// its warps' tiles, w the least for which there are enough.  Every warp finds that out for itself: which sequence its
// cluster c is given, the how manieth of its clusters it is and of how many (none where clusters are left over).
constexpr int MAX_DEALT = 128;                                 // sequences of such a launch
__device__ __forceinline__ void deal(const AttnArgs& a, int c, Item& it, int& end_tok, int& kv_len) {
    constexpr int PER = MAX_DEALT / 32;
    const int lane = threadIdx.x & 31, round = WARPS * a.shares;
    int first[PER], end[PER], len[PER], slot[PER], work[PER];
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        const int b = lane + 32 * j;
        first[j] = end[j] = len[j] = slot[j] = 0;
        if (b < a.rows) {
            first[j] = ld_now(a.cu_q + b);
            end[j] = ld_now(a.cu_q + b + 1);
            len[j] = ld_now(a.kv_len + b);
            slot[j] = ld_now(a.slots + b);
        }
    }
    int total = 0, most = 1;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        const int pos0 = len[j] - (min(end[j], a.tokens) - first[j]), from = a.window > 0 ? max(0, pos0 - a.window + 1) / KT : 0;
        work[j] = lane + 32 * j < a.rows ? min(1 << 20, max(1, ((max(0, len[j] - 1) / KT - from + 1) + round - 1) / round)) : 0;
        total += work[j];
        most = max(most, work[j]);
    }
    total = __reduce_add_sync(0xffffffffu, total);
    most = __reduce_max_sync(0xffffffffu, most);
    int lo = min(most, (total + a.dealt - 1) / a.dealt), hi = most;
    while (lo < hi) {                                          // (hi is enough: there are no fewer clusters than sequences)
        const int w = (lo + hi) >> 1;
        int need = 0;
#pragma unroll
        for (int j = 0; j < PER; ++j) need += (work[j] + w - 1) / w;
        if (__reduce_add_sync(0xffffffffu, need) <= a.dealt) hi = w;
        else lo = w + 1;
    }
    it.first_tok = it.slot = -1;
    it.span = 0;
    end_tok = kv_len = 0;
    int before = 0;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        if (32 * j >= a.rows) break;
        const int mine = (work[j] + lo - 1) / lo;
        int upto = mine;
#pragma unroll
        for (int d = 1; d < 32; d *= 2) {
            const int x = __shfl_up_sync(0xffffffffu, upto, d);
            if (lane >= d) upto += x;
        }
        const int at = c - (before + upto - mine);
        const uint32_t found = __ballot_sync(0xffffffffu, at >= 0 && at < mine);
        if (found) {
            const int from = __ffs(found) - 1;
            it.span = __shfl_sync(0xffffffffu, at, from);
            it.spans = __shfl_sync(0xffffffffu, mine, from);
            it.first_tok = __shfl_sync(0xffffffffu, first[j], from);
            end_tok = __shfl_sync(0xffffffffu, end[j], from);
            kv_len = __shfl_sync(0xffffffffu, len[j], from);
            it.slot = __shfl_sync(0xffffffffu, slot[j], from);
        }
        before += __shfl_sync(0xffffffffu, upto, 31);
    }
}

// Three round trips to memory lie before the first product: what the sequence is; its row of the tables and the queries;
// the tiles and their scales.  What one trip can fetch is asked for before anything of it is looked at.
template <int ROWS>
__device__ __forceinline__ Item find_item(const AttnArgs& a) {
    Item it;
    it.share = blockIdx.x % a.shares;
    int rest = blockIdx.x / a.shares, end_tok, kv_len;
    it.g = blockIdx.y;
    it.spans = a.spans;
    if (a.dealt > 0) {
        const int c = rest / a.row_tiles;
        it.row0 = (rest - c * a.row_tiles) * ROWS;
        it.part0 = (rest * a.n_kv + it.g) * ROWS;
        deal(a, c, it, end_tok, kv_len);
    } else {
        it.span = rest % a.spans;
        rest /= a.spans;
        const int b = rest / a.row_tiles;
        it.row0 = (rest - b * a.row_tiles) * ROWS;
        it.first_tok = ld_now(a.cu_q + b);
        end_tok = ld_now(a.cu_q + b + 1);
        kv_len = ld_now(a.kv_len + b);
        it.slot = ld_now(a.slots + b);
    }
    const int n_tok = min(end_tok, a.tokens) - it.first_tok;
    it.n_rows = it.first_tok < 0 ? 0 : (int)min((long long)ROWS, (long long)n_tok * a.group - it.row0);
    it.pos0 = kv_len - n_tok;                                  // position of the sequence's first new token
    it.pos_lo = it.pos0 + it.row0 / a.group;
    it.pos_hi = it.pos0 + (it.row0 + it.n_rows - 1) / a.group;
    it.t_begin = it.t_end = 0;
    if (it.n_rows > 0 && it.pos_hi >= 0 && it.slot >= 0 && it.slot < a.n_slots) {
        const int t_lo = a.window > 0 ? max(0, it.pos_lo - a.window + 1) / KT : 0, t_hi = it.pos_hi / KT;
        const int parts = a.shares * it.spans, per = (t_hi - t_lo + parts) / parts;
        it.t_begin = t_lo + (it.span * a.shares + it.share) * per;
        it.t_end = min(t_hi + 1, it.t_begin + per);
    }
    return it;
}

// A warp's tiles of keys and values on their way into its part of shared memory.  A tile whose place in the tables is none of
// the cache's has the value scale GONE, and nobody sees its keys.
constexpr float GONE = -1.0f;
template <int DP, int SLOTS>
struct TileRing {
    static constexpr int UNIT = KT * DP;                       // a key or value tile
    const AttnArgs& a;
    const int32_t* table;
    uint32_t base;
    int g, lane, t0, n_tiles, n_units, unit_no;
    long long place_l;                                         // of the 32 tiles that are being asked for, lane by lane: where they lie
    float sk_l, sv_l, sk_c, sv_c;                              // .. their scales, and those of the tiles that are being multiplied

    __device__ __forceinline__ TileRing(const AttnArgs& args, const Item& it, uint32_t smem, int warp, int lane_) : a(args) {
        table = a.tables + (size_t)max(it.slot, 0) * a.width;
        base = smem + warp * SLOTS * UNIT;
        g = it.g;
        lane = lane_;
        t0 = it.t_begin + warp;                                // the block's warps take tiles in turn
        n_tiles = t0 < it.t_end ? (it.t_end - t0 + WARPS - 1) / WARPS : 0;
        n_units = 2 * n_tiles;
        unit_no = 0;
        sk_c = sv_c = 0.0f;
    }
    __device__ __forceinline__ void look_up(int n) {
        place_l = 0;
        sk_l = sv_l = 0.0f;
        if (n + lane < n_tiles) {
            const long long key = (long long)(t0 + (n + lane) * WARPS) * KT;
            const int place = a.ring > 0 ? (int)(key % a.ring) : (int)key, e = place / a.block;
            int id = e < a.width ? table[e] : -1;
            const bool gone = id < 0 || id >= a.n_blocks;      // (never followed out of the cache: its tile is read elsewhere)
            if (gone) id = 0;
            const size_t bh = (size_t)id * a.n_kv + g;
            place_l = (long long)bh * a.block + (place - e * a.block);
            sv_l = GONE;
            if (!gone) {
                sk_l = a.k_scale[bh];
                sv_l = a.v_scale[bh];                          // (nothing waits for the scales before their first use)
            }
        }
    }
    __device__ __forceinline__ void load(int u) {              // key tile u / 2 or value tile u / 2 into slot u % SLOTS
        const int n = u >> 1;
        if (u > 0 && (u & 63) == 0) look_up(n);
        const long long place = __shfl_sync(0xffffffffu, place_l, n & 31);
        const int8_t* src = (u & 1 ? a.v_pages : a.k_pages) + place * a.dim;
        const uint32_t dst = base + (u % SLOTS) * UNIT;
#pragma unroll
        for (int i = 0; i < DP / 16; ++i) {
            const int piece = i * 32 + lane, row = piece / (DP / 16), c = piece % (DP / 16);
            if (c * 16 < a.dim)
                copy16(dst + (u & 1 ? value_offset<DP>(row, c) : key_offset<DP>(row, c)), src + row * a.dim + c * 16, true);
        }
    }
    __device__ __forceinline__ void start() {
        look_up(0);
#pragma unroll
        for (int u = 0; u < SLOTS - 1; ++u) {
            if (u < n_units) load(u);
            copy_commit();
        }
    }
    __device__ __forceinline__ uint32_t next() {               // waits for the next unit and asks for one more; its address
        copy_wait<SLOTS - 2>();
        __syncwarp();                                          // it has landed for all lanes; all are done with the one before
        if (unit_no + SLOTS - 1 < n_units) load(unit_no + SLOTS - 1);
        copy_commit();
        return base + (unit_no++ % SLOTS) * UNIT;
    }
    // (the scales of the next 32 tiles have been asked for when the first of them was, one or more tiles ago)
    __device__ __forceinline__ float2 scales(int n) {
        if ((n & 31) == 0) {
            const bool bad = sk_l != sk_l || sv_l != sv_l;     // a NaN block: scores of zero, values of NaN
            sk_c = bad ? 0.0f : sk_l;
            sv_c = bad ? __int_as_float(0x7fc00000) : sv_l;
        }
        return make_float2(__shfl_sync(0xffffffffu, sk_c, n & 31), __shfl_sync(0xffffffffu, sv_c, n & 31));
    }
};

// The queries of a block's rows, a warp a row, eight entries a lane.
template <typename T, int ROWS>
__device__ __forceinline__ void fetch_queries(const AttnArgs& a, const Item& it, int warp, int lane, Eight<T> (&raw)[(ROWS + WARPS - 1) / WARPS]) {
#pragma unroll
    for (int j = 0; j < (ROWS + WARPS - 1) / WARPS; ++j) {
        const int r = warp + j * WARPS, row = it.row0 + r;
        if (r < it.n_rows && lane * 8 < a.dim)
            raw[j].fetch(reinterpret_cast<const T*>(a.q) + (size_t)(it.first_tok + row / a.group) * a.q_stride +
                         (it.g * a.group + row % a.group) * a.dim + lane * 8, a.wide);
    }
}
// The exponent that brings a row's largest number to [2^top, 2^(top + 1)), within what a float's exponent can say; a row
// that is not finite gets zeros and the scale NaN.
__device__ __forceinline__ int row_exponent(float (&v)[8], int top, bool& finite) {
    float most = 0.0f;
    finite = true;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        most = fmaxf(most, fabsf(v[e]));
        finite = finite && fabsf(v[e]) < INFINITY;
    }
    most = warp_max(most);
    finite = __all_sync(0xffffffffu, finite);
    if (!finite) {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = 0.0f;
    }
    return max(min(top + 127 - (int)(__float_as_uint(most) >> 23), 120), -126);
}

// What the warps have left in shared memory (wo [WARPS][ROWS][pitch] sums, wml [WARPS][ROWS][2] maxima in log2 units and
// sums of weights) is joined over the block, then over the cluster; the result goes to the output, or, where several
// clusters share the keys, to memory for the second launch.  co, cml: room for a block's own result.
template <typename T, int ROWS, int PITCH>
__device__ __forceinline__ void merge(const AttnArgs& a, const Item& it, const float* wo, const float* wml, float* co, float* cml,
                                      const float* q_scale) {
    const int d4 = a.dim >> 2;
    for (int i = threadIdx.x; i < it.n_rows * d4; i += THREADS) {
        const int r = i / d4, d = (i - r * d4) * 4;
        float most = -INFINITY;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) most = fmaxf(most, wml[(w * ROWS + r) * 2]);
        float sum = 0.0f;
        float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
        for (int w = 0; w < WARPS; ++w) {
            const float f = most > -INFINITY ? ex2(wml[(w * ROWS + r) * 2] - most) : 0.0f;
            add_part(acc, sum, *reinterpret_cast<const float4*>(wo + (w * ROWS + r) * PITCH + d), wml[(w * ROWS + r) * 2 + 1], f);
        }
        *reinterpret_cast<float4*>(co + r * PITCH + d) = acc;
        if (d == 0) {
            cml[r * 2] = most;
            cml[r * 2 + 1] = sum;
        }
    }
    if (a.shares > 1) cluster_barrier();
    else __syncthreads();
    for (int i = it.share * THREADS + threadIdx.x; i < it.n_rows * d4; i += a.shares * THREADS) {
        const int r = i / d4, d = (i - r * d4) * 4;
        float most = -INFINITY, sum = 0.0f;
        float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (a.shares == 1) {
            most = cml[r * 2];
            sum = cml[r * 2 + 1];
            acc = *reinterpret_cast<const float4*>(co + r * PITCH + d);
        } else {
            const uint32_t o_at = smem_addr(co + r * PITCH + d), ml_at = smem_addr(cml + r * 2);
            float2 ml[MAX_SHARES];
            float4 x[MAX_SHARES];
#pragma unroll
            for (int s = 0; s < MAX_SHARES; ++s)
                if (s < a.shares) {
                    ml[s] = ld_cluster2(of_rank(ml_at, s));
                    x[s] = ld_cluster4(of_rank(o_at, s));
                }
#pragma unroll
            for (int s = 0; s < MAX_SHARES; ++s)
                if (s < a.shares) most = fmaxf(most, ml[s].x);
#pragma unroll
            for (int s = 0; s < MAX_SHARES; ++s)
                if (s < a.shares) add_part(acc, sum, x[s], ml[s].y, most > -INFINITY ? ex2(ml[s].x - most) : 0.0f);
        }
        const int row = it.row0 + r, tok = it.first_tok + row / a.group, head = it.g * a.group + row % a.group;
        if (q_scale[r] != q_scale[r]) acc.x = acc.y = acc.z = acc.w = it.pos0 + row / a.group >= 0 ? q_scale[r] : 0.0f;
        if (a.dealt > 0 && it.span == 0 && d == 0)
            a.plan[(size_t)tok * a.n_kv * a.group + head] = make_int2(it.part0 + r, it.spans);
        if (it.spans > 1) {
            const size_t at = a.dealt > 0 ? (size_t)it.part0 + r : ((size_t)tok * a.n_kv * a.group + head) * a.spans + it.span;
            *reinterpret_cast<float4*>(a.part_o + at * a.dim + d) = acc;
            if (d == 0) *reinterpret_cast<float2*>(a.part_ml + at * 2) = make_float2(most, sum);
        } else {
            store_row<T>(a.out, a.out_stride, a.dim, tok, head, d, acc, sum);
        }
    }
    if (a.shares > 1) cluster_barrier();                       // nobody leaves while its results are being read
}

// --- up to eight rows: products of whole numbers -------------------------------------------------------------------------
//
// With few rows most of an instruction's columns would be empty and turning the cache's bytes into f16 is what a warp
// spends its time on (1,380 instructions a tile of 32 keys of 256 entries, 2,870 cycles of a warp that has a scheduler to
// itself).  Here the bytes are multiplied as they are (m16n8k32, whole sums), and what is multiplied with them is whole
// numbers too, a digit of 8 bits a column:
//
//     q 2^s = sum_i d_i 256^(3 - i), four signed digits (30 bits of the row's largest number), two rows an instruction;
//     p     = sum_i e_i 256^-i,      two unsigned digits (bfloat16: 16 bits of the tile's largest weight, four rows an
//                                    instruction) or four (float32: 31 bits, two rows).
//
// A thread has two neighbouring digits' sums, joins them as whole numbers and then in floats.  Both stay below 2^31: scores are
// sums over a head's entries of products up to 127 * 128, the higher digit's times 256 (127 * 128 * 256 * 257 = 1.07e9 at 256
// entries), results are sums over a tile's 32 keys of products up to 127 * 255 (127 * 255 * 32 * 257 = 2.7e8).  The keys
// are read as the instruction wants them; of the values, four keys' bytes of an entry are gathered into a word by eight byte
// permutations for sixteen bytes.
//
// 8 sequences of 8,192 keys, 4 kv heads of 256, two query heads each, bfloat16: 29.2 us, 4.6 TB/s, with 28 % of the issue
// slots and 7 % of the tensor pipe in use (f16 products: 30.2, and for 16 sequences of unequal lengths under a window 45.6
// where these took 32.6 with the same shares); 1 of 1,280: 7.6 us, which is round trips.  A fixed number of blocks that walk
// runs of equal length over all sequences took 38.8: each further sequence of a block costs 5 us of round trips.
__device__ __forceinline__ void mma_s8(int (&d)[4], const uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_s8u8(int (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.u8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
                 : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "r"(0));
}

template <typename T, int DP, int ROWS>
struct FewShape {
    static constexpr int SEGS = DP / 64;
    static constexpr int SLOTS = DP == 256 ? 3 : DP == 192 ? 4 : DP == 128 ? 6 : 8;
    static constexpr int RING = WARPS * SLOTS * KT * DP;
    static constexpr int QT = ROWS / 2;                                    // tiles of the first product: two rows each
    static constexpr int PT = sizeof(T) == 4 ? QT : (QT + 1) / 2;          // .. of the second
    static constexpr int Q_BYTES = QT * SEGS * 512;
    static constexpr int PITCH = DP + 4;
    static constexpr int MERGE = (WARPS * ROWS * PITCH + WARPS * ROWS * 2 + ROWS * PITCH + ROWS * 2) * 4;
    static constexpr int SMEM = Q_BYTES + (RING > MERGE ? RING : MERGE);
};

template <typename T, int DP, int ROWS>
__global__ void __launch_bounds__(THREADS, 2) attn_kv8_few_kernel(AttnArgs a) {
    using SH = FewShape<T, DP, ROWS>;
    constexpr int SEGS = SH::SEGS, QT = SH::QT, PT = SH::PT, PER_WARP = (ROWS + WARPS - 1) / WARPS;
    constexpr bool EXACT = sizeof(T) == 4;
    static_assert(127ll * 128 * DP * 257 < 1ll << 31 && 127ll * 255 * KT * 257 < 1ll << 31, "joined digits' sums");
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ float q_scale[ROWS];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g8 = lane >> 2, t4 = lane & 3;
    pdl_wait();
    const Item it = find_item<ROWS>(a);
    if (it.n_rows <= 0) return;                                // (the whole cluster)
    Eight<T> raw[PER_WARP];
    fetch_queries<T, ROWS>(a, it, warp, lane, raw);
    TileRing<DP, SH::SLOTS> tiles(a, it, smem_addr(smem) + SH::Q_BYTES, warp, lane);
    tiles.start();

    // digit i of row r is column 4 (r % 2) + i of tile r / 2; a column's entries 16 t .. 16 t + 15 of a segment of 64 are
    // read by thread t of the column's four
#pragma unroll
    for (int j = 0; j < PER_WARP; ++j) {
        const int r = warp + j * WARPS;
        if (r >= ROWS) break;
        float v[8];
        raw[j].numbers(v);
        bool finite;
        const int up = row_exponent(v, 29, finite);
        const float f = power_of_two(up);
        if (lane == 0) q_scale[r] = finite ? power_of_two(-up) : __int_as_float(0x7fc00000);
        if (lane * 8 < DP) {
            uint32_t dig[4][2] = {};
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                int x = __float2int_rn(v[e] * f);
#pragma unroll
                for (int i = 3; i >= 0; --i) {
                    const int low = (int)(int8_t)(x & 255);
                    dig[i][e >> 2] |= (uint32_t)(low & 255) << (8 * (e & 3));
                    x = (x - low) >> 8;
                }
            }
            const int s = lane >> 3, t = (lane >> 1) & 3;
#pragma unroll
            for (int i = 0; i < 4; ++i)
                *reinterpret_cast<uint2*>(smem + ((r >> 1) * SEGS + s) * 512 + ((4 * (r & 1) + i) * 4 + t) * 16 + (lane & 1) * 8) =
                    make_uint2(dig[i][0], dig[i][1]);
        }
    }
    __syncthreads();

    // this thread's row of a tile: 2 q + t4 / 2 (and the two low digits of its scores where t4 is odd)
    const float unit = a.cap > 0.0f ? (EXACT ? a.scale / a.cap : a.scale / a.cap * (2.0f * LOG2E)) : a.scale * LOG2E;
    const float c1 = a.cap * LOG2E, c2 = 2.0f * a.cap * LOG2E;
    const int window = a.window > 0 ? a.window : ALL_KEYS;
    const float weight = t4 & 1 ? 1.0f : 65536.0f;
    float qf[QT], m[QT], l[QT];
    int pos[QT];
#pragma unroll
    for (int q = 0; q < QT; ++q) {
        const int r = 2 * q + (t4 >> 1);
        qf[q] = q_scale[r] * unit;
        pos[q] = r < it.n_rows ? it.pos0 + (it.row0 + r) / a.group : -1;
        m[q] = -INFINITY;
        l[q] = 0.0f;
    }
    float o[SEGS][4][PT][2];
#pragma unroll
    for (int s = 0; s < SEGS; ++s)
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int p = 0; p < PT; ++p) o[s][i][p][0] = o[s][i][p][1] = 0.0f;
    const uint32_t q_frag = smem_addr(smem) + lane * 16;

    for (int n = 0; n < tiles.n_tiles; ++n) {
        const float2 sc = tiles.scales(n);
        const int key0 = sc.y == GONE ? NOWHERE : (tiles.t0 + n * WARPS) * KT;
        uint32_t tile = tiles.next();

        // S^T: keys 16 mt + g8 (+ 8) by digits 2 t4 (+ 1); two sums where there are few, so that one need not wait for the last
        constexpr int SUMS = QT == 1 ? 2 : 1;
        int zs[SUMS][2][QT][4];
#pragma unroll
        for (int c = 0; c < SUMS; ++c)
#pragma unroll
            for (int mt = 0; mt < 2; ++mt)
#pragma unroll
                for (int q = 0; q < QT; ++q) zs[c][mt][q][0] = zs[c][mt][q][1] = zs[c][mt][q][2] = zs[c][mt][q][3] = 0;
#pragma unroll
        for (int s = 0; s < SEGS; ++s) {
            uint4 qb[QT];
#pragma unroll
            for (int q = 0; q < QT; ++q) qb[q] = lds128(q_frag + (q * SEGS + s) * 512);
#pragma unroll
            for (int mt = 0; mt < 2; ++mt) {
                const uint4 ka = lds128(tile + key_offset<DP>(16 * mt + g8, 4 * s + t4));
                const uint4 kb = lds128(tile + key_offset<DP>(16 * mt + g8 + 8, 4 * s + t4));
#pragma unroll
                for (int q = 0; q < QT; ++q) {
                    mma_s8(zs[0][mt][q], ka.x, kb.x, ka.y, kb.y, qb[q].x, qb[q].y);
                    mma_s8(zs[SUMS - 1][mt][q], ka.z, kb.z, ka.w, kb.w, qb[q].z, qb[q].w);
                }
            }
        }

        // scores in log2 units, their maximum over the tile, weights relative to it
        const bool edge = key0 + KT - 1 > it.pos_lo || key0 < it.pos_hi - window + 1;
        float alpha[QT], coef[QT];
        uint32_t digits[QT][2][2];                             // two digits of a weight, of keys 16 mt + 8 h + g8, at bits 0 and 16
#pragma unroll
        for (int q = 0; q < QT; ++q) {
            const float to_z = qf[q] * sc.x;
            float z[2][2], top = -INFINITY;
#pragma unroll
            for (int mt = 0; mt < 2; ++mt)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    int hi = zs[0][mt][q][2 * h], lo = zs[0][mt][q][2 * h + 1];
                    if constexpr (SUMS == 2) { hi += zs[1][mt][q][2 * h]; lo += zs[1][mt][q][2 * h + 1]; }
                    float x = (float)(hi * 256 + lo) * weight;
                    x += __shfl_xor_sync(0xffffffffu, x, 1);
                    z[mt][h] = x * to_z;
                }
            if (EXACT && a.cap > 0.0f) cap_exactly(reinterpret_cast<float(&)[4]>(z), c1);
#pragma unroll
            for (int mt = 0; mt < 2; ++mt)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    float x = z[mt][h];
                    if (!EXACT && a.cap > 0.0f) x = fmaf(-c2, rcp(1.0f + ex2(x)), c1);
                    if (edge) {
                        const int back = pos[q] - (key0 + 16 * mt + 8 * h + g8);
                        if (back < 0 || back >= window) x = -INFINITY;
                    }
                    z[mt][h] = x;
                    top = fmaxf(top, x);
                }
#pragma unroll
            for (int w = 4; w < 32; w *= 2) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, w));
            const bool seen = top > -INFINITY;
            const float m_new = fmaxf(m[q], top), f = seen ? ex2(top - m_new) : 0.0f, from = seen ? top : 0.0f;
            alpha[q] = m[q] == m_new ? 1.0f : ex2(m[q] - m_new);                 // (2^(-inf) = 0; both -inf: 1)
            float sum = 0.0f;
#pragma unroll
            for (int mt = 0; mt < 2; ++mt)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const float p = ex2(z[mt][h] - from);
                    sum += p;
                    uint32_t two;                              // float32: digits 0, 1 or (t4 odd) 2, 3
                    if constexpr (EXACT) {
                        const uint32_t whole = __float2uint_rn(p * 2147483648.0f);
                        two = t4 & 1 ? whole & 0xffffu : whole >> 16;
                    } else {
                        two = __float2uint_rn(p * 65535.0f);
                    }
                    digits[q][mt][h] = __byte_perm(two, 0, 0x4041);              // the high one first
                }
            m[q] = m_new;
            l[q] = fmaf(l[q], alpha[q], f * sum);
            coef[q] = seen ? sc.y * f * (EXACT ? weight * (1.0f / 2147483648.0f) : 1.0f / 65535.0f) : 0.0f;
        }
        // as the second product wants them: digit (column) g8 of keys 2 t4, 2 t4 + 1, 2 t4 + 8, 2 t4 + 9 in a word.  bfloat16:
        // threads with even t4 give the rows of tile 2 p, those with odd t4 the rows of tile 2 p + 1
        uint32_t pf[PT][2];
        float pa[PT], pc[PT];
#pragma unroll
        for (int p = 0; p < PT; ++p) {
            const int q0 = EXACT ? p : 2 * p, q1 = EXACT ? p : 2 * p + 1;
            const bool other = !EXACT && (t4 & 1);
            pa[p] = other ? (q1 < QT ? alpha[q1 < QT ? q1 : 0] : 1.0f) : alpha[q0];
            pc[p] = other ? (q1 < QT ? coef[q1 < QT ? q1 : 0] : 0.0f) : coef[q0];
#pragma unroll
            for (int mt = 0; mt < 2; ++mt) {
                uint32_t t[2];
#pragma unroll
                for (int h = 0; h < 2; ++h)
                    t[h] = transpose8x8(other ? (q1 < QT ? digits[q1 < QT ? q1 : 0][mt][h] : 0u) : digits[q0][mt][h]);
                pf[p][mt] = __byte_perm(t[0], t[1], 0x6420);
            }
        }
        bool still = true;
#pragma unroll
        for (int q = 0; q < QT; ++q) still = still && alpha[q] == 1.0f;
        if (!__all_sync(0xffffffffu, still)) {
#pragma unroll
            for (int s = 0; s < SEGS; ++s)
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int p = 0; p < PT; ++p) {
                        o[s][i][p][0] *= pa[p];
                        o[s][i][p][1] *= pa[p];
                    }
        }

        // O^T: entries 64 s + 8 g8 + 2 i (+ 1) by digits 2 t4 (+ 1)
        tile = tiles.next();
#pragma unroll
        for (int s = 0; s < SEGS; ++s) {
            uint2 v[2][4];
#pragma unroll
            for (int ks = 0; ks < 2; ++ks)
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    const int row = 16 * ks + 2 * t4 + (c & 1) + (c >> 1) * 8;
                    v[ks][c] = lds64(tile + value_offset<DP>(row, 4 * s + (g8 >> 1)) + (g8 & 1) * 8);
                }
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                uint32_t w[2][4];                              // entries 8 g8 + 4 half + 0 .. 3, four keys each
#pragma unroll
                for (int ks = 0; ks < 2; ++ks) {
                    const uint32_t w0 = half ? v[ks][0].y : v[ks][0].x, w1 = half ? v[ks][1].y : v[ks][1].x;
                    const uint32_t w2 = half ? v[ks][2].y : v[ks][2].x, w3 = half ? v[ks][3].y : v[ks][3].x;
                    const uint32_t x0 = __byte_perm(w0, w1, 0x5140), x1 = __byte_perm(w0, w1, 0x7362);
                    const uint32_t y0 = __byte_perm(w2, w3, 0x5140), y1 = __byte_perm(w2, w3, 0x7362);
                    w[ks][0] = __byte_perm(x0, y0, 0x5410);
                    w[ks][1] = __byte_perm(x0, y0, 0x7632);
                    w[ks][2] = __byte_perm(x1, y1, 0x5410);
                    w[ks][3] = __byte_perm(x1, y1, 0x7632);
                }
#pragma unroll
                for (int i2 = 0; i2 < 2; ++i2) {
                    const uint32_t af[4] = {w[0][2 * i2], w[0][2 * i2 + 1], w[1][2 * i2], w[1][2 * i2 + 1]};
#pragma unroll
                    for (int p = 0; p < PT; ++p) {
                        int d[4];
                        mma_s8u8(d, af, pf[p][0], pf[p][1]);
                        float (&acc)[2] = o[s][2 * half + i2][p];
                        acc[0] = fmaf((float)(d[0] * 256 + d[1]), pc[p], acc[0]);
                        acc[1] = fmaf((float)(d[2] * 256 + d[3]), pc[p], acc[1]);
                    }
                }
            }
        }
    }
    copy_wait<0>();
    pdl_trigger();
    __syncthreads();

    float* wo = reinterpret_cast<float*>(smem + SH::Q_BYTES);
    float* wml = wo + WARPS * ROWS * SH::PITCH;
    float* co = wml + WARPS * ROWS * 2;
    float* cml = co + ROWS * SH::PITCH;
#pragma unroll
    for (int q = 0; q < QT; ++q) {
        float sum = l[q];
#pragma unroll
        for (int w = 4; w < 32; w *= 2) sum += __shfl_xor_sync(0xffffffffu, sum, w);
        if (g8 == 0 && !(t4 & 1)) *reinterpret_cast<float2*>(wml + (warp * ROWS + 2 * q + (t4 >> 1)) * 2) = make_float2(m[q], sum);
    }
#pragma unroll
    for (int p = 0; p < PT; ++p) {
        const int r = EXACT ? 2 * p + (t4 >> 1) : 4 * p + (t4 >> 1) + 2 * (t4 & 1);
        float* dst = wo + (warp * ROWS + r) * SH::PITCH + 8 * g8;
#pragma unroll
        for (int s = 0; s < SEGS; ++s) {
            float x[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                x[e] = o[s][e >> 1][p][e & 1];
                if constexpr (EXACT) x[e] += __shfl_xor_sync(0xffffffffu, x[e], 1);      // the low digits
            }
            if (r < it.n_rows && (!EXACT || !(t4 & 1))) {
                *reinterpret_cast<float4*>(dst + 64 * s) = make_float4(x[0], x[1], x[2], x[3]);
                *reinterpret_cast<float4*>(dst + 64 * s + 4) = make_float4(x[4], x[5], x[6], x[7]);
            }
        }
    }
    __syncthreads();
    merge<T, ROWS, SH::PITCH>(a, it, wo, wml, co, cml, q_scale);
}

// --- more rows: f16 products, 16 rows a block ---------------------------------------------------------------------------
//
// int8 becomes f16 exactly and without a conversion instruction: 1024 + 128 + q has the bits 0x6400 | (q + 128), one byte
// permutation makes two of them and one subtraction takes 1152 away.  A query row is scaled by a power of two to below 2^14,
// so that it is held by one f16 a number (bfloat16 queries, exactly but for numbers 2^-38 of the row's largest) or two
// (float32: 22 bits or more).  Weights are one f16 (bfloat16) or two (float32).
//
// What bounds it is a warp's own chain, 1.9 us a tile of 32 keys of 128 entries in float32 (128 products, as many bytes to
// turn, two exponentials and a tanh a score) where a scheduler has one warp, 3.1 where it has two, and what lies around it:
// with one tile a warp or less a launch takes 8.9 us, of which the chain is 1.9.  6 sequences of 13 to 4,001 keys with five
// tokens each, 4 kv heads of 128, four query heads each, float32, take 21.7 us: dealing and joining put 2.6 on the 8.9, two
// blocks an SM and up to 11 parts a row some 4, and the longest warps' three tiles are two more than one (19.5 us in bfloat16,
// 21.0 without the cap, 22.1 with scores beyond 0.4 of it; as 5 x 1 shares of the longest 26.2, as 1 x 1 66).

template <typename T, int DP>
struct Shape {
    static constexpr int NT = 2, ROWS = 8 * NT;
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

template <typename T, int DP>
__global__ void __launch_bounds__(THREADS, 2) attn_kv8_kernel(AttnArgs a) {
    using SH = Shape<T, DP>;
    constexpr int NT = SH::NT, ROWS = SH::ROWS, PARTS = SH::PARTS, SEGS = SH::SEGS;
    constexpr bool EXACT = sizeof(T) == 4;
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ float q_scale[ROWS];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g8 = lane >> 2, t4 = lane & 3;
    pdl_wait();
    const Item it = find_item<ROWS>(a);
    if (it.n_rows <= 0) return;                                // (the whole cluster)
    Eight<T> raw[ROWS / WARPS];
    fetch_queries<T, ROWS>(a, it, warp, lane, raw);
    TileRing<DP, SH::SLOTS> tiles(a, it, smem_addr(smem) + SH::Q_BYTES, warp, lane);
    tiles.start();

    // the query rows, scaled to below 2^14 and laid out as the products read them (entry 16 t + e of a segment of 64 belongs
    // to thread t of the row's four; eight entries are 16 bytes)
#pragma unroll
    for (int j = 0; j < ROWS / WARPS; ++j) {
        const int r = warp + j * WARPS;
        float v[8];
        raw[j].numbers(v);
        bool finite;
        const int up = row_exponent(v, 13, finite);
        const float f = power_of_two(up);
        if (lane == 0) q_scale[r] = finite ? power_of_two(-up) : __int_as_float(0x7fc00000);
        if (lane * 8 < DP) {
            const int s = lane >> 3, t = (lane >> 1) & 3, half = lane & 1;
            uint8_t* dst = smem + ((((r >> 3) * SEGS + s) * 2 + half) * 32 + (r & 7) * 4 + t) * 16;
            uint32_t hi[4], lo[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float x = v[2 * e] * f, y = v[2 * e + 1] * f;
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
            pos[nt][e] = r < it.n_rows ? it.pos0 + (it.row0 + r) / a.group : -1;
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

    const int window = a.window > 0 ? a.window : ALL_KEYS;
    const uint32_t q_frag = smem_addr(smem) + lane * 16;

    for (int n = 0; n < tiles.n_tiles; ++n) {
        const float2 sc = tiles.scales(n);
        const int key0 = sc.y == GONE ? NOWHERE : (tiles.t0 + n * WARPS) * KT;
        uint32_t tile = tiles.next();

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
        const bool edge = key0 + KT - 1 > it.pos_lo || key0 < it.pos_hi - window + 1;
        float alpha[NT][2], coef[NT][2];
        uint32_t pf[PARTS][2][NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            float mt_max[2] = {-INFINITY, -INFINITY}, s8[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) s8[i] = z[i >> 2][nt][i & 3] * (qf[nt][i & 1] * sc.x);
            if (EXACT && a.cap > 0.0f) cap_exactly(s8, c1);
#pragma unroll
            for (int mt = 0; mt < 2; ++mt)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    float x = s8[4 * mt + e];
                    if (!EXACT && a.cap > 0.0f) x = fmaf(-c2, rcp(1.0f + ex2(x)), c1);
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
                coef[nt][e] = seen ? sc.y * f : 0.0f;
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
        tile = tiles.next();
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

    float* wo = reinterpret_cast<float*>(smem + SH::Q_BYTES);
    float* wml = wo + WARPS * ROWS * SH::PITCH;
    float* co = wml + WARPS * ROWS * 2;
    float* cml = co + ROWS * SH::PITCH;
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
            if (r < it.n_rows) {
                float* dst = wo + (warp * ROWS + r) * SH::PITCH + 8 * g8;
#pragma unroll
                for (int s = 0; s < SEGS; ++s) {
                    *reinterpret_cast<float4*>(dst + 64 * s) = make_float4(o[s][0][nt][e], o[s][0][nt][e + 2], o[s][1][nt][e], o[s][1][nt][e + 2]);
                    *reinterpret_cast<float4*>(dst + 64 * s + 4) = make_float4(o[s][2][nt][e], o[s][2][nt][e + 2], o[s][3][nt][e], o[s][3][nt][e + 2]);
                }
            }
        }
    __syncthreads();
    merge<T, ROWS, SH::PITCH>(a, it, wo, wml, co, cml, q_scale);
}

template <typename T>
int launch(void (*kernel)(AttnArgs), size_t smem, OncePerDevice& raised, const AttnArgs& a, int tile_rows, cudaStream_t stream) {
    const int st = allow_shared_memory(kernel, smem, raised);
    if (st) return st;
    cudaLaunchConfig_t cfg = {};
    const long long blocks = (a.dealt > 0 ? (long long)a.dealt : (long long)a.rows * a.spans) * a.row_tiles * a.shares;
    if (blocks > 0x7fffffffll) return BROLM_ERR_TOO_LARGE;
    cfg.gridDim = dim3((unsigned)blocks, a.n_kv);
    cfg.blockDim = dim3(THREADS);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = a.shares;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    // A launch that fills the device begins when the one before it has ended: let in early, its blocks land wherever that one
    // leaves room, several on one SM and none on another, and stay there (8 sequences of 8,192 keys behind a product of few
    // tokens: 42 us for 29).  A small one is let in.
    attr[1].val.programmaticStreamSerializationAllowed = pdl_enabled() && blocks * a.n_kv <= device_sm_count() ? 1 : 0;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    const int e = (int)cudaLaunchKernelEx(&cfg, kernel, a);
    if (e || (a.spans == 1 && a.dealt == 0)) return e;
    JoinArgs j{a.part_o, a.part_ml, a.out, a.cu_q, a.out_stride, a.rows, a.tokens, a.n_kv * a.group, a.dim, a.spans};
    if (a.dealt > 0) {
        j.plan = a.plan;
        j.step = a.row_tiles * a.n_kv * tile_rows;
        j.parts = a.dealt * j.step;
    }
    return launch_join<T>(j, stream);
}

template <typename T, int DP>
int launch_rows(const AttnArgs& a, int rows, cudaStream_t stream) {
    static OncePerDevice raised[4];
    if (rows == 2) return launch<T>(attn_kv8_few_kernel<T, DP, 2>, FewShape<T, DP, 2>::SMEM, raised[0], a, rows, stream);
    if (rows == 4) return launch<T>(attn_kv8_few_kernel<T, DP, 4>, FewShape<T, DP, 4>::SMEM, raised[1], a, rows, stream);
    if (rows == 8) return launch<T>(attn_kv8_few_kernel<T, DP, 8>, FewShape<T, DP, 8>::SMEM, raised[2], a, rows, stream);
    return launch<T>(attn_kv8_kernel<T, DP>, Shape<T, DP>::SMEM, raised[3], a, rows, stream);
}

template <typename T>
int launch_dim(const AttnArgs& a, int rows, cudaStream_t stream) {
    if (a.dim <= 64) return launch_rows<T, 64>(a, rows, stream);
    if (a.dim <= 128) return launch_rows<T, 128>(a, rows, stream);
    if (a.dim <= 192) return launch_rows<T, 192>(a, rows, stream);
    return launch_rows<T, 256>(a, rows, stream);
}

}  // namespace

// shares (1 .. 8): blocks of a cluster that share a row's keys; spans: clusters that do, joined by a second launch through
// part_o [tokens * n_kv * group * spans * dim] and part_ml [.. * 2].  spans < 0: -spans clusters for every kv head and tile of
// query rows are dealt out over the sequences (at most 128, and no more than clusters) by their lengths; part_o then holds
// [-spans * n_kv * tiles * rows of a tile * dim], part_ml [.. * 2] and plan [tokens * n_kv * group * 2].
struct AttnCall {
    const void* q;
    void* out;
    const void *cu_q, *kv_len, *slots, *tables, *k_pages, *v_pages, *k_scale, *v_scale;
    void *part_o, *part_ml, *plan;
    cudaStream_t stream;
    int q_stride, out_stride, dtype, tokens, rows, n_kv, group, dim, block, n_blocks, n_slots, width, ring, window, max_q_len, shares, spans;
    float scale, cap;
};

BROLM_API int brolm_attn_kv8(const AttnCall* c) {
    const int n_kv = c->n_kv, group = c->group, dim = c->dim, block = c->block;
    if (c->dtype != BROLM_F32 && c->dtype != BROLM_BF16) return BROLM_ERR_BAD_DTYPE;
    if (c->tokens < 0 || c->rows < 0 || n_kv <= 0 || group <= 0 || dim <= 0 || dim % 16 || block <= 0 || block % 32) return BROLM_ERR_BAD_SIZE;
    if (c->n_blocks <= 0 || c->n_slots <= 0 || c->width <= 0 || c->ring < 0 || c->ring % block || c->window < 0 || c->max_q_len <= 0) return BROLM_ERR_BAD_SIZE;
    if (c->shares < 1 || c->shares > MAX_SHARES || c->spans == 0 || (c->spans != 1 && (!c->part_o || !c->part_ml))) return BROLM_ERR_BAD_SIZE;
    if (c->spans < 0 && (c->rows > MAX_DEALT || c->rows > -(long long)c->spans || !c->plan)) return BROLM_ERR_BAD_SIZE;
    if (dim > MAX_DIM || block > MAX_BLOCK || (long long)n_kv * group > 65535 || (long long)c->max_q_len * group > 0x3fffffff) return BROLM_ERR_TOO_LARGE;
    if ((long long)c->n_blocks * block > 0x7fffffffll || c->tokens > 0x3fffffff) return BROLM_ERR_TOO_LARGE;
    if (((uintptr_t)c->k_pages | (uintptr_t)c->v_pages | (uintptr_t)c->part_o) & 15 || (uintptr_t)c->plan & 7) return BROLM_ERR_ALIGNMENT;
    if (c->tokens == 0 || c->rows == 0) return BROLM_OK;
    const int size = c->dtype == BROLM_F32 ? 4 : 2, most = c->max_q_len * group, per = most <= 2 ? 2 : most <= 4 ? 4 : most <= 8 ? 8 : 16;
    const int wide = ((uintptr_t)c->q & 15) == 0 && (long long)c->q_stride * size % 16 == 0;
    AttnArgs a{c->q, c->out, c->q_stride, c->out_stride, (const int32_t*)c->cu_q, (const int32_t*)c->kv_len,
               (const int32_t*)c->slots, (const int32_t*)c->tables, (const int8_t*)c->k_pages, (const int8_t*)c->v_pages,
               (const float*)c->k_scale, (const float*)c->v_scale, c->tokens, c->rows, n_kv, group, dim, block, c->n_blocks,
               c->n_slots, c->width, c->ring, min(c->window, ALL_KEYS), c->scale, c->cap, c->shares, max(c->spans, 1), (most + per - 1) / per, wide,
               max(-c->spans, 0), (float*)c->part_o, (float*)c->part_ml, (int2*)c->plan};
    if ((long long)a.dealt * a.row_tiles * n_kv * per > 0x7fffffffll) return BROLM_ERR_TOO_LARGE;
    return c->dtype == BROLM_F32 ? launch_dim<float>(a, per, c->stream) : launch_dim<bf16>(a, per, c->stream);
}
