// The end of an attention whose keys were shared out: the parts of a row, each with its maximum in log2 units, its sum of
// weights and its sum of values, become the row.
#pragma once

#include "kv8.cuh"

namespace kv8 {

constexpr float LOG2E = 1.4426950408889634f;
// What a window is where there is none, and at most: a cache has fewer than 2^31 places, and a position less this many tokens
// and a tile or two is still a whole number of 32 bits.
constexpr int ALL_KEYS = 0x7ffff000;
// Where keys lie whose place in the tables is none of the cache's: behind every token, so that none sees them.
constexpr int NOWHERE = 0x7fffff00;

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ void add_part(float4& acc, float& sum, const float4& x, float l, float f) {
    sum = fmaf(l, f, sum);
    acc.x = fmaf(x.x, f, acc.x); acc.y = fmaf(x.y, f, acc.y); acc.z = fmaf(x.z, f, acc.z); acc.w = fmaf(x.w, f, acc.w);
}
// Four entries of a row: zeros where nothing was seen, NaN where something was not a number.
template <typename T>
__device__ __forceinline__ void store_row(void* out, int out_stride, int dim, int tok, int head, int d, const float4& acc, float sum) {
    const float inv = sum > 0.0f ? 1.0f / sum : sum != 0.0f ? sum : acc.x != acc.x ? 1.0f : 0.0f;
    T* dst = reinterpret_cast<T*>(out) + (size_t)tok * out_stride + head * dim + d;
    dst[0] = from_float<T>(acc.x * inv);
    dst[1] = from_float<T>(acc.y * inv);
    dst[2] = from_float<T>(acc.z * inv);
    dst[3] = from_float<T>(acc.w * inv);
}

// Four entries of a row from its parts at, at + step, ..., in their order, and the sum of its weights:
// sum_s o_s 2^(m_s - m),  sum_s l_s 2^(m_s - m).
__device__ __forceinline__ float4 join_parts(const float* part_o, const float* part_ml, size_t at, size_t step, int spans, int dim, int d,
                                             float& sum) {
    float most = -INFINITY;
    sum = 0.0f;
    float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int s0 = 0; s0 < spans; s0 += 8) {                  // (eight parts are asked for at once)
        float2 ml[8];
        float4 x[8];
        float top = most;
#pragma unroll
        for (int s = 0; s < 8; ++s) {
            ml[s] = make_float2(-INFINITY, 0.0f);
            x[s] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            if (s0 + s < spans) {
                ml[s] = *reinterpret_cast<const float2*>(part_ml + (at + (s0 + s) * step) * 2);
                x[s] = *reinterpret_cast<const float4*>(part_o + (at + (s0 + s) * step) * dim + d);
            }
            top = fmaxf(top, ml[s].x);
        }
        const float keep = most > -INFINITY ? ex2(most - top) : 1.0f;
        most = top;
        sum *= keep;
        acc.x *= keep; acc.y *= keep; acc.z *= keep; acc.w *= keep;
#pragma unroll
        for (int s = 0; s < 8; ++s)
            if (s0 + s < spans) add_part(acc, sum, x[s], ml[s].y, top > -INFINITY ? ex2(ml[s].x - top) : 0.0f);
    }
    return acc;
}

struct JoinArgs {
    const float *part_o, *part_ml;        // [token][head][span][dim] and [..][2]
    void* out;
    const int32_t* cu_q;
    int out_stride, rows, tokens, heads, dim, spans;
    const int2* plan = nullptr;           // where given, [token][head]: the first part and how many, every `step` parts
    int step = 1, parts = 0;              // (the parts that there are: nothing is read beyond them)
};

// Rows whose keys were shared by several blocks that do not join their results themselves: a thread for four entries of a
// (token, head) adds up its parts in their order,  out = sum_s o_s 2^(m_s - m) / sum_s l_s 2^(m_s - m).
constexpr int JOIN_THREADS = 256;
template <typename T>
__global__ void __launch_bounds__(JOIN_THREADS) attn_kv8_join_kernel(JoinArgs a) {
    pdl_trigger();
    pdl_wait();
    const int per = a.dim >> 2, mine = threadIdx.x / per, d = (threadIdx.x - mine * per) * 4;
    const long long row = (long long)blockIdx.x * (JOIN_THREADS / per) + mine;
    const int tok = (int)(row / a.heads), head = (int)(row - (long long)tok * a.heads);
    if (mine >= JOIN_THREADS / per || tok >= min(a.tokens, a.cu_q[a.rows])) return;
    size_t at = ((size_t)tok * a.heads + head) * a.spans;
    int spans = a.spans;
    if (a.plan) {
        const int2 p = a.plan[(size_t)tok * a.heads + head];
        at = p.x;
        spans = p.y;
        if (spans <= 1 || p.x < 0 || p.x + (long long)(spans - 1) * a.step >= a.parts) return;     // (one part is in its place)
    }
    float sum;
    const float4 acc = join_parts(a.part_o, a.part_ml, at, a.step, spans, a.dim, d, sum);
    store_row<T>(a.out, a.out_stride, a.dim, tok, head, d, acc, sum);
}

template <typename T>
int launch_join(const JoinArgs& a, cudaStream_t stream) {
    const long long rows = (long long)a.tokens * a.heads, each = JOIN_THREADS / (a.dim >> 2), blocks = (rows + each - 1) / each;
    if (blocks > 0x7fffffffll) return BROLM_ERR_TOO_LARGE;
    return launch_pdl(attn_kv8_join_kernel<T>, dim3((unsigned)blocks), dim3(JOIN_THREADS), 0, stream, a);
}

}  // namespace kv8
