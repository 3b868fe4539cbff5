// Block tables and slot maps of a paged cache, built on the device from the lengths of a step's requests.
//
// The state is a row of block ids per slot (`tables`, of which the first `held` are the slot's) and a stack of free
// blocks (`stack`, the first `count`).  A step's row i names slot s, which holds L tokens and brings n more:
//
//     need(x) = ceil(min(x, ring or x) / P)               blocks of P tokens that x tokens take up
//     more_i  = max(0, need(L + n) - held[s])             taken from the top of the stack, rows in order
//     pos     = L + j,  place = pos (% ring)              of its j-th new token
//     row     = tables[s][place / P] * P + place % P      or -1 where pos / P + ring / P <= (L + n - 1) / P: the ring's
//                                                         newest block has already taken that block's place
//
// A row with slot -1 is padding: its tokens get position and cache row -1, its length is 0.  All or nothing: where the
// free blocks, a row of the tables or the outputs do not suffice, or a slot is wrong, the state stays as it is, every
// output reads as padding (lengths and sums 0) and `status` says why.  `refused`, where given, keeps the first status that
// was not 0: the status of a step whose results nobody waits for is soon overwritten by the next one's.
//
// What bounds it is latency: a decode step of 64 rows reads and writes 2.6 KB.  One launch does all of it: every block of
// threads of one cluster adds up all rows by itself (three short arrays out of the L2), which costs less than handing sums
// around, the cluster's barrier then lets the state be written that all have read, and tokens and new table entries are
// shared out.  A token's block is looked up in the stack where it is new, so nothing waits for the tables' new entries.
// A cluster is eight SMs, and 32,768 tokens take them 4.3 us; steps of more tokens run on all SMs without a cluster, and a
// second, small launch writes what the blocks of the first still read (300 rows of 100,559 tokens in all: 17.8 us in one
// cluster).
#include "common.cuh"

namespace {

constexpr int THREADS = 1024;
constexpr int MAX_ROWS = 4096;           // rows of a step: their sums lie in shared memory
constexpr int MAX_SLOTS = 65536;         // a bit each: a slot named twice is found in shared memory

enum : int { ST_OK = 0, ST_NO_BLOCKS = 1, ST_TABLE_WIDTH = 2, ST_TOO_MANY_TOKENS = 3, ST_BAD_ROW = 4 };

struct ExtendArgs {
    const int32_t *slots, *lengths, *fresh;        // of the step's rows
    int32_t *tables, *held, *count;
    const int32_t* stack;
    int32_t *cu_q, *kv_len, *positions, *tok_seq, *cache_rows, *status, *refused;
    int rows, n_slots, width, stack_size, block, shift, ring, tokens;      // shift: of a block that is a power of two, else -1
};

__device__ __forceinline__ void cluster_barrier() {
    asm volatile("barrier.cluster.arrive.aligned;\nbarrier.cluster.wait.aligned;\n" ::: "memory");
}

// (by one thread of a launch, and launches that share the words run one after the other)
__device__ __forceinline__ void tell(int32_t* status, int32_t* refused, int value) {
    *status = value;
    if (refused && value != ST_OK && *refused == ST_OK) *refused = value;
}

__device__ __forceinline__ int blocks_for(long long n, int block, int ring) {
    if (ring > 0 && n > ring) n = ring;
    return (int)((n + block - 1) / block);
}

// Running sums of two numbers a thread over the block of threads; `total` gets both sums.  scratch: 2 x 33 long longs.
__device__ __forceinline__ longlong2 scan2(long long a, long long b, long long (*scratch)[33], longlong2& total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const long long a0 = a, b0 = b;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long x = __shfl_up_sync(0xffffffffu, a, o), y = __shfl_up_sync(0xffffffffu, b, o);
        if (lane >= o) { a += x; b += y; }
    }
    __syncthreads();
    if (lane == 31) { scratch[0][warp] = a; scratch[1][warp] = b; }
    __syncthreads();
    if (warp == 0) {
        long long x = scratch[0][lane], y = scratch[1][lane];
        const long long x0 = x, y0 = y;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long u = __shfl_up_sync(0xffffffffu, x, o), v = __shfl_up_sync(0xffffffffu, y, o);
            if (lane >= o) { x += u; y += v; }
        }
        scratch[0][lane] = x - x0;
        scratch[1][lane] = y - y0;
        if (lane == 31) { scratch[0][32] = x; scratch[1][32] = y; }
    }
    __syncthreads();
    total = make_longlong2(scratch[0][32], scratch[1][32]);
    return make_longlong2(scratch[0][warp] + a - a0, scratch[1][warp] + b - b0);
}

// The last i in [0, n) with at[i] <= x (at ascends, at[0] <= x).
__device__ __forceinline__ int last_not_above(const int* at, int n, int x) {
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (at[mid] <= x) lo = mid;
        else hi = mid;
    }
    return lo;
}

// CLUSTER: the launch is one cluster and does everything.  Else `held`, `count` and `kv_len` (which may be `lengths`, in place)
// are left to commit_kernel.
template <bool CLUSTER>
__global__ void __launch_bounds__(THREADS) blocks_extend_kernel(ExtendArgs a) {
    extern __shared__ int rows_s[];
    int* token0 = rows_s;                       // [rows + 1] tokens ahead of the row
    int* block0 = token0 + a.rows + 1;          // [rows + 1] new blocks ahead of the row
    int* slot_s = block0 + a.rows + 1;          // [rows]
    int* held_s = slot_s + a.rows;              // [rows]
    int* before = held_s + a.rows;              // [rows] length before the step, -1 for padding
    unsigned* named = reinterpret_cast<unsigned*>(before + a.rows);      // a bit a slot
    __shared__ long long scratch[2][33];
    __shared__ int bad;
    const int words = (a.n_slots + 31) / 32;
    for (int i = threadIdx.x; i < words; i += THREADS) named[i] = 0u;
    if (threadIdx.x == 0) bad = ST_OK;
    pdl_trigger();
    pdl_wait();
    const int count = *a.count;
    __syncthreads();
    longlong2 sums = make_longlong2(0, 0);
    for (int base = 0; base < a.rows; base += THREADS) {
        const int i = base + threadIdx.x;
        int more = 0, n = 0, wrong = ST_OK;
        if (i < a.rows) {
            const int s = a.slots[i], len = a.lengths[i];
            n = a.fresh[i];
            int have = 0, from = -1;
            if (n < 0 || s < -1 || s >= a.n_slots || (s >= 0 && (len < 0 || (long long)len + n > 0x7fffffffll))) {
                wrong = ST_BAD_ROW;
                n = 0;
            } else if (s >= 0) {
                if (atomicOr(&named[s >> 5], 1u << (s & 31)) & (1u << (s & 31))) wrong = ST_BAD_ROW;
                have = a.held[s];
                if (have < 0 || have > a.width) {
                    wrong = max(wrong, (int)ST_TABLE_WIDTH);
                    have = 0;
                }
                from = len;
                const int need = blocks_for((long long)len + n, a.block, a.ring);
                if (need > a.width) wrong = max(wrong, (int)ST_TABLE_WIDTH);
                more = max(0, need - have);
            }
            slot_s[i] = s;
            held_s[i] = have;
            before[i] = from;
        }
        if (wrong) atomicMax(&bad, wrong);
        longlong2 total;
        const longlong2 at = scan2(n, more, scratch, total);
        if (i < a.rows) {                       // (where they pass 31 bits the step is refused below)
            token0[i] = (int)(sums.x + at.x);
            block0[i] = (int)(sums.y + at.y);
        }
        sums.x += total.x;
        sums.y += total.y;
    }
    if (threadIdx.x == 0) {
        token0[a.rows] = (int)sums.x;
        block0[a.rows] = (int)sums.y;
    }
    if constexpr (CLUSTER) cluster_barrier();   // everyone has read the state (and every thread's shared stores are seen)
    else __syncthreads();
    int status = bad;
    if (sums.x > a.tokens) status = max(status, (int)ST_TOO_MANY_TOKENS);
    if (sums.y > count || count > a.stack_size) status = max(status, (int)ST_NO_BLOCKS);
    const bool ok = status == ST_OK;
    const int rank = blockIdx.x, me = rank * THREADS + threadIdx.x, all = gridDim.x * THREADS;
    const int n_new = ok ? (int)sums.y : 0, n_tok = ok ? (int)sums.x : 0;
    if (me == 0) {
        tell(a.status, a.refused, status);
        if constexpr (CLUSTER) *a.count = count - n_new;
        a.cu_q[a.rows] = n_tok;
    }
    for (int i = me; i < a.rows; i += all) {
        const bool live = ok && before[i] >= 0;
        a.cu_q[i] = ok ? token0[i] : 0;
        if constexpr (CLUSTER) a.kv_len[i] = live ? before[i] + token0[i + 1] - token0[i] : 0;
        if (CLUSTER && live && block0[i + 1] != block0[i]) a.held[slot_s[i]] = held_s[i] + block0[i + 1] - block0[i];
    }
    for (int k = me; k < n_new; k += all) {
        const int i = last_not_above(block0, a.rows, k);
        a.tables[(size_t)slot_s[i] * a.width + held_s[i] + k - block0[i]] = a.stack[count - 1 - k];
    }
    // the tokens, EACH a thread and 32 EACH a warp at a time: the rows of a warp's first and last token are looked for once,
    // a token's own among them (mostly there is one)
    constexpr int EACH = CLUSTER ? 4 : 1;
    const int lane = threadIdx.x & 31;
    auto block_of = [&](int place) { return a.shift >= 0 ? place >> a.shift : place / a.block; };
    for (int base = (me >> 5) * 32 * EACH; base < a.tokens; base += all * EACH) {
        const int from = n_tok > 0 ? last_not_above(token0, a.rows, min(base, n_tok - 1)) : 0;
        const int to = n_tok > 0 ? last_not_above(token0, a.rows, min(base + 32 * EACH - 1, n_tok - 1)) : 0;
        int pos[EACH], seq[EACH], row[EACH];
        const int32_t* where[EACH];
#pragma unroll
        for (int j = 0; j < EACH; ++j) {
            const int t = base + 32 * j + lane;
            pos[j] = -1;
            seq[j] = 0;
            row[j] = -1;
            where[j] = nullptr;
            if (t >= n_tok) continue;
            const int s = from + (from < to ? last_not_above(token0 + from, to - from + 1, t) : 0);
            seq[j] = s;
            if (before[s] < 0) continue;
            const int p = before[s] + t - token0[s], last = before[s] + token0[s + 1] - token0[s] - 1;
            pos[j] = p;
            if (a.ring > 0 && block_of(p) + block_of(a.ring) <= block_of(last)) continue;
            const int place = a.ring > 0 ? (int)((unsigned)p % (unsigned)a.ring) : p, e = block_of(place);
            row[j] = place - e * a.block;
            where[j] = e < held_s[s] ? a.tables + (size_t)slot_s[s] * a.width + e : a.stack + (count - 1 - (block0[s] + e - held_s[s]));
        }
#pragma unroll
        for (int j = 0; j < EACH; ++j)
            if (where[j]) {                     // (an id that no cache of 31 bits of places has gives no place)
                const int id = *where[j];
                const long long at = (long long)id * a.block + row[j];
                row[j] = id >= 0 && at <= 0x7fffffffll ? (int)at : -1;
            }
#pragma unroll
        for (int j = 0; j < EACH; ++j) {
            const int t = base + 32 * j + lane;
            if (t < a.tokens) {
                a.positions[t] = pos[j];
                a.tok_seq[t] = seq[j];
                a.cache_rows[t] = row[j];
            }
        }
    }
}

// What blocks_extend_kernel<false> leaves: the lengths, and, if the step was taken, the slots' blocks and the stack's height.
__global__ void __launch_bounds__(THREADS) commit_kernel(ExtendArgs a) {
    __shared__ int taken;
    if (threadIdx.x == 0) taken = 0;
    __syncthreads();
    const bool ok = *a.status == ST_OK;
    int mine = 0;
    for (int i = threadIdx.x; i < a.rows; i += THREADS) {
        const int s = ok ? a.slots[i] : -1, len = s >= 0 ? a.lengths[i] + a.fresh[i] : 0;
        a.kv_len[i] = len;
        if (s < 0) continue;
        const int have = a.held[s], need = blocks_for(len, a.block, a.ring);
        if (need > have) {
            a.held[s] = need;
            mine += need - have;
        }
    }
    if (mine) atomicAdd(&taken, mine);
    __syncthreads();
    if (threadIdx.x == 0 && taken) *a.count -= taken;
}

// The blocks of the rows' slots go back to the stack, the last row's last block first: what one extend took, one release
// of the same rows puts back in its old order.  Rows with slot -1 are left out; a wrong slot changes nothing.
struct ReleaseArgs {
    const int32_t *slots, *tables;
    int32_t *held, *stack, *count, *status, *refused;
    int rows, n_slots, width, stack_size;
};

__global__ void __launch_bounds__(THREADS) blocks_release_kernel(ReleaseArgs a) {
    extern __shared__ int rows_s[];
    int* block0 = rows_s;                       // [rows + 1] blocks given back ahead of the row (rows from the last to the first)
    int* slot_s = block0 + a.rows + 1;
    unsigned* named = reinterpret_cast<unsigned*>(slot_s + a.rows);
    __shared__ long long scratch[2][33];
    __shared__ int bad;
    const int words = (a.n_slots + 31) / 32;
    for (int i = threadIdx.x; i < words; i += THREADS) named[i] = 0u;
    if (threadIdx.x == 0) bad = ST_OK;
    pdl_trigger();
    pdl_wait();
    const int count = *a.count;
    __syncthreads();
    long long sum = 0;
    for (int base = 0; base < a.rows; base += THREADS) {
        const int k = base + threadIdx.x;       // in the order of giving back
        int n = 0;
        if (k < a.rows) {
            const int s = a.slots[a.rows - 1 - k];
            if (s < -1 || s >= a.n_slots) atomicMax(&bad, (int)ST_BAD_ROW);
            else if (s >= 0) {
                if (atomicOr(&named[s >> 5], 1u << (s & 31)) & (1u << (s & 31))) atomicMax(&bad, (int)ST_BAD_ROW);
                n = a.held[s];
                if (n < 0 || n > a.width) {
                    atomicMax(&bad, (int)ST_TABLE_WIDTH);
                    n = 0;
                }
            }
            slot_s[k] = s;
        }
        longlong2 total;
        const longlong2 at = scan2(n, 0, scratch, total);
        if (k < a.rows) block0[k] = (int)(sum + at.x);
        sum += total.x;
    }
    if (threadIdx.x == 0) block0[a.rows] = (int)sum;
    cluster_barrier();
    int status = bad;
    if (count < 0 || count + sum > a.stack_size) status = max(status, (int)ST_NO_BLOCKS);
    const int me = blockIdx.x * THREADS + threadIdx.x, all = gridDim.x * THREADS;
    const int n_back = status == ST_OK ? (int)sum : 0;
    if (me == 0) {
        tell(a.status, a.refused, status);
        *a.count = count + n_back;
    }
    for (int b = me; b < n_back; b += all) {
        const int k = last_not_above(block0, a.rows, b);
        a.stack[count + b] = a.tables[(size_t)slot_s[k] * a.width + (block0[k + 1] - 1 - b)];
    }
    for (int k = me; status == ST_OK && k < a.rows; k += all)
        if (slot_s[k] >= 0) a.held[slot_s[k]] = 0;
}

__global__ void settle_kernel() {}

// One cluster of 1, 2, 4 or 8 blocks of threads: as many as give a thread a token, or an entry, of its own.
template <typename Args>
int launch_cluster(void (*kernel)(Args), const Args& a, long long work, size_t smem, OncePerDevice& raised, cudaStream_t stream) {
    const int st = allow_shared_memory(kernel, 200 * 1024, raised);
    if (st) return st;
    int blocks = 1;
    while (blocks < 8 && (long long)blocks * THREADS < work) blocks *= 2;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(blocks);
    cfg.blockDim = dim3(THREADS);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = blocks;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = pdl_enabled() ? 1 : 0;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    return (int)cudaLaunchKernelEx(&cfg, kernel, a);
}

}  // namespace

struct ExtendCall {
    const void *slots, *lengths, *fresh;
    void *tables, *held;
    const void* stack;
    void *count, *cu_q, *kv_len, *positions, *tok_seq, *cache_rows, *status, *refused;
    cudaStream_t stream;
    int rows, n_slots, width, stack_size, block, ring, tokens, settle;
};
struct ReleaseCall {
    const void *slots, *tables;
    void *held, *stack, *count, *status, *refused;
    cudaStream_t stream;
    int rows, n_slots, width, stack_size;
};

BROLM_API int brolm_blocks_extend(const ExtendCall* c) {
    if (c->rows < 0 || c->n_slots <= 0 || c->width <= 0 || c->stack_size < 0 || c->block <= 0 || c->tokens < 0) return BROLM_ERR_BAD_SIZE;
    if (c->ring < 0 || c->ring % c->block) return BROLM_ERR_BAD_SIZE;
    if (c->rows > MAX_ROWS || c->n_slots > MAX_SLOTS) return BROLM_ERR_TOO_LARGE;
    if ((long long)c->stack_size * c->block > 0x7fffffffll) return BROLM_ERR_TOO_LARGE;    // (a cache row is 31 bits)
    int shift = -1;
    for (int s = 0; s < 31; ++s)
        if (c->block == 1 << s) shift = s;
    ExtendArgs a{(const int32_t*)c->slots, (const int32_t*)c->lengths, (const int32_t*)c->fresh, (int32_t*)c->tables,
                 (int32_t*)c->held, (int32_t*)c->count, (const int32_t*)c->stack, (int32_t*)c->cu_q, (int32_t*)c->kv_len,
                 (int32_t*)c->positions, (int32_t*)c->tok_seq, (int32_t*)c->cache_rows, (int32_t*)c->status, (int32_t*)c->refused, c->rows,
                 c->n_slots, c->width, c->stack_size, c->block, shift, c->ring, c->tokens};
    static OncePerDevice raised;
    const size_t smem = (size_t)(5 * c->rows + 2 + (c->n_slots + 31) / 32) * 4;
    if (c->tokens > 8 * THREADS * 4) {
        static OncePerDevice raised_wide;
        int st = allow_shared_memory(blocks_extend_kernel<false>, 200 * 1024, raised_wide);
        if (st) return st;
        st = launch_pdl(blocks_extend_kernel<false>, dim3(min(device_sm_count(), (c->tokens + THREADS - 1) / THREADS)), dim3(THREADS), smem,
                        c->stream, a);
        if (st) return st;
        commit_kernel<<<1, THREADS, 0, c->stream>>>(a);
        st = launch_status();
        if (st || !c->settle) return st;
    } else {
        const int st = launch_cluster(blocks_extend_kernel<true>, a, c->tokens, smem, raised, c->stream);
        if (st || !c->settle) return st;
    }
    // A launch in plain stream order begins when this one has ended and its results are in memory: whatever is launched
    // behind it may read them before it waits for its predecessor, as many kernels read a step's description.
    settle_kernel<<<1, 32, 0, c->stream>>>();
    return launch_status();
}

BROLM_API int brolm_blocks_release(const ReleaseCall* c) {
    if (c->rows < 0 || c->n_slots <= 0 || c->width <= 0 || c->stack_size < 0) return BROLM_ERR_BAD_SIZE;
    if (c->rows > MAX_ROWS || c->n_slots > MAX_SLOTS) return BROLM_ERR_TOO_LARGE;
    ReleaseArgs a{(const int32_t*)c->slots, (const int32_t*)c->tables, (int32_t*)c->held, (int32_t*)c->stack, (int32_t*)c->count,
                  (int32_t*)c->status, (int32_t*)c->refused, c->rows, c->n_slots, c->width, c->stack_size};
    static OncePerDevice raised;
    const size_t smem = (size_t)(2 * c->rows + 1 + (c->n_slots + 31) / 32) * 4;
    return launch_cluster(blocks_release_kernel, a, (long long)c->rows * 16, smem, raised, c->stream);
}
