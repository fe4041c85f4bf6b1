// Log probabilities of given tokens, with rank, entropy and the best alternatives, in one pass over the logits.
//
// A row x of V logits is the distribution p_i = exp(x_i - m) / s, m = max x, s = sum exp(x_i - m).  Wanted are
//     log p(id) = x_id - m - log s,        rank(id) = #{i: x_i > x_id, or x_i = x_id and i < id},
//     entropy   = log s - u / s            with u = sum (x_i - m) exp(x_i - m)      (p = 0 contributes 0),
// and the k largest x_i with their log p, ordered by (x descending, i ascending).  Taking u about the maximum, not about
// zero, keeps the entropy exact when the logits are far from zero.
//
// A block has a slice of a row, in chunks of 4,096 logits that its threads hold in registers: every thread keeps m, s, u and
// its count (online: s and u are rescaled when m grows), joined once at the end.  The best k come from the same registers: of a
// chunk only entries above the k-th best so far can be among them, and once some chunks are through those are few.  Of the first chunk, a bound
// that k entries reach: every warp's q-th largest of its threads' maxima, q = ceil(k / 8), and of the eight warps' the least.  Where that leaves
// too many (equal logits; rising ones, later), the k-th largest of all the threads' maxima does not: entries are told apart by their index, so no
// more than k threads reach it, with 16 entries each.  Entries are 64-bit keys (the float's order, then the lower index first), so the
// order of arrival in the buffer changes nothing.
// The slices of a row are a cluster, whose first block joins them, slice after slice, out of the others' shared memory.  All sums are float32.
#include <math.h>

#include "common.cuh"

LGML_DEFINE_LAST_ERROR(lgml_logprobs)

namespace {
constexpr int THREADS = 256;
constexpr int WARPS = THREADS / 32;
constexpr int PER = 16;                       // logits a thread holds
constexpr int CHUNK = THREADS * PER;
constexpr int TOP_MAX = 32;
constexpr int BUFFER = TOP_MAX * PER;         // candidates of a chunk
constexpr int MAX_SLICES = 16;                // blocks of a cluster
constexpr float LOG2E = 1.4426950408889634f;

typedef unsigned long long Key;

__device__ __forceinline__ float ex2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
// Larger keys come first: the float's order (NaN below everything, -0 as 0), then the lower index.  0: no entry.
__device__ __forceinline__ unsigned order_of(float x) {
    const unsigned u = __float_as_uint(x + 0.f);
    return x != x ? 0u : (u & 0x80000000u) ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ Key key_of(float x, int i) { return ((Key)order_of(x) << 32) | (unsigned)(0x7fffffff - i); }
__device__ __forceinline__ int index_of(Key k) { return 0x7fffffff - (int)(unsigned)(k & 0xffffffffu); }
__device__ __forceinline__ float value_of(Key k) {
    const unsigned o = (unsigned)(k >> 32);
    return o == 0u ? __int_as_float(0x7fffffff) : __uint_as_float((o & 0x80000000u) ? o & 0x7fffffffu : ~o);
}

struct Stats {
    float m, s, u;      // maximum, sum of exp(x - m), sum of (x - m) exp(x - m)
};
// About another maximum: exp(x - M) = f exp(x - m), f = exp(m - M).
__device__ __forceinline__ Stats about(Stats a, float M) {
    if (a.m == M || a.m == -INFINITY) return Stats{M, a.s, a.u};       // (nothing but -inf so far: s and u are 0, or NaN)
    const float d = fmaxf(a.m - M, -1e30f);        // (a maximum of the type's lowest value would make the product infinite, and infinity x 0 a NaN)
    const float f = ex2(d * LOG2E);
    return Stats{M, a.s * f, (a.u + d * a.s) * f};
}
__device__ __forceinline__ Stats join(Stats a, Stats b) {
    const float M = fmaxf(a.m, b.m);
    a = about(a, M), b = about(b, M);
    return Stats{M, a.s + b.s, a.u + b.u};
}

struct Outputs {
    float *logprob;
    int *rank;
    float *entropy;
    int *top_ids;
    float *top_logprobs;
};

__device__ __forceinline__ void write_row(const Outputs &out, int r, int id, bool known, float x_id, const Stats &st, int greater) {
    const float log_s = logf(st.s);
    out.logprob[r] = known ? x_id - st.m - log_s : __int_as_float(0x7fffffff);
    out.rank[r] = known ? greater : -1;
    out.entropy[r] = log_s - st.u / st.s;
}

// Of the n keys in list (shared memory) the k largest, in order, to best; places without an entry get 0.
__device__ __forceinline__ void rank_keys(const Key *list, int n, Key *best, int k) {
    for (int i = threadIdx.x; i < n; i += THREADS) {
        const Key mine = list[i];
        int before = 0;
        for (int j = 0; j < n; ++j) before += list[j] > mine;
        if (before < k) best[before] = mine;
    }
    for (int i = n + threadIdx.x; i < k; i += THREADS) best[i] = 0;
}

__device__ __forceinline__ unsigned block_of_cluster() {
    unsigned r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_sync() { asm volatile("barrier.cluster.arrive.aligned;\nbarrier.cluster.wait.aligned;" ::: "memory"); }
// The address, in the cluster, of what block `rank` has where this block has p.
__device__ __forceinline__ uint32_t in_block(const void *p, int rank) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"((uint32_t)__cvta_generic_to_shared(p)), "r"(rank));
    return r;
}
__device__ __forceinline__ float4 load_there(uint32_t at) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(at));
    return v;
}
__device__ __forceinline__ Key load_key_there(uint32_t at) {
    Key v;
    asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(at));
    return v;
}

struct Shared {
    Key list[TOP_MAX + BUFFER];          // the best so far, then candidates; at the end, the slices' best
    Key best[TOP_MAX];
    Key thread_best[THREADS];
    float4 mine;                         // of the slice: m, s, u, the count
    Stats warp_stats[WARPS];
    int warp_count[WARPS];
    unsigned warp_bound[WARPS];
    int n_list;
    Key bound;
};

// Entries of the chunk that pass(x, i) go behind the best so far, as many as there is room for; returns how many there are.
template <typename Pass>
__device__ __forceinline__ int collect(Shared &sh, const float (&x)[PER], int first, int V, int top, Pass pass) {
    if (threadIdx.x == 0) sh.n_list = 0;
    __syncthreads();
    if (threadIdx.x < top) sh.list[threadIdx.x] = sh.best[threadIdx.x];
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        const int i = first + (j >> 2) * THREADS * 4 + (j & 3);
        if (i < V && pass(x[j], i)) {
            const int at = atomicAdd(&sh.n_list, 1);
            if (at < BUFFER) sh.list[top + at] = key_of(x[j], i);
        }
    }
    __syncthreads();
    return sh.n_list;
}

__global__ void __launch_bounds__(THREADS, 4) logprobs_kernel(const float *__restrict__ logits, long long ld, int V, const int *__restrict__ ids, int top,
                                                              int n_slices, int chunks_per_slice, int vec, Outputs out, int *__restrict__ status) {
    pdl_trigger();
    __shared__ __align__(16) Shared sh;
    const int r = blockIdx.x / n_slices, slice = n_slices > 1 ? (int)block_of_cluster() : 0, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const float *row = logits + (size_t)r * ld;
    pdl_wait();
    const int id = act_load(ids + r);
    const bool known = id >= 0 && id < V;
    if (!known && id != -1 && tid == 0) atomicExch(status, 1);
    const float x_id = known ? act_load(row + id) : __int_as_float(0x7fffffff);
    if (tid < TOP_MAX) sh.best[tid] = 0;
    __syncthreads();

    Stats st{-INFINITY, 0.f, 0.f};
    int greater = 0;
    for (int c = 0; c < chunks_per_slice; ++c) {
        const int base = (slice * chunks_per_slice + c) * CHUNK;
        if (base >= V) break;
        const int first = base + tid * 4;            // a thread's j-th entry is first + (j / 4) * 4 * THREADS + j % 4
        float x[PER];
        if (vec && V - base >= CHUNK) {
#pragma unroll
            for (int j = 0; j < PER / 4; ++j) {
                const float4 v = act_load(reinterpret_cast<const float4 *>(row + first + j * THREADS * 4));
                x[4 * j] = v.x, x[4 * j + 1] = v.y, x[4 * j + 2] = v.z, x[4 * j + 3] = v.w;
            }
        } else {
#pragma unroll
            for (int j = 0; j < PER; ++j) {
                const int i = first + (j >> 2) * THREADS * 4 + (j & 3);
                x[j] = i < V ? act_load(row + i) : -INFINITY;
            }
        }
        // ---- sums ----
        float largest = x[0];
#pragma unroll
        for (int j = 1; j < PER; ++j) largest = fmaxf(largest, x[j]);
        if (largest > st.m) st = about(st, largest);
        const float ref = st.m == -INFINITY ? 0.f : st.m;
        int above = 0, from = 0;
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            const float d = x[j] - ref, w = ex2(d * LOG2E);
            st.s += w;
            st.u += fmaxf(d, -1e30f) * w;
            above += x[j] > x_id, from += x[j] >= x_id;
        }
        if (from != above)              // (equal ones: the id itself, and a few)
#pragma unroll
            for (int j = 0; j < PER; ++j) above += x[j] == x_id && first + (j >> 2) * THREADS * 4 + (j & 3) < id;
        greater += above;
        if (top == 0) continue;
        // ---- the best ----
        // (entries of later chunks have larger indices: an equal value does not displace the k-th best)
        const Key kth = sh.best[top - 1];
        const unsigned kth_order = (unsigned)(kth >> 32);          // 0: not k yet, or NaNs among them
        int n;
        if (kth_order != 0) {
            const float least = value_of(kth);
            if (!__syncthreads_or(largest > least)) continue;
            n = collect(sh, x, first, V, top, [=](float v, int) { return v > least; });
        } else {
            unsigned left = 0, q_th = 0;              // (places past the vocabulary are none)
#pragma unroll
            for (int j = 0; j < PER; ++j)
                if (first + (j >> 2) * THREADS * 4 + (j & 3) < V) left = max(left, order_of(x[j]));
            for (int q = 0; q < (top + WARPS - 1) / WARPS; ++q) {
                q_th = __reduce_max_sync(0xffffffffu, left);
                if (lane == __ffs(__ballot_sync(0xffffffffu, left == q_th)) - 1) left = 0;
            }
            if (lane == 0) sh.warp_bound[warp] = q_th;
            __syncthreads();
            unsigned bound = sh.warp_bound[0];
#pragma unroll
            for (int w = 1; w < WARPS; ++w) bound = min(bound, sh.warp_bound[w]);
            n = collect(sh, x, first, V, top, [=](float v, int i) { return order_of(v) >= bound && key_of(v, i) > kth; });
        }
        if (n > BUFFER) {
            Key local = 0;
#pragma unroll
            for (int j = 0; j < PER; ++j) {
                const int i = first + (j >> 2) * THREADS * 4 + (j & 3);
                if (i < V) local = max(local, key_of(x[j], i));
            }
            sh.thread_best[tid] = local;
            __syncthreads();
            int before = 0;
            for (int j = 0; j < THREADS; ++j) before += sh.thread_best[j] > local || (sh.thread_best[j] == local && j < tid);
            if (before == top - 1) sh.bound = local;
            __syncthreads();
            const Key bound = sh.bound;
            n = collect(sh, x, first, V, top, [=](float v, int i) { const Key k = key_of(v, i); return k > kth && k >= bound; });
        }
        rank_keys(sh.list, top + min(n, BUFFER), sh.best, top);
        __syncthreads();
    }

    // ---- join the threads ----
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        st = join(st, Stats{__shfl_xor_sync(0xffffffffu, st.m, o), __shfl_xor_sync(0xffffffffu, st.s, o), __shfl_xor_sync(0xffffffffu, st.u, o)});
        greater += __shfl_xor_sync(0xffffffffu, greater, o);
    }
    if (lane == 0) sh.warp_stats[warp] = st, sh.warp_count[warp] = greater;
    __syncthreads();
    if (tid == 0) {
        for (int w = 1; w < WARPS; ++w) st = join(st, sh.warp_stats[w]), greater += sh.warp_count[w];
        sh.mine = make_float4(st.m, st.s, st.u, __int_as_float(greater));
    }
    // ---- and the slices ----
    if (n_slices > 1) {
        cluster_sync();
        if (slice == 0) {
            for (int i = tid; i < n_slices * top; i += THREADS) sh.list[i] = load_key_there(in_block(sh.best + i % top, i / top));
            __syncthreads();
            rank_keys(sh.list, n_slices * top, sh.thread_best, top);
            if (tid == 0) {
                for (int i = 1; i < n_slices; ++i) {
                    const float4 v = load_there(in_block(&sh.mine, i));
                    st = join(st, Stats{v.x, v.y, v.z});
                    greater += __float_as_int(v.w);
                }
                sh.mine = make_float4(st.m, st.s, st.u, 0.f);
            }
        }
        cluster_sync();                 // (the others' shared memory is read until here)
        if (slice != 0) return;
    } else {
        __syncthreads();
    }
    if (tid == 0) write_row(out, r, id, known, x_id, st, greater);
    if (tid < top) {
        const Key k = n_slices > 1 ? sh.thread_best[tid] : sh.best[tid];
        out.top_ids[(size_t)r * top + tid] = index_of(k);
        out.top_logprobs[(size_t)r * top + tid] = value_of(k) - sh.mine.x - logf(sh.mine.y);
    }
}
}  // namespace

// Into how many slices (a power of two) a row is cut.
LGML_API int lgml_token_logprobs_slices(int n_rows, int V, int n_sms) {
    const int chunks = (V + CHUNK - 1) / CHUNK;
    int slices = 1;
    while (slices < MAX_SLICES && 2 * slices <= chunks && (long long)n_rows * 2 * slices <= 4 * n_sms) slices *= 2;
    return slices;
}

LGML_API int lgml_token_logprobs(const float *logits, long long ld, int n_rows, int V, const int *ids, int top, int n_slices, float *logprob, int *rank,
                                 float *entropy, int *top_ids, float *top_logprobs, int *status, cudaStream_t stream) {
    LGML_REQUIRE(n_rows >= 0 && V > 0 && ld >= V, "token_logprobs: %d rows of %d logits, %lld apart", n_rows, V, ld);
    LGML_REQUIRE(V <= 1 << 30, "token_logprobs: a vocabulary of %d", V);
    LGML_REQUIRE(top >= 0 && top <= TOP_MAX && top <= V, "token_logprobs: %d alternatives (0 to %d, at most the vocabulary)", top, TOP_MAX);
    LGML_REQUIRE(n_slices >= 1 && n_slices <= MAX_SLICES && (n_slices & (n_slices - 1)) == 0, "token_logprobs: %d slices (a power of two up to %d)", n_slices,
                 MAX_SLICES);
    LGML_REQUIRE((long long)n_rows * n_slices <= 0x7fffffffLL, "token_logprobs: too many rows");
    if (n_rows == 0) return 0;
    const int chunks = (V + CHUNK - 1) / CHUNK, per = (chunks + n_slices - 1) / n_slices;
    const int vec = ld % 4 == 0 && ((uintptr_t)logits & 15) == 0;
    const Outputs out{logprob, rank, entropy, top_ids, top_logprobs};
    if (n_slices > 8) {
        cudaError_t e = cudaFuncSetAttribute(logprobs_kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
        if (e != cudaSuccess) LGML_FAIL("token_logprobs: no clusters of %d: %s", n_slices, cudaGetErrorString(e));
    }
    lgml_launch_cluster(logprobs_kernel, dim3(n_rows * n_slices), THREADS, 0, stream, n_slices, logits, ld, V, ids, top, n_slices, per, vec, out, status);
    return lgml_launch_status("token_logprobs");
}
