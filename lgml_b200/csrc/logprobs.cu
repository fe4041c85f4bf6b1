// Log probabilities of given tokens, with rank, entropy and the best alternatives, in one pass over the logits.
//
// A row x of V logits is the distribution p_i = exp(x_i - m) / s, m = max x, s = sum exp(x_i - m).  Wanted are
//     log p(id) = x_id - m - log s,        rank(id) = #{i: x_i > x_id, or x_i = x_id and i < id},
//     entropy   = log s - u / s            with u = sum (x_i - m) exp(x_i - m)      (p = 0 contributes 0),
// and the k largest x_i with their log p, ordered by (x descending, i ascending).  Taking u about the maximum, not about
// zero, keeps the entropy exact when the logits are far from zero.
//
// A block has a slice of a row, in chunks of 8,192 logits that its threads hold in registers: every thread keeps m, s, u and
// its count (online: s and u are rescaled when m grows), joined once at the end.  The best k come from the same registers: of a
// chunk only entries above the k-th best so far can be among them, and once some chunks are through those are few.  Where they are
// many (the first chunk; rising logits) the k-th largest of the threads' own maxima is a bound that at least k entries reach
// and, since entries are told apart by their index, that no more than k threads' 32 can: at most 32 k, which fit the buffer
// whatever the order.  Entries are 64-bit keys (the float's order, then the lower index first), so the order of arrival in the
// buffer changes nothing.  A row in several slices is joined by a second kernel, slice after slice.  All sums are float32.
#include <math.h>

#include "common.cuh"

LGML_DEFINE_LAST_ERROR(lgml_logprobs)

namespace {
constexpr int THREADS = 256;
constexpr int PER = 32;                       // logits a thread holds
constexpr int CHUNK = THREADS * PER;
constexpr int TOP_MAX = 32;
constexpr int BUFFER = TOP_MAX * PER + TOP_MAX;      // candidates of a chunk, and the best so far
constexpr int MAX_SLICES = 64;
constexpr float LOG2E = 1.4426950408889634f;

typedef unsigned long long Key;

// Larger keys come first: the float's order (NaN below everything, -0 as 0), then the lower index.  0: no entry.
__device__ __forceinline__ Key key_of(float x, int i) {
    const unsigned u = __float_as_uint(x + 0.f);
    const unsigned o = x != x ? 0u : (u & 0x80000000u) ? ~u : u | 0x80000000u;
    return ((Key)o << 32) | (unsigned)(0x7fffffff - i);
}
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
    const float f = exp2f(d * LOG2E);
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

__global__ void __launch_bounds__(THREADS) logprobs_kernel(const float *__restrict__ logits, long long ld, int V, const int *__restrict__ ids, int top,
                                                           int n_slices, int chunks_per_slice, int vec, float4 *__restrict__ part, Key *__restrict__ part_keys,
                                                           Outputs out, int *__restrict__ status) {
    pdl_trigger();
    pdl_wait();
    __shared__ Key list[BUFFER];
    __shared__ Key best[TOP_MAX];
    __shared__ Key thread_best[THREADS];
    __shared__ Stats warp_stats[THREADS / 32];
    __shared__ int warp_count[THREADS / 32];
    __shared__ int n_list;
    __shared__ Key bound;
    const int r = blockIdx.x / n_slices, slice = blockIdx.x - r * n_slices, tid = threadIdx.x;
    const float *row = logits + (size_t)r * ld;
    const int id = act_load(ids + r);
    const bool known = id >= 0 && id < V;
    if (!known && id != -1 && tid == 0) atomicExch(status, 1);
    const float x_id = known ? act_load(row + id) : __int_as_float(0x7fffffff);
    if (tid < TOP_MAX) best[tid] = 0;
    __syncthreads();

    Stats st{-INFINITY, 0.f, 0.f};
    int greater = 0;
    for (int c = 0; c < chunks_per_slice; ++c) {
        const int base = (slice * chunks_per_slice + c) * CHUNK;
        if (base >= V) break;
        float x[PER];
        const bool whole = vec && V - base >= CHUNK;
#pragma unroll
        for (int j = 0; j < PER / 4; ++j) {
            const int at = base + (j * THREADS + tid) * 4;
            if (whole) {
                const float4 v = act_load(reinterpret_cast<const float4 *>(row + at));
                x[4 * j] = v.x, x[4 * j + 1] = v.y, x[4 * j + 2] = v.z, x[4 * j + 3] = v.w;
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) x[4 * j + e] = at + e < V ? act_load(row + at + e) : -INFINITY;
            }
        }
        // ---- sums ----
        float M = st.m;
#pragma unroll
        for (int j = 0; j < PER; ++j) M = fmaxf(M, x[j]);
        st = about(st, M);
        const float ref = M == -INFINITY ? 0.f : M;
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            const float d = x[j] - ref, w = exp2f(d * LOG2E);
            st.s += w;
            st.u += fmaxf(d, -1e30f) * w;
            const int i = base + ((j >> 2) * THREADS + tid) * 4 + (j & 3);
            greater += x[j] > x_id || (x[j] == x_id && i < id);
        }
        if (top == 0) continue;
        // ---- the best ----
        // (entries of later chunks have larger indices: an equal value does not displace the k-th best)
        const Key kth = best[top - 1];
        int mine = 0;
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            const int i = base + ((j >> 2) * THREADS + tid) * 4 + (j & 3);
            mine += i < V && key_of(x[j], i) > kth;
        }
        int total = mine;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
        if ((tid & 31) == 0) warp_count[tid >> 5] = total;
        if (!__syncthreads_or(mine)) continue;
        total = 0;
        for (int w = 0; w < THREADS / 32; ++w) total += warp_count[w];
        Key floor_key = kth;            // entries above it go to the buffer
        if (total > TOP_MAX * PER) {
            Key local = 0;
#pragma unroll
            for (int j = 0; j < PER; ++j) {
                const int i = base + ((j >> 2) * THREADS + tid) * 4 + (j & 3);
                if (i < V) local = max(local, key_of(x[j], i));
            }
            thread_best[tid] = local;
            __syncthreads();
            int before = 0;
            for (int j = 0; j < THREADS; ++j) before += thread_best[j] > local || (thread_best[j] == local && j < tid);
            if (before == top - 1) bound = local;
            __syncthreads();
            if (bound != 0 && bound - 1 > floor_key) floor_key = bound - 1;       // entries from the bound on
        }
        if (tid == 0) n_list = 0;
        __syncthreads();
        if (tid < top) list[tid] = best[tid];
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            const int i = base + ((j >> 2) * THREADS + tid) * 4 + (j & 3);
            const Key k = key_of(x[j], i);
            if (i < V && k > floor_key) {
                const int at = atomicAdd(&n_list, 1);
                if (at < TOP_MAX * PER) list[top + at] = k;
            }
        }
        __syncthreads();
        const int n = top + min(n_list, TOP_MAX * PER);
        rank_keys(list, n, best, top);
        __syncthreads();
    }

    // ---- join the threads ----
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        st = join(st, Stats{__shfl_xor_sync(0xffffffffu, st.m, o), __shfl_xor_sync(0xffffffffu, st.s, o), __shfl_xor_sync(0xffffffffu, st.u, o)});
        greater += __shfl_xor_sync(0xffffffffu, greater, o);
    }
    __syncthreads();
    if ((tid & 31) == 0) warp_stats[tid >> 5] = st, warp_count[tid >> 5] = greater;
    __syncthreads();
    if (tid == 0) {
        st = warp_stats[0], greater = warp_count[0];
        for (int w = 1; w < THREADS / 32; ++w) st = join(st, warp_stats[w]), greater += warp_count[w];
        warp_stats[0] = st;
        if (n_slices == 1) write_row(out, r, id, known, x_id, st, greater);
        else part[(size_t)r * n_slices + slice] = make_float4(st.m, st.s, st.u, __int_as_float(greater));
    }
    __syncthreads();
    if (tid >= top) return;
    if (n_slices == 1) {
        const Key k = best[tid];
        out.top_ids[(size_t)r * top + tid] = index_of(k);
        out.top_logprobs[(size_t)r * top + tid] = value_of(k) - warp_stats[0].m - logf(warp_stats[0].s);
    } else {
        part_keys[((size_t)r * n_slices + slice) * top + tid] = best[tid];
    }
}

// A row's slices together, in their order.
__global__ void __launch_bounds__(THREADS) logprobs_join_kernel(const float *__restrict__ logits, long long ld, int V, const int *__restrict__ ids, int top,
                                                                int n_slices, const float4 *__restrict__ part, const Key *__restrict__ part_keys,
                                                                Outputs out) {
    pdl_trigger();
    pdl_wait();
    __shared__ Key list[MAX_SLICES * TOP_MAX];
    __shared__ Key best[TOP_MAX];
    __shared__ Stats slices[MAX_SLICES];
    __shared__ int counts[MAX_SLICES];
    const int r = blockIdx.x, tid = threadIdx.x;
    for (int i = tid; i < n_slices; i += THREADS) {
        const float4 p = act_load(part + (size_t)r * n_slices + i);
        slices[i] = Stats{p.x, p.y, p.z};
        counts[i] = __float_as_int(p.w);
    }
    const int n = n_slices * top;
    for (int i = tid; i < n; i += THREADS) list[i] = __ldcg(part_keys + (size_t)r * n + i);
    __syncthreads();
    rank_keys(list, n, best, top);
    if (tid == 0) {
        Stats st = slices[0];
        int greater = counts[0];
        for (int i = 1; i < n_slices; ++i) st = join(st, slices[i]), greater += counts[i];
        const int id = act_load(ids + r);
        const bool known = id >= 0 && id < V;
        write_row(out, r, id, known, known ? act_load(logits + (size_t)r * ld + id) : 0.f, st, greater);
        slices[0] = st;
    }
    __syncthreads();
    if (tid < top) {
        const Key k = best[tid];
        out.top_ids[(size_t)r * top + tid] = index_of(k);
        out.top_logprobs[(size_t)r * top + tid] = value_of(k) - slices[0].m - logf(slices[0].s);
    }
}
}  // namespace

// Into how many slices a row is cut, and the bytes of scratch that takes.
LGML_API int lgml_token_logprobs_slices(int n_rows, int V, int n_sms) {
    const int chunks = (V + CHUNK - 1) / CHUNK;
    int slices = n_rows > 0 ? (4 * n_sms) / n_rows : 1;
    if (slices > chunks) slices = chunks;
    if (slices > MAX_SLICES) slices = MAX_SLICES;
    if (slices < 1) slices = 1;
    const int per = (chunks + slices - 1) / slices;
    return (chunks + per - 1) / per;
}
LGML_API long long lgml_token_logprobs_scratch(int n_rows, int top, int n_slices) {
    return n_slices <= 1 ? 0 : (long long)n_rows * n_slices * (16 + 8 * top);
}

LGML_API int lgml_token_logprobs(const float *logits, long long ld, int n_rows, int V, const int *ids, int top, int n_slices, void *scratch, float *logprob,
                                 int *rank, float *entropy, int *top_ids, float *top_logprobs, int *status, cudaStream_t stream) {
    LGML_REQUIRE(n_rows >= 0 && V > 0 && ld >= V, "token_logprobs: %d rows of %d logits, %lld apart", n_rows, V, ld);
    LGML_REQUIRE(V <= 1 << 30, "token_logprobs: a vocabulary of %d", V);
    LGML_REQUIRE(top >= 0 && top <= TOP_MAX && top <= V, "token_logprobs: %d alternatives (0 to %d, at most the vocabulary)", top, TOP_MAX);
    LGML_REQUIRE(n_slices >= 1 && n_slices <= MAX_SLICES, "token_logprobs: %d slices (1 to %d)", n_slices, MAX_SLICES);
    LGML_REQUIRE(n_slices == 1 || (scratch != nullptr && ((uintptr_t)scratch & 15) == 0), "token_logprobs: several slices need scratch memory on 16 bytes");
    LGML_REQUIRE((long long)n_rows * n_slices <= 0x7fffffffLL, "token_logprobs: too many rows");
    if (n_rows == 0) return 0;
    const int chunks = (V + CHUNK - 1) / CHUNK, per = (chunks + n_slices - 1) / n_slices;
    const int vec = ld % 4 == 0 && ((uintptr_t)logits & 15) == 0;
    float4 *part = (float4 *)scratch;
    Key *keys = (Key *)(part + (size_t)n_rows * n_slices);
    const Outputs out{logprob, rank, entropy, top_ids, top_logprobs};
    lgml_launch(logprobs_kernel, dim3(n_rows * n_slices), THREADS, 0, stream, logits, ld, V, ids, top, n_slices, per, vec, part, keys, out, status);
    int rc = lgml_launch_status("token_logprobs");
    if (rc || n_slices == 1) return rc;
    lgml_launch(logprobs_join_kernel, dim3(n_rows), THREADS, 0, stream, logits, ld, V, ids, top, n_slices, part, keys, out);
    return lgml_launch_status("token_logprobs_join");
}
