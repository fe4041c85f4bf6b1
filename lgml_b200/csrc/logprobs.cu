// Log probabilities of given tokens, with rank, entropy and the best alternatives, in one pass over the logits.
//
// A row x of V logits is the distribution p_i = exp(x_i - m) / s, m = max x, s = sum exp(x_i - m).  Wanted are
//     log p(id) = x_id - m - log s,        rank(id) = #{i: x_i > x_id, or x_i = x_id and i < id},
//     entropy   = log s - u / s            with u = sum (x_i - m) exp(x_i - m)      (p = 0 contributes 0),
// and the k largest x_i with their log p, ordered by (x descending, i ascending).  Taking u about the maximum, not about
// zero, keeps the entropy exact when the logits are far from zero.
//
// A block has a slice of a row, in chunks of 4,096 logits that come by bulk copies through a ring of stages (a row that starts off 16 bytes: from the
// boundary ahead on, the groups of four that it shares with its neighbours by loads): every thread keeps m, s, u and its count (online: s and u are rescaled when m grows), joined once at the end.  The best k come from the same pass: of a
// chunk only entries above the k-th best so far can be among them; they go to a list, which is ranked when it has grown (an entry's rank is how many
// of the list are above it), so most chunks cost one barrier.  Of the first chunk, a bound that k entries reach: every warp's q-th largest of its
// threads' maxima, q = ceil(k / 8), and of the eight warps' the least.  Where that leaves too many (equal logits; rising ones, later), the k-th largest of all the
// threads' maxima does not: entries are told apart by their index, so no more than k threads reach it, with 16 entries each.  Entries are 64-bit
// keys (the float's order, then the lower index first), so the order of arrival in the list changes nothing.
// The slices of a row are a cluster, whose first block joins them, slice after slice, out of the others' shared memory.  All sums are float32.
//
// What bounds it is instructions (0.67 of the cycles issue one; maximum, exponential, two sums, the comparisons, a chunk's ranking) and the chunks' barriers, then memory:
// 1,021 rows of 128,256 logits with 20 alternatives take 130 us (524 MB, 4.0 TB/s, 0.61 of the measured copy rate; without alternatives 86, 0.93); 8 rows 12.5 us, a cluster of 16 blocks a row.
// For those 1,021 rows: loads through registers and a ranking with every chunk 179; PER_SM blocks an SM: 2 224, 3 175, 4 133, 5 138, 6 190 (registers spill); two
// stages 133; the list ranked with every entry that comes 132, from RANK_AT = 16 on 133, from 64 on 140 (what it saves is barriers where few entries come).
#include <math.h>

#include "common.cuh"

LGML_DEFINE_LAST_ERROR(lgml_logprobs)

namespace {
constexpr int THREADS = 256;
constexpr int WARPS = THREADS / 32;
constexpr int PER = 16;                       // logits a thread holds
constexpr int CHUNK = THREADS * PER;
constexpr int TOP_MAX = 32;
constexpr int BUFFER = TOP_MAX * PER;         // entries of the list
constexpr int RANK_AT = 16;                   // ... and this many more than the best are ranked
constexpr int STAGES = 3;
constexpr int PER_SM = 4;                     // blocks that an SM holds
constexpr int MAX_SLICES = 16;                // blocks of a cluster
constexpr float LOG2E = 1.4426950408889634f;

typedef unsigned long long Key;

__device__ __forceinline__ float ex2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
// The larger one, or NaN if either is.
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
// two float32 sums, products, or products-and-sums, in one instruction
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    uint64_t d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(*reinterpret_cast<uint64_t *>(&a)), "l"(*reinterpret_cast<uint64_t *>(&b)));
    return *reinterpret_cast<float2 *>(&d);
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    uint64_t d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(*reinterpret_cast<uint64_t *>(&a)), "l"(*reinterpret_cast<uint64_t *>(&b)));
    return *reinterpret_cast<float2 *>(&d);
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(*reinterpret_cast<uint64_t *>(&a)), "l"(*reinterpret_cast<uint64_t *>(&b)), "l"(*reinterpret_cast<uint64_t *>(&c)));
    return *reinterpret_cast<float2 *>(&d);
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

// Of the n keys in list (shared memory) the k largest, in order, to best; places without an entry get 0.  Eight neighbouring threads count for a key.
__device__ __forceinline__ void rank_keys(const Key *list, int n, Key *best, int k) {
    const int part = threadIdx.x & 7;
    for (int i0 = 0; i0 < n; i0 += THREADS / 8) {
        const int i = i0 + (threadIdx.x >> 3);
        const Key mine = i < n ? list[i] : 0;
        int before = 0;
#pragma unroll 4
        for (int j = part; j < n; j += 8) before += list[j] > mine;
        before += __shfl_xor_sync(0xffffffffu, before, 1);
        before += __shfl_xor_sync(0xffffffffu, before, 2);
        before += __shfl_xor_sync(0xffffffffu, before, 4);
        if (part == 0 && i < n && before < k) best[before] = mine;
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
    Key list[TOP_MAX + BUFFER];          // entries above the k-th best when they came, and room for the best; at the end, the slices' best
    Key best[TOP_MAX];
    Key thread_best[THREADS];
    float4 mine;                         // of the slice: m, s, u, the count
    Stats warp_stats[WARPS];
    int warp_count[WARPS];
    unsigned warp_bound[WARPS];
    int came[3];                         // entries of a chunk (by its number modulo 3: one is counted, one read, one cleared)
    Key bound;
    unsigned long long full[STAGES];
};

__device__ __forceinline__ bool stage_full(unsigned long long *bar, unsigned parity) {
    unsigned ok;
    asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                 : "=r"(ok) : "r"((uint32_t)__cvta_generic_to_shared(bar)), "r"(parity), "r"(1000u) : "memory");
    return ok != 0;
}

// The list's entries and the best so far -> the best.
__device__ __forceinline__ void rank_list(Shared &sh, int n, int top) {
    if (threadIdx.x < top) sh.list[n + threadIdx.x] = sh.best[threadIdx.x];
    __syncthreads();
    rank_keys(sh.list, n + top, sh.best, top);
    __syncthreads();
}

__global__ void __launch_bounds__(THREADS, PER_SM) logprobs_kernel(const float *__restrict__ logits, long long ld, int V, const int *__restrict__ ids, int top,
                                                                   int n_slices, int chunks_per_slice, Outputs out, int *__restrict__ status) {
    pdl_trigger();
    extern __shared__ __align__(128) float ring[];          // [STAGES][CHUNK]
    __shared__ __align__(16) Shared sh;
    const int r = blockIdx.x / n_slices, slice = n_slices > 1 ? (int)block_of_cluster() : 0, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const float *row = logits + (size_t)r * ld;
    // Places are counted from the 16-byte boundary at or ahead of the row's start: logit i is at place i + off.
    const int off = (int)(((uintptr_t)row >> 2) & 3);
    const float *from0 = row - off;
    const int begin = (int)min((long long)V + off, (long long)slice * chunks_per_slice * CHUNK);
    const int end = (int)min((long long)V + off, (long long)(slice + 1) * chunks_per_slice * CHUNK), n_chunks = (end - begin + CHUNK - 1) / CHUNK;
    if (tid == 0) {
        for (int i = 0; i < STAGES; ++i) asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"((uint32_t)__cvta_generic_to_shared(&sh.full[i])));
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (tid < TOP_MAX) sh.best[tid] = 0;
    if (tid < 3) sh.came[tid] = 0;
    pdl_wait();
    // Chunk c on its way to stage c % STAGES: its groups of four that are the row's alone (one thread).
    auto ask = [&](int c) {
        const int base = begin + c * CHUNK, lo = base == 0 && off ? 4 : base, hi = min(base + CHUNK, end) & ~3;
        const int bytes = max(hi - lo, 0) * 4;
        const uint32_t bar = (uint32_t)__cvta_generic_to_shared(&sh.full[c % STAGES]);
        asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
        if (bytes > 0)
            asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                             (uint32_t)__cvta_generic_to_shared(ring + (c % STAGES) * CHUNK + (lo - base))), "l"(from0 + lo), "r"(bytes), "r"(bar) : "memory");
    };
    if (tid == 0)
        for (int c = 0; c < min(STAGES, n_chunks); ++c) ask(c);
    const int id = act_load(ids + r);
    const bool known = id >= 0 && id < V;
    if (!known && id != -1 && tid == 0) atomicExch(status, 1);
    const float x_id = known ? act_load(row + id) : __int_as_float(0x7fffffff);
    __syncthreads();

    Stats st{-INFINITY, 0.f, 0.f};
    int greater = 0, n_list = 0;
    for (int c = 0; c < n_chunks; ++c) {
        // a thread's j-th logit is first + (j / 4) 4 THREADS + j % 4
        const int base = begin + c * CHUNK, first = base - off + tid * 4, last = end - off;
        float x[PER];
        unsigned polls = 0;         // (of a microsecond each: about a second)
        while (!stage_full(&sh.full[c % STAGES], (c / STAGES) & 1) && ++polls < (1u << 20)) {
        }
        if (polls == (1u << 20)) atomicExch(status, 15);
        const bool inner = first >= 0 && base + CHUNK <= end;
#pragma unroll
        for (int j = 0; j < PER / 4; ++j) {
            const int i = first + j * THREADS * 4;
            if (inner || (i >= 0 && i + 3 < last)) {
                const float4 v = *reinterpret_cast<const float4 *>(ring + (c % STAGES) * CHUNK + (j * THREADS + tid) * 4);
                x[4 * j] = v.x, x[4 * j + 1] = v.y, x[4 * j + 2] = v.z, x[4 * j + 3] = v.w;
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) x[4 * j + e] = i + e >= 0 && i + e < last ? act_load(row + i + e) : -INFINITY;
            }
        }
        // ---- sums ----
        float largest4[PER / 4], largest = -INFINITY;
#pragma unroll
        for (int j = 0; j < PER / 4; ++j) {
            largest4[j] = fmaxf(fmaxf(x[4 * j], x[4 * j + 1]), fmaxf(x[4 * j + 2], x[4 * j + 3]));
            largest = fmaxf(largest, largest4[j]);
        }
        if (largest > st.m) st = about(st, largest);
        const float ref = st.m == -INFINITY ? 0.f : st.m;
        float2 s2 = make_float2(0.f, 0.f), u2 = s2;
#pragma unroll
        for (int j = 0; j < PER / 2; ++j) {
            // (in powers of two; what is under 2^-200 of the largest is nothing, and -inf x 0 would be NaN)
            float2 d = mul2(add2(make_float2(x[2 * j], x[2 * j + 1]), make_float2(-ref, -ref)), make_float2(LOG2E, LOG2E));
            d.x = max_nan(d.x, -200.f), d.y = max_nan(d.y, -200.f);
            const float2 w = make_float2(ex2(d.x), ex2(d.y));
            s2 = add2(s2, w);
            u2 = fma2(d, w, u2);
        }
        st.s += s2.x + s2.y;
        st.u += (u2.x + u2.y) * 0.6931471805599453f;
        if (largest >= x_id) {          // (mostly nobody: the given token is one of the best)
            // (an equal one counts if its index is lower: all of a chunk ahead of the id's, none of one behind it)
            const int chunk_from = base - off;
            float2 above = make_float2(0.f, 0.f);
            if (chunk_from > id) {
#pragma unroll
                for (int j = 0; j < PER; j += 2) above = add2(above, make_float2(x[j] > x_id ? 1.f : 0.f, x[j + 1] > x_id ? 1.f : 0.f));
            } else if (chunk_from >= 0 && chunk_from + CHUNK <= id) {
#pragma unroll
                for (int j = 0; j < PER; j += 2) above = add2(above, make_float2(x[j] >= x_id ? 1.f : 0.f, x[j + 1] >= x_id ? 1.f : 0.f));
            } else {
#pragma unroll
                for (int j = 0; j < PER; ++j) {
                    const int i = first + (j >> 2) * THREADS * 4 + (j & 3);           // (below 0: -inf ahead of a row that starts off 16 bytes, which is no entry)
                    above.x += x[j] > x_id || (x[j] == x_id && i >= 0 && i < id) ? 1.f : 0.f;
                }
            }
            greater += (int)(above.x + above.y);
        }
        // ---- the best ----
        auto collect = [&](int *count, auto pass) {
#pragma unroll
            for (int j = 0; j < PER; ++j) {
                const int i = first + (j >> 2) * THREADS * 4 + (j & 3);
                if (i >= 0 && i < last && pass(x[j], i)) {
                    const int at = n_list + atomicAdd(count, 1);
                    if (at < BUFFER) sh.list[at] = key_of(x[j], i);
                }
            }
        };
        int *count = &sh.came[c % 3];
        if (tid == 0) sh.came[(c + 1) % 3] = 0;
        const Key kth = top > 0 ? sh.best[top - 1] : 0;
        const unsigned kth_order = (unsigned)(kth >> 32);          // 0: not k yet, or NaNs among them
        if (top > 0 && kth_order != 0) {
            // (entries of later chunks have larger indices: an equal value does not displace the k-th best)
            const float least = value_of(kth);
            if (largest > least) {              // (a few threads, and of those mostly one group of four)
#pragma unroll
                for (int j = 0; j < PER / 4; ++j) {
                    if (!(largest4[j] > least)) continue;
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (x[4 * j + e] > least) {
                            const int at = n_list + atomicAdd(count, 1);
                            if (at < BUFFER) sh.list[at] = key_of(x[4 * j + e], first + j * THREADS * 4 + e);
                        }
                }
            }
        } else if (top > 0) {
            unsigned left = 0, q_th = 0;              // (places past the slice are none)
#pragma unroll
            for (int j = 0; j < PER; ++j)
                if (first + (j >> 2) * THREADS * 4 + (j & 3) >= 0 && first + (j >> 2) * THREADS * 4 + (j & 3) < last) left = max(left, order_of(x[j]));
            for (int q = 0; q < (top + WARPS - 1) / WARPS; ++q) {
                q_th = __reduce_max_sync(0xffffffffu, left);
                if (lane == __ffs(__ballot_sync(0xffffffffu, left == q_th)) - 1) left = 0;
            }
            if (lane == 0) sh.warp_bound[warp] = q_th;
            __syncthreads();
            unsigned bound = sh.warp_bound[0];
#pragma unroll
            for (int w = 1; w < WARPS; ++w) bound = min(bound, sh.warp_bound[w]);
            collect(count, [=](float v, int i) { return order_of(v) >= bound && key_of(v, i) > kth; });
        }
        __syncthreads();                // the stage has been read, the chunk's entries are in the list
        if (tid == 0 && c + STAGES < n_chunks) ask(c + STAGES);
        if (top == 0) continue;
        const int came = *count;
        if (n_list + came > BUFFER) {
            // too many: the list without them, then this chunk's by the bound that holds
            rank_list(sh, n_list, top);
            n_list = 0;
            const Key now = sh.best[top - 1];
            Key local = 0;
#pragma unroll
            for (int j = 0; j < PER; ++j) {
                const int i = first + (j >> 2) * THREADS * 4 + (j & 3);
                if (i >= 0 && i < last) local = max(local, key_of(x[j], i));
            }
            sh.thread_best[tid] = local;
            if (tid == 0) *count = 0;
            __syncthreads();
            int before = 0;
            for (int j = 0; j < THREADS; ++j) before += sh.thread_best[j] > local || (sh.thread_best[j] == local && j < tid);
            if (before == top - 1) sh.bound = local;
            __syncthreads();
            const Key bound = sh.bound;
            collect(count, [=](float v, int i) { const Key k = key_of(v, i); return k > now && k >= bound; });
            __syncthreads();
            n_list = *count;
        } else {
            n_list += came;
        }
        // (the first time the k-th best is what the chunks behind go by)
        if (n_list > (kth_order != 0 ? top + RANK_AT : 0)) {
            rank_list(sh, n_list, top);
            n_list = 0;
        }
    }
    if (top > 0 && n_list > 0) rank_list(sh, n_list, top);

    // ---- join the threads ----
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        st = join(st, Stats{__shfl_xor_sync(0xffffffffu, st.m, o), __shfl_xor_sync(0xffffffffu, st.s, o), __shfl_xor_sync(0xffffffffu, st.u, o)});
        greater += __shfl_xor_sync(0xffffffffu, greater, o);
    }
    __syncthreads();
    if (lane == 0) sh.warp_stats[warp] = st, sh.warp_count[warp] = greater;
    __syncthreads();
    if (tid == 0) {
        for (int w = 1; w < WARPS; ++w) st = join(st, sh.warp_stats[w]), greater += sh.warp_count[w];
        sh.mine = make_float4(st.m, st.s, st.u, __int_as_float(greater));
    }
    // ---- and the slices ----
    if (n_slices > 1) {
        __syncwarp();                   // (the barrier takes whole warps)
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
        __syncwarp();
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

// Into how many slices (a power of two) a row is cut: what takes the fewest rounds of blocks, each as long as its chunks and what a slice costs beside them.
LGML_API int lgml_token_logprobs_slices(int n_rows, int V, int n_sms) {
    const int chunks = (V + 3 + CHUNK - 1) / CHUNK, slots = PER_SM * n_sms, beside = 2;
    int best = 1;
    long long least = 0;
    for (int s = 1; s <= MAX_SLICES && s <= chunks; s *= 2) {
        const long long cost = (((long long)n_rows * s + slots - 1) / slots) * ((chunks + s - 1) / s + beside);
        if (s == 1 || cost < least) best = s, least = cost;
    }
    return best;
}

LGML_API int lgml_token_logprobs(const float *logits, long long ld, int n_rows, int V, const int *ids, int top, int n_slices, float *logprob, int *rank,
                                 float *entropy, int *top_ids, float *top_logprobs, int *status, cudaStream_t stream) {
    LGML_REQUIRE(n_rows >= 0 && V > 0 && ld >= V, "token_logprobs: %d rows of %d logits, %lld apart", n_rows, V, ld);
    LGML_REQUIRE(V <= 1 << 30, "token_logprobs: a vocabulary of %d", V);
    LGML_REQUIRE(top >= 0 && top <= TOP_MAX && top <= V, "token_logprobs: %d alternatives (0 to %d, at most the vocabulary)", top, TOP_MAX);
    LGML_REQUIRE(((uintptr_t)logits & 3) == 0, "token_logprobs: logits off 4 bytes");
    LGML_REQUIRE(n_slices >= 1 && n_slices <= MAX_SLICES && (n_slices & (n_slices - 1)) == 0, "token_logprobs: %d slices (a power of two up to %d)", n_slices,
                 MAX_SLICES);
    LGML_REQUIRE((long long)n_rows * n_slices <= 0x7fffffffLL, "token_logprobs: too many rows");
    if (n_rows == 0) return 0;
    const int chunks = (V + 3 + CHUNK - 1) / CHUNK, per = (chunks + n_slices - 1) / n_slices;          // (a row may start 3 places behind a boundary)
    const size_t smem = sizeof(float) * STAGES * CHUNK;
    const Outputs out{logprob, rank, entropy, top_ids, top_logprobs};
    cudaError_t e = cudaFuncSetAttribute(logprobs_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e == cudaSuccess && n_slices > 8) e = cudaFuncSetAttribute(logprobs_kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e != cudaSuccess) LGML_FAIL("token_logprobs: no blocks of %zu bytes in clusters of %d: %s", smem, n_slices, cudaGetErrorString(e));
    lgml_launch_cluster(logprobs_kernel, dim3(n_rows * n_slices), THREADS, smem, stream, n_slices, logits, ld, V, ids, top, n_slices, per, out, status);
    return lgml_launch_status("token_logprobs");
}
