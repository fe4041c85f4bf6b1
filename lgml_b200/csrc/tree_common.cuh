// What the kernels of tree_attention share (attention_tree.cu for few rows, attention_tree_tall.cu for many): the join of the ranges of a
// request's pages, inside a cluster or through scratch memory.
#pragma once
#include <cuda_fp16.h>
#include <math.h>

#include "common.cuh"

namespace {
constexpr int PAGE = 64;
constexpr int MAX_NEW = 64;             // bits of a mask
constexpr int MAX_SPLITS = 256, MAX_CLUSTER = 8;

__device__ __forceinline__ float power_of_two(int e) { return __uint_as_float((unsigned)(e + 127) << 23); }
__device__ __forceinline__ unsigned half2_of_codes(unsigned short two) {
    unsigned r;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(two));
    return r;
}
__device__ __forceinline__ float ex2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ uint32_t smem_u32(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void copy_16(uint32_t dst, const void *src, bool there) {
    const int bytes = there ? 16 : 0;            // 0: zeros
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ unsigned block_of_cluster() {
    unsigned r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_sync() { asm volatile("barrier.cluster.arrive.aligned;\nbarrier.cluster.wait.aligned;" ::: "memory"); }
// What block `rank` of the cluster has where this block has p.
__device__ __forceinline__ float2 load_there(const float *p, int rank) {
    uint32_t at;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_u32(p)), "r"(rank));
    float2 v;
    asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(at));
    return v;
}

// What a part with maximum m counts for beside others up to M (nothing seen: 0, or NaN, which stays one).
__device__ __forceinline__ float share_of(float m, float M) { return m == -INFINITY ? (M == -INFINITY ? 1.f : 0.f) : ex2(m - M); }
__device__ __forceinline__ void store_row(__nv_bfloat16 *dst, float2 o, float l) {
    const float inv = 1.f / l;
    *reinterpret_cast<__nv_bfloat162 *>(dst) = l == 0.f ? __floats2bfloat162_rn(0.f, 0.f) : __floats2bfloat162_rn(o.x * inv, o.y * inv);
}
// Where entry d of row r (token r / group, head r % group of a KV head) of a request's result lies.
__device__ __forceinline__ __nv_bfloat16 *row_at(__nv_bfloat16 *out, int ldo, int row0, int r, int group, int kvh, int D, int d) {
    return out + (size_t)(row0 + r / group) * ldo + (size_t)(kvh * group + r % group) * D + d;
}

// Every block of a cluster has its range's outputs in merge [ROWS][D + 2] and (maximum, sum) in fin: each joins a share of the rows, in the ranges' order.
template <int ROWS, int D, int THREADS, typename At>
__device__ __forceinline__ void join_cluster(const float *merge, const float (*fin)[2], int n_splits, int n_rows, At at) {
    for (int i = (int)block_of_cluster() * THREADS + (int)threadIdx.x; i < ROWS * (D / 2); i += n_splits * THREADS) {
        const int row = i / (D / 2), d = 2 * (i - row * (D / 2));
        if (row >= n_rows) break;
        float2 ml[MAX_CLUSTER], part[MAX_CLUSTER];
#pragma unroll
        for (int j = 0; j < MAX_CLUSTER; ++j)
            if (j < n_splits) ml[j] = load_there(fin[row], j), part[j] = load_there(merge + (size_t)row * (D + 2) + d, j);
        float M = -INFINITY, l = 0.f;
        float2 o = make_float2(0.f, 0.f);
#pragma unroll
        for (int j = 0; j < MAX_CLUSTER; ++j)
            if (j < n_splits) M = fmaxf(M, ml[j].x);
#pragma unroll
        for (int j = 0; j < MAX_CLUSTER; ++j)
            if (j < n_splits) {
                const float f = share_of(ml[j].x, M);
                l += ml[j].y * f;
                o.x += part[j].x * f, o.y += part[j].y * f;
            }
        store_row(at(row, d), o, l);
    }
}

// The ranges of one (token, head) in their order: a warp each.
constexpr int JOIN_WARPS = 2;
__global__ void __launch_bounds__(JOIN_WARPS * 32) tree_join_kernel(const float *__restrict__ part_o, const float2 *__restrict__ part_ml,
                                                                    const int *__restrict__ seq_start, int least, int limit, int n_tokens, __nv_bfloat16 *__restrict__ out,
                                                                    int ldo, int n_splits, int H, int D) {
    pdl_trigger();
    pdl_wait();
    const int s = blockIdx.x / limit, j = blockIdx.x - s * limit, lane = threadIdx.x & 31;
    const int head = blockIdx.y * JOIN_WARPS + (threadIdx.x >> 5);
    const int row0 = act_load(seq_start + s), n = act_load(seq_start + s + 1) - row0;
    if (j >= n || n < least || n > limit || head >= H || row0 < 0 || row0 + n > n_tokens) return;
    const size_t at = ((size_t)(row0 + j) * H + head) * n_splits;
    // lane i has the maxima and sums of ranges i, i + 32, ..; eight ranges' outputs are under way at a time
    constexpr int PER_LANE = MAX_SPLITS / 32;
    float2 ml[PER_LANE];
    float M = -INFINITY, l = 0.f;
#pragma unroll
    for (int p = 0; p < PER_LANE; ++p) {
        ml[p] = lane + 32 * p < n_splits ? act_load(part_ml + at + lane + 32 * p) : make_float2(-INFINITY, 0.f);
        M = fmaxf(M, ml[p].x);
    }
    M = warp_max(M);
#pragma unroll
    for (int p = 0; p < PER_LANE; ++p) {
        ml[p].x = share_of(ml[p].x, M);
        l += ml[p].y * ml[p].x;
    }
    l = warp_sum(l);
    float2 o[2] = {};
#pragma unroll
    for (int p = 0; p < PER_LANE; ++p)
        for (int i0 = 32 * p; i0 < min(n_splits, 32 * p + 32); i0 += 8) {
            float2 v[8][2];
#pragma unroll
            for (int e = 0; e < 8; ++e)
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    const int d = 2 * (lane + 32 * u);
                    v[e][u] = i0 + e < n_splits && d < D ? act_load(reinterpret_cast<const float2 *>(part_o + (at + i0 + e) * D + d)) : make_float2(0.f, 0.f);
                }
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float f = __shfl_sync(0xffffffffu, ml[p].x, (i0 + e) & 31);
#pragma unroll
                for (int u = 0; u < 2; ++u) o[u].x += v[e][u].x * f, o[u].y += v[e][u].y * f;
            }
        }
#pragma unroll
    for (int u = 0; u < 2; ++u) {
        const int d = 2 * (lane + 32 * u);
        if (d < D) store_row(out + (size_t)(row0 + j) * ldo + (size_t)head * D + d, o[u], l);
    }
}
int tree_join(const float *part_o, const float2 *part_ml, const int *seq_start, int n_seqs, int least, int limit, int n_tokens, void *out, int ldo, int n_splits, int H, int D,
              cudaStream_t stream) {
    lgml_launch(tree_join_kernel, dim3(n_seqs * limit, (H + JOIN_WARPS - 1) / JOIN_WARPS), JOIN_WARPS * 32, 0, stream, part_o, part_ml, seq_start, least, limit, n_tokens,
                (__nv_bfloat16 *)out, ldo, n_splits, H, D);
    return lgml_launch_status("tree_attention_join");
}
}  // namespace
