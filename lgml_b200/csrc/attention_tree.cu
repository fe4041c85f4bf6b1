// Attention of a few new tokens a request over its paged cache, in bfloat16 or in e4m3 with one power of two a vector:
// a token a request when decoding, a short portion, or drafted tokens that form a tree.
//
// Request s brings the rows seq_start[s] .. seq_start[s + 1] of q; its cells 0 .. pos0 - 1 hold what earlier steps wrote and cell
// pos0 + j the key and value of its j-th new token.  A token sees every old cell and those new cells whose bit of its mask is
// set (without masks: new cells up to its own); with a window, of these the cells whose position is over its own less the window
// (an old cell's position is its number, a new one's is its token's).
//     o = sum_c p_c v_c / sum_c p_c,   p_c = exp2(scale log2(e) q.k_c - m)      over the visible cells; none: zeros
//
// Rows: a request's (token, head of the KV head) pairs, 8 NT of them a block.  The keys are the M side of the tensor-core tiles
// (mma.sync m16n8k16), so that a token's few heads fill an N of 8:
//     S^T[16 keys, 8 rows] = K[16, D] . Q^T        O^T[D, 8 rows] += V^T[D, 16] . P^T
// Each of a block's four warps is a pipeline of its own: of every page it takes a quarter, 16 cells, through a ring of stages in shared memory that
// 16-byte asynchronous copies fill (rows 16 bytes apart from a multiple of 128, so that neither products' reads meet a bank twice).  The order of the D entries
// inside a product, and of the D rows of O^T, is free: a thread's entries of a row are neighbours, and it reads 16 bytes at a time.
// The ranges of a request's pages are a cluster of up to 8 blocks, which join through one another's shared memory; where there are more,
// through scratch memory and a second kernel.
//
// e4m3: codes are exact in float16, so the products are of float16 (q is scaled per row by a power of two so that its largest
// entry is in [2^14, 2^15): rounding it to float16 loses nothing above 2^-39 of that).  A key's power of two multiplies its score, exactly.  A value's joins
// the exponent of its weight in the numerator: with w = log2 of the value's power, p'_c = 2^15 exp2(score + w_c - m'), m' the maximum of score + w, is
// at most 2^15 and is rounded to float16: half a step, 2^-11 of it, down to 2^-29 of the largest, and 2^-40 of the largest under that.  The sum of the weights is another matter: a
// value of zeros, or a small one, may have most of the weight, and beside it p' says nothing of that.  So it is of exp2(score - m) in float32, about a maximum of
// the scores alone (every thread has one of its own, which needs no exchange), and the two meet at the end: o = exp2(m' - m) sum p' code / sum p.
// bfloat16: p is rounded to bfloat16 (2^-8), and the sum takes the rounded ones.  Maxima, sums and outputs are float32.
//
// A value that is not finite must not reach a row that does not see it (0 x NaN): in blocks of 16 cells that not every row sees whole,
// values are looked at, and where one is not finite the block's products are formed one by one.
//
// What bounds it: with a token a request, memory, and for small caches the way there and back (a launch, a trip to the table, the cells, the join).  32 heads on 8
// of 128, e4m3: 64 requests of up to 4,097 cells 86 us (403 MB, 4.7 TB/s: 0.72 of the measured copy rate; the requests' lengths differ, so the last
// blocks run alone), of 4,096 cells each 96 (541 MB, 5.6 TB/s: 0.86); eight of 2,176 cells 17 us (36 MB; 8.6 of them with cells on their way); one of 1,001 cells 6.9.
// (The sum of the weights by itself, ahead of the weights for the values, is 1 to 2 % of these, 6 % of four tokens of 64 requests.)  A tile of rows keeps two stages a
// warp in flight, so that four blocks share an SM; more tiles three.  Taking the codes into mma.sync.m16n8k32 as they are, in place of converting them, measured
// the same (the conversions hide behind the loads) and is not here.
#include <cuda_fp16.h>
#include <math.h>

#include "tree_common.cuh"

LGML_DEFINE_LAST_ERROR(lgml_attention_tree)

namespace {
constexpr int WARPS = 4;
constexpr int THREADS = WARPS * 32;

__device__ __forceinline__ unsigned transpose8(unsigned a) {
    unsigned r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(a));
    return r;
}
template <bool Q8>
__device__ __forceinline__ void mma(float (&c)[4], unsigned a0, unsigned a1, unsigned a2, unsigned a3, unsigned b0, unsigned b1) {
    if (Q8)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// N 32-bit words of shared memory, at most four at a time.
template <int N>
__device__ __forceinline__ void read_words(unsigned (&r)[N], const uint8_t *p) {
    if (N % 4 == 0) {
#pragma unroll
        for (int i = 0; i < N; i += 4) {
            const uint4 v = *reinterpret_cast<const uint4 *>(p + 4 * i);
            r[i] = v.x, r[(i + 1) % N] = v.y, r[(i + 2) % N] = v.z, r[(i + 3) % N] = v.w;
        }
    } else if (N == 2) {
        const uint2 v = *reinterpret_cast<const uint2 *>(p);
        r[0] = v.x, r[N - 1] = v.y;
    } else {
        r[0] = *reinterpret_cast<const unsigned *>(p);
    }
}

// Which entries of a row a thread has, for rows of KS x 16 entries.
//   keys: thread c = lane % 4 has, of every 4 E neighbouring entries, E: as the columns of E / 4 products
//   values: thread g = lane / 4 has, of every 8 E neighbouring entries, E: as rows g and g + 8 of E / 2 products
template <int KS, int NT, bool Q8> struct Cut {
    static constexpr int SIZE = Q8 ? 1 : 2;
    static constexpr int KE = Q8 ? (KS % 8 == 0 ? 32 : KS % 4 == 0 ? 16 : KS % 2 == 0 ? 8 : 4) : (KS % 4 == 0 ? 16 : KS % 2 == 0 ? 8 : 4);
    static constexpr int VE = Q8 ? (KS % 8 == 0 ? 16 : KS % 4 == 0 ? 8 : KS % 2 == 0 ? 4 : 2) : (KS % 4 == 0 ? 8 : KS % 2 == 0 ? 4 : 2);
    static constexpr int KW = KE * SIZE / 4, VW = VE * SIZE / 4;       // words of these (a value's 2 codes of e4m3: half a word)
    static constexpr int ROW = KS * 16 * SIZE, PITCH = ROW + 16;       // bytes of a row, and from row to row in a stage
    static constexpr int STAGE = 32 * PITCH + 32;                      // 16 keys, 16 values, their exponents
    static constexpr int STAGES = NT == 1 ? 2 : 3;                     // (one tile of rows: more blocks on an SM are worth more than a third stage)
    static __device__ __forceinline__ int key_entry(int ks, int c) { return (ks / (KE / 4)) * 4 * KE + c * KE + (ks % (KE / 4)) * 4; }
    static __device__ __forceinline__ int value_entry(int mt, int g) { return (mt / (VE / 2)) * 8 * VE + g * VE + (mt % (VE / 2)) * 2; }
};

template <int KS, int NT, bool Q8>
__global__ void __launch_bounds__(THREADS) tree_attention_kernel(
    const __nv_bfloat16 *__restrict__ q, int ldq, const int *__restrict__ positions, const int *__restrict__ seq_start, const int *__restrict__ seq_pos0,
    const long long *__restrict__ visible, const int *__restrict__ block_table, int max_blocks, const uint8_t *__restrict__ k_pages,
    const uint8_t *__restrict__ v_pages, const uint8_t *__restrict__ k_exps, const uint8_t *__restrict__ v_exps, int n_pages, __nv_bfloat16 *__restrict__ out,
    int ldo, float *__restrict__ part_o, float2 *__restrict__ part_ml, int n_splits, int clustered, int n_tokens, int H, int Hkv, int n_chunks, int least, int limit,
    float scale, int window, int *__restrict__ status) {
    pdl_trigger();
    constexpr int D = KS * 16, ROWS = 8 * NT;
    constexpr float P_UP = Q8 ? 15.f : 0.f;               // the numerator's weights are times 2^this
    using C = Cut<KS, NT, Q8>;
    extern __shared__ __align__(16) uint8_t smem[];                // the warps' stages; at the end [WARPS][ROWS][D + 2] floats
    __shared__ int row_pos[ROWS];
    __shared__ long long row_mask[ROWS];
    __shared__ __align__(8) float fin[ROWS][2];
    __shared__ int stage_page[WARPS][C::STAGES];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, c = lane & 3;
    const int s = blockIdx.x / n_splits, split = blockIdx.x - s * n_splits, kvh = blockIdx.y / n_chunks, chunk = blockIdx.y - kvh * n_chunks;
    // (the step's description, down to the first pages' numbers, is read while the kernels ahead may still run)
    const int row0 = early_int(seq_start + s), n = early_int(seq_start + s + 1) - row0, pos0 = early_int(seq_pos0 + s);
    const int group = H / Hkv, n_rows = n * group, r0 = chunk * ROWS;
    // (The first block waits also where it leaves: a grid none of whose blocks waited could be over before the kernels ahead are, and the kernel behind waits for this
    // grid alone.  The others that leave make room at once; where they waited too, one request of 64 tokens beside 64 decoding ones took 20 us more.)
    const bool misplaced = row0 < 0 || row0 + n > n_tokens || pos0 < 0;
    if (n < least || n > limit || r0 >= n_rows || misplaced) {
        const bool report = misplaced && n >= least && n <= limit;
        if (report || (blockIdx.x == 0 && blockIdx.y == 0)) pdl_wait();
        if (report && tid == 0) atomicExch(status, 3);
        return;
    }
    if (tid < ROWS) {
        const int r = min(r0 + tid, n_rows - 1), tok = r / group;
        row_pos[tid] = early_int(positions + row0 + tok);
        row_mask[tid] = visible ? __ldcg(visible + row0 + tok) : (long long)(~0ull >> (63 - tok));
    }
    __syncthreads();

    // the cells of this split, in whole pages
    const int n_cells = pos0 + n;
    int low = 0, all_from = 0;              // none of the rows sees a cell below the first, every row sees the old cells from the second on
    if (window > 0) {
        int lowest = row_pos[0], highest = row_pos[0];
        for (int i = 1; i < ROWS; ++i) lowest = min(lowest, row_pos[i]), highest = max(highest, row_pos[i]);
        low = min(max(lowest - window + 1, 0), pos0);
        all_from = highest - window + 1;
    }
    const int first_page = low / PAGE, end_page = (n_cells + PAGE - 1) / PAGE;
    const int pps = (end_page - first_page + n_splits - 1) / n_splits;
    const int pb = first_page + split * pps, n_it = max(min(pps, end_page - pb), 0);

    // ---- the copies: this warp's quarter of page pb + it into stage it % STAGES ----
    uint8_t *ring = smem + (size_t)warp * C::STAGES * C::STAGE;
    auto table_from = [&](int it) { return it + lane < n_it && pb + it + lane < max_blocks ? early_int(block_table + (size_t)s * max_blocks + pb + it + lane) : -1; };
    int pages_ahead = table_from(0);        // the table's entry for iteration (it / 32) * 32 + lane
    auto fetch = [&](int it) {
        if ((it & 31) == 0 && it > 0) pages_ahead = table_from(it);
        int page = __shfl_sync(0xffffffffu, pages_ahead, it & 31);
        const int cell0 = (pb + it) * PAGE + warp * 16, left = n_cells - cell0;
        if (left <= 0 || cell0 + 16 <= low) {
            page = -1;                      // nothing there that a row could see
        } else if (page < 0 || page >= n_pages) {
            if (lane == 0) atomicExch(status, 3);
            page = -1;
        }
        uint8_t *stage = ring + (it % C::STAGES) * C::STAGE;
        if (lane == 0) stage_page[warp][it % C::STAGES] = page;
        if (page < 0) return;
        const size_t vec0 = ((size_t)page * Hkv + kvh) * PAGE + warp * 16;
        const uint8_t *kt = k_pages + vec0 * C::ROW, *vt = v_pages + vec0 * C::ROW;
        constexpr int PER_ROW = C::ROW / 16;
#pragma unroll
        for (int u = lane; u < 16 * PER_ROW; u += 32) {
            const int row = u / PER_ROW, col = (u - row * PER_ROW) * 16;
            const uint32_t to = smem_u32(stage + row * C::PITCH + col);
            copy_16(to, kt + row * C::ROW + col, row < left);
            copy_16(to + 16 * C::PITCH, vt + row * C::ROW + col, row < left);
        }
        if (Q8 && lane < 2) copy_16(smem_u32(stage + 32 * C::PITCH + 16 * lane), (lane ? v_exps : k_exps) + vec0, true);
    };
    // Q^T as B fragments: row g of n-tile nt, the entries that the keys' fragments have in this thread
    pdl_wait();
    unsigned qb[NT][KS][2];
    float q_unscale[NT][2];          // 2^-(row's scaling) of rows 2 c and 2 c + 1
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        const int r = r0 + nt * 8 + g;
        const bool there = r < n_rows;
        const __nv_bfloat16 *qrow = q + (size_t)(row0 + (there ? r / group : 0)) * ldq + (size_t)(kvh * group + (there ? r % group : 0)) * D;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            const unsigned *p = reinterpret_cast<const unsigned *>(qrow + C::key_entry(ks, c));
            qb[nt][ks][0] = there ? act_load(p) : 0u;
            qb[nt][ks][1] = there ? act_load(p + 1) : 0u;
        }
    }
#pragma unroll
    for (int it = 0; it < C::STAGES - 1; ++it) {
        if (it < n_it) fetch(it);
        copies_commit();
    }

    if (Q8)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            float amax = 0.f;
#pragma unroll
            for (int ks = 0; ks < KS; ++ks)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const float2 f = __bfloat1622float2(*reinterpret_cast<__nv_bfloat162 *>(&qb[nt][ks][e]));
                    amax = fmaxf(amax, fmaxf(fabsf(f.x), fabsf(f.y)));
                }
            amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
            amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
            // 2^x so that amax 2^x is in [2^14, 2^15); x within what float32 holds (an infinite amax: whatever, the row is NaN)
            const int x = min(max(14 - ((int)(__float_as_uint(amax) >> 23) - 127), -114), 100);
            const float up = power_of_two(x), down = power_of_two(-x);
#pragma unroll
            for (int ks = 0; ks < KS; ++ks)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const float2 f = __bfloat1622float2(*reinterpret_cast<__nv_bfloat162 *>(&qb[nt][ks][e]));
                    const __half2 h = __floats2half2_rn(f.x * up, f.y * up);
                    qb[nt][ks][e] = *reinterpret_cast<const unsigned *>(&h);
                }
            q_unscale[nt][0] = __shfl_sync(0xffffffffu, down, 8 * c);            // thread (g = 2 c, any) has row 2 c
            q_unscale[nt][1] = __shfl_sync(0xffffffffu, down, 8 * c + 4);
        }

    const float scale_log2 = scale * 1.4426950408889634f;
    float m_run[NT][2], l_run[NT][2], oacc[NT][KS][4];
    float m_sum[NT][2];              // (e4m3) the maximum that l_run is about: of this thread's scores
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        m_run[nt][0] = m_run[nt][1] = m_sum[nt][0] = m_sum[nt][1] = -INFINITY, l_run[nt][0] = l_run[nt][1] = 0.f;
#pragma unroll
        for (int i = 0; i < KS; ++i) oacc[nt][i][0] = oacc[nt][i][1] = oacc[nt][i][2] = oacc[nt][i][3] = 0.f;
    }

    for (int it = 0; it < n_it; ++it) {
        if (it + C::STAGES - 1 < n_it) fetch(it + C::STAGES - 1);
        copies_commit();
        copies_wait<C::STAGES - 1>();
        __syncwarp();
        const int page = stage_page[warp][it % C::STAGES];
        if (page < 0) {
            __syncwarp();
            continue;
        }
        const uint8_t *stage = ring + (it % C::STAGES) * C::STAGE, *vs = stage + 16 * C::PITCH, *es = stage + 32 * C::PITCH;
        const int cell0 = (pb + it) * PAGE + warp * 16, left = n_cells - cell0;
        int ke[2] = {0, 0}, ve[2] = {0, 0};
        if (Q8)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                ke[h] = min((int)es[g + 8 * h], 246) - 127;          // (246: the largest that is written)
                ve[h] = min((int)es[16 + g + 8 * h], 246) - 127;
            }

        // ---- S^T ----
        // (in two sums where there is one tile of rows: a product waits for the one before it in its sum)
        constexpr int SUMS = NT == 1 ? 2 : 1;
        float sc[NT][4], sums[SUMS][NT][4] = {};
#pragma unroll
        for (int i = 0; i < KS * 4 / C::KE; ++i) {
            unsigned kw[2][C::KW];
#pragma unroll
            for (int h = 0; h < 2; ++h) read_words(kw[h], stage + (g + 8 * h) * C::PITCH + (i * 4 * C::KE + c * C::KE) * C::SIZE);
#pragma unroll
            for (int u = 0; u < C::KE / 4; ++u) {
                unsigned a[4];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    if (Q8) a[h] = half2_of_codes((unsigned short)kw[h][u % C::KW]), a[2 + h] = half2_of_codes((unsigned short)(kw[h][u % C::KW] >> 16));
                    else a[h] = kw[h][(2 * u) % C::KW], a[2 + h] = kw[h][(2 * u + 1) % C::KW];
                }
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) mma<Q8>(sums[u % SUMS][nt], a[0], a[1], a[2], a[3], qb[nt][i * (C::KE / 4) + u][0], qb[nt][i * (C::KE / 4) + u][1]);
            }
        }
        // ---- which of them are seen: bit i of seen[nt] for sc[nt][i] ----
        const bool whole = cell0 + 16 <= pos0 && cell0 >= all_from;
        unsigned seen[NT];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            seen[nt] = 15u;
            if (!whole) {
                seen[nt] = 0u;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int cell = cell0 + g + 8 * (i >> 1), row = nt * 8 + 2 * c + (i & 1), j = cell - pos0;
                    if (cell >= n_cells) continue;
                    const int at = j < 0 ? cell : act_load(positions + row0 + j);
                    const bool yes = (j < 0 || ((row_mask[row] >> j) & 1)) && (window <= 0 || at > row_pos[row] - window);
                    if (yes) seen[nt] |= 1u << i;
                }
            }
        }
        // ---- probabilities ----
        const float kf[2] = {Q8 ? scale_log2 * power_of_two(ke[0]) : scale_log2, Q8 ? scale_log2 * power_of_two(ke[1]) : scale_log2};
        unsigned pb0[NT], pb1[NT];
        bool grown = false;
        float corr[NT][2], pr[NT][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float x = (SUMS == 2 ? sums[0][nt][i] + sums[SUMS - 1][nt][i] : sums[0][nt][i]) * kf[i >> 1];
                if (Q8) x *= q_unscale[nt][i & 1];
                sc[nt][i] = (seen[nt] >> i) & 1 ? x : -INFINITY;
            }
            if (Q8) {
                // the weights, and then the scores with the values' powers
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const float m_new = fmaxf(m_sum[nt][e], fmaxf(sc[nt][e], sc[nt][2 + e])), ref = m_new == -INFINITY ? 0.f : m_new;
                    l_run[nt][e] = l_run[nt][e] * ex2(m_sum[nt][e] - ref) + (ex2(sc[nt][e] - ref) + ex2(sc[nt][2 + e] - ref));
                    m_sum[nt][e] = m_new;
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) sc[nt][i] += (float)ve[i >> 1];
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) mx[i & 1] = fmaxf(mx[i & 1], sc[nt][i]);
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                mx[e] = fmaxf(mx[e], __shfl_xor_sync(0xffffffffu, mx[e], 4));
                mx[e] = fmaxf(mx[e], __shfl_xor_sync(0xffffffffu, mx[e], 8));
                mx[e] = fmaxf(mx[e], __shfl_xor_sync(0xffffffffu, mx[e], 16));
                const float m_new = fmaxf(m_run[nt][e], mx[e]);
                corr[nt][e] = m_new == m_run[nt][e] ? 1.f : ex2(m_run[nt][e] - m_new);
                grown |= m_new != m_run[nt][e];
                m_run[nt][e] = m_new;
                if (!Q8) l_run[nt][e] *= corr[nt][e];
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float m = m_run[nt][i & 1];
                pr[nt][i] = ex2(sc[nt][i] - (m == -INFINITY ? 0.f : m - P_UP));          // (unseen: exp2(-inf) = 0)
            }
            unsigned lo, hi;
            if (Q8) {
                const __half2 a = __floats2half2_rn(pr[nt][0], pr[nt][1]), b = __floats2half2_rn(pr[nt][2], pr[nt][3]);
                lo = *reinterpret_cast<const unsigned *>(&a), hi = *reinterpret_cast<const unsigned *>(&b);
                const float2 fa = __half22float2(a), fb = __half22float2(b);
                pr[nt][0] = fa.x, pr[nt][1] = fa.y, pr[nt][2] = fb.x, pr[nt][3] = fb.y;
            } else {
                const __nv_bfloat162 a = __floats2bfloat162_rn(pr[nt][0], pr[nt][1]), b = __floats2bfloat162_rn(pr[nt][2], pr[nt][3]);
                lo = *reinterpret_cast<const unsigned *>(&a), hi = *reinterpret_cast<const unsigned *>(&b);
                const float2 fa = __bfloat1622float2(a), fb = __bfloat1622float2(b);
                pr[nt][0] = fa.x, pr[nt][1] = fa.y, pr[nt][2] = fb.x, pr[nt][3] = fb.y;
            }
            if (!Q8)
#pragma unroll
                for (int i = 0; i < 4; ++i) l_run[nt][i & 1] += pr[nt][i];
            pb0[nt] = transpose8(lo);
            pb1[nt] = transpose8(hi);
        }
        if (__any_sync(0xffffffffu, grown)) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int mt = 0; mt < KS; ++mt)
#pragma unroll
                    for (int i = 0; i < 4; ++i) oacc[nt][mt][i] *= corr[nt][i & 1];
        }
        // ---- values that are not finite, among cells that not every row sees ----
        if (!whole) {
            bool odd = false;
            for (int u = lane; u < 16 * C::ROW / 4; u += 32) {
                const unsigned x = *reinterpret_cast<const unsigned *>(vs + (u / (C::ROW / 4)) * C::PITCH + (u % (C::ROW / 4)) * 4);
                if (Q8) odd |= (((x & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) != 0;
                else odd |= (x & 0x7f80u) == 0x7f80u || (x & 0x7f800000u) == 0x7f800000u;
            }
            if (__any_sync(0xffffffffu, odd)) {
                for (int key = 0; key < min(left, 16); ++key) {
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        const int from = (key & 7) * 4 + c;
                        const float p_a = __shfl_sync(0xffffffffu, key < 8 ? pr[nt][0] : pr[nt][2], from);
                        const float p_b = __shfl_sync(0xffffffffu, key < 8 ? pr[nt][1] : pr[nt][3], from);
                        const unsigned bits = __shfl_sync(0xffffffffu, seen[nt], from) >> (key < 8 ? 0 : 2);
#pragma unroll
                        for (int mt = 0; mt < KS; ++mt) {
                            const int d = C::value_entry(mt, g);
                            float2 v;
                            if (Q8) {
                                const unsigned h2 = half2_of_codes(*reinterpret_cast<const unsigned short *>(vs + key * C::PITCH + d));
                                v = __half22float2(*reinterpret_cast<const __half2 *>(&h2));
                            } else {
                                const unsigned b2 = *reinterpret_cast<const unsigned *>(vs + key * C::PITCH + 2 * d);
                                v = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162 *>(&b2));
                            }
                            if (bits & 1u) oacc[nt][mt][0] += p_a * v.x, oacc[nt][mt][2] += p_a * v.y;
                            if (bits & 2u) oacc[nt][mt][1] += p_b * v.x, oacc[nt][mt][3] += p_b * v.y;
                        }
                    }
                }
                __syncwarp();
                continue;
            }
        }
        // ---- O^T += V^T P^T ----
        constexpr int VWORDS = C::VW > 0 ? C::VW : 1;
#pragma unroll
        for (int i = 0; i < KS * 2 / C::VE; ++i) {
            unsigned vw[4][VWORDS];               // of cells 2 c, 2 c + 1, 2 c + 8, 2 c + 9
#pragma unroll
            for (int h = 0; h < 4; ++h) {
                const uint8_t *p = vs + (2 * c + (h & 1) + (h >> 1) * 8) * C::PITCH + (i * 8 * C::VE + g * C::VE) * C::SIZE;
                if (C::VW > 0) read_words(vw[h], p);
                else vw[h][0] = *reinterpret_cast<const unsigned short *>(p);
            }
#pragma unroll
            for (int u = 0; u < C::VE / 2; ++u) {
                unsigned a[4];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    if (Q8) {
                        const unsigned both = __byte_perm(vw[2 * h][u / 2], vw[2 * h + 1][u / 2], u % 2 ? 0x7362 : 0x5140);      // an entry of both cells, the next entry's
                        a[2 * h] = half2_of_codes((unsigned short)both), a[2 * h + 1] = half2_of_codes((unsigned short)(both >> 16));
                    } else {
                        a[2 * h] = __byte_perm(vw[2 * h][u % VWORDS], vw[2 * h + 1][u % VWORDS], 0x5410);
                        a[2 * h + 1] = __byte_perm(vw[2 * h][u % VWORDS], vw[2 * h + 1][u % VWORDS], 0x7632);
                    }
                }
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) mma<Q8>(oacc[nt][i * (C::VE / 2) + u], a[0], a[1], a[2], a[3], pb0[nt], pb1[nt]);
            }
        }
        __syncwarp();
    }
    copies_wait<0>();
    __syncthreads();                        // every warp is done with its stages

    // ---- the four warps together ----
    float *merge = reinterpret_cast<float *>(smem), *mine = merge + (size_t)warp * ROWS * (D + 2);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            float l = l_run[nt][e], m = m_run[nt][e], up = 1.f;
            if (Q8) {
                // the eight threads' sums about one maximum m, and the outputs about the same; both times 2^-24, so that sums of the largest values stay finite
                m = fmaxf(m_sum[nt][e], __shfl_xor_sync(0xffffffffu, m_sum[nt][e], 4));
                m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 8));
                m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 16));
                const bool none = m == -INFINITY;
                l *= ex2((none ? 0.f : m_sum[nt][e] - m) - 24.f);
                up = none ? 1.f : ex2(m_run[nt][e] - m - P_UP - 24.f);
            }
            l += __shfl_xor_sync(0xffffffffu, l, 4);
            l += __shfl_xor_sync(0xffffffffu, l, 8);
            l += __shfl_xor_sync(0xffffffffu, l, 16);
            float *row = mine + (size_t)(nt * 8 + 2 * c + e) * (D + 2);
#pragma unroll
            for (int mt = 0; mt < KS; ++mt) {
                const int d = C::value_entry(mt, g);
                *reinterpret_cast<float2 *>(row + d) = Q8 ? make_float2(oacc[nt][mt][e] * up, oacc[nt][mt][2 + e] * up) : make_float2(oacc[nt][mt][e], oacc[nt][mt][2 + e]);
            }
            if (g == 0) *reinterpret_cast<float2 *>(row + D) = make_float2(m, l);
        }
    __syncthreads();
    for (int i = tid; i < ROWS * (D / 2); i += THREADS) {
        const int row = i / (D / 2), d = 2 * (i - row * (D / 2));
        if (r0 + row >= n_rows) break;
        float M = -INFINITY, l = 0.f;
        float2 o = make_float2(0.f, 0.f);
#pragma unroll
        for (int w = 0; w < WARPS; ++w) M = fmaxf(M, merge[((size_t)w * ROWS + row) * (D + 2) + D]);
#pragma unroll
        for (int w = 0; w < WARPS; ++w) {
            const float *p = merge + ((size_t)w * ROWS + row) * (D + 2);
            const float f = share_of(p[D], M);
            l += p[D + 1] * f;
            o.x += p[d] * f, o.y += p[d + 1] * f;
        }
        if (n_splits == 1) {
            store_row(row_at(out, ldo, row0, r0 + row, group, kvh, D, d), o, l);
        } else if (clustered) {
            *reinterpret_cast<float2 *>(merge + (size_t)row * (D + 2) + d) = o;         // (no other thread reads it here)
            if (d == 0) fin[row][0] = M, fin[row][1] = l;
        } else {
            const size_t at = ((size_t)(row0 + (r0 + row) / group) * H + kvh * group + (r0 + row) % group) * n_splits + split;
            *reinterpret_cast<float2 *>(part_o + at * D + d) = o;
            if (d == 0) part_ml[at] = make_float2(M, l);
        }
    }
    if (!clustered) return;
    // ---- the cluster's ranges together: each block joins a share of the results ----
    __syncwarp();
    cluster_sync();
    join_cluster<ROWS, D, THREADS>(merge, fin, n_splits, n_rows - r0, [&](int row, int d) { return row_at(out, ldo, row0, r0 + row, group, kvh, D, d); });
    __syncwarp();
    cluster_sync();                         // (the others' shared memory is read until here)
}

template <int KS, int NT, bool Q8, typename... Args>
int launch_one(dim3 grid, int cluster, cudaStream_t stream, Args... args) {
    using C = Cut<KS, NT, Q8>;
    const size_t stages = (size_t)WARPS * C::STAGES * C::STAGE, merge = sizeof(float) * WARPS * 8 * NT * (KS * 16 + 2);
    const size_t smem = stages > merge ? stages : merge;
    cudaError_t e = cudaFuncSetAttribute(tree_attention_kernel<KS, NT, Q8>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) LGML_FAIL("tree_attention: cannot have %zu bytes of shared memory: %s", smem, cudaGetErrorString(e));
    lgml_launch_cluster(tree_attention_kernel<KS, NT, Q8>, grid, THREADS, smem, stream, cluster, args...);
    return lgml_launch_status("tree_attention");
}
template <int KS, bool Q8, typename... Args>
int launch_rows(int nt, Args... args) {
    return nt == 1 ? launch_one<KS, 1, Q8>(args...) : nt == 2 ? launch_one<KS, 2, Q8>(args...) : launch_one<KS, 4, Q8>(args...);
}
template <bool Q8, typename... Args>
int launch_dim(int ks, Args... args) {
    switch (ks) {
        case 1: return launch_rows<1, Q8>(args...);
        case 2: return launch_rows<2, Q8>(args...);
        case 3: return launch_rows<3, Q8>(args...);
        case 4: return launch_rows<4, Q8>(args...);
        case 5: return launch_rows<5, Q8>(args...);
        case 6: return launch_rows<6, Q8>(args...);
        case 7: return launch_rows<7, Q8>(args...);
        case 8: return launch_rows<8, Q8>(args...);
    }
    LGML_FAIL("tree_attention: head_dim %d not handled", 16 * ks);
}
}  // namespace

// least, limit: requests that bring fewer or more tokens than this are left alone (their rows of out too).  k_exps null: pages in bfloat16.
LGML_API int lgml_tree_attention(const void *q, int ldq, const int *positions, const int *seq_start, const int *seq_pos0, const long long *visible,
                                 const int *block_table, int n_seqs, int max_blocks, const void *k_pages, const void *v_pages, const void *k_exps,
                                 const void *v_exps, int n_pages, int page_size, void *out, int ldo, float *scratch, int n_splits, int n_tokens, int least, int limit, int H,
                                 int Hkv, int D, float scale, int window, int *status, cudaStream_t stream) {
    LGML_REQUIRE(n_tokens >= 0 && n_seqs >= 0 && H > 0 && Hkv > 0 && max_blocks > 0 && n_pages >= 0, "tree_attention: bad sizes");
    LGML_REQUIRE(page_size == PAGE, "tree_attention: pages of %d tokens, this kernel takes %d", page_size, PAGE);
    LGML_REQUIRE(H % Hkv == 0, "tree_attention: %d heads are no multiple of %d KV heads", H, Hkv);
    LGML_REQUIRE(D >= 16 && D <= 128 && D % 16 == 0, "tree_attention: head_dim %d must be a multiple of 16 up to 128", D);
    LGML_REQUIRE(least >= 1 && least <= limit && limit <= MAX_NEW, "tree_attention: %d to %d new tokens a request (1 to %d)", least, limit, MAX_NEW);
    LGML_REQUIRE(n_splits >= 1 && n_splits <= MAX_SPLITS, "tree_attention: %d key ranges (1 to %d)", n_splits, MAX_SPLITS);
    LGML_REQUIRE(n_splits <= MAX_CLUSTER || (scratch != nullptr && ((uintptr_t)scratch & 7) == 0), "tree_attention: several ranges need scratch memory");
    LGML_REQUIRE((k_exps == nullptr) == (v_exps == nullptr), "tree_attention: exponents for keys and values, or for neither");
    LGML_REQUIRE((((uintptr_t)k_pages | (uintptr_t)v_pages | (uintptr_t)k_exps | (uintptr_t)v_exps) & 15) == 0, "tree_attention: the cache must be 16-byte aligned");
    LGML_REQUIRE(ldq % 2 == 0 && ((uintptr_t)q & 3) == 0 && ldo % 2 == 0 && ((uintptr_t)out & 3) == 0,
                 "tree_attention: q and out must be 4-byte aligned with even row strides");
    LGML_REQUIRE((long long)n_seqs * (limit > n_splits ? limit : n_splits) <= 0x7fffffffLL, "tree_attention: too many requests");
    if (n_tokens == 0 || n_seqs == 0) return 0;
    const int rows = limit * (H / Hkv);
    const int nt = rows <= 8 ? 1 : rows <= 16 ? 2 : 4;
    const int n_chunks = (rows + 8 * nt - 1) / (8 * nt);
    LGML_REQUIRE((long long)Hkv * n_chunks <= 65535, "tree_attention: too many heads");
    const int clustered = n_splits > 1 && n_splits <= MAX_CLUSTER;
    dim3 grid(n_seqs * n_splits, Hkv * n_chunks);
    float *part_o = scratch;
    float2 *part_ml = scratch ? reinterpret_cast<float2 *>(scratch + (size_t)n_tokens * H * n_splits * D) : nullptr;
#define LGML_ARGS D / 16, nt, grid, clustered ? n_splits : 1, stream, (const __nv_bfloat16 *)q, ldq, positions, seq_start, seq_pos0, visible, block_table, max_blocks,            \
                  (const uint8_t *)k_pages, (const uint8_t *)v_pages, (const uint8_t *)k_exps, (const uint8_t *)v_exps, n_pages, (__nv_bfloat16 *)out, ldo, \
                  part_o, part_ml, n_splits, clustered, n_tokens, H, Hkv, n_chunks, least, limit, scale, window, status
    int rc = k_exps ? launch_dim<true>(LGML_ARGS) : launch_dim<false>(LGML_ARGS);
#undef LGML_ARGS
    if (rc || n_splits <= MAX_CLUSTER) return rc;
    return tree_join(part_o, part_ml, seq_start, n_seqs, least, limit, n_tokens, out, ldo, n_splits, H, D, stream);
}
