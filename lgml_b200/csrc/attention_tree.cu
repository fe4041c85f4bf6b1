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
// A warp takes 16 cells at a time and holds their part of everything in registers; keys and values go from memory to the fragments
// without shared memory, since the order of the D entries inside a product, and of the D rows of O^T, is free: a thread's entries of
// a row are neighbours, so its loads are 16 bytes wide, and a warp's loads whole rows.
//
// e4m3: codes are exact in float16, so the products are of float16 (q is scaled per row by a power of two so that its largest
// entry is in [2^14, 2^15): rounding it to float16 loses nothing above 2^-39 of that).  A key's power of two multiplies its score, exactly.  A value's joins
// the probability's exponent: with w = log2 of the value's power, p'_c = exp2(score + w_c - m'), m' the maximum of score + w; p' is at most 1 and is
// rounded to float16 (half a step: 2^-12), and the sum takes the rounded p' times 2^-w.  bfloat16: p is rounded to bfloat16 (2^-9), and the sum takes the rounded
// ones.  Maxima, sums and outputs are float32.
//
// A value that is not finite must not reach a row that does not see it (0 x NaN): in blocks of 16 cells that not every row sees whole,
// values are looked at, and where one is not finite the block's products are formed one by one.
#include <cuda_fp16.h>
#include <math.h>

#include "common.cuh"

LGML_DEFINE_LAST_ERROR(lgml_attention_tree)

namespace {
constexpr int PAGE = 64;
constexpr int WARPS = 4;
constexpr int THREADS = WARPS * 32;
constexpr int MAX_NEW = 64;             // bits of a mask
constexpr int MAX_SPLITS = 256;

__device__ __forceinline__ float power_of_two(int e) { return __uint_as_float((unsigned)(e + 127) << 23); }
__device__ __forceinline__ unsigned half2_of_codes(unsigned short two) {
    unsigned r;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(two));
    return r;
}
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

// N 32-bit words from p, by loads of W words (what has been written by the kernels ahead goes through L2).
template <int N, int W>
__device__ __forceinline__ void load_words(unsigned (&r)[N], const uint8_t *p, bool there) {
#pragma unroll
    for (int i = 0; i < N; i += W) {
        if (W == 4) {
            const uint4 v = there ? __ldcg(reinterpret_cast<const uint4 *>(p + 4 * i)) : make_uint4(0, 0, 0, 0);
            r[i] = v.x, r[(i + 1) % N] = v.y, r[(i + 2) % N] = v.z, r[(i + 3) % N] = v.w;
        } else if (W == 2) {
            const uint2 v = there ? __ldcg(reinterpret_cast<const uint2 *>(p + 4 * i)) : make_uint2(0, 0);
            r[i] = v.x, r[(i + 1) % N] = v.y;
        } else {
            r[i] = there ? __ldcg(reinterpret_cast<const unsigned *>(p + 4 * i)) : 0u;
        }
    }
}

// Which entries of a row a thread has, for rows of KS x 16 entries.
//   keys: thread c = lane % 4 has, of every 4 E neighbouring entries, E: as the columns of E / 4 products
//   values: thread g = lane / 4 has, of every 8 E neighbouring entries, E: as rows g and g + 8 of E / 2 products
template <int KS, bool Q8> struct Cut {
    static constexpr int SIZE = Q8 ? 1 : 2;
    static constexpr int KE = Q8 ? (KS % 4 == 0 ? 16 : KS % 2 == 0 ? 8 : 4) : (KS % 2 == 0 ? 8 : 4);
    static constexpr int VE = Q8 ? (KS % 8 == 0 ? 16 : KS % 4 == 0 ? 8 : KS % 2 == 0 ? 4 : 2) : (KS % 4 == 0 ? 8 : KS % 2 == 0 ? 4 : 2);
    static constexpr int KW = KE * SIZE / 4, VW = VE * SIZE / 4;       // words of a load (a value's 2 codes of e4m3: half a word)
    static __device__ __forceinline__ int key_entry(int ks, int c) { return (ks / (KE / 4)) * 4 * KE + c * KE + (ks % (KE / 4)) * 4; }
    static __device__ __forceinline__ int value_entry(int mt, int g) { return (mt / (VE / 2)) * 8 * VE + g * VE + (mt % (VE / 2)) * 2; }
};

template <int KS, int NT, bool Q8>
__global__ void __launch_bounds__(THREADS) tree_attention_kernel(
    const __nv_bfloat16 *__restrict__ q, int ldq, const int *__restrict__ positions, const int *__restrict__ seq_start, const int *__restrict__ seq_pos0,
    const long long *__restrict__ visible, const int *__restrict__ block_table, int max_blocks, const uint8_t *__restrict__ k_pages,
    const uint8_t *__restrict__ v_pages, const uint8_t *__restrict__ k_exps, const uint8_t *__restrict__ v_exps, int n_pages, __nv_bfloat16 *__restrict__ out,
    int ldo, float *__restrict__ part_o, float2 *__restrict__ part_ml, int n_splits, int n_tokens, int H, int Hkv, int n_chunks, int limit, float scale,
    int window, int *__restrict__ status) {
    pdl_trigger();
    constexpr int D = KS * 16, ROWS = 8 * NT;
    using C = Cut<KS, Q8>;
    extern __shared__ __align__(16) float merge[];                 // [WARPS][ROWS][D + 2] at the end
    __shared__ int row_pos[ROWS];
    __shared__ long long row_mask[ROWS];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, c = lane & 3;
    const int s = blockIdx.x, kvh = blockIdx.y / n_chunks, chunk = blockIdx.y - kvh * n_chunks, split = blockIdx.z;
    pdl_wait();
    const int row0 = act_load(seq_start + s), n = act_load(seq_start + s + 1) - row0, pos0 = act_load(seq_pos0 + s);
    const int group = H / Hkv, n_rows = n * group, r0 = chunk * ROWS;
    if (n <= 0 || n > limit || r0 >= n_rows) return;
    if (row0 < 0 || row0 + n > n_tokens || pos0 < 0) {
        if (tid == 0) atomicExch(status, 3);
        return;
    }
    if (tid < ROWS) {
        const int r = min(r0 + tid, n_rows - 1), tok = r / group;
        row_pos[tid] = act_load(positions + row0 + tok);
        row_mask[tid] = visible ? __ldcg(visible + row0 + tok) : (long long)(~0ull >> (63 - tok));
    }
    __syncthreads();

    // Q^T as B fragments: row g of n-tile nt, the entries that the keys' fragments have in this thread
    unsigned qb[NT][KS][2];
    float q_unscale[NT][2];          // 2^-(row's scaling) of rows 2 c and 2 c + 1
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        const int r = r0 + nt * 8 + g;
        const bool there = r < n_rows;
        const __nv_bfloat16 *qrow = q + (size_t)(row0 + (there ? r / group : 0)) * ldq + (size_t)(kvh * group + (there ? r % group : 0)) * D;
        float amax = 0.f;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            const unsigned *p = reinterpret_cast<const unsigned *>(qrow + C::key_entry(ks, c));
            qb[nt][ks][0] = there ? act_load(p) : 0u;
            qb[nt][ks][1] = there ? act_load(p + 1) : 0u;
            if (Q8)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const float2 f = __bfloat1622float2(*reinterpret_cast<__nv_bfloat162 *>(&qb[nt][ks][e]));
                    amax = fmaxf(amax, fmaxf(fabsf(f.x), fabsf(f.y)));
                }
        }
        if (Q8) {
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
    }

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
    const int pb = first_page + split * pps, pe = min(pb + pps, end_page);
    const int t_end = min(4 * pe, (n_cells + 15) / 16);

    const float scale_log2 = scale * 1.4426950408889634f;
    float m_run[NT][2], l_run[NT][2], oacc[NT][KS][4];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        m_run[nt][0] = m_run[nt][1] = -INFINITY, l_run[nt][0] = l_run[nt][1] = 0.f;
#pragma unroll
        for (int i = 0; i < KS; ++i) oacc[nt][i][0] = oacc[nt][i][1] = oacc[nt][i][2] = oacc[nt][i][3] = 0.f;
    }

    for (int tile = 4 * pb + warp; tile < t_end; tile += WARPS) {
        const int cell0 = tile * 16;
        const int blk = tile >> 2;
        int page = blk < max_blocks ? act_load(block_table + (size_t)s * max_blocks + blk) : -1;
        if (page < 0 || page >= n_pages) {
            if (lane == 0 && cell0 + 16 > low) atomicExch(status, 3);
            continue;
        }
        const size_t vec0 = ((size_t)page * Hkv + kvh) * PAGE + (tile & 3) * 16;
        const uint8_t *kt = k_pages + vec0 * D * C::SIZE, *vt = v_pages + vec0 * D * C::SIZE;
        const int left = n_cells - cell0;                          // cells of the tile that there are
        const int vkey[4] = {2 * c, 2 * c + 1, 2 * c + 8, 2 * c + 9};

        // ---- loads: keys g and g + 8; values of keys 2 c, 2 c + 1, 2 c + 8, 2 c + 9 ----
        constexpr int KL = KS * 4 / C::KE, VL = KS * 2 / C::VE;          // loads of a row
        unsigned kw[2][KL][C::KW];
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int i = 0; i < KL; ++i)
                load_words<C::KW, C::KW>(kw[h][i], kt + ((size_t)(g + 8 * h) * D + i * 4 * C::KE + c * C::KE) * C::SIZE, g + 8 * h < left);
        constexpr int VWORDS = C::VW > 0 ? C::VW : 1;
        unsigned vw[4][VL][VWORDS];
#pragma unroll
        for (int h = 0; h < 4; ++h)
#pragma unroll
            for (int i = 0; i < VL; ++i) {
                const uint8_t *p = vt + ((size_t)vkey[h] * D + i * 8 * C::VE + g * C::VE) * C::SIZE;
                if (C::VW > 0) load_words<VWORDS, VWORDS>(vw[h][i], p, vkey[h] < left);
                else vw[h][i][0] = vkey[h] < left ? (unsigned)__ldcg(reinterpret_cast<const unsigned short *>(p)) : 0u;
            }
        int ke[2] = {0, 0}, ve[2] = {0, 0};
        if (Q8)
#pragma unroll
            for (int h = 0; h < 2; ++h)
                if (g + 8 * h < left) {
                    ke[h] = min((int)__ldcg(k_exps + vec0 + g + 8 * h), 246) - 127;          // (246: the largest that is written)
                    ve[h] = min((int)__ldcg(v_exps + vec0 + g + 8 * h), 246) - 127;
                }

        // ---- S^T ----
        float sc[NT][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) sc[nt][0] = sc[nt][1] = sc[nt][2] = sc[nt][3] = 0.f;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            const int i = ks / (C::KE / 4), u = ks % (C::KE / 4);
            unsigned a[4];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                if (Q8) {
                    const unsigned w = kw[h][i][u];
                    a[h] = half2_of_codes((unsigned short)w), a[2 + h] = half2_of_codes((unsigned short)(w >> 16));
                } else {
                    a[h] = kw[h][i][(2 * u) % C::KW], a[2 + h] = kw[h][i][(2 * u + 1) % C::KW];
                }
            }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) mma<Q8>(sc[nt], a[0], a[1], a[2], a[3], qb[nt][ks][0], qb[nt][ks][1]);
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
        const float vf[2] = {Q8 ? power_of_two(-ve[0]) : 1.f, Q8 ? power_of_two(-ve[1]) : 1.f};
        unsigned pb0[NT], pb1[NT];
        bool grown = false;
        float corr[NT][2], pr[NT][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float x = sc[nt][i] * kf[i >> 1];
                if (Q8) x = x * q_unscale[nt][i & 1] + (float)ve[i >> 1];
                sc[nt][i] = (seen[nt] >> i) & 1 ? x : -INFINITY;
                mx[i & 1] = fmaxf(mx[i & 1], sc[nt][i]);
            }
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                mx[e] = fmaxf(mx[e], __shfl_xor_sync(0xffffffffu, mx[e], 4));
                mx[e] = fmaxf(mx[e], __shfl_xor_sync(0xffffffffu, mx[e], 8));
                mx[e] = fmaxf(mx[e], __shfl_xor_sync(0xffffffffu, mx[e], 16));
                const float m_new = fmaxf(m_run[nt][e], mx[e]);
                corr[nt][e] = m_new == m_run[nt][e] ? 1.f : exp2f(m_run[nt][e] - m_new);
                grown |= m_new != m_run[nt][e];
                m_run[nt][e] = m_new;
                l_run[nt][e] *= corr[nt][e];
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float m = m_run[nt][i & 1];
                pr[nt][i] = exp2f(sc[nt][i] - (m == -INFINITY ? 0.f : m));        // (unseen: exp2(-inf) = 0)
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
#pragma unroll
            for (int i = 0; i < 4; ++i) l_run[nt][i & 1] += pr[nt][i] * vf[i >> 1];
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
#pragma unroll
            for (int h = 0; h < 4; ++h)
#pragma unroll
                for (int i = 0; i < VL; ++i)
#pragma unroll
                    for (int w = 0; w < VWORDS; ++w) {
                        const unsigned x = vw[h][i][w];
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
                                const unsigned h2 = half2_of_codes(__ldcg(reinterpret_cast<const unsigned short *>(vt + (size_t)key * D + d)));
                                v = __half22float2(*reinterpret_cast<const __half2 *>(&h2));
                            } else {
                                const unsigned b2 = __ldcg(reinterpret_cast<const unsigned *>(vt + ((size_t)key * D + d) * 2));
                                v = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162 *>(&b2));
                            }
                            if (bits & 1u) oacc[nt][mt][0] += p_a * v.x, oacc[nt][mt][2] += p_a * v.y;
                            if (bits & 2u) oacc[nt][mt][1] += p_b * v.x, oacc[nt][mt][3] += p_b * v.y;
                        }
                    }
                }
                continue;
            }
        }
        // ---- O^T += V^T P^T ----
#pragma unroll
        for (int mt = 0; mt < KS; ++mt) {
            const int i = mt / (C::VE / 2), u = mt % (C::VE / 2);
            unsigned a[4];
#pragma unroll
            for (int h = 0; h < 2; ++h) {             // keys 2 c and 2 c + 1, then 2 c + 8 and 2 c + 9
                if (Q8) {
                    const unsigned wa = vw[2 * h][i][u / 2], wb = vw[2 * h + 1][i][u / 2];
                    const unsigned both = __byte_perm(wa, wb, u % 2 ? 0x7362 : 0x5140);          // entry of one key, of the other, the next entry's
                    a[2 * h] = half2_of_codes((unsigned short)both), a[2 * h + 1] = half2_of_codes((unsigned short)(both >> 16));
                } else {
                    const unsigned wa = vw[2 * h][i][u], wb = vw[2 * h + 1][i][u];
                    a[2 * h] = __byte_perm(wa, wb, 0x5410), a[2 * h + 1] = __byte_perm(wa, wb, 0x7632);
                }
            }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) mma<Q8>(oacc[nt][mt], a[0], a[1], a[2], a[3], pb0[nt], pb1[nt]);
        }
    }

    // ---- the four warps together ----
    float *mine = merge + (size_t)warp * ROWS * (D + 2);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            float l = l_run[nt][e];
            l += __shfl_xor_sync(0xffffffffu, l, 4);
            l += __shfl_xor_sync(0xffffffffu, l, 8);
            l += __shfl_xor_sync(0xffffffffu, l, 16);
            float *row = mine + (size_t)(nt * 8 + 2 * c + e) * (D + 2);
#pragma unroll
            for (int mt = 0; mt < KS; ++mt) {
                const int d = C::value_entry(mt, g);
                *reinterpret_cast<float2 *>(row + d) = make_float2(oacc[nt][mt][e], oacc[nt][mt][2 + e]);
            }
            if (g == 0) *reinterpret_cast<float2 *>(row + D) = make_float2(m_run[nt][e], l);
        }
    __syncthreads();
    for (int i = tid; i < ROWS * (D / 2); i += THREADS) {
        const int row = i / (D / 2), d = 2 * (i - row * (D / 2)), r = r0 + row;
        if (r >= n_rows) break;
        float M = -INFINITY, l = 0.f;
        float2 o = make_float2(0.f, 0.f);
#pragma unroll
        for (int w = 0; w < WARPS; ++w) M = fmaxf(M, merge[((size_t)w * ROWS + row) * (D + 2) + D]);
#pragma unroll
        for (int w = 0; w < WARPS; ++w) {
            const float *p = merge + ((size_t)w * ROWS + row) * (D + 2);
            const float f = p[D] == -INFINITY ? (M == -INFINITY ? 1.f : 0.f) : exp2f(p[D] - M);         // (nothing seen: 0, or NaN, which stays one)
            l += p[D + 1] * f;
            o.x += p[d] * f, o.y += p[d + 1] * f;
        }
        const size_t tok = row0 + r / group, head = kvh * group + r % group;
        if (n_splits == 1) {
            const float inv = l == 0.f ? 0.f : 1.f / l;
            *reinterpret_cast<__nv_bfloat162 *>(out + tok * ldo + head * D + d) =
                l == 0.f ? __floats2bfloat162_rn(0.f, 0.f) : __floats2bfloat162_rn(o.x * inv, o.y * inv);
        } else {
            const size_t at = (tok * H + head) * n_splits + split;
            *reinterpret_cast<float2 *>(part_o + at * D + d) = o;
            if (d == 0) part_ml[at] = make_float2(M, l);
        }
    }
}

// The ranges of one (token, head) in their order: a warp each.
constexpr int JOIN_WARPS = 4;
__global__ void __launch_bounds__(JOIN_WARPS * 32) tree_join_kernel(const float *__restrict__ part_o, const float2 *__restrict__ part_ml,
                                                                    const int *__restrict__ seq_start, int limit, int n_tokens, __nv_bfloat16 *__restrict__ out,
                                                                    int ldo, int n_splits, int H, int D) {
    pdl_trigger();
    pdl_wait();
    const int s = blockIdx.x / limit, j = blockIdx.x - s * limit, lane = threadIdx.x & 31;
    const int head = blockIdx.y * JOIN_WARPS + (threadIdx.x >> 5);
    const int row0 = act_load(seq_start + s), n = act_load(seq_start + s + 1) - row0;
    if (j >= n || n > limit || head >= H || row0 < 0 || row0 + n > n_tokens) return;
    const size_t at = ((size_t)(row0 + j) * H + head) * n_splits;
    float M = -INFINITY;
    for (int i = lane; i < n_splits; i += 32) M = fmaxf(M, act_load(part_ml + at + i).x);
    M = warp_max(M);
    float l = 0.f;
    float2 o[4] = {};
    for (int i = 0; i < n_splits; ++i) {
        const float2 ml = act_load(part_ml + at + i);
        const float f = ml.x == -INFINITY ? (M == -INFINITY ? 1.f : 0.f) : exp2f(ml.x - M);
        l += ml.y * f;
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int d = 2 * (lane + 32 * u);
            if (d < D) {
                const float2 v = act_load(reinterpret_cast<const float2 *>(part_o + (at + i) * D + d));
                o[u].x += v.x * f, o[u].y += v.y * f;
            }
        }
    }
    const float inv = 1.f / l;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
        const int d = 2 * (lane + 32 * u);
        if (d < D)
            *reinterpret_cast<__nv_bfloat162 *>(out + (size_t)(row0 + j) * ldo + (size_t)head * D + d) =
                l == 0.f ? __floats2bfloat162_rn(0.f, 0.f) : __floats2bfloat162_rn(o[u].x * inv, o[u].y * inv);
    }
}

template <int KS, int NT, bool Q8, typename... Args>
int launch_one(dim3 grid, cudaStream_t stream, Args... args) {
    const size_t smem = sizeof(float) * WARPS * 8 * NT * (KS * 16 + 2);
    if (smem > 48 * 1024) {
        cudaError_t e = cudaFuncSetAttribute(tree_attention_kernel<KS, NT, Q8>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        if (e != cudaSuccess) LGML_FAIL("tree_attention: cannot have %zu bytes of shared memory: %s", smem, cudaGetErrorString(e));
    }
    lgml_launch(tree_attention_kernel<KS, NT, Q8>, grid, THREADS, smem, stream, args...);
    return lgml_launch_status("tree_attention");
}
template <int KS, bool Q8, typename... Args>
int launch_rows(int nt, Args... args) {
    return nt == 1 ? launch_one<KS, 1, Q8>(args...) : launch_one<KS, 4, Q8>(args...);
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

LGML_API long long lgml_tree_attention_scratch_floats(int n_tokens, int H, int D, int n_splits) {
    return n_splits <= 1 ? 0 : (long long)n_tokens * H * n_splits * (D + 2);
}

// limit: requests that bring more tokens than this are left alone (their rows of out too).  k_exps null: pages in bfloat16.
LGML_API int lgml_tree_attention(const void *q, int ldq, const int *positions, const int *seq_start, const int *seq_pos0, const long long *visible,
                                 const int *block_table, int n_seqs, int max_blocks, const void *k_pages, const void *v_pages, const void *k_exps,
                                 const void *v_exps, int n_pages, int page_size, void *out, int ldo, float *scratch, int n_splits, int n_tokens, int limit, int H,
                                 int Hkv, int D, float scale, int window, int *status, cudaStream_t stream) {
    LGML_REQUIRE(n_tokens >= 0 && n_seqs >= 0 && H > 0 && Hkv > 0 && max_blocks > 0 && n_pages >= 0, "tree_attention: bad sizes");
    LGML_REQUIRE(page_size == PAGE, "tree_attention: pages of %d tokens, this kernel takes %d", page_size, PAGE);
    LGML_REQUIRE(H % Hkv == 0, "tree_attention: %d heads are no multiple of %d KV heads", H, Hkv);
    LGML_REQUIRE(D >= 16 && D <= 128 && D % 16 == 0, "tree_attention: head_dim %d must be a multiple of 16 up to 128", D);
    LGML_REQUIRE(limit >= 1 && limit <= MAX_NEW, "tree_attention: %d new tokens a request (1 to %d)", limit, MAX_NEW);
    LGML_REQUIRE(n_splits >= 1 && n_splits <= MAX_SPLITS, "tree_attention: %d key ranges (1 to %d)", n_splits, MAX_SPLITS);
    LGML_REQUIRE(n_splits == 1 || (scratch != nullptr && ((uintptr_t)scratch & 7) == 0), "tree_attention: several ranges need scratch memory");
    LGML_REQUIRE((k_exps == nullptr) == (v_exps == nullptr), "tree_attention: exponents for keys and values, or for neither");
    LGML_REQUIRE((((uintptr_t)k_pages | (uintptr_t)v_pages) & 15) == 0, "tree_attention: the cache must be 16-byte aligned");
    LGML_REQUIRE(ldq % 2 == 0 && ((uintptr_t)q & 3) == 0 && ldo % 2 == 0 && ((uintptr_t)out & 3) == 0,
                 "tree_attention: q and out must be 4-byte aligned with even row strides");
    LGML_REQUIRE((long long)n_seqs * limit <= 0x7fffffffLL, "tree_attention: too many requests");
    if (n_tokens == 0 || n_seqs == 0) return 0;
    const int rows = limit * (H / Hkv);
    const int nt = rows <= 8 ? 1 : 4;
    const int n_chunks = (rows + 8 * nt - 1) / (8 * nt);
    LGML_REQUIRE((long long)Hkv * n_chunks <= 65535, "tree_attention: too many heads");
    dim3 grid(n_seqs, Hkv * n_chunks, n_splits);
    float *part_o = scratch;
    float2 *part_ml = reinterpret_cast<float2 *>(scratch + (size_t)n_tokens * H * n_splits * D);
#define LGML_ARGS D / 16, nt, grid, stream, (const __nv_bfloat16 *)q, ldq, positions, seq_start, seq_pos0, visible, block_table, max_blocks,            \
                  (const uint8_t *)k_pages, (const uint8_t *)v_pages, (const uint8_t *)k_exps, (const uint8_t *)v_exps, n_pages, (__nv_bfloat16 *)out, ldo, \
                  part_o, part_ml, n_splits, n_tokens, H, Hkv, n_chunks, limit, scale, window, status
    int rc = k_exps ? launch_dim<true>(LGML_ARGS) : launch_dim<false>(LGML_ARGS);
#undef LGML_ARGS
    if (rc || n_splits == 1) return rc;
    lgml_launch(tree_join_kernel, dim3(n_seqs * limit, (H + JOIN_WARPS - 1) / JOIN_WARPS), JOIN_WARPS * 32, 0, stream, part_o, part_ml, seq_start, limit,
                n_tokens, (__nv_bfloat16 *)out, ldo, n_splits, H, D);
    return lgml_launch_status("tree_attention_join");
}
