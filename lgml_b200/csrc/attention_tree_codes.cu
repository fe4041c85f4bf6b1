// Attention of new tokens over pages of e4m3 (attention_tree.cu has the definition) where a KV head has up to 8 rows, tokens x heads: decoding above all.
// The codes go into the tensor cores as they are (mma.sync m16n8k32 of e4m3), so nothing of the cache is converted: what bounds a step here is how many
// instructions a cell costs, and converting every code to 16 bits was half of them.
//
// The keys are the M side, the rows the N side:
//     S^T[16 keys, 8] = K[16, D] . Q^T          O^T[D, 8] += V^T[D, 32 keys] . P^T
// Queries and probabilities are two codes each, a number's nearest code and what that leaves, times 2^4 (queries) and 2^5 (probabilities), as columns of their
// own: up to four rows in the first and the last four columns of one tile (PACK), up to eight in two tiles.  A bfloat16 query has eight significant
// bits and two codes hold four each: with the row scaled by a power of two so that its largest entry is in (224, 448], entries down to 2^-15 of that
// are exact, smaller ones off by 2^-24 of it at most.  A probability (its row's largest so far is 1) is taken 256 times: off by 2^-8 of itself, or by 2^-23 where
// it is under 2^-14.  The sum takes the probability itself.  Keys' powers of two multiply the scores, values' join the probabilities' exponents, as there.
//
// Each of a block's four warps is a pipeline of its own: of every other page it takes half, 32 cells, through two stages in shared memory that 16-byte
// asynchronous copies fill (rows 16 bytes apart from a multiple of 128).  The order of the D entries inside a product, of the D rows of O^T and of the 32 cells is
// free: a thread reads neighbours, and the values' bytes are transposed four cells by four entries in registers.
#include "tree_common.cuh"

LGML_DEFINE_LAST_ERROR(lgml_attention_tree_codes)

namespace {
constexpr int WARPS = 4;
constexpr int THREADS = WARPS * 32;
constexpr int CELLS = 32;                // of a warp's turn
constexpr int STAGES = 2;
constexpr float P_SCALE = 256.f, P_LOW = 32.f, Q_LOW = 16.f;

__device__ __forceinline__ void mma_codes(float (&c)[4], unsigned a0, unsigned a1, unsigned a2, unsigned a3, unsigned b0, unsigned b1) {
    asm volatile("mma.sync.aligned.m16n8k32.row.col.f32.e4m3.e4m3.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ unsigned transpose8(unsigned a) {
    unsigned r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(a));
    return r;
}
// Two codes, the first in the low byte (numbers up to 448; NaN stays NaN).
__device__ __forceinline__ unsigned short codes_of(float a, float b) {
    unsigned short r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(b), "f"(a));
    return r;
}
__device__ __forceinline__ float2 numbers_of(unsigned short two) {
    const unsigned h = half2_of_codes(two);
    return __half22float2(*reinterpret_cast<const __half2 *>(&h));
}
__device__ __forceinline__ float finite_or_nan(float x) { return fabsf(x) <= 3.402823466e38f ? x : __int_as_float(0x7fffffff); }

// Which entries of a row of 32 KS codes a thread has.
//   keys: thread c = lane % 4 has, of every 4 E neighbouring entries, E, four to a register
//   values: thread g = lane / 4 has, of every 8 E neighbouring entries, E: as rows g and g + 8 of E / 2 products
template <int KS> struct Cut {
    static constexpr int D = 32 * KS;
    static constexpr int KE = KS % 4 == 0 ? 32 : KS % 2 == 0 ? 16 : 8, VE = KS % 4 == 0 ? 16 : KS % 2 == 0 ? 8 : 4;
    static constexpr int PITCH = D + 16, STAGE = 2 * CELLS * PITCH + 2 * CELLS;       // keys, values, their exponents
    static __device__ __forceinline__ int key_entry(int word, int c) { return (word / (KE / 4)) * 4 * KE + c * KE + (word % (KE / 4)) * 4; }
    static __device__ __forceinline__ int value_entry(int mt, int g) { return (mt / (VE / 2)) * 8 * VE + g * VE + (mt % (VE / 2)) * 2; }
};
template <int N> __device__ __forceinline__ void read_words(unsigned (&r)[N], const uint8_t *p) {
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

template <int KS, bool PACK>
__global__ void __launch_bounds__(THREADS) tree_attention_codes_kernel(
    const __nv_bfloat16 *__restrict__ q, int ldq, const int *__restrict__ positions, const int *__restrict__ seq_start, const int *__restrict__ seq_pos0,
    const long long *__restrict__ visible, const int *__restrict__ block_table, int max_blocks, const uint8_t *__restrict__ k_pages,
    const uint8_t *__restrict__ v_pages, const uint8_t *__restrict__ k_exps, const uint8_t *__restrict__ v_exps, int n_pages, __nv_bfloat16 *__restrict__ out,
    int ldo, float *__restrict__ part_o, float2 *__restrict__ part_ml, int n_splits, int clustered, int n_tokens, int H, int Hkv, int limit, float scale,
    int window, int *__restrict__ status) {
    pdl_trigger();
    using C = Cut<KS>;
    constexpr int D = C::D, ROWS = PACK ? 4 : 8, NQ = PACK ? 1 : 2, MT = D / 16;
    extern __shared__ __align__(16) uint8_t smem[];                // the warps' stages; at the end [WARPS][ROWS][D + 2] floats
    __shared__ int row_pos[8];
    __shared__ long long row_mask[8];
    __shared__ __align__(8) float fin[ROWS][2];
    __shared__ int stage_page[WARPS][STAGES];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, c = lane & 3;
    const int s = blockIdx.x / n_splits, split = blockIdx.x - s * n_splits, kvh = blockIdx.y;
    // (the step's description, down to the first pages' numbers, is read while the kernels ahead may still run)
    const int row0 = early_int(seq_start + s), n = early_int(seq_start + s + 1) - row0, pos0 = early_int(seq_pos0 + s);
    const int group = H / Hkv, n_rows = n * group;
    if (n <= 0 || n > limit) return;
    if (row0 < 0 || row0 + n > n_tokens || pos0 < 0) {
        if (tid == 0) atomicExch(status, 3);
        return;
    }
    if (tid < 8) {
        const int tok = min(tid, n_rows - 1) / group;
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
    const int pb = first_page + split * pps, n_pg = max(min(pps, end_page - pb), 0), n_it = (n_pg + 1) / 2;

    // ---- the copies: half (warp % 2) of page pb + 2 it + warp / 2 into stage it % STAGES ----
    uint8_t *ring = smem + (size_t)warp * STAGES * C::STAGE;
    const int half = (warp & 1) * CELLS, first_pg = warp >> 1;
    auto table_from = [&](int it) {
        const int p = 2 * (it + lane) + first_pg;
        return p < n_pg && pb + p < max_blocks ? early_int(block_table + (size_t)s * max_blocks + pb + p) : -1;
    };
    int pages_ahead = table_from(0);        // the table's entry for turn (it / 32) * 32 + lane
    auto fetch = [&](int it) {
        if ((it & 31) == 0 && it > 0) pages_ahead = table_from(it);
        int page = __shfl_sync(0xffffffffu, pages_ahead, it & 31);
        const int p = 2 * it + first_pg, cell0 = (pb + p) * PAGE + half, left = n_cells - cell0;
        if (p >= n_pg || left <= 0 || cell0 + CELLS <= low) {
            page = -1;                      // nothing there that a row could see
        } else if (page < 0 || page >= n_pages) {
            if (lane == 0) atomicExch(status, 3);
            page = -1;
        }
        uint8_t *stage = ring + (it % STAGES) * C::STAGE;
        if (lane == 0) stage_page[warp][it % STAGES] = page;
        if (page < 0) return;
        const size_t vec0 = ((size_t)page * Hkv + kvh) * PAGE + half;
        constexpr int PER_ROW = D / 16, ROWS_A_TURN = 32 / PER_ROW > 0 ? 32 / PER_ROW : 1;
        if (32 % PER_ROW == 0) {
            // a lane keeps its 16 bytes of the row and goes down ROWS_A_TURN rows a copy
            const int row = lane / PER_ROW, col = (lane % PER_ROW) * 16;
            const uint8_t *kt = k_pages + vec0 * D + row * D + col, *vt = v_pages + vec0 * D + row * D + col;
            const uint32_t to = smem_u32(stage + row * C::PITCH + col);
#pragma unroll
            for (int u = 0; u < CELLS / ROWS_A_TURN; ++u) {
                const bool there = row + u * ROWS_A_TURN < left;
                copy_16(to + u * ROWS_A_TURN * C::PITCH, kt + u * ROWS_A_TURN * D, there);
                copy_16(to + (CELLS + u * ROWS_A_TURN) * C::PITCH, vt + u * ROWS_A_TURN * D, there);
            }
        } else {
            for (int u = lane; u < CELLS * PER_ROW; u += 32) {
                const int row = u / PER_ROW, col = (u - row * PER_ROW) * 16;
                const uint32_t to = smem_u32(stage + row * C::PITCH + col);
                copy_16(to, k_pages + (vec0 + row) * D + col, row < left);
                copy_16(to + CELLS * C::PITCH, v_pages + (vec0 + row) * D + col, row < left);
            }
        }
        if (lane < 4) copy_16(smem_u32(stage + 2 * CELLS * C::PITCH + 16 * lane), (lane & 2 ? v_exps : k_exps) + vec0 + 16 * (lane & 1), true);
    };

    // Q^T as B fragments: column g, the entries that the keys' registers have in this thread
    pdl_wait();
    const int q_row = PACK ? g & 3 : g;                  // (PACK: columns 4 to 7 are the first four's second codes)
    unsigned qb[NQ][KS][2];
    float q_up[2];                                       // 2^(row's scaling) of this thread's two rows of S, times the score's factor
    {
        const bool there = q_row < n_rows;
        const __nv_bfloat16 *src = q + (size_t)(row0 + (there ? q_row / group : 0)) * ldq + (size_t)(kvh * group + (there ? q_row % group : 0)) * D;
        uint2 raw[KS][2];
#pragma unroll
        for (int w = 0; w < 2 * KS; ++w) {
            const unsigned *p = reinterpret_cast<const unsigned *>(src + C::key_entry(w, c));
            raw[w / 2][w & 1] = there ? make_uint2(act_load(p), act_load(p + 1)) : make_uint2(0, 0);
        }
#pragma unroll
        for (int it = 0; it < STAGES - 1; ++it) {
            if (it < n_it) fetch(it);
            copies_commit();
        }
        float amax = 0.f;
        float2 x[2 * KS][2];
#pragma unroll
        for (int w = 0; w < 2 * KS; ++w) {
            x[w][0] = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162 *>(&raw[w / 2][w & 1].x));
            x[w][1] = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162 *>(&raw[w / 2][w & 1].y));
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const float a = fabsf(x[w][e].x), b = fabsf(x[w][e].y);
                amax = fmaxf(amax, fmaxf(a <= 3.402823466e38f ? a : 0.f, b <= 3.402823466e38f ? b : 0.f));
            }
        }
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
        // 2^-e puts the largest entry into (224, 448]: 448 = 1.75 x 2^8
        const unsigned bits = __float_as_uint(amax);
        const int e = min(max((int)(bits >> 23) - 127 - ((bits & 0x7fffffu) <= 0x600000u ? 8 : 7), -100), 120);
        const float inv = power_of_two(-e), up = power_of_two(e);
#pragma unroll
        for (int w = 0; w < 2 * KS; ++w) {
            unsigned short hi[2], lo[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const float a = finite_or_nan(x[w][h].x) * inv, b = finite_or_nan(x[w][h].y) * inv;
                hi[h] = codes_of(a, b);
                const float2 n = numbers_of(hi[h]);
                lo[h] = codes_of((a - n.x) * Q_LOW, (b - n.y) * Q_LOW);
            }
            const unsigned first = hi[0] | (unsigned)hi[1] << 16, second = lo[0] | (unsigned)lo[1] << 16;
            if (PACK) qb[0][w / 2][w & 1] = g < 4 ? first : second;
            else qb[0][w / 2][w & 1] = first, qb[NQ - 1][w / 2][w & 1] = second;
        }
        const float scale_log2 = scale * 1.4426950408889634f;
        const int r = PACK ? 2 * (c & 1) : 2 * c;           // this thread's rows of S are r and r + 1
        q_up[0] = __shfl_sync(0xffffffffu, up, 4 * r) * scale_log2;
        q_up[1] = __shfl_sync(0xffffffffu, up, 4 * r + 4) * scale_log2;
    }
    const int my_row = PACK ? 2 * (c & 1) : 2 * c;
    const float first_codes = !PACK || c < 2 ? 1.f : 0.f, own = PACK && c >= 2 ? 1.f / Q_LOW : 1.f;

    float m_run[2] = {-INFINITY, -INFINITY}, l_run[2] = {0.f, 0.f}, oacc[NQ][MT][4];
#pragma unroll
    for (int i = 0; i < NQ; ++i)
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) oacc[i][mt][0] = oacc[i][mt][1] = oacc[i][mt][2] = oacc[i][mt][3] = 0.f;

    for (int it = 0; it < n_it; ++it) {
        if (it + STAGES - 1 < n_it) fetch(it + STAGES - 1);
        copies_commit();
        copies_wait<STAGES - 1>();
        __syncwarp();
        if (stage_page[warp][it % STAGES] < 0) {
            __syncwarp();
            continue;
        }
        const uint8_t *ks = ring + (it % STAGES) * C::STAGE, *vs = ks + CELLS * C::PITCH, *es = ks + 2 * CELLS * C::PITCH;
        const int cell0 = (pb + 2 * it + first_pg) * PAGE + half;

        // ---- S^T: cells 16 t + g and 16 t + g + 8, rows my_row and my_row + 1 ----
        float sc[2][4];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            float sum[NQ][4] = {};
#pragma unroll
            for (int i = 0; i < D / (4 * C::KE); ++i) {
                unsigned kw[2][C::KE / 4];
#pragma unroll
                for (int h = 0; h < 2; ++h) read_words(kw[h], ks + (16 * t + g + 8 * h) * C::PITCH + i * 4 * C::KE + c * C::KE);
#pragma unroll
                for (int u = 0; u < C::KE / 8; ++u)
#pragma unroll
                    for (int j = 0; j < NQ; ++j)
                        mma_codes(sum[j], kw[0][2 * u], kw[1][2 * u], kw[0][2 * u + 1], kw[1][2 * u + 1], qb[j][i * (C::KE / 8) + u][0], qb[j][i * (C::KE / 8) + u][1]);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (PACK) {
                    const float x = sum[0][i] * own;
                    sc[t][i] = x + __shfl_xor_sync(0xffffffffu, x, 2);
                } else {
                    sc[t][i] = sum[0][i] + sum[NQ - 1][i] * (1.f / Q_LOW);
                }
            }
        }
        // ---- scores, and which of them are seen: bit 4 t + i for sc[t][i] ----
        const bool whole = cell0 + CELLS <= pos0 && cell0 >= all_from;
        unsigned seen = 0xffu;
        if (!whole) {
            seen = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int cell = cell0 + 16 * (i >> 2) + g + 8 * ((i >> 1) & 1), row = my_row + (i & 1), j = cell - pos0;
                if (cell >= n_cells) continue;
                const int at = j < 0 ? cell : window > 0 ? act_load(positions + row0 + j) : 0;
                if ((j < 0 || ((row_mask[row] >> j) & 1)) && (window <= 0 || at > row_pos[row] - window)) seen |= 1u << i;
            }
        }
        float vf[2][2];
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int ke = min((int)es[16 * t + g + 8 * h], 246) - 127, ve = min((int)es[CELLS + 16 * t + g + 8 * h], 246) - 127;      // (246: the largest that is written)
                const float kf = power_of_two(ke), add = (float)ve;
                vf[t][h] = power_of_two(-ve);
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const float x = fmaf(sc[t][2 * h + e] * q_up[e], kf, add);
                    sc[t][2 * h + e] = (seen >> (4 * t + 2 * h + e)) & 1 ? x : -INFINITY;
                }
            }
        // ---- probabilities ----
        float corr[2];
        bool grown = false;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            float mx = fmaxf(fmaxf(sc[0][e], sc[0][2 + e]), fmaxf(sc[1][e], sc[1][2 + e]));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
            const float m_new = fmaxf(m_run[e], mx);
            corr[e] = m_new == m_run[e] ? 1.f : ex2(m_run[e] - m_new);
            grown |= m_new != m_run[e];
            m_run[e] = m_new;
            l_run[e] *= corr[e];
        }
        if (__any_sync(0xffffffffu, grown)) {
#pragma unroll
            for (int j = 0; j < NQ; ++j)
#pragma unroll
                for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                    for (int i = 0; i < 4; ++i) oacc[j][mt][i] *= corr[i & 1];
        }
        unsigned pb_[NQ][2];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            unsigned short hi[2], lo[2];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const float m = m_run[e] == -INFINITY ? 0.f : m_run[e];
                const float a = ex2(sc[t][e] - m) * P_SCALE, b = ex2(sc[t][2 + e] - m) * P_SCALE;          // (unseen: exp2(-inf) = 0)
                sc[t][e] = a, sc[t][2 + e] = b;             // from here on, probabilities
                l_run[e] = fmaf(a, vf[t][0], fmaf(b, vf[t][1], l_run[e]));
                hi[e] = codes_of(a, b);
                const float2 n = numbers_of(hi[e]);
                lo[e] = codes_of((a - n.x) * P_LOW, (b - n.y) * P_LOW);
            }
            const unsigned first = hi[0] | (unsigned)hi[1] << 16, second = lo[0] | (unsigned)lo[1] << 16;
            // a thread then has, of column g, cells 2 c, 2 c + 8, 2 c + 1 and 2 c + 9 of the tile
            if (PACK) pb_[0][t] = transpose8(c < 2 ? first : second);
            else pb_[0][t] = transpose8(first), pb_[NQ - 1][t] = transpose8(second);
        }
        // ---- values that are not finite, among cells that not every row sees ----
        if (!whole) {
            bool odd = false;
            for (int u = lane; u < CELLS * D / 4; u += 32) {
                const unsigned x = *reinterpret_cast<const unsigned *>(vs + (u / (D / 4)) * C::PITCH + (u % (D / 4)) * 4);
                odd |= (((x & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) != 0;
            }
            if (__any_sync(0xffffffffu, odd)) {
                for (int cell = 0; cell < min(n_cells - cell0, CELLS); ++cell) {
                    const int from = (cell & 7) * 4 + c, which = cell >> 3;        // tile 0 rows g, g + 8, tile 1 rows g, g + 8
                    const float p_a = __shfl_sync(0xffffffffu, which == 0 ? sc[0][0] : which == 1 ? sc[0][2] : which == 2 ? sc[1][0] : sc[1][2], from);
                    const float p_b = __shfl_sync(0xffffffffu, which == 0 ? sc[0][1] : which == 1 ? sc[0][3] : which == 2 ? sc[1][1] : sc[1][3], from);
                    const unsigned bits = __shfl_sync(0xffffffffu, seen, from) >> (2 * which);
                    if (first_codes == 0.f) continue;              // (the second codes' columns take none of it)
#pragma unroll
                    for (int mt = 0; mt < MT; ++mt) {
                        const float2 v = numbers_of(*reinterpret_cast<const unsigned short *>(vs + cell * C::PITCH + C::value_entry(mt, g)));
                        if (bits & 1u) oacc[0][mt][0] += p_a * v.x, oacc[0][mt][2] += p_a * v.y;
                        if (bits & 2u) oacc[0][mt][1] += p_b * v.x, oacc[0][mt][3] += p_b * v.y;
                    }
                }
                __syncwarp();
                continue;
            }
        }
        // ---- O^T += V^T P^T ----
#pragma unroll
        for (int i = 0; i < D / (8 * C::VE); ++i) {
            unsigned vw[2][4][C::VE / 4];             // of cells 2 c, 2 c + 8, 2 c + 1, 2 c + 9 of both tiles
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int h = 0; h < 4; ++h) read_words(vw[t][h], vs + (16 * t + 2 * c + (h >> 1) + 8 * (h & 1)) * C::PITCH + i * 8 * C::VE + g * C::VE);
#pragma unroll
            for (int w = 0; w < C::VE / 4; ++w) {
                unsigned o[2][4];                     // four entries, each of the tile's four cells
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    const unsigned a = __byte_perm(vw[t][0][w], vw[t][1][w], 0x5140), b = __byte_perm(vw[t][2][w], vw[t][3][w], 0x5140);
                    const unsigned d = __byte_perm(vw[t][0][w], vw[t][1][w], 0x7362), e = __byte_perm(vw[t][2][w], vw[t][3][w], 0x7362);
                    o[t][0] = __byte_perm(a, b, 0x5410), o[t][1] = __byte_perm(a, b, 0x7632), o[t][2] = __byte_perm(d, e, 0x5410), o[t][3] = __byte_perm(d, e, 0x7632);
                }
                const int mt = i * (C::VE / 2) + 2 * w;
#pragma unroll
                for (int j = 0; j < NQ; ++j) {
                    mma_codes(oacc[j][mt], o[0][0], o[0][1], o[1][0], o[1][1], pb_[j][0], pb_[j][1]);
                    mma_codes(oacc[j][mt + 1], o[0][2], o[0][3], o[1][2], o[1][3], pb_[j][0], pb_[j][1]);
                }
            }
        }
        __syncwarp();
    }
    copies_wait<0>();
    __syncthreads();                        // every warp is done with its stages

    // ---- the four warps together ----
    float *merge = reinterpret_cast<float *>(smem), *mine = merge + (size_t)warp * ROWS * (D + 2);
#pragma unroll
    for (int e = 0; e < 2; ++e) {
        float l = l_run[e];
        l += __shfl_xor_sync(0xffffffffu, l, 4);
        l += __shfl_xor_sync(0xffffffffu, l, 8);
        l += __shfl_xor_sync(0xffffffffu, l, 16);
        float *row = mine + (size_t)(my_row + e) * (D + 2);
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
            float2 o = make_float2(oacc[0][mt][e], oacc[0][mt][2 + e]);
            if (PACK) {
                o.x *= c < 2 ? 1.f : 1.f / P_LOW, o.y *= c < 2 ? 1.f : 1.f / P_LOW;
                o.x += __shfl_xor_sync(0xffffffffu, o.x, 2), o.y += __shfl_xor_sync(0xffffffffu, o.y, 2);
            } else {
                o.x += oacc[NQ - 1][mt][e] * (1.f / P_LOW), o.y += oacc[NQ - 1][mt][2 + e] * (1.f / P_LOW);
            }
            if (!PACK || c < 2) *reinterpret_cast<float2 *>(row + C::value_entry(mt, g)) = o;
        }
        if (g == 0 && (!PACK || c < 2)) *reinterpret_cast<float2 *>(row + D) = make_float2(m_run[e], l);
    }
    __syncthreads();
    for (int i = tid; i < ROWS * (D / 2); i += THREADS) {
        const int row = i / (D / 2), d = 2 * (i - row * (D / 2));
        if (row >= n_rows) break;
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
            store_row(row_at(out, ldo, row0, row, group, kvh, D, d), o, l);
        } else if (clustered) {
            *reinterpret_cast<float2 *>(merge + (size_t)row * (D + 2) + d) = o;         // (no other thread reads it here)
            if (d == 0) fin[row][0] = M, fin[row][1] = l;
        } else {
            const size_t at = ((size_t)(row0 + row / group) * H + kvh * group + row % group) * n_splits + split;
            *reinterpret_cast<float2 *>(part_o + at * D + d) = o;
            if (d == 0) part_ml[at] = make_float2(M, l);
        }
    }
    if (!clustered) return;
    // ---- the cluster's ranges together: each block joins a share of the results ----
    __syncwarp();
    cluster_sync();
    join_cluster<ROWS, D, THREADS>(merge, fin, n_splits, n_rows, [&](int row, int d) { return row_at(out, ldo, row0, row, group, kvh, D, d); });
    __syncwarp();
    cluster_sync();                         // (the others' shared memory is read until here)
}

template <int KS, bool PACK, typename... Args>
int launch_one(dim3 grid, int cluster, cudaStream_t stream, Args... args) {
    const size_t stages = (size_t)WARPS * STAGES * Cut<KS>::STAGE, merge = sizeof(float) * WARPS * (PACK ? 4 : 8) * (KS * 32 + 2);
    const size_t smem = stages > merge ? stages : merge;
    cudaError_t e = cudaFuncSetAttribute(tree_attention_codes_kernel<KS, PACK>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) LGML_FAIL("tree_attention: cannot have %zu bytes of shared memory: %s", smem, cudaGetErrorString(e));
    lgml_launch_cluster(tree_attention_codes_kernel<KS, PACK>, grid, THREADS, smem, stream, cluster, args...);
    return lgml_launch_status("tree_attention");
}
template <bool PACK, typename... Args>
int launch_dim(int D, Args... args) {
    switch (D) {
        case 32: return launch_one<1, PACK>(args...);
        case 64: return launch_one<2, PACK>(args...);
        case 96: return launch_one<3, PACK>(args...);
        case 128: return launch_one<4, PACK>(args...);
    }
    LGML_FAIL("tree_attention: head_dim %d not handled", D);
}
}  // namespace

// As lgml_tree_attention, for pages of e4m3, head sizes in steps of 32 up to 128 and up to 8 rows (tokens x heads of a KV head) a request.
LGML_API int lgml_tree_attention_codes(const void *q, int ldq, const int *positions, const int *seq_start, const int *seq_pos0, const long long *visible,
                                       const int *block_table, int n_seqs, int max_blocks, const void *k_pages, const void *v_pages, const void *k_exps,
                                       const void *v_exps, int n_pages, int page_size, void *out, int ldo, float *scratch, int n_splits, int n_tokens, int limit,
                                       int H, int Hkv, int D, float scale, int window, int *status, cudaStream_t stream) {
    LGML_REQUIRE(n_tokens >= 0 && n_seqs >= 0 && H > 0 && Hkv > 0 && max_blocks > 0 && n_pages >= 0, "tree_attention: bad sizes");
    LGML_REQUIRE(page_size == PAGE, "tree_attention: pages of %d tokens, this kernel takes %d", page_size, PAGE);
    LGML_REQUIRE(H % Hkv == 0, "tree_attention: %d heads are no multiple of %d KV heads", H, Hkv);
    LGML_REQUIRE(D >= 32 && D <= 128 && D % 32 == 0, "tree_attention: head_dim %d must be a multiple of 32 up to 128 here", D);
    LGML_REQUIRE(limit >= 1 && (long long)limit * (H / Hkv) <= 8, "tree_attention: %d tokens of %d heads a KV head are over 8 rows", limit, H / Hkv);
    LGML_REQUIRE(n_splits >= 1 && n_splits <= MAX_SPLITS, "tree_attention: %d key ranges (1 to %d)", n_splits, MAX_SPLITS);
    LGML_REQUIRE(n_splits <= MAX_CLUSTER || (scratch != nullptr && ((uintptr_t)scratch & 7) == 0), "tree_attention: several ranges need scratch memory");
    LGML_REQUIRE(k_exps != nullptr && v_exps != nullptr, "tree_attention: pages of e4m3 come with their exponents");
    LGML_REQUIRE((((uintptr_t)k_pages | (uintptr_t)v_pages | (uintptr_t)k_exps | (uintptr_t)v_exps) & 15) == 0, "tree_attention: the cache must be 16-byte aligned");
    LGML_REQUIRE(ldq % 2 == 0 && ((uintptr_t)q & 3) == 0 && ldo % 2 == 0 && ((uintptr_t)out & 3) == 0,
                 "tree_attention: q and out must be 4-byte aligned with even row strides");
    LGML_REQUIRE((long long)n_seqs * (limit > n_splits ? limit : n_splits) <= 0x7fffffffLL && Hkv <= 65535, "tree_attention: too many requests or heads");
    if (n_tokens == 0 || n_seqs == 0) return 0;
    const int clustered = n_splits > 1 && n_splits <= MAX_CLUSTER;
    dim3 grid(n_seqs * n_splits, Hkv);
    float *part_o = scratch;
    float2 *part_ml = scratch ? reinterpret_cast<float2 *>(scratch + (size_t)n_tokens * H * n_splits * D) : nullptr;
#define LGML_ARGS D, grid, clustered ? n_splits : 1, stream, (const __nv_bfloat16 *)q, ldq, positions, seq_start, seq_pos0, visible, block_table, max_blocks,    \
                  (const uint8_t *)k_pages, (const uint8_t *)v_pages, (const uint8_t *)k_exps, (const uint8_t *)v_exps, n_pages, (__nv_bfloat16 *)out, ldo, part_o, \
                  part_ml, n_splits, clustered, n_tokens, H, Hkv, limit, scale, window, status
    const int rc = limit * (H / Hkv) <= 4 ? launch_dim<true>(LGML_ARGS) : launch_dim<false>(LGML_ARGS);
#undef LGML_ARGS
    if (rc || n_splits <= MAX_CLUSTER) return rc;
    return tree_join(part_o, part_ml, seq_start, n_seqs, limit, n_tokens, out, ldo, n_splits, H, D, stream);
}
