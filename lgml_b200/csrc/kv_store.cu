// Rotary positions and the write of keys and values into cells that are given apart from the positions, and the
// reading back of pages that hold eight bits a value.
//
// A vector (the key or the value of one token and KV head) in e4m3 comes with one power of two:
//     e = clamp(ceil(log2(amax / 448)), -60, 119)     amax over the vector's finite entries; all zero: -60
//     code_i = e4m3(x_i 2^-e), to nearest;  NaN and infinities: NaN
// so the largest entry lands in (224, 448], and x 2^-e and code 2^e are exact in float32 and, the second, in bfloat16: a
// vector is rounded once, when it is written (half a step of four bits, 2^-4 of an entry's size, or 2^-10 2^e for entries under 2^-6 2^e).  A key that is to
// be codes is turned in float64: float32's last bit would put a few of 10^6 entries on the other side of a border between codes.  Reading back rounds nothing, and a vector that is read back and
// written again keeps its codes.  The exponent is kept as a byte, e + 127, in an array of its own: 1 byte on 128.
//
// Cells and positions differ for drafted tokens that stand side by side at one position: the cell is where a token's key
// lies (table[cell / 64], cell % 64), the position what it is turned by.  The cells of a call differ (two tokens in one cell leave either's entries there).
//
// Both directions are memory's: every entry is read and written once.  What they take (32 heads on 8 of 128, launches back to back): one token e4m3 1.5 us,
// 8 tokens 1.6, 2,048 tokens 11.3 (46 MB, 4.1 TB/s; 10.2 with the rotation in float32) in e4m3 and 9.1 (50 MB, 5.5 TB/s) in bfloat16; reading 1,531 pages back
// 98 us (604 MB, 6.2 TB/s, 0.94 of the measured copy rate), 34 pages 5.4.
#include <cuda_fp16.h>
#include <math.h>

#include "common.cuh"

LGML_DEFINE_LAST_ERROR(lgml_kv_store)

namespace {
constexpr int PAGE = 64;
constexpr int WARPS = 8;
constexpr int MAX_D = 256;
constexpr int LOWEST = -60, HIGHEST = 119;

// The exponent of a vector whose largest finite entry is amax: 448 = 1.75 x 2^8.
__device__ __forceinline__ int vector_exponent(float amax) {
    const unsigned u = __float_as_uint(amax);
    const int e = (int)(u >> 23) - 127 - ((u & 0x7fffffu) <= 0x600000u ? 8 : 7);       // (zero and denormal numbers: far below LOWEST)
    return min(max(e, LOWEST), HIGHEST);
}
__device__ __forceinline__ float power_of_two(int e) { return __uint_as_float((unsigned)(e + 127) << 23); }
__device__ __forceinline__ float finite_abs(float x) { return fabsf(x) <= 3.402823466e38f ? fabsf(x) : 0.f; }
// Two codes, the first in the low byte.
__device__ __forceinline__ unsigned short e4m3_pair(float a, float b, float inv) {
    a = fabsf(a) <= 3.402823466e38f ? a * inv : __int_as_float(0x7fffffff);
    b = fabsf(b) <= 3.402823466e38f ? b * inv : __int_as_float(0x7fffffff);
    unsigned short r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(b), "f"(a));
    return r;
}

// The sine and cosine of pos (f + f_lo), in float64.
__device__ __forceinline__ void sincos_64(int pos, float f, float f_lo, double *s, double *c) {
    const double a = (double)pos * ((double)f + (double)f_lo), k = rint(a * 0.15915494309189535);
    sincos(fma(-k, 2.4492935982947064e-16, fma(-k, 6.283185307179586, a)), s, c);            // (2 pi in two parts)
}

// Few tokens, and any head size: a warp a head of a token; a lane holds pairs lane, lane + 32, .. (PAIRS at most) of the head, so the vector's
// largest entry is one warp reduction.  pairing and the treatment of entries past n_rot as in rope_cache.cu.
template <typename TS, bool Q8, int PAIRS>
__global__ void __launch_bounds__(WARPS * 32) kv_store_kernel(
    const TS *__restrict__ src, int lds, int n_parts, long long part_stride, const float *__restrict__ bias, __nv_bfloat16 *__restrict__ q_out, int ldq,
    const int *__restrict__ positions, const int *__restrict__ cells, const int *__restrict__ seq_of_token, const int *__restrict__ block_table,
    int n_seqs, int max_blocks, const float *__restrict__ inv_freq, const float *__restrict__ inv_freq_lo, int n_rot, int pairing, void *__restrict__ k_pages,
    void *__restrict__ v_pages, uint8_t *__restrict__ k_exps, uint8_t *__restrict__ v_exps, int n_pages, int H, int Hkv, int D, int n_heads,
    int *__restrict__ status) {
    pdl_trigger();
    const int t = blockIdx.x, lane = threadIdx.x & 31;
    const int head = blockIdx.y * WARPS + (threadIdx.x >> 5);
    if (head >= n_heads) return;
    const int half_d = D / 2, half_rot = n_rot / 2;
    const int pos = early_int(positions + t);
    int page = -1, cell = 0;
    if (head >= H) {
        cell = cells ? early_int(cells + t) : pos;
        const int seq = early_int(seq_of_token + t);
        const int blk = cell / PAGE;
        if (cell >= 0 && blk < max_blocks && seq >= 0 && seq < n_seqs) page = early_int(block_table + (size_t)seq * max_blocks + blk);
    }
    const size_t col = (size_t)head * D;
    const TS *row = src + (size_t)t * lds + col;
    float a[PAIRS], b[PAIRS];
    int d0[PAIRS], d1[PAIRS];
    float sn[PAIRS], cs[PAIRS];
    double sn64[Q8 ? PAIRS : 1], cs64[Q8 ? PAIRS : 1];
    const bool turns = head < H + Hkv, coded = Q8 && head >= H;
#pragma unroll
    for (int i = 0; i < PAIRS; ++i) {
        const int j = lane + 32 * i;
        if (j >= half_d) continue;
        sn[i] = 0.f, cs[i] = 1.f;
        if (turns && j < half_rot) {
            d0[i] = pairing ? 2 * j : j;
            d1[i] = pairing ? 2 * j + 1 : j + half_rot;
            const float f = early_weight(inv_freq + j), f_lo = inv_freq_lo ? early_weight(inv_freq_lo + j) : 0.f;
            if (coded) sincos_64(pos, f, f_lo, &sn64[Q8 ? i : 0], &cs64[Q8 ? i : 0]);
            else rope_sincos(pos, f, f_lo, &sn[i], &cs[i]);
        } else {
            d0[i] = 2 * j;
            d1[i] = d0[i] + 1;
        }
    }
    pdl_wait();
#pragma unroll
    for (int i = 0; i < PAIRS; ++i) {
        if (lane + 32 * i >= half_d) continue;
        a[i] = to_f32(act_load(row + d0[i]));
        b[i] = to_f32(act_load(row + d1[i]));
    }
    for (int p = 1; p < n_parts; ++p)
#pragma unroll
        for (int i = 0; i < PAIRS; ++i) {
            if (lane + 32 * i >= half_d) continue;
            a[i] += to_f32(act_load(row + (size_t)p * part_stride + d0[i]));
            b[i] += to_f32(act_load(row + (size_t)p * part_stride + d1[i]));
        }
    float amax = 0.f;
#pragma unroll
    for (int i = 0; i < PAIRS; ++i) {
        const int j = lane + 32 * i;
        if (j >= half_d) continue;
        if (bias) a[i] += bias[col + d0[i]], b[i] += bias[col + d1[i]];
        if (turns && j < half_rot) {
            if (coded) {
                const double x = a[i], y = b[i], sn_i = sn64[Q8 ? i : 0], cs_i = cs64[Q8 ? i : 0];
                a[i] = (float)(x * cs_i - y * sn_i), b[i] = (float)(x * sn_i + y * cs_i);
            } else {
                const float x = a[i] * cs[i] - b[i] * sn[i], y = a[i] * sn[i] + b[i] * cs[i];
                a[i] = x, b[i] = y;
            }
        }
        if (Q8) amax = fmaxf(amax, fmaxf(finite_abs(a[i]), finite_abs(b[i])));
    }
    if (head < H) {
        __nv_bfloat16 *dst = q_out + (size_t)t * ldq + col;
#pragma unroll
        for (int i = 0; i < PAIRS; ++i)
            if (lane + 32 * i < half_d) dst[d0[i]] = __float2bfloat16_rn(a[i]), dst[d1[i]] = __float2bfloat16_rn(b[i]);
        return;
    }
    if (page < 0 || page >= n_pages) {      // the host reserves pages first; never write outside the pool
        if (lane == 0) atomicExch(status, 2);
        return;
    }
    const bool is_k = head < H + Hkv;
    const size_t vec = ((size_t)page * Hkv + (is_k ? head - H : head - H - Hkv)) * PAGE + cell % PAGE;
    if (Q8) {
        const int e = vector_exponent(warp_max(amax));
        const float inv = power_of_two(-e);
        uint8_t *dst = reinterpret_cast<uint8_t *>(is_k ? k_pages : v_pages) + vec * D;
#pragma unroll
        for (int i = 0; i < PAIRS; ++i) {
            if (lane + 32 * i >= half_d) continue;
            const unsigned short c = e4m3_pair(a[i], b[i], inv);
            dst[d0[i]] = (uint8_t)(c & 0xff), dst[d1[i]] = (uint8_t)(c >> 8);
        }
        if (lane == 0) (is_k ? k_exps : v_exps)[vec] = (uint8_t)(e + 127);
    } else {
        __nv_bfloat16 *dst = reinterpret_cast<__nv_bfloat16 *>(is_k ? k_pages : v_pages) + vec * D;
#pragma unroll
        for (int i = 0; i < PAIRS; ++i)
            if (lane + 32 * i < half_d) dst[d0[i]] = __float2bfloat16_rn(a[i]), dst[d1[i]] = __float2bfloat16_rn(b[i]);
    }
}

// The same for many tokens, bfloat16 in, heads of 64 or 128 entries that turn whole: a block a token, whose angles are computed once for all its
// heads; sixteen lanes a head, each with P = D / 32 neighbouring entries of the first half of the head and P of the second ("half"), or 2 P
// neighbouring entries ("adjacent"): either way the pairs that turn together are in one thread, and loads and stores are 4 P and 2 P bytes wide.
// A thread's first loads set out ahead of the trip to the block table.  (us this way and by a warp a head, heads of 128: 64 tokens e4m3 2.5 / 2.3, bfloat16
// 1.9 / 2.0; 128 tokens 2.8 / 3.7 and 2.3 / 3.5; 2,048 tokens 11 / 39 and 9 / 37.  Two or four heads on their way instead of three: 2 and 1.5 us more at 2,048.
// Heads of 128 in codes, five blocks an SM instead of the four that the registers would leave: 11.3 for 12.4 at 2,048, 46 for 50 at 8,192, 4.4 for 3.8 at 512;
// six: 12.0, 44, 5.3.)
constexpr int WIDE_THREADS = 256, WIDE_FROM = 65, WIDE_HEADS = 3;      // (heads a thread has on their way)
template <int P> struct Vec;
template <> struct Vec<2> { using type = unsigned; };
template <> struct Vec<4> { using type = uint2; };
template <int P, bool Q8, bool ADJACENT>
__global__ void __launch_bounds__(WIDE_THREADS, Q8 && P == 4 ? 5 : 1) kv_store_wide_kernel(
    const __nv_bfloat16 *__restrict__ src, int lds, __nv_bfloat16 *__restrict__ q_out, int ldq, const int *__restrict__ positions, const int *__restrict__ cells,
    const int *__restrict__ seq_of_token, const int *__restrict__ block_table, int n_seqs, int max_blocks, const float *__restrict__ inv_freq,
    const float *__restrict__ inv_freq_lo, void *__restrict__ k_pages, void *__restrict__ v_pages, uint8_t *__restrict__ k_exps, uint8_t *__restrict__ v_exps,
    int n_pages, int H, int Hkv, int n_heads, int *__restrict__ status) {
    pdl_trigger();
    constexpr int D = 32 * P;
    using Half = typename Vec<P>::type;
    __shared__ float2 turn[D / 2];           // (cos, sin) of pair i
    __shared__ double2 turn64[Q8 ? D / 2 : 1];
    const int t = blockIdx.x, tid = threadIdx.x, l = tid & 15;
    const int pos = early_int(positions + t), cell = cells ? early_int(cells + t) : pos, seq = early_int(seq_of_token + t), blk = cell / PAGE;
    if (tid < D / 2) {
        float sn, cs;
        const float f = early_weight(inv_freq + tid), f_lo = inv_freq_lo ? early_weight(inv_freq_lo + tid) : 0.f;
        if (Q8) {
            double sn64, cs64;
            sincos_64(pos, f, f_lo, &sn64, &cs64);
            turn64[tid] = make_double2(cs64, sn64);
            sn = (float)sn64, cs = (float)cs64;
        } else {
            rope_sincos(pos, f, f_lo, &sn, &cs);
        }
        turn[tid] = make_float2(cs, sn);
    }
    pdl_wait();
    // entries e of the first run and of the second; pair i of the thread is (x[i], x[P + i]) or, adjacent, (x[2 i], x[2 i + 1])
    const int run0 = ADJACENT ? 2 * P * l : P * l, run1 = ADJACENT ? run0 + P : run0 + D / 2;
    constexpr int UNITS = WIDE_THREADS / 16;
    bool there = false;
    int page = -1;
    for (int base = 0; base < n_heads; base += WIDE_HEADS * UNITS) {       // (both heads of a warp go round as often)
        const int head = base + tid / 16;
        Half raw[WIDE_HEADS][2];
#pragma unroll
        for (int k = 0; k < WIDE_HEADS; ++k)
            if (head + k * UNITS < n_heads) {
                const __nv_bfloat16 *p = src + (size_t)t * lds + (size_t)(head + k * UNITS) * D;
                raw[k][0] = __ldcg(reinterpret_cast<const Half *>(p + run0)), raw[k][1] = __ldcg(reinterpret_cast<const Half *>(p + run1));
            }
        if (base == 0) {
            // (behind the first loads: a trip to the table and the other threads' angles)
            page = cell >= 0 && blk < max_blocks && seq >= 0 && seq < n_seqs ? early_int(block_table + (size_t)seq * max_blocks + blk) : -1;
            there = page >= 0 && page < n_pages;
            if (!there && n_heads > H && tid == 0) atomicExch(status, 2);      // the host reserves pages first; never write outside the pool
            __syncthreads();
        }
#pragma unroll
        for (int k = 0; k < WIDE_HEADS; ++k) {
            const int h = head + k * UNITS;
            const bool mine = h < n_heads;              // (the lanes of a head are together in this, and in the reduction below)
            float x[2 * P];
#pragma unroll
            for (int i = 0; i < 2 * P; ++i) x[i] = mine ? __bfloat162float(reinterpret_cast<const __nv_bfloat16 *>(raw[k])[i]) : 0.f;
            if (Q8 && h >= H && h < H + Hkv) {
#pragma unroll
                for (int i = 0; i < P; ++i) {
                    const int a = ADJACENT ? 2 * i : i, b = ADJACENT ? 2 * i + 1 : P + i;
                    const double2 f = turn64[Q8 ? P * l + i : 0];
                    const double u = x[a], v = x[b];
                    x[a] = (float)(u * f.x - v * f.y), x[b] = (float)(u * f.y + v * f.x);
                }
            } else if (h < H + Hkv) {
#pragma unroll
                for (int i = 0; i < P; ++i) {
                    const int a = ADJACENT ? 2 * i : i, b = ADJACENT ? 2 * i + 1 : P + i;
                    const float2 f = turn[P * l + i];
                    const float u = x[a] * f.x - x[b] * f.y, v = x[a] * f.y + x[b] * f.x;
                    x[a] = u, x[b] = v;
                }
            }
            const size_t vec = there ? ((size_t)page * Hkv + (h < H + Hkv ? h - H : h - H - Hkv)) * PAGE + cell % PAGE : 0;
            if (Q8 && (h | 1) >= H) {              // (one of the warp's two heads is a key or a value)
                float amax = 0.f;
#pragma unroll
                for (int i = 0; i < 2 * P; ++i) amax = fmaxf(amax, finite_abs(x[i]));
#pragma unroll
                for (int o = 8; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
                if (mine && h >= H && there) {
                    const int e = vector_exponent(amax);
                    const float inv = power_of_two(-e);
                    unsigned short c[P];
#pragma unroll
                    for (int i = 0; i < P; ++i) c[i] = e4m3_pair(x[2 * i], x[2 * i + 1], inv);
                    uint8_t *dst = reinterpret_cast<uint8_t *>(h < H + Hkv ? k_pages : v_pages) + vec * D;
                    if (ADJACENT) {
                        if (P == 4) *reinterpret_cast<uint2 *>(dst + run0) = make_uint2(c[0] | (unsigned)c[1 % P] << 16, c[2 % P] | (unsigned)c[3 % P] << 16);
                        else *reinterpret_cast<unsigned *>(dst + run0) = c[0] | (unsigned)c[1] << 16;
                    } else if (P == 4) {
                        *reinterpret_cast<unsigned *>(dst + run0) = c[0] | (unsigned)c[1 % P] << 16;
                        *reinterpret_cast<unsigned *>(dst + run1) = c[2 % P] | (unsigned)c[3 % P] << 16;
                    } else {
                        *reinterpret_cast<unsigned short *>(dst + run0) = c[0];
                        *reinterpret_cast<unsigned short *>(dst + run1) = c[1];
                    }
                    if (l == 0) (h < H + Hkv ? k_exps : v_exps)[vec] = (uint8_t)(e + 127);
                }
            }
            if (!mine || (h >= H && (Q8 || !there))) continue;
            __nv_bfloat16 *dst = h < H ? q_out + (size_t)t * ldq + (size_t)h * D : reinterpret_cast<__nv_bfloat16 *>(h < H + Hkv ? k_pages : v_pages) + vec * D;
            Half y[2];
#pragma unroll
            for (int i = 0; i < P; ++i) reinterpret_cast<__nv_bfloat162 *>(y)[i] = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
            *reinterpret_cast<Half *>(dst + run0) = y[0];
            *reinterpret_cast<Half *>(dst + run1) = y[1];
        }
    }
}

// Page list[i] of the pool as bfloat16 page i of the output: a block per (page, KV head, keys or values), 16 codes a thread and turn.
// An entry below zero leaves its page of the output as it is; one past the pool does too, and sets the status.  (Nothing is used twice: what counts is that
// every thread's four or eight loads are 16 bytes wide and on their way together.)
constexpr int READ_THREADS = 128;
__global__ void __launch_bounds__(READ_THREADS) kv_read_kernel(const uint8_t *__restrict__ k_pages, const uint8_t *__restrict__ v_pages,
                                                               const uint8_t *__restrict__ k_exps, const uint8_t *__restrict__ v_exps, int n_pages,
                                                               const int *__restrict__ list, __nv_bfloat16 *__restrict__ k_out,
                                                               __nv_bfloat16 *__restrict__ v_out, int Hkv, int D, int *__restrict__ status) {
    pdl_trigger();
    pdl_wait();
    const int i = blockIdx.x / Hkv, h = blockIdx.x - i * Hkv;
    const bool is_k = blockIdx.y == 0;
    const int page = act_load(list + i);
    if (page < 0 || page >= n_pages) {
        if (page >= n_pages && threadIdx.x == 0) atomicExch(status, 3);
        return;
    }
    const size_t from = ((size_t)page * Hkv + h) * PAGE, to = ((size_t)i * Hkv + h) * PAGE;
    const uint4 *src = reinterpret_cast<const uint4 *>((is_k ? k_pages : v_pages) + from * D);
    const uint8_t *exps = (is_k ? k_exps : v_exps) + from;
    uint4 *dst = reinterpret_cast<uint4 *>((is_k ? k_out : v_out) + to * D);
    const int per_row = D / 16;
    for (int u = threadIdx.x; u < PAGE * per_row; u += READ_THREADS) {
        const uint4 raw = act_load(src + u);
        const float f = power_of_two((int)__ldcg(exps + u / per_row) - 127);
        const unsigned w[4] = {raw.x, raw.y, raw.z, raw.w};
        unsigned o[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const unsigned short two = (unsigned short)(w[j >> 1] >> (16 * (j & 1)));
            unsigned h2;
            asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h2) : "h"(two));
            const float2 x = __half22float2(*reinterpret_cast<__half2 *>(&h2));
            __nv_bfloat162 y = __floats2bfloat162_rn(x.x * f, x.y * f);
            o[j] = *reinterpret_cast<unsigned *>(&y);
        }
        dst[2 * u] = make_uint4(o[0], o[1], o[2], o[3]);
        dst[2 * u + 1] = make_uint4(o[4], o[5], o[6], o[7]);
    }
}

template <typename TS, bool Q8, typename... Args>
int launch_store(int D, dim3 grid, cudaStream_t stream, const void *src, Args... args) {
    if (D <= 64) lgml_launch(kv_store_kernel<TS, Q8, 1>, grid, WARPS * 32, 0, stream, (const TS *)src, args...);
    else if (D <= 128) lgml_launch(kv_store_kernel<TS, Q8, 2>, grid, WARPS * 32, 0, stream, (const TS *)src, args...);
    else lgml_launch(kv_store_kernel<TS, Q8, 4>, grid, WARPS * 32, 0, stream, (const TS *)src, args...);
    return lgml_launch_status("rope_kv_store");
}
template <int P, typename... Args>
int launch_wide(bool q8, bool adjacent, int n_tokens, cudaStream_t stream, Args... args) {
    if (q8 && adjacent) lgml_launch(kv_store_wide_kernel<P, true, true>, dim3(n_tokens), WIDE_THREADS, 0, stream, args...);
    else if (q8) lgml_launch(kv_store_wide_kernel<P, true, false>, dim3(n_tokens), WIDE_THREADS, 0, stream, args...);
    else if (adjacent) lgml_launch(kv_store_wide_kernel<P, false, true>, dim3(n_tokens), WIDE_THREADS, 0, stream, args...);
    else lgml_launch(kv_store_wide_kernel<P, false, false>, dim3(n_tokens), WIDE_THREADS, 0, stream, args...);
    return lgml_launch_status("rope_kv_store");
}
}  // namespace

// src_type: 0 float32 (n_parts of them, part_stride apart), 1 bfloat16.  cells null: the positions.  k_exps null: pages in bfloat16.
LGML_API int lgml_rope_kv_store(const void *src, int src_type, int lds, int n_parts, long long part_stride, const float *bias, void *q_out, int ldq,
                                const int *positions, const int *cells, const int *seq_of_token, const int *block_table, int n_seqs, int max_blocks,
                                const float *inv_freq, const float *inv_freq_lo, int n_rot, int pairing, void *k_pages, void *v_pages, void *k_exps,
                                void *v_exps, int n_pages, int page_size, int n_tokens, int H, int Hkv, int D, int write_kv, int *status,
                                cudaStream_t stream) {
    LGML_REQUIRE(n_tokens >= 0 && H > 0 && Hkv > 0 && n_parts >= 1 && max_blocks > 0 && n_seqs >= 0, "rope_kv_store: bad sizes");
    LGML_REQUIRE(page_size == PAGE, "rope_kv_store: pages of %d tokens, this kernel takes %d", page_size, PAGE);
    LGML_REQUIRE(D >= 16 && D <= MAX_D && D % 16 == 0, "rope_kv_store: head_dim %d must be a multiple of 16 up to %d", D, MAX_D);
    LGML_REQUIRE(n_rot >= 0 && n_rot <= D && n_rot % 2 == 0, "rope_kv_store: n_rot %d must be even and at most head_dim", n_rot);
    LGML_REQUIRE((k_exps == nullptr) == (v_exps == nullptr), "rope_kv_store: exponents for keys and values, or for neither");
    if (n_tokens == 0) return 0;
    const int n_heads = write_kv ? H + 2 * Hkv : H;
    LGML_REQUIRE((n_heads + WARPS - 1) / WARPS <= 65535, "rope_kv_store: too many heads");
    // many tokens whose heads turn whole, everything on the width of a thread's loads and stores
    if (src_type == LGML_BF16 && n_tokens >= WIDE_FROM && n_rot == D && (D == 64 || D == 128) && lds % 8 == 0 && ldq % 8 == 0 &&
        (((uintptr_t)src | (uintptr_t)q_out | (uintptr_t)k_pages | (uintptr_t)v_pages) & 15) == 0) {
#define LGML_ARGS k_exps != nullptr, pairing != 0, n_tokens, stream, (const __nv_bfloat16 *)src, lds, (__nv_bfloat16 *)q_out, ldq, positions, cells, seq_of_token, \
                  block_table, n_seqs, max_blocks, inv_freq, inv_freq_lo, k_pages, v_pages, (uint8_t *)k_exps, (uint8_t *)v_exps, n_pages, H, Hkv, n_heads, status
        return D == 64 ? launch_wide<2>(LGML_ARGS) : launch_wide<4>(LGML_ARGS);
#undef LGML_ARGS
    }
    dim3 grid(n_tokens, (n_heads + WARPS - 1) / WARPS);
#define LGML_ARGS D, grid, stream, src, lds, n_parts, part_stride, bias, (__nv_bfloat16 *)q_out, ldq, positions, cells, seq_of_token, block_table, n_seqs,  \
                  max_blocks, inv_freq, inv_freq_lo, n_rot, pairing, k_pages, v_pages, (uint8_t *)k_exps, (uint8_t *)v_exps, n_pages, H, Hkv, D, n_heads, \
                  status
    if (src_type == LGML_F32) return k_exps ? launch_store<float, true>(LGML_ARGS) : launch_store<float, false>(LGML_ARGS);
    if (src_type == LGML_BF16) return k_exps ? launch_store<__nv_bfloat16, true>(LGML_ARGS) : launch_store<__nv_bfloat16, false>(LGML_ARGS);
#undef LGML_ARGS
    LGML_FAIL("rope_kv_store: element type %d", src_type);
}

LGML_API int lgml_kv_read(const void *k_pages, const void *v_pages, const void *k_exps, const void *v_exps, int n_pages, int page_size,
                          const int *list, int n_list, void *k_out, void *v_out, int Hkv, int D, int *status, cudaStream_t stream) {
    LGML_REQUIRE(n_list >= 0 && Hkv > 0 && n_pages >= 0, "kv_read: bad sizes");
    LGML_REQUIRE(page_size == PAGE, "kv_read: pages of %d tokens, this kernel takes %d", page_size, PAGE);
    LGML_REQUIRE(D >= 16 && D <= MAX_D && D % 16 == 0, "kv_read: head_dim %d must be a multiple of 16 up to %d", D, MAX_D);
    LGML_REQUIRE((((uintptr_t)k_pages | (uintptr_t)v_pages | (uintptr_t)k_out | (uintptr_t)v_out) & 15) == 0, "kv_read: pages must be 16-byte aligned");
    LGML_REQUIRE((long long)n_list * Hkv <= 0x7fffffffLL, "kv_read: too many pages");
    if (n_list == 0) return 0;
    lgml_launch(kv_read_kernel, dim3(n_list * Hkv, 2), READ_THREADS, 0, stream, (const uint8_t *)k_pages, (const uint8_t *)v_pages, (const uint8_t *)k_exps,
                (const uint8_t *)v_exps, n_pages, list, (__nv_bfloat16 *)k_out, (__nv_bfloat16 *)v_out, Hkv, D, status);
    return lgml_launch_status("kv_read");
}
