// Attention of the new tokens of a request over its paged cache (attention_tree.cu has the definition) where a KV head has many rows: tokens x heads
// of 33 and more.  There the products are what takes time, so they are on tcgen05, 128 rows a block:
//     S[128, 64] = Q[128, D] . K_page^T        O[128, D] += P[128, 64] . V_page        accumulators in tensor memory
// Warps 0-7 do the softmax, two threads a row (half a page's columns each; they tell one another their maxima), and write P back into tensor memory, over the
// scores it came from; warps 8 and 9 bring the keys, 10 and 11 the values, into two stages each; the first thread of warp 12 issues the products.  There are
// two buffers of scores: those of page it + 2 are issued behind the P V product of page it, which read the buffer they go to, so a page's scores are there
// before the softmax of the page ahead of it is done, and the only chain is softmax after softmax.  (Products of one thread complete in the order of
// issue.)  Operands lie in shared memory in rows of 128 bytes, swizzled; V is the N-major operand.  The running output stays in tensor
// memory; the softmax threads correct it only when a row's maximum has grown by more than 2^8 since its sums'.
// Every mbarrier is of one parity of pages, and what its next phase needs comes after its waiters have seen this one, so none is missed.
// Tensor memory is taken behind the wait for the kernels ahead, so it is never held against one of them, and the kernels behind start when this one is done.
//
// Pages of e4m3 become float16 on the way to shared memory, exactly: 16 codes a load, a page ahead in registers, converted by the threads that loaded
// them.  Their powers of two stay outside: a key's multiplies its column of scores, a value's joins its column's
// exponent, and q is scaled row by row, as in attention_tree.cu (a row whose largest entry is
// between 2^-2 and 2^15 stays as it is: what float16 then rounds is under 2^-23 of that).  Pages in bfloat16 are copied as they are, a page ahead.
//
// Every column that a row may not see is a bit of a 64-bit word, tested only in pages that some row does not see whole.  There, values that are
// not finite become zeros before the product (0 x NaN), and are added at the end to the rows that see them.
// Two blocks share an SM.  Waits on mbarriers are bounded (status 14).
#include "tree_common.cuh"

LGML_DEFINE_LAST_ERROR(lgml_attention_tree_tall)

namespace {
constexpr int ROWS = 128;
constexpr int THREADS = 416;
constexpr int SOFTMAX = 256;                 // threads of warps 0-7
constexpr int LOADERS = 64;                  // threads that bring the keys, and the values
constexpr int KEYS = 256, VALUES = 320, ISSUER = 384;        // first thread of warps 8, 10 and 12
constexpr uint32_t SPIN_LIMIT = 1u << 20;    // polls of up to WAIT_HINT_NS each: about a second
constexpr uint32_t WAIT_HINT_NS = 1000;
constexpr int STATUS_TIMEOUT = 14;
constexpr uint32_t TMEM_COLS = 256, S1_COL = 64, O_COL = 128;      // scores of even pages at column 0, of odd ones at 64, the output at 128
constexpr float RESCALE_STEP = 8.f;

// shared memory written by threads becomes visible to the tensor core's reads
__device__ __forceinline__ void fence_async_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ void st_shared_16(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
__device__ __forceinline__ void mbar_arrive(uint64_t *bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
// A whole warp's: one arrival for its 32 threads (each would be an operation of its own on the barrier, one after the other).
__device__ __forceinline__ void warp_arrive(uint64_t *bar) {
    __syncwarp();
    if ((threadIdx.x & 31) == 0) mbar_arrive(bar);
}
__device__ __forceinline__ uint4 ld_shared_16(uint32_t addr) {
    uint4 v;
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ void mbar_init(uint64_t *bar, uint32_t count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(bar)), "r"(count));
}
__device__ __forceinline__ bool mbar_try_wait(uint64_t *bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok) : "r"(smem_u32(bar)), "r"(parity), "r"(WAIT_HINT_NS) : "memory");
    return ok != 0;
}
__device__ __forceinline__ bool mbar_wait(uint64_t *bar, uint32_t parity, volatile int *abort_flag, int *status) {
    for (uint32_t i = 0; i < SPIN_LIMIT; ++i) {
        if (mbar_try_wait(bar, parity)) return true;
        if ((i & 1023u) == 1023u && *abort_flag) return false;
        __nanosleep(100);
    }
    *abort_flag = 1;
    atomicExch(status, STATUS_TIMEOUT);
    return false;
}
__device__ __forceinline__ void tcgen05_alloc(uint32_t *dst_smem, uint32_t ncols) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(dst_smem)), "r"(ncols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tcgen05_dealloc(uint32_t taddr, uint32_t ncols) {
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(ncols) : "memory");
}
__device__ __forceinline__ void tcgen05_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tcgen05_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tcgen05_commit(uint64_t *bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void tcgen05_mma_f16(uint32_t tmem_d, uint64_t desc_a, uint64_t desc_b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
        ::"r"(tmem_d), "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(accumulate) : "memory");
}
// A in tensor memory: its row i in lane i, two 16-bit elements of K a 32-bit column
__device__ __forceinline__ void tcgen05_mma_f16_ts(uint32_t tmem_d, uint32_t tmem_a, uint64_t desc_b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
        ::"r"(tmem_d), "r"(tmem_a), "l"(desc_b), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void tcgen05_ld_16(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
          "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr) : "memory");
}
__device__ __forceinline__ void tcgen05_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tcgen05_st_16(uint32_t taddr, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
        ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
          "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}
__device__ __forceinline__ void tcgen05_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Shared-memory matrix descriptor, 128-byte swizzle, version 1.  Offsets in units of 16 bytes.
//   K-major operand (rows of 128 bytes, 8-row groups of 1024 bytes): leading 1 (unused), stride 1024.
//   N-major operand (64 elements of N contiguous in 128 bytes, 8 rows of K per 1024 bytes):
//   leading = distance between blocks of 64 along N, stride = distance between groups of 8 along K.
__device__ __forceinline__ uint64_t make_desc(uint32_t smem_addr, uint32_t leading_bytes, uint32_t stride_bytes) {
    uint64_t d = 0;
    d |= (uint64_t)((smem_addr >> 4) & 0x3fff);
    d |= (uint64_t)((leading_bytes >> 4) & 0x3fff) << 16;
    d |= (uint64_t)((stride_bytes >> 4) & 0x3fff) << 32;
    d |= (uint64_t)1 << 46;
    d |= (uint64_t)2 << 61;
    return d;
}
// kind::f16 instruction descriptor: float32 accumulator, both operands bfloat16 or both float16, A K-major; B K-major or N-major
__host__ __device__ constexpr uint32_t make_idesc(int m, int n, int b_n_major, int bf16) {
    return (1u << 4) | ((uint32_t)bf16 << 7) | ((uint32_t)bf16 << 10) | ((uint32_t)b_n_major << 16) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}
// byte offset of 16-byte chunk `chunk` (0..7) of row `row` inside a swizzled block of 128-byte rows
__device__ __forceinline__ uint32_t swz(int row, int chunk) { return (uint32_t)((row >> 3) * 1024 + (row & 7) * 128 + ((chunk ^ (row & 7)) << 4)); }

// two float32 products-and-sums, products, or sums, in one instruction
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(*reinterpret_cast<uint64_t *>(&a)), "l"(*reinterpret_cast<uint64_t *>(&b)), "l"(*reinterpret_cast<uint64_t *>(&c)));
    return *reinterpret_cast<float2 *>(&d);
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    uint64_t d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(*reinterpret_cast<uint64_t *>(&a)), "l"(*reinterpret_cast<uint64_t *>(&b)));
    return *reinterpret_cast<float2 *>(&d);
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    uint64_t d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(*reinterpret_cast<uint64_t *>(&a)), "l"(*reinterpret_cast<uint64_t *>(&b)));
    return *reinterpret_cast<float2 *>(&d);
}

// A pair of numbers that are not finite becomes zeros, and `odd` says so.
__device__ __forceinline__ uint32_t finite_pair(uint32_t x, uint32_t inf, bool &odd) {
    const uint32_t lo = inf & 0xffffu, hi = inf & 0xffff0000u;
    if ((x & lo) == lo) x &= 0xffff0000u, odd = true;
    if ((x & hi) == hi) x &= 0xffffu, odd = true;
    return x;
}

template <int D, bool Q8>
__global__ void __launch_bounds__(THREADS, 2) tree_attention_tall_kernel(
    const __nv_bfloat16 *__restrict__ q, int ldq, const int *__restrict__ positions, const int *__restrict__ seq_start, const int *__restrict__ seq_pos0,
    const long long *__restrict__ visible, const int *__restrict__ block_table, int max_blocks, const uint8_t *__restrict__ k_pages,
    const uint8_t *__restrict__ v_pages, const uint8_t *__restrict__ k_exps, const uint8_t *__restrict__ v_exps, int n_pages, __nv_bfloat16 *__restrict__ out,
    int ldo, float *__restrict__ part_o, float2 *__restrict__ part_ml, int n_splits, int clustered, int n_tokens, int H, int Hkv, int n_chunks, int limit,
    float scale, int window, int *__restrict__ status) {
    constexpr int KB = D / 64;                        // 64-element blocks along the head
    constexpr uint32_t Q_BYTES = KB * ROWS * 128, K_BYTES = KB * PAGE * 128;
    constexpr int HALF = D / 2;
    constexpr int SIZE = Q8 ? 1 : 2, PER_ROW = D * SIZE / 16, LOADS = PAGE * PER_ROW / LOADERS;       // 16-byte loads of a page's keys: a row's, a thread's
    constexpr int STEP = LOADERS / PER_ROW;           // rows from one load of a thread to its next: 4, 8 or 16
    extern __shared__ uint8_t smem_raw[];
    uint8_t *base = (uint8_t *)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    uint8_t *Qs = base, *Ks = Qs + Q_BYTES, *Vs = Ks + 2 * K_BYTES;         // two stages of keys, two of values
    __shared__ __align__(16) float kf_s[4][PAGE], add_s[4][PAGE], vf_s[4][PAGE];      // per column of page it (it % 4): its scores' factor, what is added to them,
                                                                                      // and what its probability counts for in the sum
    __shared__ float max_s[2][2][ROWS], sum_s[2][ROWS];   // by the page's parity and the half: a row's maximum; its sum, at the end
    __shared__ __align__(8) float fin[ROWS][2];
    __shared__ float unscale_s[ROWS];
    __shared__ uint64_t k_full[2], v_full[2], s_full[2], p_full[2], o_done[2];        // by the page's parity
    __shared__ uint32_t tmem_base_s;
    __shared__ int abort_s, odd_s, ok_s[4];               // ok_s[it % 4]: whether page it is there
    volatile int *abort_flag = &abort_s;

    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int s = blockIdx.x / n_splits, split = blockIdx.x - s * n_splits, kvh = blockIdx.y / n_chunks, chunk = blockIdx.y - kvh * n_chunks;
    const int row0 = early_int(seq_start + s), n = early_int(seq_start + s + 1) - row0, pos0 = early_int(seq_pos0 + s);
    const int group = H / Hkv, n_rows = n * group, r0 = chunk * ROWS;
    if (n <= 0 || n > limit || r0 >= n_rows) return;
    if (row0 < 0 || row0 + n > n_tokens || pos0 < 0) {
        if (tid == 0) atomicExch(status, 3);
        return;
    }
    // ---- this thread's row ----
    const int quarter = warp & 3, half = (warp >> 2) & 1, row = quarter * 32 + lane;         // (tensor memory: a warp reads its quarter of the lanes)
    const bool row_valid = r0 + row < n_rows;
    const int my_tok = min(r0 + row, n_rows - 1) / group;
    const int my_pos = early_int(positions + row0 + my_tok);
    const unsigned long long all_new = ~0ull >> (64 - n);
    unsigned long long my_mask = (visible ? (unsigned long long)__ldcg(visible + row0 + my_tok) : ~0ull >> (63 - my_tok)) & all_new;
    const int n_cells = pos0 + n;
    int low = 0, all_from = 0;              // none of the rows sees a cell below the first, every row sees the old cells from the second on
    if (window > 0) {
        const int t0 = r0 / group, t1 = (min(r0 + ROWS, n_rows) - 1) / group;
        int lowest = 0x7fffffff, highest = -0x7fffffff;
        for (int j = 0; j < n; ++j) {
            const int at = early_int(positions + row0 + j);
            if (j >= t0 && j <= t1) lowest = min(lowest, at), highest = max(highest, at);
            if (at <= my_pos - window) my_mask &= ~(1ull << j);
        }
        low = min(max(lowest - window + 1, 0), pos0);
        all_from = highest - window + 1;
    }
    // Which of page pg's cells the row sees.
    auto seen_of = [&](int pg) -> unsigned long long {
        const int old = pos0 - pg * PAGE, from = window > 0 ? my_pos - window + 1 - pg * PAGE : 0;
        unsigned long long v = old >= PAGE ? ~0ull : old <= 0 ? 0ull : ~0ull >> (PAGE - old);
        if (from > 0) v = from >= PAGE ? 0ull : v & (~0ull << from);
        if (old < PAGE && old > -PAGE) v |= old >= 0 ? my_mask << old : my_mask >> -old;
        return v;
    };
    auto whole = [&](int pg) { return (pg + 1) * PAGE <= pos0 && pg * PAGE >= all_from; };
    const int first_page = low / PAGE, end_page = (n_cells + PAGE - 1) / PAGE;
    const int pps = (end_page - first_page + n_splits - 1) / n_splits;
    const int pb = first_page + split * pps, n_it = max(min(pps, end_page - pb), 0);

    if (tid == 0) {
        for (int i = 0; i < 2; ++i) {
            mbar_init(&k_full[i], LOADERS / 32);
            mbar_init(&v_full[i], LOADERS / 32);
            mbar_init(&s_full[i], 1);
            mbar_init(&p_full[i], SOFTMAX / 32);
            mbar_init(&o_done[i], 1);
        }
        abort_s = odd_s = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    pdl_wait();
    if (warp == 1) tcgen05_alloc(&tmem_base_s, TMEM_COLS);
    {
        // queries: row r = (token, head) r0 + r; through L2, they were just written
        constexpr int CH = D / 8;
#pragma unroll
        for (int c = tid; c < ROWS * CH; c += THREADS) {
            const int r = c / CH, ch = c - r * CH, rr = r0 + r;
            uint4 v = make_uint4(0, 0, 0, 0);
            if (rr < n_rows) v = __ldcg(reinterpret_cast<const uint4 *>(q + (size_t)(row0 + rr / group) * ldq + (size_t)(kvh * group + rr % group) * D + ch * 8));
            if (Q8) {
                uint32_t w[4] = {v.x, v.y, v.z, v.w};
                float amax = 0.f;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float2 f = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162 *>(&w[j]));
                    amax = fmaxf(amax, fmaxf(fabsf(f.x), fabsf(f.y)));
                }
#pragma unroll
                for (int o = CH / 2; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));       // (CH neighbouring threads have a row)
                // 2^x so that amax 2^x is in [2^14, 2^15), unless it is well within float16 already
                const int e = (int)(__float_as_uint(amax) >> 23) - 127, x = e >= -2 && e <= 14 ? 0 : min(max(14 - e, -114), 100);
                const float up = power_of_two(x);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float2 f = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162 *>(&w[j]));
                    const __half2 h = __floats2half2_rn(f.x * up, f.y * up);
                    w[j] = *reinterpret_cast<const uint32_t *>(&h);
                }
                v = make_uint4(w[0], w[1], w[2], w[3]);
                if (ch == 0) unscale_s[r] = power_of_two(-x);
            }
            *reinterpret_cast<uint4 *>(Qs + (ch >> 3) * (ROWS * 128) + swz(r, ch & 7)) = v;
        }
    }
    fence_async_smem();
    tcgen05_fence_before();
    __syncthreads();
    tcgen05_fence_after();
    const uint32_t tmem_base = tmem_base_s, lane_addr = tmem_base + ((uint32_t)(quarter * 32) << 16);
    const float scale_log2 = scale * 1.4426950408889634f;
    bool alive = true;

    // ---- the pages ----
    const int l = tid & (LOADERS - 1);
    auto page_of = [&](int it) {
        const int page = it < n_it && pb + it < max_blocks ? early_int(block_table + (size_t)s * max_blocks + pb + it) : -1;
        return page >= 0 && page < n_pages ? page : -1;
    };
    // Load u of a thread: 16 bytes from chunk l % PER_ROW of row l / PER_ROW + STEP u on.
    const int l_row = l / PER_ROW, l_chunk = l - l_row * PER_ROW;
    // Where 16-byte chunk `chunk` of that row lies in a stage.
    auto place = [&](int chunk, int u) -> uint32_t {
        const int r = l_row + STEP * u;
        return (uint32_t)((chunk >> 3) * (PAGE * 128)) + swz(r, chunk & 7);
    };
    auto fetch = [&](uint4 (&raw)[LOADS], const uint8_t *pages, int it, int page) {
        const int left = n_cells - (pb + it) * PAGE;
        const uint8_t *src = pages + ((size_t)max(page, 0) * Hkv + kvh) * PAGE * D;
#pragma unroll
        for (int u = 0; u < LOADS; ++u)
            raw[u] = page >= 0 && l_row + STEP * u < left ? __ldcg(reinterpret_cast<const uint4 *>(src) + l + LOADERS * u) : make_uint4(0, 0, 0, 0);
    };
    // ... as float16 in shared memory; in a page that not every row sees whole (check), without what is not finite.
    auto convert = [&](uint32_t dst, const uint4 (&raw)[LOADS], bool check) {
        bool odd = false;
#pragma unroll
        for (int u = 0; u < LOADS; ++u) {
            const uint32_t w[4] = {raw[u].x, raw[u].y, raw[u].z, raw[u].w};
            uint32_t h[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) h[j] = half2_of_codes((unsigned short)(w[j >> 1] >> (16 * (j & 1))));
            if (check) {
#pragma unroll
                for (int j = 0; j < 8; ++j) h[j] = finite_pair(h[j], 0x7c007c00u, odd);
            }
            st_shared_16(dst + place(2 * l_chunk, u), h[0], h[1], h[2], h[3]);
            st_shared_16(dst + place(2 * l_chunk + 1, u), h[4], h[5], h[6], h[7]);
        }
        if (odd) odd_s = 1;
    };
    // What the softmax of page it has to know of its columns: the exponents of column l, as bytes ...
    auto exponents = [&](int it, int page) -> int2 {
        if (!Q8 || page < 0 || (pb + it) * PAGE + l >= n_cells) return make_int2(127, 127);
        const size_t vec = ((size_t)page * Hkv + kvh) * PAGE + l;
        return make_int2((int)__ldcg(k_exps + vec), (int)__ldcg(v_exps + vec));
    };
    // ... and what it makes of them.
    auto columns = [&](int it, int page, int2 e) {
        if (l == 0) ok_s[it & 3] = page >= 0;
        if (l == 0 && page < 0) atomicExch(status, 3);
        if (Q8) {
            const int ke = min(e.x, 246) - 127, ve = min(e.y, 246) - 127;
            kf_s[it & 3][l] = scale_log2 * power_of_two(ke);
            add_s[it & 3][l] = (float)ve;
            vf_s[it & 3][l] = power_of_two(-ve);
        }
    };
    // bfloat16: asynchronous copies
    auto copy_page = [&](uint32_t dst, const uint8_t *pages, int it, int page) {
        const int left = n_cells - (pb + it) * PAGE;
        const uint8_t *src = pages + ((size_t)max(page, 0) * Hkv + kvh) * PAGE * D * 2;
#pragma unroll
        for (int u = 0; u < LOADS; ++u) copy_16(dst + place(l_chunk, u), src + (size_t)(l + LOADERS * u) * 16, page >= 0 && l_row + STEP * u < left);
        copies_commit();
    };
    auto ask_l2 = [&](const uint8_t *pages, int page) {
        if (page < 0) return;
        const uint8_t *src = pages + ((size_t)page * Hkv + kvh) * PAGE * D * SIZE;
#pragma unroll
        for (int u = 0; u < (PAGE * D * SIZE / 128 + LOADERS - 1) / LOADERS; ++u)
            if (l + LOADERS * u < PAGE * D * SIZE / 128) asm volatile("prefetch.global.L2 [%0];" ::"l"(src + (size_t)(l + LOADERS * u) * 128));
    };
    const uint32_t ks0 = smem_u32(Ks), vs0 = smem_u32(Vs);
    float m_ref = -INFINITY, l_run = 0.f;
    if (tid >= KEYS && tid < ISSUER) {
        // ---- the keys, or the values: page it's stage is free when the products of page it - 2 have read it ----
        // (page numbers come four pages ahead and ask L2 for their pages, codes and exponents one page ahead: each is a trip to L2 or beyond)
        const bool keys = tid < VALUES;
        const uint8_t *pages = keys ? k_pages : v_pages;
        const uint32_t stages = keys ? ks0 : vs0;
        uint64_t *full = keys ? k_full : v_full, *read = keys ? s_full : o_done;
        int next[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) next[i] = page_of(i);
#pragma unroll
        for (int i = Q8 ? 1 : 2; i < 4; ++i) ask_l2(pages, next[i]);
        if (Q8) {
            uint4 raw[LOADS];
            int2 exps = make_int2(127, 127);
            if (n_it > 0) {
                if (keys) exps = exponents(0, next[0]);
                fetch(raw, pages, 0, next[0]);
            }
            for (int it = 0; it < n_it; ++it) {
                const int coming = page_of(it + 4);
                if (it >= 2 && !__all_sync(0xffffffffu, mbar_wait(&read[it & 1], ((it - 2) >> 1) & 1, abort_flag, status))) break;
                if (keys) columns(it, next[0], exps);
                convert(stages + (it & 1) * K_BYTES, raw, !keys && !whole(pb + it));
                fence_async_smem();
                warp_arrive(&full[it & 1]);
                if (it + 1 < n_it) {
                    if (keys) exps = exponents(it + 1, next[1]);
                    fetch(raw, pages, it + 1, next[1]);
                }
                next[0] = next[1], next[1] = next[2], next[2] = next[3], next[3] = coming;
                ask_l2(pages, coming);
            }
        } else {
            for (int it = 0; it < 2; ++it) {
                if (it < n_it) copy_page(stages + it * K_BYTES, pages, it, next[it]);
                else copies_commit();
            }
            for (int it = 0; it < n_it; ++it) {
                const int coming = page_of(it + 4);
                if (keys) columns(it, next[0], make_int2(127, 127));
                copies_wait<1>();
                if (!keys && !whole(pb + it)) {
                    bool odd = false;
#pragma unroll
                    for (int u = 0; u < LOADS; ++u) {
                        const uint32_t where = vs0 + (it & 1) * K_BYTES + place(l_chunk, u);
                        const uint4 v = ld_shared_16(where);
                        st_shared_16(where, finite_pair(v.x, 0x7f807f80u, odd), finite_pair(v.y, 0x7f807f80u, odd), finite_pair(v.z, 0x7f807f80u, odd),
                                     finite_pair(v.w, 0x7f807f80u, odd));
                    }
                    if (odd) odd_s = 1;
                }
                fence_async_smem();
                warp_arrive(&full[it & 1]);
                // the stage is free again when this page's products have read it: the page after the next
                if (it + 2 < n_it) {
                    if (!__all_sync(0xffffffffu, mbar_wait(&read[it & 1], (it >> 1) & 1, abort_flag, status))) break;
                    copy_page(stages + (it & 1) * K_BYTES, pages, it + 2, next[2]);
                } else {
                    copies_commit();
                }
                next[0] = next[1], next[1] = next[2], next[2] = next[3], next[3] = coming;
                ask_l2(pages, coming);
            }
        }
    } else if (tid == ISSUER) {
        // ---- the products ----
        constexpr uint32_t idesc_qk = make_idesc(ROWS, PAGE, 0, Q8 ? 0 : 1), idesc_pv = make_idesc(ROWS, D, 1, Q8 ? 0 : 1);
        const uint64_t desc_q0 = make_desc(smem_u32(Qs), 16, 1024), desc_k0 = make_desc(ks0, 16, 1024), desc_v0 = make_desc(vs0, PAGE * 128, 1024);
        auto issue_scores = [&](int it) {
            const uint64_t dk = desc_k0 + (uint64_t)(((it & 1) * K_BYTES) >> 4);
#pragma unroll
            for (int ks = 0; ks < D / 16; ++ks) {
                const uint64_t da = desc_q0 + (uint64_t)(((ks >> 2) * (ROWS * 128) + (ks & 3) * 32) >> 4);
                const uint64_t db = dk + (uint64_t)(((ks >> 2) * (PAGE * 128) + (ks & 3) * 32) >> 4);
                tcgen05_mma_f16(tmem_base + (uint32_t)(it & 1) * S1_COL, da, db, idesc_qk, ks > 0 ? 1u : 0u);
            }
            tcgen05_commit(&s_full[it & 1]);
        };
        for (int it = 0; it < n_it && it < 2 && alive; ++it) {
            alive = mbar_wait(&k_full[it], 0, abort_flag, status);
            tcgen05_fence_after();
            if (alive) issue_scores(it);
        }
        for (int it = 0; it < n_it && alive; ++it) {
            const uint32_t ph = (it >> 1) & 1;
            alive = mbar_wait(&v_full[it & 1], ph, abort_flag, status) && mbar_wait(&p_full[it & 1], ph, abort_flag, status);
            tcgen05_fence_after();
            if (!alive) break;
            const uint64_t dv = desc_v0 + (uint64_t)(((it & 1) * K_BYTES) >> 4);
#pragma unroll
            for (int k2 = 0; k2 < PAGE / 16; ++k2)
                tcgen05_mma_f16_ts(tmem_base + O_COL, tmem_base + (uint32_t)(it & 1) * S1_COL + (uint32_t)k2 * 8u, dv + (uint64_t)((k2 * 2048) >> 4), idesc_pv,
                                   (it > 0 || k2 > 0) ? 1u : 0u);
            tcgen05_commit(&o_done[it & 1]);
            if (it + 2 < n_it) {
                alive = mbar_wait(&k_full[it & 1], ((it + 2) >> 1) & 1, abort_flag, status);
                tcgen05_fence_after();
                if (alive) issue_scores(it + 2);
            }
        }
    } else if (tid < SOFTMAX) {
        // ---- softmax: columns 32 half .. 32 half + 31 of this row ----
        constexpr int COLS = PAGE / 2;
        const int c_first = half * COLS;
        const float unscale = Q8 ? unscale_s[row] : 1.f;
        const bool any_scaled = Q8 && __any_sync(0xffffffffu, unscale != 1.f);
        for (int it = 0; it < n_it; ++it) {
            const int pg = pb + it;
            const uint32_t s_addr = lane_addr + (uint32_t)(it & 1) * S1_COL;
            // (a warp gives up as one, and then goes through its pages without waiting: its partner meets it in each)
            alive = __all_sync(0xffffffffu, alive && mbar_wait(&s_full[it & 1], (it >> 1) & 1, abort_flag, status));
            tcgen05_fence_after();
            const bool there = ok_s[it & 3] != 0, edge = !whole(pg) || !there;
            union {
                uint32_t u[COLS];
                float2 f[COLS / 2];
            } r;
            tcgen05_ld_16(s_addr + (uint32_t)c_first, *reinterpret_cast<uint32_t(*)[16]>(&r.u[0]));
            tcgen05_ld_16(s_addr + (uint32_t)c_first + 16u, *reinterpret_cast<uint32_t(*)[16]>(&r.u[16]));
            tcgen05_wait_ld();
            if (Q8) {
                if (any_scaled) {
#pragma unroll
                    for (int c = 0; c < COLS / 2; ++c) r.f[c] = mul2(r.f[c], make_float2(unscale, unscale));
                }
#pragma unroll
                for (int c = 0; c < COLS; c += 4) {
                    const float4 kf = *reinterpret_cast<const float4 *>(&kf_s[it & 3][c_first + c]), ad = *reinterpret_cast<const float4 *>(&add_s[it & 3][c_first + c]);
                    r.f[c / 2] = fma2(r.f[c / 2], make_float2(kf.x, kf.y), make_float2(ad.x, ad.y));
                    r.f[c / 2 + 1] = fma2(r.f[c / 2 + 1], make_float2(kf.z, kf.w), make_float2(ad.z, ad.w));
                }
            } else {
#pragma unroll
                for (int c = 0; c < COLS / 2; ++c) r.f[c] = mul2(r.f[c], make_float2(scale_log2, scale_log2));
            }
            if (edge) {
                const uint32_t v = there ? (uint32_t)(seen_of(pg) >> c_first) : 0u;
#pragma unroll
                for (int c = 0; c < COLS; ++c)
                    if (!((v >> c) & 1u)) r.u[c] = __float_as_uint(-INFINITY);
            }
            float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
            for (int c = 0; c < COLS; ++c) mx4[c & 3] = fmaxf(mx4[c & 3], __uint_as_float(r.u[c]));
            const float mine = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3]));
            // the row's other thread is in the warp four further: the two warps meet here.  (Behind this both have their scores, so P may be written over them.)
            max_s[it & 1][half][row] = mine;
            asm volatile("bar.sync %0, 64;" ::"r"(1 + quarter) : "memory");
            const float m_new = fmaxf(mine, max_s[it & 1][half ^ 1][row]);
            float corr = 1.f;
            if (m_ref == -INFINITY) {
                m_ref = m_new;                       // nothing summed yet: nothing to correct
            } else if (m_new > m_ref + RESCALE_STEP) {
                corr = ex2(m_ref - m_new);
                m_ref = m_new;
                l_run *= corr;
            }
            if (__any_sync(0xffffffffu, corr != 1.f)) {
                // ---- correct this half of the running output (rare): the product of the page before must be done, this page's has to wait for P ----
                // (a correction implies an earlier page)
                alive = __all_sync(0xffffffffu, alive && mbar_wait(&o_done[(it - 1) & 1], ((it - 1) >> 1) & 1, abort_flag, status));
                tcgen05_fence_after();
#pragma unroll
                for (int c0 = 0; c0 < HALF; c0 += 16) {
                    uint32_t o[16];
                    tcgen05_ld_16(lane_addr + O_COL + (uint32_t)(half * HALF + c0), o);
                    tcgen05_wait_ld();
#pragma unroll
                    for (int j = 0; j < 16; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * corr);
                    tcgen05_st_16(lane_addr + O_COL + (uint32_t)(half * HALF + c0), o);
                }
            }
            const float neg_m = m_ref == -INFINITY ? 0.f : -m_ref;
            float2 sum2[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
            uint32_t packed[16];
#pragma unroll
            for (int c = 0; c < COLS / 2; ++c) {
                const float2 x = add2(r.f[c], make_float2(neg_m, neg_m)), e = make_float2(ex2(x.x), ex2(x.y));
                if (Q8) {
                    sum2[c & 1] = fma2(e, *reinterpret_cast<const float2 *>(&vf_s[it & 3][c_first + 2 * c]), sum2[c & 1]);
                    const __half2 h2 = __floats2half2_rn(e.x, e.y);
                    packed[c] = *reinterpret_cast<const uint32_t *>(&h2);
                } else {
                    sum2[c & 1] = add2(sum2[c & 1], e);
                    const __nv_bfloat162 h2 = __floats2bfloat162_rn(e.x, e.y);
                    packed[c] = *reinterpret_cast<const uint32_t *>(&h2);
                }
            }
            tcgen05_st_16(s_addr + (uint32_t)(c_first >> 1), packed);
            l_run += (sum2[0].x + sum2[0].y) + (sum2[1].x + sum2[1].y);
            tcgen05_wait_st();
            tcgen05_fence_before();
            warp_arrive(&p_full[it & 1]);
        }
        // (the last scores were seen, and were issued behind the product two pages before: the barrier is at most a phase away)
        if (n_it > 0 && alive && !mbar_wait(&o_done[(n_it - 1) & 1], ((n_it - 1) >> 1) & 1, abort_flag, status)) alive = false;
        sum_s[half][row] = l_run;
        if (half == 0) fin[row][0] = m_ref;
    }
    copies_wait<0>();
    __syncthreads();
    tcgen05_fence_after();
    alive = abort_s == 0;
    if (tid < ROWS) fin[row][1] = sum_s[0][row] + sum_s[1][row];

    // ---- the result: every thread half the columns of its row ----
    float *merge = reinterpret_cast<float *>(base);          // [ROWS][D + 2], where the operands were
    if (tid < SOFTMAX) {
        const float M = fin[row][0], sum = sum_s[0][row] + sum_s[1][row];
        const int col0 = half * HALF;
        __nv_bfloat16 *dst = row_at(out, ldo, row0, min(r0 + row, n_rows - 1), group, kvh, D, 0);
        const size_t part = ((size_t)(row0 + my_tok) * H + kvh * group + min(r0 + row, n_rows - 1) % group) * n_splits + split;
        const bool odd = odd_s != 0;
#pragma unroll
        for (int c0 = 0; c0 < HALF; c0 += 16) {
            uint32_t r[16];
            if (n_it > 0) {
                tcgen05_ld_16(lane_addr + O_COL + (uint32_t)(col0 + c0), r);
                tcgen05_wait_ld();
            } else {
#pragma unroll
                for (int j = 0; j < 16; ++j) r[j] = 0u;
            }
            if (odd && row_valid) {
                // (rare) what was taken out of the values, for the cells this row sees
                for (int it = 0; it < n_it; ++it) {
                    const int page = page_of(it);
                    if (page < 0 || whole(pb + it)) continue;
                    const unsigned long long v = seen_of(pb + it);
                    for (int c = 0; c < PAGE; ++c) {
                        if (!((v >> c) & 1)) continue;
                        const uint8_t *p = v_pages + ((((size_t)page * Hkv + kvh) * PAGE + c) * D + col0 + c0) * SIZE;
                        for (int j = 0; j < 16; ++j) {
                            float x;
                            if (Q8) x = (__ldcg(p + j) & 0x7f) == 0x7f ? __int_as_float(0x7fffffff) : 0.f;
                            else x = __bfloat162float(__ldcg(reinterpret_cast<const __nv_bfloat16 *>(p) + j));
                            if (!(fabsf(x) <= 3.402823466e38f)) {
#pragma unroll
                                for (int k = 0; k < 16; ++k)
                                    if (k == j) r[k] = __float_as_uint(__uint_as_float(r[k]) + x);
                            }
                        }
                    }
                }
            }
            if (n_splits == 1) {
                if (row_valid && alive) {
                    const float inv = 1.f / sum;
                    uint32_t h[8];
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const __nv_bfloat162 two = sum == 0.f ? __floats2bfloat162_rn(0.f, 0.f)
                                                              : __floats2bfloat162_rn(__uint_as_float(r[2 * j]) * inv, __uint_as_float(r[2 * j + 1]) * inv);
                        h[j] = *reinterpret_cast<const uint32_t *>(&two);
                    }
                    *reinterpret_cast<uint4 *>(dst + col0 + c0) = make_uint4(h[0], h[1], h[2], h[3]);
                    *reinterpret_cast<uint4 *>(dst + col0 + c0 + 8) = make_uint4(h[4], h[5], h[6], h[7]);
                }
            } else if (clustered) {
#pragma unroll
                for (int j = 0; j < 16; j += 2)
                    *reinterpret_cast<float2 *>(merge + (size_t)row * (D + 2) + col0 + c0 + j) = make_float2(__uint_as_float(r[j]), __uint_as_float(r[j + 1]));
            } else if (row_valid) {
#pragma unroll
                for (int j = 0; j < 16; j += 2)
                    *reinterpret_cast<float2 *>(part_o + part * D + col0 + c0 + j) = make_float2(__uint_as_float(r[j]), __uint_as_float(r[j + 1]));
                if (col0 + c0 == 0) part_ml[part] = make_float2(M, sum);
            }
        }
    }
    tcgen05_fence_before();
    pdl_trigger();      // at the end: a block that takes half an SM keeps the next kernel back until it is done
    __syncthreads();
    if (warp == 1) {
        tcgen05_fence_after();
        tcgen05_dealloc(tmem_base, TMEM_COLS);
    }
    if (!clustered) return;
    __syncwarp();
    cluster_sync();
    join_cluster<ROWS, D, THREADS>(merge, fin, n_splits, n_rows - r0, [&](int r, int d) { return row_at(out, ldo, row0, r0 + r, group, kvh, D, d); });
    __syncwarp();
    cluster_sync();                         // (the others' shared memory is read until here)
}

template <int D, bool Q8, typename... Args>
int launch(dim3 grid, int cluster, cudaStream_t stream, Args... args) {
    constexpr size_t smem = (size_t)(D / 64) * (ROWS + 4 * PAGE) * 128 + 1024;
    cudaError_t e = cudaFuncSetAttribute(tree_attention_tall_kernel<D, Q8>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) LGML_FAIL("tree_attention: cannot have %zu bytes of shared memory: %s", smem, cudaGetErrorString(e));
    lgml_launch_cluster(tree_attention_tall_kernel<D, Q8>, grid, THREADS, smem, stream, cluster, args...);
    return lgml_launch_status("tree_attention");
}
}  // namespace

// As lgml_tree_attention, for head sizes of 64 and 128 and rows of q and out on 16 bytes.
LGML_API int lgml_tree_attention_tall(const void *q, int ldq, const int *positions, const int *seq_start, const int *seq_pos0, const long long *visible,
                                      const int *block_table, int n_seqs, int max_blocks, const void *k_pages, const void *v_pages, const void *k_exps,
                                      const void *v_exps, int n_pages, int page_size, void *out, int ldo, float *scratch, int n_splits, int n_tokens, int limit,
                                      int H, int Hkv, int D, float scale, int window, int *status, cudaStream_t stream) {
    LGML_REQUIRE(n_tokens >= 0 && n_seqs >= 0 && H > 0 && Hkv > 0 && max_blocks > 0 && n_pages >= 0, "tree_attention: bad sizes");
    LGML_REQUIRE(page_size == PAGE, "tree_attention: pages of %d tokens, this kernel takes %d", page_size, PAGE);
    LGML_REQUIRE(H % Hkv == 0, "tree_attention: %d heads are no multiple of %d KV heads", H, Hkv);
    LGML_REQUIRE(D == 64 || D == 128, "tree_attention: head_dim %d must be 64 or 128 here", D);
    LGML_REQUIRE(limit >= 1 && limit <= MAX_NEW, "tree_attention: %d new tokens a request (1 to %d)", limit, MAX_NEW);
    LGML_REQUIRE(n_splits >= 1 && n_splits <= MAX_SPLITS, "tree_attention: %d key ranges (1 to %d)", n_splits, MAX_SPLITS);
    LGML_REQUIRE(n_splits <= MAX_CLUSTER || (scratch != nullptr && ((uintptr_t)scratch & 7) == 0), "tree_attention: several ranges need scratch memory");
    LGML_REQUIRE((k_exps == nullptr) == (v_exps == nullptr), "tree_attention: exponents for keys and values, or for neither");
    LGML_REQUIRE((((uintptr_t)k_pages | (uintptr_t)v_pages) & 15) == 0, "tree_attention: the cache must be 16-byte aligned");
    LGML_REQUIRE(ldq % 8 == 0 && ldo % 8 == 0 && (((uintptr_t)q | (uintptr_t)out) & 15) == 0, "tree_attention: q and out must be 16-byte aligned here");
    LGML_REQUIRE((long long)n_seqs * (limit > n_splits ? limit : n_splits) <= 0x7fffffffLL, "tree_attention: too many requests");
    if (n_tokens == 0 || n_seqs == 0) return 0;
    const int n_chunks = (limit * (H / Hkv) + ROWS - 1) / ROWS;
    LGML_REQUIRE((long long)Hkv * n_chunks <= 65535, "tree_attention: too many heads");
    const int clustered = n_splits > 1 && n_splits <= MAX_CLUSTER;
    dim3 grid(n_seqs * n_splits, Hkv * n_chunks);
    float *part_o = scratch;
    float2 *part_ml = scratch ? reinterpret_cast<float2 *>(scratch + (size_t)n_tokens * H * n_splits * D) : nullptr;
#define LGML_ARGS grid, clustered ? n_splits : 1, stream, (const __nv_bfloat16 *)q, ldq, positions, seq_start, seq_pos0, visible, block_table, max_blocks, \
                  (const uint8_t *)k_pages, (const uint8_t *)v_pages, (const uint8_t *)k_exps, (const uint8_t *)v_exps, n_pages, (__nv_bfloat16 *)out, ldo,  \
                  part_o, part_ml, n_splits, clustered, n_tokens, H, Hkv, n_chunks, limit, scale, window, status
    const int rc = D == 64 ? (k_exps ? launch<64, true>(LGML_ARGS) : launch<64, false>(LGML_ARGS)) : (k_exps ? launch<128, true>(LGML_ARGS) : launch<128, false>(LGML_ARGS));
#undef LGML_ARGS
    if (rc || n_splits <= MAX_CLUSTER) return rc;
    return tree_join(part_o, part_ml, seq_start, n_seqs, limit, n_tokens, out, ldo, n_splits, H, D, stream);
}
