// Attention of the new tokens of a request over its paged cache (attention_tree.cu has the definition) where a KV head has many rows: tokens x heads
// of 17 or 33 and more.  There the products are what takes time, so they are on tcgen05, one tile of 128 rows a block, or two where there are more rows:
//     S[128, 64] = Q[128, D] . K_page^T        O[128, D] += P[128, 64] . V_page        accumulators in tensor memory
// A thread a row does the softmax and writes P back into tensor memory, over the scores it came from; groups of two warps bring pages' keys and values into
// stages of shared memory, which the tiles share; a warp a tile issues its products.  A tile has two buffers of scores: those of page it + 2 are issued behind the
// P V product of page it, which read the buffer they go to, so a page's scores are there before the softmax of the page ahead of it is done, and a
// tile's only chain is softmax after softmax.  (Products of one thread complete in the order of issue.)  Operands lie in shared memory in rows of 128 bytes,
// swizzled; V is the N-major operand.  The running output stays in tensor memory; the softmax corrects it only when a row's maximum has grown by more than
// 2^8 since its sums'.  The maximum is of the products as they are, so a score is one multiply-and-add; the scale has to be above zero.
// P is rounded for the product, to float16 beside codes (half a step: 2^-11 of it) and to bfloat16 beside bfloat16 (2^-8), as the types of a product must be; sums are float32, of
// the probabilities before that (of the rounded bfloat16 ones, which attention_tree.cu takes: 3 to 10 % more time here).  Beside codes a probability is times its value's
// power of two, so the sum is about a maximum of its own, of the scores alone: powers that are 2^100 apart, or values of zeros, take nothing from it.
// Every mbarrier is of one stage, or one parity of pages, and what its next phase needs comes after its waiters have seen this one, so none is missed.
// Tensor memory is taken behind the wait for the kernels ahead, so it is never held against one of them, and the kernels behind start when this one is done.
//
// Pages of e4m3 become float16 on the way to shared memory, exactly: 16 codes a load, which set out as the unit before them goes in.  Where a page's
// powers of two lie close together (powers_of), its rows are multiplied by theirs below the largest, which the whole page is scaled by; q is scaled row by row, as
// in attention_tree.cu (a row whose largest entry is between 2^-2 and 2^15 stays as it is: what float16 then rounds is under 2^-23 of that).
// Pages in bfloat16 are copied as they are, one or three pages ahead.
//
// Every column that a row may not see is a bit of a 64-bit word, tested only in pages that some row does not see whole.  There, values that are
// not finite become zeros before the product (0 x NaN), and are added at the end to the rows that see them.
//
// What bounds it is the chain of a tile's softmax, page after page: 2,100 cycles from one page's scores to the next (150 until they are seen, 110 to load them, 300 for
// scale and maximum, 1,300 for the exponentials of two warps a scheduler, 150 to hand P over), of which the products are 512.  No pipe is full: the one of the
// exponentials and conversions is busy for 26 % of the time, the tensor cores for 23 %, an instruction is issued in 38 % of the cycles (of an SM that has a block;
// 20 of 148 have none), and conversions by integer arithmetic, which leave that pipe alone, measured the same.  Two tiles a block convert a page once for 256 rows.
// Three groups bring pages to two tiles, since sixteen warps are as many as leave a thread 128 registers.  Measured, four requests of up to 8,256 cells, 64
// drafted tokens, 32 heads on 8 of 128, e4m3: 50.4 us (one tile a block, two threads a row, columns scaled one by one: 75; four groups at 96 registers: 59); 27 drafted
// tokens of one request over 2,203 cells, bfloat16: 15.3.  Of those 50: 2 until the queries are in, 36 for 25 pages, 4 to join the ranges; the rest is blocks
// that start after others.  (A value that is not finite, in a page that not every row sees whole, takes its rows through the cells one by one: 420 us.)
// Two tiles a block from 129 rows on, and a block an SM, against one tile and two blocks (us, each at its best cut; 2,064 cells, eight requests): 256 rows e4m3 38 / 58,
// bfloat16 36 / 44, heads of 64 27 / 29; 132 rows e4m3 35 / 53, bfloat16 31 / 40; one request of 256 rows bfloat16 20 / 18; 512 rows, two of 8,256 cells: e4m3 61 / 89,
// bfloat16 51 / 67.
// That form is also the better one for a single tile where blocks have SMs to themselves (its second tile stays empty): 20 rows of one request e4m3 14.4 / 13.6 us, 108 of
// one of 32,027 cells 82 / 61, bfloat16 46 / 43; not where two would share an SM: 36 rows of 64 requests of 1,009 cells 98 / 118.  (Both sides of these e4m3 pairs without
// the sum's own maximum, which adds 0.5 us to two tiles' 50 and nothing to one tile's 97.)
// Waits on mbarriers are bounded (status 14).
#include "tree_common.cuh"

LGML_DEFINE_LAST_ERROR(lgml_attention_tree_tall)

namespace {
constexpr int ROWS = 128;
// With TILES tiles of 128 rows: the softmax threads of the tiles, the loaders, a warp a tile that issues its products.
template <int TILES, bool Q8> struct Roles {
    static constexpr int LOADERS = 64, GROUPS = Q8 && TILES == 2 ? 3 : 2;        // threads that bring a page's keys, or its values; groups of them
    static constexpr int BRING = ROWS * TILES, ISSUERS = BRING + LOADERS * GROUPS, THREADS = ISSUERS + 32 * TILES;       // first threads of the loaders, the issuers
    static constexpr int STAGES = TILES == 1 ? 2 : 4;        // pages of keys, and of values, in shared memory
};
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
__device__ __forceinline__ bool elect_one() {
    uint32_t ok;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(ok));
    return ok != 0;
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
__device__ __forceinline__ bool mbar_test(uint64_t *bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok) : "r"(smem_u32(bar)), "r"(parity) : "memory");
    return ok != 0;
}
__device__ __forceinline__ bool mbar_wait(uint64_t *bar, uint32_t parity, volatile int *abort_flag, int *status) {
    if (mbar_test(bar, parity)) return true;
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
__device__ __forceinline__ void tcgen05_ld_32(uint32_t taddr, uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]),
          "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]),
          "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
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

__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}

// Four numbers that block `rank` of the cluster has where this block has p.
__device__ __forceinline__ float4 load_there_16(const float *p, int rank) {
    uint32_t at;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_u32(p)), "r"(rank));
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(at));
    return v;
}

// A pair of numbers that are not finite becomes zeros, and `odd` says so.
__device__ __forceinline__ uint32_t finite_pair(uint32_t x, uint32_t inf, bool &odd) {
    const uint32_t lo = inf & 0xffffu, hi = inf & 0xffff0000u;
    if ((x & lo) == lo) x &= 0xffff0000u, odd = true;
    if ((x & hi) == hi) x &= 0xffffu, odd = true;
    return x;
}

template <int D, bool Q8, int TILES>
__global__ void __launch_bounds__(Roles<TILES, Q8>::THREADS, TILES == 1 ? 2 : 1) tree_attention_tall_kernel(
    const __nv_bfloat16 *__restrict__ q, int ldq, const int *__restrict__ positions, const int *__restrict__ seq_start, const int *__restrict__ seq_pos0,
    const long long *__restrict__ visible, const int *__restrict__ block_table, int max_blocks, const uint8_t *__restrict__ k_pages,
    const uint8_t *__restrict__ v_pages, const uint8_t *__restrict__ k_exps, const uint8_t *__restrict__ v_exps, int n_pages, __nv_bfloat16 *__restrict__ out,
    int ldo, float *__restrict__ part_o, float2 *__restrict__ part_ml, int n_splits, int clustered, int n_tokens, int H, int Hkv, int n_chunks, int least, int limit,
    float scale, int window, int *__restrict__ status) {
    constexpr int KB = D / 64;                        // 64-element blocks along the head
    constexpr float P_UP = Q8 ? 7.f : 0.f;            // probabilities times 2^this in the products: at most 2^15, float16 has numbers down to 2^-24
    using R = Roles<TILES, Q8>;
    constexpr int THREADS = R::THREADS, LOADERS = R::LOADERS, GROUPS = R::GROUPS, STAGES = R::STAGES, ALL_ROWS = TILES * ROWS;
    constexpr uint32_t Q_BYTES = KB * ROWS * 128, K_BYTES = KB * PAGE * 128;          // of a tile's queries, of a page's keys
    constexpr int SIZE = Q8 ? 1 : 2, PER_ROW = D * SIZE / 16, LOADS = PAGE * PER_ROW / LOADERS;       // 16-byte loads of a page's keys: a row's, a thread's
    constexpr int STEP = LOADERS / PER_ROW;           // rows from one load of a thread to its next (bfloat16)
    constexpr int STEP8 = LOADERS / 4, TURNS = PAGE / STEP8;      // ... and of codes, in which four threads load 64 bytes of a row; a thread's loads in 64 columns
    extern __shared__ uint8_t smem_raw[];
    uint8_t *base = (uint8_t *)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    uint8_t *Qs = base, *Ks = Qs + TILES * Q_BYTES, *Vs = Ks + STAGES * K_BYTES;
    constexpr int RING = 2 * STAGES;                      // pages whose columns are described (a page is described again when the softmax of RING pages before is done)
    __shared__ __align__(16) float kf_s[RING][PAGE], add_s[RING][PAGE];      // per column of page it (it % RING): its scores' factor, its value's power of two
    __shared__ __align__(8) float fin[ALL_ROWS][2];
    __shared__ int unscale_s[ALL_ROWS];                   // q was multiplied by 2 to the minus this
    __shared__ __align__(16) int4 page_s[RING];           // of page it: the powers of two its keys and its values were divided by, whether they are in column by
                                                          // column (and above), whether it is there
    __shared__ uint64_t k_full[STAGES], v_full[STAGES], k_free[STAGES], v_free[STAGES];        // by the page's stage (the free ones with two tiles)
    __shared__ uint64_t s_full[TILES][2], p_full[TILES][2], o_done[TILES][2];                  // by the tile and the page's parity
    __shared__ uint32_t tmem_base_s;
    __shared__ int abort_s, odd_s;
    volatile int *abort_flag = &abort_s;

    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int s = blockIdx.x / n_splits, split = blockIdx.x - s * n_splits, kvh = blockIdx.y / n_chunks, chunk = blockIdx.y - kvh * n_chunks;
    const int row0 = early_int(seq_start + s), n = early_int(seq_start + s + 1) - row0, pos0 = early_int(seq_pos0 + s);
    const int group = H / Hkv, n_rows = n * group, r0 = chunk * ALL_ROWS;
    // (The first block waits also where it leaves: a grid none of whose blocks waited could be over before the kernels ahead are, and the kernel behind waits for this
    // grid alone.  The others that leave make room at once; where they waited too, one request of 64 tokens beside 64 decoding ones took 20 us more.)
    const bool misplaced = row0 < 0 || row0 + n > n_tokens || pos0 < 0;
    if (n < least || n > limit || r0 >= n_rows || misplaced) {
        const bool report = misplaced && n >= least && n <= limit;
        if (report || (blockIdx.x == 0 && blockIdx.y == 0)) pdl_wait();
        if (report && tid == 0) atomicExch(status, 3);
        return;
    }
    // ---- this thread's row ----
    const int tile = TILES == 1 ? 0 : min(warp >> 2, TILES - 1), quarter = warp & 3;         // (tensor memory: a warp reads its quarter of the lanes)
    const int row = tile * ROWS + quarter * 32 + lane;
    const int n_tiles = min(TILES, (n_rows - r0 + ROWS - 1) / ROWS);              // that have rows
    const bool row_valid = r0 + row < n_rows;
    const int my_tok = min(r0 + row, n_rows - 1) / group;
    const int my_pos = early_int(positions + row0 + my_tok);
    const unsigned long long all_new = ~0ull >> (64 - n);
    unsigned long long my_mask = (visible ? (unsigned long long)__ldcg(visible + row0 + my_tok) : ~0ull >> (63 - my_tok)) & all_new;
    const int n_cells = pos0 + n;
    int low = 0, all_from = 0;              // none of the rows sees a cell below the first, every row sees the old cells from the second on
    if (window > 0) {
        const int t0 = r0 / group, t1 = (min(r0 + ALL_ROWS, n_rows) - 1) / group;
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
        for (int i = 0; i < STAGES; ++i) {
            mbar_init(&k_full[i], LOADERS / 32);
            mbar_init(&v_full[i], LOADERS / 32);
            mbar_init(&k_free[i], n_tiles);
            mbar_init(&v_free[i], n_tiles);
        }
        for (int i = 0; i < 2 * TILES; ++i) {
            mbar_init(&s_full[i >> 1][i & 1], 1);
            mbar_init(&p_full[i >> 1][i & 1], ROWS / 32);
            mbar_init(&o_done[i >> 1][i & 1], 1);
        }
        abort_s = odd_s = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncthreads();
    pdl_wait();
    if (tid < R::BRING) {
        if (warp == 0) tcgen05_alloc(&tmem_base_s, TILES * TMEM_COLS);
        // queries: row r = (token, head) r0 + r; through L2, they were just written; QN loads of a thread at a time
        constexpr int CH = D / 8, QN = 8;
        for (int c0 = tid; c0 < ALL_ROWS * CH; c0 += QN * R::BRING) {
            uint4 v[QN];
#pragma unroll
            for (int k = 0; k < QN; ++k) {
                const int c = c0 + k * R::BRING, r = c / CH, ch = c - r * CH, rr = r0 + r;
                v[k] = make_uint4(0, 0, 0, 0);
                if (rr < n_rows) v[k] = __ldcg(reinterpret_cast<const uint4 *>(q + (size_t)(row0 + rr / group) * ldq + (size_t)(kvh * group + rr % group) * D + ch * 8));
            }
#pragma unroll
            for (int k = 0; k < QN; ++k) {
                const int c = c0 + k * R::BRING, r = c / CH, ch = c - r * CH;
                if (Q8) {
                    uint32_t w[4] = {v[k].x, v[k].y, v[k].z, v[k].w};
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
                    v[k] = make_uint4(w[0], w[1], w[2], w[3]);
                    if (ch == 0) unscale_s[r] = -x;
                }
                *reinterpret_cast<uint4 *>(Qs + (r / ROWS) * Q_BYTES + (ch >> 3) * (ROWS * 128) + swz(r % ROWS, ch & 7)) = v[k];
            }
        }
        static_assert(ALL_ROWS * CH % (QN * R::BRING) == 0, "whole turns of the loop above");
        fence_async_smem();
    }
    if (tid < R::BRING || tid >= R::ISSUERS) {
        // the queries and tensor memory are there, for those that use them
        tcgen05_fence_before();
        asm volatile("bar.sync 1, %0;" ::"n"(R::BRING + R::THREADS - R::ISSUERS) : "memory");
        tcgen05_fence_after();
    }
    const uint32_t tmem_base = *reinterpret_cast<volatile uint32_t *>(&tmem_base_s), lane_addr = tmem_base + (uint32_t)tile * TMEM_COLS + ((uint32_t)(quarter * 32) << 16);
    const float scale_log2 = scale * 1.4426950408889634f;
    bool alive = true;

    // ---- the pages ----
    const int l = tid & (LOADERS - 1);
    auto page_of = [&](int it) {
        const int page = it < n_it && pb + it < max_blocks ? early_int(block_table + (size_t)s * max_blocks + pb + it) : -1;
        return page >= 0 && page < n_pages ? page : -1;
    };
    // bfloat16: load u of a thread is 16 bytes from chunk l % PER_ROW of row l / PER_ROW + STEP u on, which lie in a stage at:
    const int l_row = l / PER_ROW, l_chunk = l - l_row * PER_ROW;
    auto place = [&](int u) -> uint32_t { return (uint32_t)((l_chunk >> 3) * (PAGE * 128)) + swz(l_row + STEP * u, l_chunk & 7); };
    // e4m3: 16 codes, chunk l % 4 of 64 columns u / TURNS, of row l / 4 + STEP8 (u % TURNS); eight threads store to all banks.
    const uint32_t l_place = swz(l >> 2, 2 * (l & 3));
    auto fetch = [&](uint4 &raw, const uint8_t *src, int left, int u) {
        const int r = (l >> 2) + STEP8 * (u % TURNS);
        raw = r < left ? __ldcg(reinterpret_cast<const uint4 *>(src + (size_t)r * D + (u / TURNS) * 64) + (l & 3)) : make_uint4(0, 0, 0, 0);
    };
    auto codes_of = [&](const uint8_t *pages, int page) { return pages + ((size_t)max(page, 0) * Hkv + kvh) * PAGE * D; };
    auto cells_of = [&](int it, int page) { return page >= 0 && it < n_it ? n_cells - (pb + it) * PAGE : 0; };
    // ... as float16 in shared memory; in a page that not every row sees whole (check), without what is not finite.
    auto convert = [&](uint32_t dst, const uint4 (&raw)[LOADS], bool check, const uint32_t (&times)[TURNS]) {
        bool odd = false;
#pragma unroll
        for (int u = 0; u < LOADS; ++u) {
            const uint32_t w[4] = {raw[u].x, raw[u].y, raw[u].z, raw[u].w};
            uint32_t h[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const uint32_t two = half2_of_codes((unsigned short)(w[j >> 1] >> (16 * (j & 1))));
                const __half2 y = __hmul2(*reinterpret_cast<const __half2 *>(&two), *reinterpret_cast<const __half2 *>(&times[u % TURNS]));
                h[j] = *reinterpret_cast<const uint32_t *>(&y);
            }
            if (check) {
#pragma unroll
                for (int j = 0; j < 8; ++j) h[j] = finite_pair(h[j], 0x7c007c00u, odd);
            }
            const uint32_t to = dst + l_place + (uint32_t)((u / TURNS) * (PAGE * 128) + (u % TURNS) * STEP8 * 128);
            st_shared_16(to, h[0], h[1], h[2], h[3]);
            st_shared_16(to ^ 16u, h[4], h[5], h[6], h[7]);
        }
        if (odd) odd_s = 1;
    };
    // The powers of two of page it, four bytes of a lane: cells lane and lane + 32, keys and values.  (0: no such cell.)
    auto exponents = [&](int it, int page) -> uint32_t {
        if (!Q8) return 0;
        const int left = cells_of(it, page);
        const size_t vec = ((size_t)max(page, 0) * Hkv + kvh) * PAGE + lane;
        uint32_t e = 0;
        if (lane < left) e = max((uint32_t)__ldcg(k_exps + vec), 1u) | max((uint32_t)__ldcg(v_exps + vec), 1u) << 16;
        if (lane + 32 < left) e |= max((uint32_t)__ldcg(k_exps + vec + 32), 1u) << 8 | max((uint32_t)__ldcg(v_exps + vec + 32), 1u) << 24;
        return e;
    };
    // What becomes of them: a page's codes times 2^k are exact in float16 for k from -15 to 7.  So if its keys' powers of two are within 22 of their largest, and
    // its values' within 7, the largest is the page's, and a row is multiplied by 2^(7 - what it is below it).  If not, its codes are as they are, and the
    // softmax takes the powers column by column.  (7: a probability is as large as its value's power of two makes it, and float16 loses what is under 2^-32 of the
    // largest, so what is lost stays under 2^-25 of what counts most.)
    struct Powers {
        int largest, own[2];         // of the keys, or the values: their largest, this lane's cells'
        bool apart;
    };
    auto powers_of = [&](int it, int page, uint32_t e, bool keys) -> Powers {
        auto beyond = [&](int a, int b, int &largest, int reach) {
            largest = max(__reduce_max_sync(0xffffffffu, max(a, b)), 8);
            return largest - __reduce_min_sync(0xffffffffu, min(a ? a : 255, b ? b : 255)) > reach;
        };
        const int k0 = min(e & 255u, 246u), k1 = min((e >> 8) & 255u, 246u), v0 = min((e >> 16) & 255u, 246u), v1 = min(e >> 24, 246u);
        int k_largest, v_largest;
        const bool k_apart = beyond(k0, k1, k_largest, 22), v_apart = beyond(v0, v1, v_largest, 7), apart = k_apart || v_apart;
        if (keys) {
            if (l == 0) page_s[it % RING] = make_int4(k_largest - 127 - 7, v_largest - 127 - 7, apart, page >= 0);
            if (apart) {
                const int ke = (l < 32 ? k0 : k1) - 127, ve = (l < 32 ? v0 : v1) - 127;
                kf_s[it % RING][l] = scale_log2 * power_of_two(max(ke, -126));
                add_s[it % RING][l] = (float)ve;
            }
        }
        return keys ? Powers{k_largest, {k0, k1}, apart} : Powers{v_largest, {v0, v1}, apart};
    };
    // bfloat16: asynchronous copies
    auto copy_page = [&](uint32_t dst, const uint8_t *pages, int it, int page) {
        const int left = n_cells - (pb + it) * PAGE;
        const uint8_t *src = pages + ((size_t)max(page, 0) * Hkv + kvh) * PAGE * D * 2;
#pragma unroll
        for (int u = 0; u < LOADS; ++u) copy_16(dst + place(u), src + (size_t)(l + LOADERS * u) * 16, page >= 0 && l_row + STEP * u < left);
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
    // Output and sum are about maxima of their own where pages hold codes: m_ref is of scores and their values' powers together, m_sum of the scores alone.
    float m_ref = -INFINITY, m_sum = -INFINITY, l_run = 0.f, up = 1.f;
    if (tid >= R::BRING && tid < R::ISSUERS) {
        // ---- the keys and the values: a stage is free when the products of the page that was in it have read it ----
        // (page numbers come ahead and ask L2 for their pages, codes and exponents set out as what is before them goes in: each is a trip to L2 or beyond)
        const int group_of = (tid - R::BRING) / LOADERS;
        // (a warp waits, or gives up, as one)
        auto products_of = [&](bool keys, int it) {
            uint64_t *read = TILES == 1 ? (keys ? s_full[0] : o_done[0]) : keys ? k_free : v_free;
            return __all_sync(0xffffffffu, mbar_wait(&read[it % STAGES], (it / STAGES) & 1, abort_flag, status));
        };
        if (Q8) {
            // unit 2 i is page i's keys, 2 i + 1 its values: the groups take the units in turn
            uint4 raw[LOADS];
            auto pages_of = [&](int unit) { return unit & 1 ? v_pages : k_pages; };
            auto bring = [&](int unit, int page) {
#pragma unroll
                for (int u = 0; u < LOADS; ++u) fetch(raw[u], codes_of(pages_of(unit), page), cells_of(unit >> 1, page), u);
            };
            int page = page_of(group_of >> 1), next = page_of((group_of + GROUPS) >> 1);
            ask_l2(pages_of(group_of + GROUPS), next);
            uint32_t exps = exponents(group_of >> 1, page);
            bring(group_of, page);
            for (int unit = group_of; unit < 2 * n_it; unit += GROUPS) {
                const int it = unit >> 1, coming = page_of((unit + 2 * GROUPS) >> 1);
                const bool keys = !(unit & 1);
                if (it >= STAGES && !products_of(keys, it - STAGES)) break;
                if (keys && l == 0 && page < 0) atomicExch(status, 3);
                const Powers powers = powers_of(it, page, exps, keys);
                exps = exponents((unit + GROUPS) >> 1, next);
                uint32_t times[TURNS];
#pragma unroll
                for (int t = 0; t < TURNS; ++t) {
                    const int r = (l >> 2) + STEP8 * t, below = powers.largest - __shfl_sync(0xffffffffu, powers.own[STEP8 * t / 32], r & 31);
                    times[t] = powers.apart ? 0x3c003c00u : (below >= 22 ? 0x0200u : (uint32_t)(22 - below) << 10) * 0x10001u;
                }
                convert((keys ? ks0 : vs0) + (it % STAGES) * K_BYTES, raw, !keys && !whole(pb + it), times);
                fence_async_smem();
                warp_arrive(&(keys ? k_full : v_full)[it % STAGES]);
                bring(unit + GROUPS, next);
                page = next, next = coming;
                ask_l2(pages_of(unit + 2 * GROUPS), coming);
            }
        } else {
            const bool keys = group_of == 0;
            const uint8_t *pages = keys ? k_pages : v_pages;
            const uint32_t stages = keys ? ks0 : vs0;
            constexpr int LAG = STAGES / 2;          // a page is handed over when the copies of as many behind it have set out
            int next[4];                 // numbers of this page and the next
#pragma unroll
            for (int i = 0; i < 4; ++i) next[i] = page_of(i), ask_l2(pages, next[i]);
            for (int at = 0; at < n_it + LAG; ++at) {
                if (at < n_it) {
                    const int coming = page_of(at + 4);
                    if (at >= STAGES && !products_of(keys, at - STAGES)) break;
                    if (keys && l == 0) {
                        page_s[at % RING] = make_int4(0, 0, 0, next[0] >= 0);
                        if (next[0] < 0) atomicExch(status, 3);
                    }
                    copy_page(stages + (at % STAGES) * K_BYTES, pages, at, next[0]);
                    next[0] = next[1], next[1] = next[2], next[2] = next[3], next[3] = coming;
                    ask_l2(pages, coming);
                } else {
                    copies_commit();
                }
                const int it = at - LAG;
                if (it < 0) continue;
                copies_wait<LAG>();
                if (!keys && !whole(pb + it)) {
                    bool odd = false;
#pragma unroll
                    for (int u = 0; u < LOADS; ++u) {
                        const uint32_t where = vs0 + (it % STAGES) * K_BYTES + place(u);
                        const uint4 v = ld_shared_16(where);
                        st_shared_16(where, finite_pair(v.x, 0x7f807f80u, odd), finite_pair(v.y, 0x7f807f80u, odd), finite_pair(v.z, 0x7f807f80u, odd),
                                     finite_pair(v.w, 0x7f807f80u, odd));
                    }
                    if (odd) odd_s = 1;
                }
                fence_async_smem();
                warp_arrive(&(keys ? k_full : v_full)[it % STAGES]);
            }
        }
    } else if (tid >= R::ISSUERS && (tid - R::ISSUERS) / 32 < n_tiles) {
        // ---- the products of a tile: the warp goes through its pages as one, one thread issues (so that what an issue takes is the same in all threads) ----
        const int mine = __shfl_sync(0xffffffffu, (tid - R::ISSUERS) / 32, 0);
        const bool elected = elect_one();
        auto wait_for = [&](uint64_t *bar, uint32_t parity) { return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag, status)) != 0; };
        const uint32_t tile_base = tmem_base + (uint32_t)mine * TMEM_COLS;
        constexpr uint32_t idesc_qk = make_idesc(ROWS, PAGE, 0, Q8 ? 0 : 1), idesc_pv = make_idesc(ROWS, D, 1, Q8 ? 0 : 1);
        const uint64_t desc_q0 = make_desc(smem_u32(Qs + mine * Q_BYTES), 16, 1024), desc_k0 = make_desc(ks0, 16, 1024), desc_v0 = make_desc(vs0, PAGE * 128, 1024);
        auto issue_scores = [&](int it) {
            const uint64_t dk = desc_k0 + (uint64_t)(((it % STAGES) * K_BYTES) >> 4);
#pragma unroll
            for (int ks = 0; ks < D / 16; ++ks) {
                const uint64_t da = desc_q0 + (uint64_t)(((ks >> 2) * (ROWS * 128) + (ks & 3) * 32) >> 4);
                const uint64_t db = dk + (uint64_t)(((ks >> 2) * (PAGE * 128) + (ks & 3) * 32) >> 4);
                tcgen05_mma_f16(tile_base + (uint32_t)(it & 1) * S1_COL, da, db, idesc_qk, ks > 0 ? 1u : 0u);
            }
            tcgen05_commit(&s_full[mine][it & 1]);
            if (TILES > 1) tcgen05_commit(&k_free[it % STAGES]);
        };
        for (int it = 0; it < n_it && it < 2 && alive; ++it) {
            alive = wait_for(&k_full[it % STAGES], 0);
            tcgen05_fence_after();
            if (alive && elected) issue_scores(it);
            __syncwarp();
        }
        for (int it = 0; it < n_it && alive; ++it) {
            alive = wait_for(&v_full[it % STAGES], (it / STAGES) & 1) && wait_for(&p_full[mine][it & 1], (it >> 1) & 1);
            tcgen05_fence_after();
            if (!alive) break;
            const uint64_t dv = desc_v0 + (uint64_t)(((it % STAGES) * K_BYTES) >> 4);
            if (elected) {
#pragma unroll
                for (int k2 = 0; k2 < PAGE / 16; ++k2)
                    tcgen05_mma_f16_ts(tile_base + O_COL, tile_base + (uint32_t)(it & 1) * S1_COL + (uint32_t)k2 * 8u, dv + (uint64_t)((k2 * 2048) >> 4), idesc_pv,
                                       (it > 0 || k2 > 0) ? 1u : 0u);
                tcgen05_commit(&o_done[mine][it & 1]);
                if (TILES > 1) tcgen05_commit(&v_free[it % STAGES]);
            }
            __syncwarp();
            if (it + 2 < n_it) {
                alive = wait_for(&k_full[(it + 2) % STAGES], ((it + 2) / STAGES) & 1);
                tcgen05_fence_after();
                if (alive && elected) issue_scores(it + 2);
                __syncwarp();
            }
        }
    } else if (tid < R::BRING && tile < n_tiles) {
        // ---- softmax: a thread a row ----
        const int unscale = Q8 ? unscale_s[row] : 0;
        for (int it = 0; it < n_it; ++it) {
            const int pg = pb + it;
            const uint32_t s_addr = lane_addr + (uint32_t)(it & 1) * S1_COL;
            // (a warp gives up as one)
            alive = __all_sync(0xffffffffu, mbar_wait(&s_full[tile][it & 1], (it >> 1) & 1, abort_flag, status));
            if (!alive) break;
            tcgen05_fence_after();
            const int4 page = page_s[it % RING];
            const bool there = page.w != 0, edge = !whole(pg) || !there;
            union {
                uint32_t u[PAGE];
                float2 f[PAGE / 2];
            } r;
            tcgen05_ld_32(s_addr, *reinterpret_cast<uint32_t(*)[32]>(&r.u[0]));
            tcgen05_ld_32(s_addr + 32u, *reinterpret_cast<uint32_t(*)[32]>(&r.u[32]));
            tcgen05_wait_ld();
            // a score (in powers of two, of what the values are multiplied by too) is r times + plus
            float times = scale_log2, plus = 0.f;
            if (Q8) {
                if (page.z) {
                    // (rare) column by column
                    const float f = power_of_two(unscale);
#pragma unroll
                    for (int c = 0; c < PAGE; c += 4) {
                        const float4 kf = *reinterpret_cast<const float4 *>(&kf_s[it % RING][c]), ad = *reinterpret_cast<const float4 *>(&add_s[it % RING][c]);
                        r.f[c / 2] = fma2(mul2(r.f[c / 2], make_float2(f, f)), make_float2(kf.x, kf.y), make_float2(ad.x, ad.y));
                        r.f[c / 2 + 1] = fma2(mul2(r.f[c / 2 + 1], make_float2(f, f)), make_float2(kf.z, kf.w), make_float2(ad.z, ad.w));
                    }
                    times = 1.f;
                } else {
                    times = scale_log2 * power_of_two(min(max(page.x + unscale, -120), 120));
                    plus = (float)page.y;
                }
            }
            if (edge) {
                const unsigned long long seen = there ? seen_of(pg) : 0ull;
                const uint32_t v[2] = {(uint32_t)seen, (uint32_t)(seen >> 32)};
#pragma unroll
                for (int c = 0; c < PAGE; ++c)
                    if (!((v[c >> 5] >> (c & 31)) & 1u)) r.u[c] = __float_as_uint(-INFINITY);
            }
            float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
            for (int c = 0; c < PAGE; c += 2) mx4[(c >> 1) & 3] = max3(mx4[(c >> 1) & 3], __uint_as_float(r.u[c]), __uint_as_float(r.u[c + 1]));
            const float largest = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3])), m_new = fmaf(largest, times, plus);
            float corr = 1.f;
            if (m_ref == -INFINITY) {
                m_ref = m_new;                       // nothing summed yet: nothing to correct
            } else if (m_new > m_ref + RESCALE_STEP) {
                corr = ex2(m_ref - m_new);
                m_ref = m_new;
                if (!Q8) l_run *= corr;
            }
            if (__any_sync(0xffffffffu, corr != 1.f)) {
                // ---- correct the running output (rare): the product of the page before must be done, this page's has to wait for P ----
                // (a correction implies an earlier page)
                alive = __all_sync(0xffffffffu, mbar_wait(&o_done[tile][(it - 1) & 1], ((it - 1) >> 1) & 1, abort_flag, status));
                if (!alive) break;
                tcgen05_fence_after();
                for (int c0 = 0; c0 < D; c0 += 16) {
                    uint32_t o[16];
                    tcgen05_ld_16(lane_addr + O_COL + (uint32_t)c0, o);
                    tcgen05_wait_ld();
#pragma unroll
                    for (int j = 0; j < 16; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * corr);
                    tcgen05_st_16(lane_addr + O_COL + (uint32_t)c0, o);
                }
            }
            // The sum.  The probabilities below come with their values' powers of two; one factor takes those out again, unless they differ by column, or leave too
            // little of them: then (rare) the weights are formed on their own, from the scores as they still are in tensor memory.
            float out_of = 1.f;
            bool apart = false;
            if (Q8) {
                auto raise = [&](float s_new) {
                    if (m_sum == -INFINITY) {
                        m_sum = s_new;
                    } else if (s_new > m_sum + RESCALE_STEP) {
                        l_run *= ex2(m_sum - s_new);
                        m_sum = s_new;
                    }
                };
                const bool little = m_new < m_ref - 60.f;
                apart = page.z || (little && m_new > -INFINITY);
                if (__any_sync(0xffffffffu, apart)) {
                    const unsigned long long seen = edge ? (there ? seen_of(pg) : 0ull) : ~0ull;
                    const float f = page.z ? power_of_two(unscale) : times;
#pragma unroll 1
                    for (int c0 = 0; c0 < PAGE; c0 += 16) {
                        uint32_t x[16];
                        tcgen05_ld_16(s_addr + (uint32_t)c0, x);
                        tcgen05_wait_ld();
                        float most = -INFINITY, part = 0.f;
#pragma unroll
                        for (int j = 0; j < 16; ++j) {
                            const float y = (seen >> (c0 + j)) & 1 ? __uint_as_float(x[j]) * f * (page.z ? kf_s[it % RING][c0 + j] : 1.f) : -INFINITY;
                            x[j] = __float_as_uint(y);
                            most = fmaxf(most, y);
                        }
                        if (apart) raise(most);
                        const float ref = m_sum == -INFINITY ? 0.f : m_sum;
#pragma unroll
                        for (int j = 0; j < 16; ++j) part += ex2(__uint_as_float(x[j]) - ref);
                        if (apart) l_run += part;
                    }
                }
                if (!apart) {
                    raise(largest * times);
                    // (little of nothing seen: 0, whatever the factor)
                    if (!little) out_of = ex2((m_ref == -INFINITY ? 0.f : m_ref) - plus - P_UP - (m_sum == -INFINITY ? 0.f : m_sum));
                }
            }
            const float less = (m_ref == -INFINITY ? plus : plus - m_ref) + P_UP;
            float2 sum2[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
            // P over the scores, which this row's thread alone reads
#pragma unroll
            for (int c0 = 0; c0 < PAGE / 2; c0 += 16) {
                uint32_t packed[16];
#pragma unroll
                for (int c = c0; c < c0 + 16; ++c) {
                    const float2 x = fma2(r.f[c], make_float2(times, times), make_float2(less, less)), e = make_float2(ex2(x.x), ex2(x.y));
                    sum2[c & 1] = add2(sum2[c & 1], e);
                    if (Q8) {
                        const __half2 h2 = __floats2half2_rn(e.x, e.y);
                        packed[c - c0] = *reinterpret_cast<const uint32_t *>(&h2);
                    } else {
                        const __nv_bfloat162 h2 = __floats2bfloat162_rn(e.x, e.y);
                        packed[c - c0] = *reinterpret_cast<const uint32_t *>(&h2);
                    }
                }
                tcgen05_st_16(s_addr + (uint32_t)c0, packed);
            }
            const float sum = (sum2[0].x + sum2[0].y) + (sum2[1].x + sum2[1].y);
            if (!apart) l_run += Q8 ? sum * out_of : sum;
            tcgen05_wait_st();
            tcgen05_fence_before();
            warp_arrive(&p_full[tile][it & 1]);
        }
        // (the last scores were seen, and were issued behind the product two pages before: the barrier is at most a phase away)
        if (n_it > 0 && alive && !mbar_wait(&o_done[tile][(n_it - 1) & 1], ((n_it - 1) >> 1) & 1, abort_flag, status)) alive = false;
        if (Q8) {
            // (both times 2^-24, so that sums of the largest values stay finite)
            if (m_sum != -INFINITY) up = ex2(m_ref - m_sum - P_UP - 24.f);
            m_ref = m_sum;
            l_run *= 5.9604644775390625e-8f;
        }
        fin[row][0] = m_ref;
        fin[row][1] = l_run;
    }
    copies_wait<0>();
    __syncthreads();
    tcgen05_fence_after();
    alive = abort_s == 0;

    // ---- the result ----
    constexpr int LDM = D + 4;
    float *merge = reinterpret_cast<float *>(base);          // [ALL_ROWS][LDM], where the operands were; behind it the ranges' shares
    if (tid < R::BRING && tile < n_tiles) {
        const float M = m_ref, sum = l_run;
        __nv_bfloat16 *dst = row_at(out, ldo, row0, min(r0 + row, n_rows - 1), group, kvh, D, 0);
        const size_t part = ((size_t)(row0 + my_tok) * H + kvh * group + min(r0 + row, n_rows - 1) % group) * n_splits + split;
        const bool odd = odd_s != 0;
#pragma unroll
        for (int c0 = 0; c0 < D; c0 += 16) {
            uint32_t r[16];
            if (n_it > 0) {
                tcgen05_ld_16(lane_addr + O_COL + (uint32_t)c0, r);
                tcgen05_wait_ld();
                if (Q8)
#pragma unroll
                    for (int j = 0; j < 16; ++j) r[j] = __float_as_uint(__uint_as_float(r[j]) * up);
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
                        const uint8_t *p = v_pages + ((((size_t)page * Hkv + kvh) * PAGE + c) * D + c0) * SIZE;
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
                    *reinterpret_cast<uint4 *>(dst + c0) = make_uint4(h[0], h[1], h[2], h[3]);
                    *reinterpret_cast<uint4 *>(dst + c0 + 8) = make_uint4(h[4], h[5], h[6], h[7]);
                }
            } else if (clustered) {
#pragma unroll
                for (int j = 0; j < 16; j += 4) *reinterpret_cast<uint4 *>(merge + (size_t)row * LDM + c0 + j) = make_uint4(r[j], r[j + 1], r[j + 2], r[j + 3]);
            } else if (row_valid) {
#pragma unroll
                for (int j = 0; j < 16; j += 2)
                    *reinterpret_cast<float2 *>(part_o + part * D + c0 + j) = make_float2(__uint_as_float(r[j]), __uint_as_float(r[j + 1]));
                if (c0 == 0) part_ml[part] = make_float2(M, sum);
            }
        }
    }
    tcgen05_fence_before();
    pdl_trigger();      // at the end: a block that takes half an SM keeps the next kernel back until it is done
    __syncthreads();
    if (warp == 0) {
        tcgen05_fence_after();
        tcgen05_dealloc(tmem_base, TILES * TMEM_COLS);
    }
    if (!clustered) return;
    __syncwarp();
    cluster_sync();
    {
        // The cluster's blocks share out the rows; a thread has four columns of a row.  First the shares of a row's ranges in its result, a thread a row.
        const int rows = min(n_rows - r0, ALL_ROWS), per_block = (rows + n_splits - 1) / n_splits, from = (int)block_of_cluster() * per_block;
        const int mine = max(min(per_block, rows - from), 0);
        float *shares = merge + (size_t)ALL_ROWS * LDM;      // [ALL_ROWS][MAX_CLUSTER]
        for (int i = tid; i < mine; i += THREADS) {
            float2 ml[MAX_CLUSTER];
#pragma unroll
            for (int j = 0; j < MAX_CLUSTER; ++j) ml[j] = j < n_splits ? load_there(fin[from + i], j) : make_float2(-INFINITY, 0.f);
            float M = -INFINITY, sum = 0.f;
#pragma unroll
            for (int j = 0; j < MAX_CLUSTER; ++j) M = fmaxf(M, ml[j].x);
#pragma unroll
            for (int j = 0; j < MAX_CLUSTER; ++j) ml[j].x = j < n_splits ? share_of(ml[j].x, M) : 0.f, sum += ml[j].y * ml[j].x;
            const float inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
            for (int j = 0; j < MAX_CLUSTER; ++j) shares[i * MAX_CLUSTER + j] = ml[j].x * inv;
        }
        __syncthreads();
        constexpr int QUADS = D / 4;
        for (int i = tid; i < mine * QUADS; i += THREADS) {
            const int r = i / QUADS, d = 4 * (i - r * QUADS);
            float4 part[MAX_CLUSTER];
#pragma unroll
            for (int j = 0; j < MAX_CLUSTER; ++j)
                if (j < n_splits) part[j] = load_there_16(merge + (size_t)(from + r) * LDM + d, j);
            float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int j = 0; j < MAX_CLUSTER; ++j)
                if (j < n_splits) {
                    const float f = shares[r * MAX_CLUSTER + j];
                    o.x += part[j].x * f, o.y += part[j].y * f, o.z += part[j].z * f, o.w += part[j].w * f;
                }
            const __nv_bfloat162 lo = __floats2bfloat162_rn(o.x, o.y), hi = __floats2bfloat162_rn(o.z, o.w);
            *reinterpret_cast<uint2 *>(row_at(out, ldo, row0, r0 + from + r, group, kvh, D, d)) =
                make_uint2(*reinterpret_cast<const uint32_t *>(&lo), *reinterpret_cast<const uint32_t *>(&hi));
        }
    }
    __syncwarp();
    cluster_sync();                         // (the others' shared memory is read until here)
}

template <int D, bool Q8, int TILES, typename... Args>
int launch(dim3 grid, int cluster, cudaStream_t stream, Args... args) {
    constexpr size_t operands = (size_t)(D / 64) * (TILES * ROWS + 2 * Roles<TILES, Q8>::STAGES * PAGE) * 128, merge = sizeof(float) * TILES * ROWS * (D + 4 + MAX_CLUSTER);
    constexpr size_t smem = (operands > merge ? operands : merge) + 1024;
    cudaError_t e = cudaFuncSetAttribute(tree_attention_tall_kernel<D, Q8, TILES>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) LGML_FAIL("tree_attention: cannot have %zu bytes of shared memory: %s", smem, cudaGetErrorString(e));
    lgml_launch_cluster(tree_attention_tall_kernel<D, Q8, TILES>, grid, Roles<TILES, Q8>::THREADS, smem, stream, cluster, args...);
    return lgml_launch_status("tree_attention");
}
template <int TILES, typename... Args>
int launch_tiles(int D, bool q8, Args... args) {
    if (D == 64) return q8 ? launch<64, true, TILES>(args...) : launch<64, false, TILES>(args...);
    return q8 ? launch<128, true, TILES>(args...) : launch<128, false, TILES>(args...);
}
}  // namespace

// As lgml_tree_attention, for head sizes of 64 and 128 and rows of q and out on 16 bytes.
LGML_API int lgml_tree_attention_tall(const void *q, int ldq, const int *positions, const int *seq_start, const int *seq_pos0, const long long *visible,
                                      const int *block_table, int n_seqs, int max_blocks, const void *k_pages, const void *v_pages, const void *k_exps,
                                      const void *v_exps, int n_pages, int page_size, void *out, int ldo, float *scratch, int n_splits, int n_tokens, int least, int limit,
                                      int H, int Hkv, int D, float scale, int window, int *status, cudaStream_t stream) {
    LGML_REQUIRE(n_tokens >= 0 && n_seqs >= 0 && H > 0 && Hkv > 0 && max_blocks > 0 && n_pages >= 0, "tree_attention: bad sizes");
    LGML_REQUIRE(page_size == PAGE, "tree_attention: pages of %d tokens, this kernel takes %d", page_size, PAGE);
    LGML_REQUIRE(H % Hkv == 0, "tree_attention: %d heads are no multiple of %d KV heads", H, Hkv);
    LGML_REQUIRE(D == 64 || D == 128, "tree_attention: head_dim %d must be 64 or 128 here", D);
    LGML_REQUIRE(least >= 1 && least <= limit && limit <= MAX_NEW, "tree_attention: %d to %d new tokens a request (1 to %d)", least, limit, MAX_NEW);
    LGML_REQUIRE(n_splits >= 1 && n_splits <= MAX_SPLITS, "tree_attention: %d key ranges (1 to %d)", n_splits, MAX_SPLITS);
    LGML_REQUIRE(n_splits <= MAX_CLUSTER || (scratch != nullptr && ((uintptr_t)scratch & 7) == 0), "tree_attention: several ranges need scratch memory");
    LGML_REQUIRE((k_exps == nullptr) == (v_exps == nullptr), "tree_attention: exponents for keys and values, or for neither");
    LGML_REQUIRE((((uintptr_t)k_pages | (uintptr_t)v_pages) & 15) == 0, "tree_attention: the cache must be 16-byte aligned");
    LGML_REQUIRE(ldq % 8 == 0 && ldo % 8 == 0 && (((uintptr_t)q | (uintptr_t)out) & 15) == 0, "tree_attention: q and out must be 16-byte aligned here");
    LGML_REQUIRE((long long)n_seqs * (limit > n_splits ? limit : n_splits) <= 0x7fffffffLL, "tree_attention: too many requests");
    if (n_tokens == 0 || n_seqs == 0) return 0;
    static const int n_sms = [] {
        int dev = 0, n = 0;
        cudaGetDevice(&dev);
        cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
        return n;
    }();
    // one block an SM, two tiles, deeper rings and more loaders: for more rows than a tile has, and where a block has an SM to itself anyway
    const int rows = limit * (H / Hkv), tiles = rows > ROWS || (long long)n_seqs * n_splits * Hkv <= n_sms ? 2 : 1;
    const int n_chunks = (rows + tiles * ROWS - 1) / (tiles * ROWS);
    LGML_REQUIRE((long long)Hkv * n_chunks <= 65535, "tree_attention: too many heads");
    const int clustered = n_splits > 1 && n_splits <= MAX_CLUSTER;
    dim3 grid(n_seqs * n_splits, Hkv * n_chunks);
    float *part_o = scratch;
    float2 *part_ml = scratch ? reinterpret_cast<float2 *>(scratch + (size_t)n_tokens * H * n_splits * D) : nullptr;
#define LGML_ARGS D, k_exps != nullptr, grid, clustered ? n_splits : 1, stream, (const __nv_bfloat16 *)q, ldq, positions, seq_start, seq_pos0, visible, block_table, \
                  max_blocks, (const uint8_t *)k_pages, (const uint8_t *)v_pages, (const uint8_t *)k_exps, (const uint8_t *)v_exps, n_pages,                     \
                  (__nv_bfloat16 *)out, ldo, part_o, part_ml, n_splits, clustered, n_tokens, H, Hkv, n_chunks, least, limit, scale, window, status
    const int rc = tiles == 2 ? launch_tiles<2>(LGML_ARGS) : launch_tiles<1>(LGML_ARGS);
#undef LGML_ARGS
    if (rc || n_splits <= MAX_CLUSTER) return rc;
    return tree_join(part_o, part_ml, seq_start, n_seqs, least, limit, n_tokens, out, ldo, n_splits, H, D, stream);
}
