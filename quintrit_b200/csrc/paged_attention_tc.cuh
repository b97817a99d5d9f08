// Attention of many new tokens over a paged cache on the 5th-generation tensor cores (the mathematics: paged_attention.cuh).
//
// A block of threads takes one KV head of one sequence, 256 rows of queries (128 where a head has 256 values, or where there are no more; a row is a (token, head of the group)) and a
// range of positions, in tiles of 128 positions (64 where a head has 256 values). Units of work, a row tile and a tile of positions, take two score buffers in tensor memory in turn. For a unit one thread issues S = Q K^T (tcgen05.mma, operands in shared memory; Q of a single row tile in tensor memory), a warpgroup
// with a row per thread (two warpgroups where there is one row tile: two threads per row, half of the positions each, which speak to each other when a maximum grew) turns S into
// weights (maximum, exponentials, sum) and writes them as 16-bit values over S, and O += P V takes them from
// there. The tensor cores work on the other buffer meanwhile: the score products that take a buffer next follow the value products that took its weights. O stays in tensor memory and is rescaled, by its
// warpgroups, only when a row's maximum grew by more than 2^8.
//
// F16 / BF16: one warp brings the pages' rows by bulk copies straight into the operands' places, since they lie in the cache in the 128-byte swizzle already (keys as a K-major,
// values as an MN-major operand). Q8: it brings codes and scales to a ring of their own, and four or eight warps widen the codes to F16 operands and prepare the scales.
//
// Bound by the tensor cores (4 head_dim flops per row and position) and, for heads of up to 128 values, as much by the exponentials: 16 a clock and
// multiprocessor, so that 128 x 128 scores take 1024 cycles, and the two products 8 head_dim. (Tiles of 64
// positions and four buffers kept the threads busier and the tensor cores less: an instruction over 64 positions took 87 cycles, one over 128 took 100. 64-value heads apart, 2048 tokens behind 14336:
// 461 us against 318 us.)
//
// Measured: 296 query heads of 128 over 37 KV heads, 256 tokens behind 16384, whole waves: F16 1141 TFLOP/s (70% of the library's matrix product), Q8 851; 2048 tokens of 20 heads of 128 behind
// 14336: F16 314 us, 1027 TFLOP/s, Q8 398 us, 809; 12 heads of 256: F16 382 us, 1013. With one score buffer to a row tile its products and its exponentials, 3200 cycles
// a tile with Q8's scales, follow one another (two threads to a row there too, of 96 registers each: Q8 528 us, F16 342).
#pragma once
#include "packed_f32.cuh"
#include "paged_attention.cuh"

namespace qtb {

// Which rows and ranges the blocks of a launch take. Where all sequences have as many new tokens, row blocks count from the last one of a sequence, which sees most (order 0, 1, ...), and m = KV heads x
// sequences have each order. Where they differ (a prompt among sequences that answer), the row blocks that are there count through the sequences, each from its last one, and m = KV heads have each
// (orders and sequences would be mostly blocks without rows: with 257 tokens next to seven single ones 1152 blocks were launched for 144 with work, 35 us instead of 27, and 21 instead of 7 to join them). One block of threads
// per multiprocessor, so that what matters is the last of them to end: as long as row blocks fill whole waves they are taken whole; the rest, or all where there are too few,
// are cut into ranges of equal length, whose results meet in the workspace.
constexpr int kPagedMapped = 160;  // most (row block, range) pairs of a mapped schedule
struct PagedSchedule {
    int m, whole, cut;                       // blocks x m: order x < whole, all of its range; else order whole + (x - whole) / cut, range (x - whole) % cut of cut
    int even;                                // all sequences have as many new tokens
    int orders;                              // row blocks that there are at most (times m)
    int mapped;                              // few row blocks, of different lengths: order[x], range[x] of ranges[x] instead
    unsigned char order[kPagedMapped], range[kPagedMapped], ranges[kPagedMapped], at[kPagedMapped];  // at: the first x of an order
    float* part_o;                           // [x - whole][m][rows of a block][head_dim] for what is cut; mapped: [range][KV head][packed tokens x group][head_dim]
    float2* part_ml;
};
struct PagedPart {
    int order, range, ranges, slot;  // slot: of the workspace
};
__device__ __forceinline__ PagedPart paged_part(const PagedSchedule& g, int x) {
    if (g.mapped) return PagedPart{g.order[x], g.range[x], g.ranges[x], x};
    if (x < g.whole) return PagedPart{x, 0, 1, 0};
    return PagedPart{g.whole + (x - g.whole) / g.cut, (x - g.whole) % g.cut, g.cut, x - g.whole};
}
// The row blocks of sequence s that this launch serves.
__device__ __forceinline__ int paged_row_blocks(const PagedAttnArgs& a, int s, int rows) {
    const PagedSequence q = paged_sequence(a.c, a.r, s);
    if (q.news > a.r.most) atomicOr(a.c.status, kPagedBadPosition);
    return q.ok && q.news >= a.few && q.news <= a.many ? (q.news * a.group + rows - 1) / rows : 0;
}
// The sequence that has the x-th row block of all, and which of its own it is, or the sequence -1; by all lanes of a warp. And the row blocks of the sequences before s.
__device__ __forceinline__ int2 paged_row_block(const PagedAttnArgs& a, int x, int rows) {
    const int lane = threadIdx.x & 31;
    long long sum = 0;
    for (int s0 = 0; s0 < a.r.sequences; s0 += 32) {
        const int mine = s0 + lane < a.r.sequences ? paged_row_blocks(a, s0 + lane, rows) : 0;
        const long long until = sum + paged_detail::prefix(mine);
        const unsigned int there = __ballot_sync(0xffffffffu, until > x);
        if (there) {
            const int first = __ffs(there) - 1;
            return make_int2(s0 + first, static_cast<int>(x - __shfl_sync(0xffffffffu, until - mine, first)));
        }
        sum = __shfl_sync(0xffffffffu, until, 31);
    }
    return make_int2(-1, 0);
}
__device__ __forceinline__ long long paged_row_blocks_before(const PagedAttnArgs& a, int s, int rows) {
    const int lane = threadIdx.x & 31;
    long long sum = 0;
    for (int s0 = 0; s0 < s; s0 += 32) sum += __shfl_sync(0xffffffffu, paged_detail::prefix(s0 + lane < s ? paged_row_blocks(a, s0 + lane, rows) : 0), 31);
    return sum;
}
// The row of the workspace that has the result of row r (`local` of its block) for a part.
__device__ __forceinline__ size_t paged_part_row(const PagedAttnArgs& a, const PagedSchedule& g, const PagedSequence& q, const PagedPart& part, int which, int kvh, int r, int local, int rows) {
    if (g.mapped) return (static_cast<size_t>(part.range) * a.c.kv_heads + kvh) * (static_cast<size_t>(a.r.tokens) * a.group) + static_cast<size_t>(q.first) * a.group + r;
    return (static_cast<size_t>(part.slot) * g.m + which) * rows + local;
}
// Range `part` of `parts` of what rows of tokens [t0, t1) see; begin is a multiple of 64.
__device__ __forceinline__ PagedRange paged_part_range(const PagedAttnArgs& a, const PagedSequence& q, int t0, int t1, int part, int parts, int tile) {
    const int p0 = q.length - q.news, low = paged_first_seen(a, q, t0) & ~(kPagedTile - 1), high = max(low, max(0, p0 + t1));
    const int tiles = (high - low + tile - 1) / tile, per = (tiles + parts - 1) / parts;
    return PagedRange{min(high, low + part * per * tile), min(high, low + (part + 1) * per * tile)};
}

template <int TYPE, int BLOCKS, int NT>  // NT: row tiles of a block, 1 or 2 (1 where a head has 256 values)
struct PagedMany {
    static constexpr bool Q8 = TYPE == kPagedQ8, BF = TYPE == kPagedBf16;
    static constexpr int HD = BLOCKS * kPagedBlock;
    static constexpr int KT = BLOCKS == 4 ? 64 : 128, NB = 2;                  // positions of a tile; score buffers
    static constexpr int kRows = 128 * NT;
    static constexpr int kSlot = KT * HD * 2, kSlots = Q8 ? 3 : 4;             // operand tiles: keys and values in turn
    static constexpr int kRaw = KT * HD, kRaws = Q8 ? (NT == 1 ? 4 : 3) : 0;                   // Q8: the codes; those of keys with the scales of keys and values
    static constexpr int kRawStride = Q8 ? kRaw + KT * 8 : 0;
    static constexpr int kFactors = Q8 ? 4 : 0;                                // sets of KT x (key scale, log2 of the value scale, its reciprocal)
    static constexpr bool kQTmem = NT == 1;
    // A warp's rows go through 32 rows of 144 bytes, so that they are read and written in whole pieces: queries on their way to tensor memory, results on their way out (over the queries in shared
    // memory, which nothing reads any more by then).
    static constexpr int kStagePitch = 144, kStageBytes = 4 * NT * (NT == 1 ? 2 : 1) * 32 * kStagePitch, kStageOwn = kQTmem ? kStageBytes : 0;
    static constexpr int kQBytes = kQTmem ? 0 : NT * 128 * HD * 2 > kStageBytes ? NT * 128 * HD * 2 : (kStageBytes + 1023) / 1024 * 1024;
    static constexpr int SIDES = NT == 1 ? 2 : 1;                              // threads of a row
    static constexpr int kWidenWarps = Q8 ? 8 / NT : 0;
    static constexpr int kSoftWarps = 4 * NT * SIDES, kLoadWarp = kSoftWarps, kMmaWarp = kSoftWarps + 1, kWidenWarp = kSoftWarps + 4;
    static constexpr int kThreads = (kSoftWarps + 4 + kWidenWarps) * 32;
    // registers: 384 threads are launched with 168 each, 512 with 128; the warpgroups with the scores of two row tiles take some of the others'
    static constexpr bool kSplitRegs = NT == 2;
    static constexpr int kLaunchRegs = Q8 ? 128 : 168, kSoftRegs = Q8 ? 200 : 216, kRestRegs = Q8 ? 56 : 72;
    static_assert(!kSplitRegs || kSoftWarps * 32 * kSoftRegs + (kThreads - kSoftWarps * 32) * kRestRegs <= kThreads * kLaunchRegs, "more registers than the block was launched with");
    static constexpr int kBars = 2 * kSlots + 2 * kRaws + 3 * NB + 3;
    static constexpr int kNeed = 1024 + kQBytes + kSlots * kSlot + kRaws * kRawStride + kFactors * KT * 12 + (SIDES == 2 ? 2048 : 0) + NT * 512 + kStageOwn + kBars * 8 + 16;
    static constexpr int kSmem = kNeed > 116 * 1024 ? kNeed : 116 * 1024;  // one block per multiprocessor: it takes all of its tensor memory
    static constexpr int kOCol = 0, kSCol = 256, kQCol = BLOCKS == 4 ? 384 : 128;  // tensor memory columns: O (of row tile i at 128 i), S (buffer b at KT b behind), Q
};

namespace paged_detail {

__device__ __forceinline__ void tmem_load32(uint32_t addr, uint32_t (&v)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, "
        "%29, %30, %31}, [%32];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]),
          "=r"(v[14]), "=r"(v[15]), "=r"(v[16]), "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]), "=r"(v[25]), "=r"(v[26]),
          "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
        : "r"(addr));
}
__device__ __forceinline__ void tmem_store16(uint32_t addr, const uint32_t (&v)[16]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(addr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]),
                 "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
                 : "memory");
}
__device__ __forceinline__ void tmem_wait_load() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_store() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
// kind::f16: F32 accumulator (1 at bit 4), A and B F16 or BF16 (1 at bits 7 and 10), B transposed (MN-major) at bit 16, N / 8 at bit 17, M / 16 at bit 24.
__host__ __device__ constexpr uint32_t instr_desc_16(bool bf16, bool b_mn, int n) {
    return (1u << 4) | (bf16 ? (1u << 7) | (1u << 10) : 0u) | (b_mn ? 1u << 16 : 0u) | (uint32_t(n >> 3) << 17) | (uint32_t(128 >> 4) << 24);
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
        "r"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
}
template <int N> __device__ __forceinline__ void registers_up() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N> __device__ __forceinline__ void registers_down() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }

}  // namespace paged_detail

template <int TYPE, int BLOCKS, int NT, bool FAR>  // FAR: the cap is far above the scores
__global__ void __launch_bounds__(PagedMany<TYPE, BLOCKS, NT>::kThreads, 1) paged_many_kernel(const __grid_constant__ PagedAttnArgs a, const __grid_constant__ PagedSchedule g) {
    using namespace gemm_detail;
    using namespace paged_detail;
    using M = PagedMany<TYPE, BLOCKS, NT>;
    constexpr bool Q8 = M::Q8;
    constexpr int HD = M::HD, NB = M::NB, SIDES = M::SIDES, KT = M::KT, RS = M::kSlots, RW = Q8 ? M::kRaws : 1, kRow = paged_row_bytes(TYPE);
    extern __shared__ unsigned char many_smem_raw[];
    const uint32_t base = (smem_u32(many_smem_raw) + 1023u) & ~1023u;
    unsigned char* smem = many_smem_raw + (base - smem_u32(many_smem_raw));
    const uint32_t q_at = base, slots = base + M::kQBytes, raws = slots + RS * M::kSlot;
    unsigned char* raw_smem = smem + M::kQBytes + RS * M::kSlot;
    float* factors = reinterpret_cast<float*>(raw_smem + M::kRaws * M::kRawStride);  // [kFactors][3][KT]
    float2* exchange = reinterpret_cast<float2*>(factors + M::kFactors * 3 * KT);  // [2][128]: between the two threads of a row
    float* row_factor = reinterpret_cast<float*>(exchange + (SIDES == 2 ? 256 : 0));  // [NT * 128]
    unsigned char* staging = M::kQTmem ? reinterpret_cast<unsigned char*>(row_factor + NT * 128) : smem;
    uint64_t* bars = reinterpret_cast<uint64_t*>(reinterpret_cast<unsigned char*>(row_factor + NT * 128) + M::kStageOwn);
    const uint32_t bar0 = smem_u32(bars);
    auto full = [&](int s) { return bar0 + 8u * s; };                       // an operand tile is there
    auto empty = [&](int s) { return bar0 + 8u * (RS + s); };               // the products that read it are done
    auto raw_full = [&](int s) { return bar0 + 8u * (2 * RS + s); };
    auto raw_empty = [&](int s) { return bar0 + 8u * (2 * RS + M::kRaws + s); };
    const uint32_t tail = bar0 + 8u * (2 * RS + 2 * M::kRaws);
    auto s_full = [&](int b) { return tail + 8u * b; };                     // scores of a buffer
    auto p_full = [&](int b) { return tail + 8u * (NB + b); };               // weights of a buffer
    auto o_done = [&](int b) { return tail + 8u * (2 * NB + b); };               // the value products of a buffer's weights
    const uint32_t q_full = tail + 8u * (3 * NB), drained = q_full + 8u, pages_known = drained + 8u;  // the last: every page number was looked at
    volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(bars + M::kBars);
    volatile unsigned int *abort_flag = reinterpret_cast<volatile unsigned int*>(tmem_slot + 1), *bad_flag = abort_flag + 1;  // bad: the sequence has a page that is not there
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

    const PagedPart part = paged_part(g, static_cast<int>(blockIdx.x) / g.m);
    const int which = static_cast<int>(blockIdx.x) % g.m, kvh = which % a.c.kv_heads;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");  // the join may come up beside the last wave; it waits for this launch's end before it reads
    const int2 own = g.even ? make_int2(which / a.c.kv_heads, part.order) : paged_row_block(a, part.order, M::kRows);
    if (own.x < 0) return;
    const PagedSequence sq = paged_sequence(a.c, a.r, own.x);
    if (!sq.ok || sq.news < a.few || sq.news > a.many) {
        if (sq.news > a.r.most && tid == 0) atomicOr(a.c.status, kPagedBadPosition);
        return;
    }
    const int rows = sq.news * a.group, block = (rows + M::kRows - 1) / M::kRows - 1 - own.y, r0 = block * M::kRows, r1 = min(rows, r0 + M::kRows);
    if (block < 0) return;
    const PagedRange range = paged_part_range(a, sq, r0 / a.group, (r1 - 1) / a.group + 1, part.range, part.ranges, KT);
    const int p0 = sq.length - sq.news, tiles = range.end > range.begin ? (range.end - range.begin + KT - 1) / KT : 0, units = tiles * NT;

    if (tid == 0) {
        for (int s = 0; s < RS; ++s) mbar_init(full(s), Q8 ? M::kWidenWarps : 1), mbar_init(empty(s), 1);
        for (int s = 0; s < M::kRaws; ++s) mbar_init(raw_full(s), 1), mbar_init(raw_empty(s), M::kWidenWarps);
        for (int b = 0; b < NB; ++b) mbar_init(s_full(b), 1), mbar_init(p_full(b), 4 * SIDES), mbar_init(o_done(b), 1);
        mbar_init(q_full, M::kSoftWarps);
        mbar_init(drained, 1), mbar_init(pages_known, 1);
        *abort_flag = 0, *bad_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == M::kMmaWarp) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(const_cast<uint32_t*>(tmem_slot))), "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = *tmem_slot;

    if (warp >= M::kSoftWarps) {
        if constexpr (M::kSplitRegs) registers_down<M::kRestRegs>();
        if (warp == M::kLoadWarp) {
            // ---- pages to shared memory: per tile of positions the keys' rows, then the values' ----
            const int* table = a.r.table + static_cast<size_t>(own.x) * a.r.stride;
            const int P = 1 << a.c.page_log2, PR = min(P, kPagedTile);
            constexpr int kRing = Q8 ? RW : RS;
            PagedPages<KT> pages_of(a.c, table, range.begin, range.end, paged_first_seen(a, sq, r0 / a.group));
            int n = 0;
            bool okay = true;
            for (int j = 0; j < tiles && okay; ++j) {
                const int k0 = range.begin + j * KT, pages = pages_of.of(j), pieces = (min(KT, range.end - k0) + PR - 1) / PR;
                for (int value = 0; value < 2; ++value, ++n) {
                    const int s = n % kRing;
                    const uint32_t bar = Q8 ? raw_full(s) : full(s), to = Q8 ? raws + s * M::kRawStride : slots + s * M::kSlot;
                    if (!(okay = __all_sync(0xffffffffu, mbar_wait(Q8 ? raw_empty(s) : empty(s), ((n / kRing) & 1) ^ 1, abort_flag, a.spin_limit)))) break;
                    if (!Q8 && value && pieces * PR < KT) {  // rows that no page brings: their weights are zeros, their values must be numbers
                        for (int i = pieces * PR * 8 + lane; i < KT * 8; i += 32)
                            for (int b = 0; b < BLOCKS; ++b)
                                *reinterpret_cast<uint4*>(smem + (to - base) + paged_row_at(TYPE, BLOCKS, b, i >> 3) + (i & 7) * 16) = make_uint4(0, 0, 0, 0);
                        fence_async_shared();
                        __syncwarp();
                    }
                    if (lane == 0) mbar_expect_tx(bar, pieces * PR * (BLOCKS * kRow + (Q8 && !value ? 8 : 0)));
                    __syncwarp();
                    const unsigned char* store = value ? a.c.v : a.c.k;
                    if (lane < pieces) bulk_load(to + lane * PR * BLOCKS * kRow, store + paged_rows_at(a.c, TYPE, pages, kvh, (k0 + lane * PR) & (P - 1)), PR * BLOCKS * kRow, bar);
                    if constexpr (Q8) {
                        if (!value && lane < pieces) {
                            const size_t from = paged_scales_at(a.c, pages, kvh) + ((k0 + lane * PR) & (P - 1));
                            bulk_load(to + M::kRaw + lane * PR * 4, a.c.ks + from, PR * 4, bar);
                            bulk_load(to + M::kRaw + (KT + lane * PR) * 4, a.c.vs + from, PR * 4, bar);
                        }
                    }
                }
            }
            if (pages_of.bad) *bad_flag = 1;
            __syncwarp();
            if (lane == 0) mbar_arrive(pages_known);
            for (int back = max(0, n - kRing); back < n; ++back) mbar_wait(Q8 ? raw_full(back % kRing) : full(back % kRing), (back / kRing) & 1, abort_flag, a.spin_limit, false);
        } else if (warp == M::kMmaWarp) {
            // ---- all products: one thread issues them, but the warp stays together, so that descriptors live in uniform registers (issued by a lane on its own, eight products took as long to issue
            // as sixteen to run) ----
            constexpr uint32_t kScores = instr_desc_16(M::BF, false, KT), kValues = instr_desc_16(M::BF, true, HD);
            // descriptors: the upper word does not change
            const uint64_t q_desc = smem_desc(0, 16, 1024, 2), k_desc = smem_desc(0, 16, BLOCKS * 1024, 2), v_desc = smem_desc(0, 1024, BLOCKS * 1024, 2);
            auto at = [](uint64_t desc, uint32_t addr) { return desc | static_cast<uint64_t>((addr & 0x3FFFFu) >> 4); };
            bool okay = units == 0 || __all_sync(0xffffffffu, mbar_wait(q_full, 0, abort_flag, a.spin_limit));
            fence_after();
            int have = 0;  // operand tiles waited for: tile n of the sequence keys 0, values 0, keys 1, ...
            auto need = [&](int n) {
                for (; okay && have <= n; ++have) okay = __all_sync(0xffffffffu, mbar_wait(full(have % RS), (have / RS) & 1, abort_flag, a.spin_limit));
                fence_after();
                return okay;
            };
            auto scores = [&](int u) {  // S of unit u; the keys are given back behind the last unit that reads them
                const int j = u / NT, i = u % NT, b = u % NB;
                if (!need(2 * j)) return;
                const uint32_t d = tmem + M::kSCol + b * KT;
                const uint64_t keys = at(k_desc, slots + (2 * j % RS) * M::kSlot), queries = at(q_desc, q_at + i * BLOCKS * 128 * 128);
                if (elect_one()) {
#pragma unroll
                    for (int k = 0; k < HD / 16; ++k) {
                        const uint64_t kd = keys + ((k >> 2) * 1024 >> 4) + 2 * (k & 3);
                        if constexpr (M::kQTmem) mma_ts(d, tmem + M::kQCol + k * 8, kd, kScores, k > 0);
                        else mma_ss(d, queries + ((k >> 2) * 128 * 128 >> 4) + 2 * (k & 3), kd, kScores, k > 0);
                    }
                    mma_commit(s_full(b));
                    if (i == NT - 1) mma_commit(empty(2 * j % RS));
                }
                __syncwarp();
            };
            for (int u = 0; u < NB && u < units && okay; ++u) scores(u);
            for (int u = 0; u < units && okay; ++u) {
                const int j = u / NT, i = u % NT, b = u % NB;
                if (!need(2 * j + 1) || !(okay = __all_sync(0xffffffffu, mbar_wait(p_full(b), (u / NB) & 1, abort_flag, a.spin_limit)))) break;
                fence_after();
                const uint64_t values = at(v_desc, slots + ((2 * j + 1) % RS) * M::kSlot);
                const uint32_t first = j > 0;
                if (elect_one()) {
#pragma unroll
                    for (int k = 0; k < KT / 16; ++k) mma_ts(tmem + M::kOCol + i * 128, tmem + M::kSCol + b * KT + k * 8, values + (k * 2 * BLOCKS * 1024 >> 4), kValues, k > 0 ? 1u : first);
                    mma_commit(o_done(b));
                    if (i == NT - 1) mma_commit(empty((2 * j + 1) % RS));
                }
                __syncwarp();
                if (u + NB < units) scores(u + NB);
            }
            if (elect_one()) mma_commit(drained);  // nothing is under way when the block leaves
            __syncwarp();
            mbar_wait(drained, 0, abort_flag, a.spin_limit, false);
        } else if (Q8 && warp >= M::kWidenWarp) {
            // ---- codes to F16 operands ----
            if constexpr (Q8) {
                const int w = tid - M::kWidenWarp * 32;
                const float scale = fmaxf(fabsf(a.scale), 1e-37f);
                bool okay = true;
                for (int n = 0; n < 2 * tiles && okay; ++n) {
                    const int j = n >> 1, value = n & 1, rs = n % RW, s = n % RS, left = range.end - (range.begin + j * KT);  // rows of the tile that are there
                    okay = __all_sync(0xffffffffu, mbar_wait(raw_full(rs), (n / RW) & 1, abort_flag, a.spin_limit) && mbar_wait(empty(s), ((n / RS) & 1) ^ 1, abort_flag, a.spin_limit));
                    if (!okay) break;
                    const uint32_t from = raws + rs * M::kRawStride;
                    unsigned char* to = smem + M::kQBytes + s * M::kSlot;
                    if (!value && w < KT) {
                        const float* d = reinterpret_cast<const float*>(raw_smem + rs * M::kRawStride + M::kRaw) + w;
                        float* f = factors + (j & 3) * 3 * KT + w;
                        f[0] = w < left ? d[0] * scale : 0.0f, f[KT] = w < left ? lg2(d[KT]) : 0.0f, f[2 * KT] = w < left ? rcp(d[KT]) : 0.0f;
                    }
                    constexpr int kPieces = KT * BLOCKS * 4 / (M::kWidenWarps * 32), kAtOnce = kPieces > 4 ? 4 : kPieces;  // pieces of sixteen codes of a thread, and those under way together
#pragma unroll
                    for (int k0 = 0; k0 < kPieces; k0 += kAtOnce) {
                        uint32_t v[kAtOnce][4];
#pragma unroll
                        for (int k = 0; k < kAtOnce; ++k)
                            asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                                         : "=r"(v[k][0]), "=r"(v[k][1]), "=r"(v[k][2]), "=r"(v[k][3])
                                         : "r"(from + (w + (k0 + k) * M::kWidenWarps * 32) * 16)
                                         : "memory");
#pragma unroll
                        for (int k = 0; k < kAtOnce; ++k) {
                            const int i = w + (k0 + k) * M::kWidenWarps * 32, row = i >> 2, r = (row / (8 * BLOCKS)) * 8 + (row & 7), c = (i & 3) ^ ((r >> 1) & 3);  // row: 128 bytes of the operand, in the order of the codes' 64
                            uint32_t o[8];
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                const uint32_t u = r < left ? v[k][e] ^ 0x80808080u : 0x80808080u;
                                o[2 * e] = codes_to_half2(u, 0x4140), o[2 * e + 1] = codes_to_half2(u, 0x4342);
                            }
                            *reinterpret_cast<uint4*>(to + row * 128 + (((2 * c) ^ (r & 7)) << 4)) = make_uint4(o[0], o[1], o[2], o[3]);
                            *reinterpret_cast<uint4*>(to + row * 128 + (((2 * c + 1) ^ (r & 7)) << 4)) = make_uint4(o[4], o[5], o[6], o[7]);
                        }
                    }
                    fence_async_shared();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(full(s)), mbar_arrive(raw_empty(rs));
                }
            }
        }
    } else {
        if constexpr (M::kSplitRegs) registers_up<M::kSoftRegs>();
        // ---- a row of queries for a thread, or for two, which have half of a tile's positions each: warps w and w + 4 ----
        const int i = SIDES == 2 ? 0 : warp >> 2, side = SIDES == 2 ? warp >> 2 : 0, local = (warp & 3) * 32 + lane, r = r0 + i * 128 + local, t = r / a.group;
        const uint32_t lanes = uint32_t((warp & 3) * 32) << 16;
        const bool live = r < r1;
        constexpr int KH = KT / SIDES, HH = HD / SIDES;
        // the two warps meet at a barrier of their own; both come to it the same number of times whatever happens, as all other waits end by themselves
        const int meet = 1 + (warp & 3);
        volatile float2* mine = exchange + side * 128 + local;
        volatile float2* theirs = exchange + (side ^ 1) * 128 + local;
        auto meet_sync = [&]() { asm volatile("barrier.cta.sync %0, 64;" ::"r"(meet) : "memory"); };
        auto meet_any = [&](bool x) {
            if constexpr (SIDES == 1) return __any_sync(0xffffffffu, x) != 0;
            uint32_t any;
            asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbarrier.cta.red.or.pred q, %2, 64, p;\n\tselp.u32 %0, 1, 0, q;\n\t}" : "=r"(any) : "r"(x ? 1u : 0u), "r"(meet) : "memory");
            return any != 0;
        };
        unsigned char* stage = staging + warp * 32 * M::kStagePitch;
        {   // queries: lanes side by side along a row
            constexpr int kLanes = HD / 8, kAtOnce = 32 / kLanes;  // 16-byte pieces of a row; rows at once
            const int wr = r0 + i * 128 + (warp & 3) * 32, sub = lane / kLanes, e = lane % kLanes * 8;  // the warp's first row
            const float sign = a.scale < 0.0f ? -1.0f : 1.0f, scale = fmaxf(fabsf(a.scale), 1e-37f);  // (times minus infinity, where a mask hides a score, it stays that)
            // the byte offset of the warp's row `lane`; the last row's where there are no more
            const int own = min(wr + lane, r1 - 1);
            const size_t own_at = ((static_cast<size_t>(sq.first) + own / a.group) * a.q_token + (kvh * a.group + own % a.group) * a.q_head) * paged_size_of(a.q_type);
            auto load = [&](auto of) {  // by the queries' type, so that the loads of a batch of rows are under way together
                constexpr int T = decltype(of)::value;
                auto fetch = [&](int row, int e) { return paged_raw<T>(static_cast<const unsigned char*>(a.q) + __shfl_sync(0xffffffffu, own_at, row), e); };
                auto power = [&](const float (&x)[8]) {  // of the row's maximum, as the bits of a power of two; 1 for zeros, denormals and what is not finite
                    float top = 0.0f;
#pragma unroll
                    for (int c = 0; c < 8; ++c) top = fmaxf(top, fabsf(x[c]));
#pragma unroll
                    for (int o = kLanes / 2; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
                    const uint32_t ex = __float_as_uint(top) >> 23;
                    return (T != kPagedF16 && ex > 1 && ex < 254 ? ex : 127u) << 23;  // (F16 queries go in as they are)
                };
                if constexpr (!M::kQTmem) {
                    constexpr int kBatch = T == kPagedF32 ? 4 : 8;
#pragma unroll 1
                    for (int k0 = 0; k0 < 32; k0 += kBatch * kAtOnce) {
                        PagedRaw<T> raw[kBatch];
#pragma unroll
                        for (int k = 0; k < kBatch; ++k) raw[k] = fetch(k0 + k * kAtOnce + sub, e);
#pragma unroll
                        for (int k = 0; k < kBatch; ++k) {
                            const int mine = k0 + k * kAtOnce + sub, row = (warp & 3) * 32 + mine;
                            float x[8], f = sign, factor = Q8 ? 1.0f : scale;
                            paged_load8(raw[k].v, T, x);
                            if constexpr (Q8) {
                                const uint32_t bits = power(x);
                                factor *= __uint_as_float(bits), f *= __uint_as_float((254u << 23) - bits);  // (the reciprocal of a power of two)
                            }
#pragma unroll
                            for (int c = 0; c < 8; ++c) x[c] = wr + mine < r1 ? x[c] * f : 0.0f;
                            paged_store8(smem + ((i * BLOCKS + e / 64) * 128 + row) * 128 + (((e / 8 & 7) ^ (row & 7)) << 4), M::BF ? kPagedBf16 : kPagedF16, x);
                            if (lane % kLanes == 0) row_factor[i * 128 + row] = factor;
                        }
                    }
                    fence_async_shared();
                } else {
                    if constexpr (Q8) {  // both warps of a row look at all of it
                        constexpr int kBatch = T == kPagedF32 ? 4 : 8;
#pragma unroll 1
                        for (int k0 = 0; k0 < 32 && wr + k0 < r1; k0 += kBatch * kAtOnce) {
                            PagedRaw<T> raw[kBatch];
#pragma unroll
                            for (int k = 0; k < kBatch; ++k) raw[k] = fetch(min(k0 + k * kAtOnce + sub, 31), e);
#pragma unroll
                            for (int k = 0; k < kBatch; ++k) {
                                float x[8];
                                paged_load8(raw[k].v, T, x);
                                const uint32_t bits = power(x);
                                if (lane % kLanes == 0 && k0 + k * kAtOnce + sub < 32) reinterpret_cast<uint32_t*>(stage + (k0 + k * kAtOnce + sub) * M::kStagePitch)[32] = bits;  // behind the row's 128 bytes
                            }
                        }
                    }
                    __syncwarp();
                    constexpr int kPart = HH < 64 ? HH : 64, kPartLanes = kPart / 8, kRowsAtOnce = 32 / kPartLanes;  // values of a row that fit the staging's row
                    constexpr int kAhead = Q8 ? 1 : HH / kPart;  // parts whose reads are under way together (1024 tokens of 256-value heads: 26.7 us one after the other, 25.5 so; Q8 has no registers for it)
#pragma unroll 1
                    for (int c1 = side * HH; c1 < (side + 1) * HH; c1 += kPart * kAhead) {
                        PagedRaw<T> raw[kAhead][kPartLanes];
#pragma unroll
                        for (int p = 0; p < kAhead; ++p)
#pragma unroll
                            for (int k = 0; k < kPartLanes; ++k) raw[p][k] = fetch(k * kRowsAtOnce + lane / kPartLanes, c1 + p * kPart + lane % kPartLanes * 8);
#pragma unroll
                        for (int p = 0; p < kAhead; ++p) {
                        const int c0 = c1 + p * kPart;
#pragma unroll
                        for (int k = 0; k < kPartLanes; ++k) {
                            const int row = k * kRowsAtOnce + lane / kPartLanes;
                            float x[8], f = sign;
                            paged_load8(raw[p][k].v, T, x);
                            if constexpr (Q8) f *= __uint_as_float((254u << 23) - reinterpret_cast<const uint32_t*>(stage + row * M::kStagePitch)[32]);
#pragma unroll
                            for (int c = 0; c < 8; ++c) x[c] = wr + row < r1 ? x[c] * f : 0.0f;
                            paged_store8(stage + row * M::kStagePitch + lane % kPartLanes * 16, M::BF ? kPagedBf16 : kPagedF16, x);
                        }
                        __syncwarp();
                        uint32_t v[kPart / 2];
#pragma unroll
                        for (int k = 0; k < kPart / 8; ++k) {
                            const uint4 w = *reinterpret_cast<const uint4*>(stage + lane * M::kStagePitch + k * 16);
                            v[4 * k] = w.x, v[4 * k + 1] = w.y, v[4 * k + 2] = w.z, v[4 * k + 3] = w.w;
                        }
                        if constexpr (kPart == 64) tmem_store32(tmem + lanes + M::kQCol + c0 / 2, v);
                        else tmem_store16(tmem + lanes + M::kQCol + c0 / 2, v);
                        __syncwarp();
                        }
                    }
                    if (side == 0) row_factor[local] = Q8 ? __uint_as_float(reinterpret_cast<const uint32_t*>(stage + lane * M::kStagePitch)[32]) : scale;
                    tmem_wait_store();
                }
            };
            if constexpr (TYPE != kPagedQ8) load(PagedTag<TYPE>());
            else if (a.q_type == kPagedF16) load(PagedTag<kPagedF16>());
            else if (a.q_type == kPagedBf16) load(PagedTag<kPagedBf16>());
            else load(PagedTag<kPagedF32>());
            fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(q_full);
            if constexpr (SIDES == 2) meet_sync();
        }
        const float rowf = row_factor[i * 128 + local];  // what the row's scores are multiplied by: positive, the queries took the sign
        // (a row that is not there, of zeros, sees everything, so that it makes no masks necessary: a row tile of 20 rows that masked every tile for the others took 58 us instead of 47)
        const int p = p0 + t, last = live ? min(p, range.end - 1) : range.end - 1, first = live ? paged_first_seen(a, sq, t) : 0;
        const bool some = r0 + i * 128 + (warp & 3) * 32 < r1;  // the same for the two warps that meet
        float m = -INFINITY, l = 0.0f;  // l: over this thread's positions
        bool okay = true;
        // The value products of unit u. A wait tells phases apart by their parity alone, so each buffer has a barrier: those of unit u - NB, the phase before, are done, as the scores
        // of unit u (asked for behind them) were waited for, and those of unit u + NB cannot have begun.
        auto values_done = [&](int u) { return __all_sync(0xffffffffu, mbar_wait(o_done(u % NB), (u / NB) & 1, abort_flag, a.spin_limit)); };
#pragma unroll 1
        for (int j = 0; j < tiles; ++j) {
            const int u = j * NT + i, b = u % NB, k0 = range.begin + j * KT + side * KH;
            const uint32_t s_at = tmem + lanes + M::kSCol + b * KT;
            if (okay) okay = __all_sync(0xffffffffu, mbar_wait(s_full(b), (u / NB) & 1, abort_flag, a.spin_limit));
            fence_after();
            if constexpr (SIDES == 2) {
                if (!some) {  // a warp without rows of its own (they are the last ones: a few rows are in the first warp): its weights multiply nothing that is read
                    if (lane == 0 && okay) mbar_arrive(p_full(b));
                    continue;
                }
            }
            uint32_t s[KH / 32][32];
#pragma unroll
            for (int c = 0; c < KH / 32; ++c) tmem_load32(s_at + side * KH + c * 32, s[c]);
            tmem_wait_load();
            // v in s, so that a weight is 2^(v mul - m): the products themselves, where only the scale is to come; else the whole exponent
            float mul = 1.0f;
            const float4* f = reinterpret_cast<const float4*>(factors + (j & 3) * 3 * KT + side * KH);
            auto pair = [&](int c, int e) { return pack_f32x2(__uint_as_float(s[c][e]), __uint_as_float(s[c][e + 1])); };
            auto put = [&](int c, int e, unsigned long long v) {
                const float2 x = unpack_f32x2(v);
                s[c][e] = __float_as_uint(x.x), s[c][e + 1] = __float_as_uint(x.y);
            };
            const unsigned long long row2 = pack_f32x2(rowf, rowf);
            if (a.cap > 0.0f) {
#pragma unroll
                for (int c = 0; c < KH / 32; ++c)
#pragma unroll
                    for (int e = 0; e < 32; ++e) {
                        float x = __uint_as_float(s[c][e]);
                        if constexpr (Q8) x *= reinterpret_cast<const float*>(f)[c * 32 + e];
                        x = a.cap * tanh_of<FAR>(x * rowf);
                        if constexpr (Q8) x += reinterpret_cast<const float*>(f)[KT + c * 32 + e];
                        s[c][e] = __float_as_uint(x);
                    }
            } else if (Q8 && a.q_type == kPagedF16) {  // every row's factor is 1
#pragma unroll
                for (int c = 0; c < KH / 32; ++c)
#pragma unroll
                    for (int e = 0; e < 32; e += 4) {
                        const float4 ks = f[(c * 32 + e) / 4], lv = f[(KT + c * 32 + e) / 4];
                        put(c, e, fma_f32x2(pair(c, e), pack_f32x2(ks.x, ks.y), pack_f32x2(lv.x, lv.y)));
                        put(c, e + 2, fma_f32x2(pair(c, e + 2), pack_f32x2(ks.z, ks.w), pack_f32x2(lv.z, lv.w)));
                    }
            } else if constexpr (Q8) {
#pragma unroll
                for (int c = 0; c < KH / 32; ++c)
#pragma unroll
                    for (int e = 0; e < 32; e += 4) {
                        const float4 ks = f[(c * 32 + e) / 4], lv = f[(KT + c * 32 + e) / 4];
                        put(c, e, fma_f32x2(mul_f32x2(pair(c, e), pack_f32x2(ks.x, ks.y)), row2, pack_f32x2(lv.x, lv.y)));
                        put(c, e + 2, fma_f32x2(mul_f32x2(pair(c, e + 2), pack_f32x2(ks.z, ks.w)), row2, pack_f32x2(lv.z, lv.w)));
                    }
            } else {
                mul = rowf;
            }
            if (__any_sync(0xffffffffu, k0 + KH - 1 > last || k0 < first)) {
                const int lo = first - k0, hi = last - k0;
#pragma unroll
                for (int c = 0; c < KH / 32; ++c)
#pragma unroll
                    for (int e = 0; e < 32; ++e) s[c][e] = c * 32 + e >= lo && c * 32 + e <= hi ? s[c][e] : 0xff800000u;  // minus infinity
            }
            float tops[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};  // four at a time: a chain of maxima or sums takes four cycles a link
#pragma unroll
            for (int c = 0; c < KH / 32; ++c)
#pragma unroll
                for (int e = 0; e < 32; ++e) tops[e & 3] = fmaxf(tops[e & 3], __uint_as_float(s[c][e]));
            float top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3])) * mul;
            // (also: both have read their scores, so that the weights may be written over them)
            if (meet_any(!okay || top > m + kPagedLazy || (m == -INFINITY && top > -INFINITY))) {
                if constexpr (SIDES == 2) {
                    mine->x = top, mine->y = okay ? 0.0f : 1.0f;
                    meet_sync();
                    const float other = theirs->x, theirs_okay = theirs->y;
                    meet_sync();  // before either writes the next one
                    okay = __all_sync(0xffffffffu, okay && theirs_okay == 0.0f);  // the same in both warps: a warp is of one mind, and hears of the other's
                    top = fmaxf(top, other);
                }
                if (!okay) break;
                const bool grew = top > m + kPagedLazy || (m == -INFINITY && top > -INFINITY);
                const float keep = grew ? ex2(m - top) : 1.0f;  // 0 the first time
                if (grew) m = top, l *= keep;
                if (j > 0 && __any_sync(0xffffffffu, grew)) {
                    okay = values_done(u - NT);
                    fence_after();
#pragma unroll 1
                    for (int c = side * HH; c < (side + 1) * HH; c += 32) {
                        uint32_t o[32];
                        tmem_load32(tmem + lanes + M::kOCol + i * 128 + c, o);
                        tmem_wait_load();
#pragma unroll
                        for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * keep);
                        tmem_store32(tmem + lanes + M::kOCol + i * 128 + c, o);
                    }
                }
            }
            const float ref = m == -INFINITY ? 0.0f : -m;
            const unsigned long long mul2 = pack_f32x2(mul, mul), ref2 = pack_f32x2(ref, ref);
            unsigned long long sums[2] = {0ull, 0ull};
#pragma unroll
            for (int c = 0; c < KH / 32; ++c) {
                uint32_t w[16];
#pragma unroll
                for (int e = 0; e < 16; e += 2) {
                    const int k = 2 * e;
                    float2 x = unpack_f32x2(fma_f32x2(pair(c, k), mul2, ref2)), y = unpack_f32x2(fma_f32x2(pair(c, k + 2), mul2, ref2));
                    x.x = ex2(x.x), x.y = ex2(x.y), y.x = ex2(y.x), y.y = ex2(y.y);
                    if constexpr (Q8) {
                        const float4 iv = f[(2 * KT + c * 32 + k) / 4];
                        sums[0] = fma_f32x2(pack_f32x2(x.x, x.y), pack_f32x2(iv.x, iv.y), sums[0]);
                        sums[1] = fma_f32x2(pack_f32x2(y.x, y.y), pack_f32x2(iv.z, iv.w), sums[1]);
                    } else {
                        sums[0] = add_f32x2(sums[0], pack_f32x2(x.x, x.y)), sums[1] = add_f32x2(sums[1], pack_f32x2(y.x, y.y));
                    }
                    w[e] = paged_pack2<M::BF ? kPagedBf16 : kPagedF16>(x.x, x.y), w[e + 1] = paged_pack2<M::BF ? kPagedBf16 : kPagedF16>(y.x, y.y);
                }
                tmem_store16(s_at + side * (KH / 2) + c * 16, w);
            }
            const float2 sum = unpack_f32x2(add_f32x2(sums[0], sums[1]));
            l += sum.x + sum.y;
            tmem_wait_store();
            fence_before();
            __syncwarp();
            if (lane == 0 && okay) mbar_arrive(p_full(b));
        }
        if (okay && tiles > 0) okay = values_done((tiles - 1) * NT + i);
        if constexpr (!M::kQTmem) {  // results go out over the queries: the products that were waited for have read them; without any, the warps wait for one another's
            if (tiles == 0) asm volatile("barrier.cta.sync 5, %0;" ::"n"(M::kSoftWarps * 32) : "memory");
        }
        if (okay) okay = __all_sync(0xffffffffu, mbar_wait(pages_known, 0, abort_flag, a.spin_limit));
        okay = __all_sync(0xffffffffu, okay && *abort_flag == 0);
        if constexpr (SIDES == 2) {
            mine->x = l, mine->y = okay ? 0.0f : 1.0f;
            meet_sync();
            okay = __all_sync(0xffffffffu, okay && theirs->y == 0.0f);
            l += theirs->x;
        }
        if (!okay && lane == 0) atomicOr(a.c.status, kPagedGaveUp);
        if (okay) {
            fence_after();
            const bool left_out = *bad_flag != 0;
            const float inv = part.ranges > 1 ? 1.0f : l > 0.0f ? 1.0f / l : l == 0.0f ? 0.0f : l;
            const int wr = r0 + i * 128 + (warp & 3) * 32;  // the warp's first row
            const size_t row = paged_part_row(a, g, sq, part, which, kvh, r, i * 128 + local, M::kRows);
            if (!left_out && (tiles > 0 || part.ranges == 1)) {  // (of a range in which the rows see nothing only the sums below are read)
#pragma unroll 1
                for (int c = side * HH; c < (side + 1) * HH; c += 32) {
                    uint32_t o[32];
                    if (tiles > 0) {
                        tmem_load32(tmem + lanes + M::kOCol + i * 128 + c, o);
                        tmem_wait_load();
                    } else {
#pragma unroll
                        for (int e = 0; e < 32; ++e) o[e] = 0u;
                    }
                    __syncwarp();
#pragma unroll
                    for (int e = 0; e < 32; e += 4)
                        *reinterpret_cast<float4*>(stage + lane * M::kStagePitch + e * 4) =
                            make_float4(__uint_as_float(o[e]) * inv, __uint_as_float(o[e + 1]) * inv, __uint_as_float(o[e + 2]) * inv, __uint_as_float(o[e + 3]) * inv);
                    __syncwarp();
#pragma unroll
                    for (int k = 0; k < 32; k += 8) {  // four lanes a row
                        const int rr = k + (lane >> 2), e = (lane & 3) * 8;
                        if (wr + rr >= r1) continue;
                        float x[8];
                        paged_load8(stage + rr * M::kStagePitch + e * 4, kPagedF32, x);
                        if (part.ranges == 1) {
                            const size_t token = static_cast<size_t>(sq.first) + (wr + rr) / a.group;
                            paged_store8(static_cast<unsigned char*>(a.out) + (token * a.o_token + (kvh * a.group + (wr + rr) % a.group) * a.o_head + c + e) * paged_size_of(a.out_type), a.out_type, x);
                        } else {
                            paged_store8(g.part_o + (row - lane + rr) * HD + c + e, kPagedF32, x);
                        }
                    }
                }
            }
            if (live && part.ranges > 1 && side == 0) g.part_ml[row] = left_out ? paged_left_out() : make_float2(m, l);
        }
    }
    fence_before();
    __syncthreads();
    if (warp == M::kMmaWarp) {
        fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
    }
}

// Joins the ranges of the row blocks that were cut, in the order of the ranges: a warp takes four query heads of a packed token, whose reads overlap (bound by their latency: with a head to
// a warp a mixed batch's 8448 rows of four ranges took 2 to 4 us longer). Grid: packed tokens x groups of heads, eight to a block.
constexpr int kPagedJoinRows = 4;
template <int BLOCKS>
__global__ void __launch_bounds__(256) paged_join_kernel(const __grid_constant__ PagedAttnArgs a, const __grid_constant__ PagedSchedule g, int kRows) {
    using namespace paged_detail;
    constexpr int HD = BLOCKS * kPagedBlock, kPer = HD / 32, ROWS = kPagedJoinRows;
    const int heads = a.group * a.c.kv_heads, units = (heads + ROWS - 1) / ROWS, lane = threadIdx.x & 31;
    const int item = static_cast<int>(blockIdx.x) * 8 + (threadIdx.x >> 5), token = item / units, h0 = item % units * ROWS;
    const int seq = token < a.r.tokens ? paged_sequence_of(a.r, token) : -1;
    PagedSequence sq{};
    if (seq >= 0) sq = paged_sequence(a.c, a.r, seq);
    const int rows = sq.news * a.group, blocks = (rows + kRows - 1) / kRows;
    const long long before = g.even || seq < 0 ? 0 : paged_row_blocks_before(a, seq, kRows);
    asm volatile("griddepcontrol.wait;" ::: "memory");  // what was read above is input. Every block waits, so that none ends before the launch that it joins
    if (!sq.ok || sq.news < a.few || sq.news > a.many || token < sq.first || token >= sq.first + sq.news) return;
    int ranges[ROWS], most = 1;
    size_t from[ROWS], step[ROWS];  // the first range's row of the workspace, and from one range to the next
#pragma unroll
    for (int k = 0; k < ROWS; ++k) {
        const int h = min(h0 + k, heads - 1), kvh = h / a.group, r = (token - sq.first) * a.group + h % a.group;
        const long long order = before + blocks - 1 - r / kRows;
        const bool known = h0 + k < heads && order < g.orders;
        const int x = !known ? 0 : g.mapped ? g.at[order] : static_cast<int>(order - g.whole) * g.cut;
        ranges[k] = !known ? 1 : g.mapped ? g.ranges[x] : x < 0 ? 1 : g.cut;
        auto at = [&](int i) { return paged_part_row(a, g, sq, PagedPart{0, i, ranges[k], x + i}, g.even ? seq * a.c.kv_heads + kvh : kvh, kvh, r, r % kRows, kRows); };
        from[k] = ranges[k] > 1 ? at(0) : 0, step[k] = ranges[k] > 1 ? at(1) - at(0) : 0;
        most = max(most, ranges[k]);
    }
    if (most == 1) return;
    // a lane holds the sums of a range, of 32 at a time: their maximum over all, then their weights
    auto sums_of = [&](int k, int i) { return i < ranges[k] && ranges[k] > 1 ? g.part_ml[from[k] + i * step[k]] : make_float2(-INFINITY, 0.0f); };
    float top[ROWS], total[ROWS] = {}, x[ROWS][kPer] = {};
    float2 ml[ROWS];
    bool left_out[ROWS];
#pragma unroll
    for (int k = 0; k < ROWS; ++k) ml[k] = sums_of(k, lane);
#pragma unroll
    for (int k = 0; k < ROWS; ++k) {
        top[k] = ml[k].x, left_out[k] = ml[k].y < 0.0f;
        for (int i = lane + 32; i < most; i += 32) {
            const float2 v = sums_of(k, i);
            top[k] = fmaxf(top[k], v.x), left_out[k] = left_out[k] || v.y < 0.0f;
        }
        left_out[k] = __any_sync(0xffffffffu, left_out[k]);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) top[k] = fmaxf(top[k], __shfl_xor_sync(0xffffffffu, top[k], o));
    }
    for (int i0 = 0; i0 < most; i0 += 32) {
        float weight[ROWS];
#pragma unroll
        for (int k = 0; k < ROWS; ++k) {
            if (i0 > 0) ml[k] = sums_of(k, i0 + lane);
            weight[k] = ml[k].x == -INFINITY && ml[k].y == 0.0f ? -1.0f : ex2(ml[k].x - top[k]);  // -1: a range in which nothing was visible has no values
        }
        for (int i = i0; i < min(most, i0 + 32); ++i) {
            float v[ROWS][kPer], w[ROWS];
#pragma unroll
            for (int k = 0; k < ROWS; ++k) {
                w[k] = __shfl_sync(0xffffffffu, weight[k], i - i0);
                const float* p = g.part_o + (from[k] + i * step[k]) * HD + lane * kPer;
#pragma unroll
                for (int e = 0; e < kPer; ++e) v[k][e] = w[k] != -1.0f ? p[e] : 0.0f;
            }
#pragma unroll
            for (int k = 0; k < ROWS; ++k) {
                if (w[k] == -1.0f) continue;
                total[k] = fmaf(w[k], __shfl_sync(0xffffffffu, ml[k].y, i - i0), total[k]);
#pragma unroll
                for (int e = 0; e < kPer; ++e) x[k][e] = fmaf(w[k], v[k][e], x[k][e]);
            }
        }
    }
#pragma unroll
    for (int k = 0; k < ROWS; ++k) {
        if (ranges[k] == 1 || left_out[k]) continue;
        const float inv = total[k] > 0.0f ? 1.0f / total[k] : total[k] == 0.0f ? 0.0f : total[k];
#pragma unroll
        for (int e = 0; e < kPer; ++e) x[k][e] *= inv;
        paged_store_row(static_cast<unsigned char*>(a.out) + (static_cast<size_t>(token) * a.o_token + (h0 + k) * a.o_head + lane * kPer) * paged_size_of(a.out_type), a.out_type, x[k]);
    }
}

}  // namespace qtb
