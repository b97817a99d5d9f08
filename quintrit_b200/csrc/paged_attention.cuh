// Attention of new tokens over a paged cache, a few rows of queries at a time.
//
// For token i of a sequence at position p and query head h with KV head h / G: z_j = scale q.k_j, or cap tanh(scale q.k_j / cap), over the visible
// positions j <= p and, with a window, j > p - window; out = sum_j exp(z_j) v_j / sum_j exp(z_j), zeros where no position is visible. One pass over the
// rows: a running maximum m, the weights exp(z_j - m) and their sum l, and the products rescaled when m grows (only when it grows by more than 2^8,
// so that weights stay below 256 and a rescale is rare). Logarithms are to base 2: log2(e) goes into the scale.
//
// Q8 rows: k_j = ks_j a_j, v_j = vs_j b_j with integer codes. The codes go into the products as they are (exact in F16), ks_j multiplies the score, and
// vs_j goes into the exponent: with y_j = z_j + log2(vs_j) the weights w_j = 2^(y_j - m), m the maximum of y, are what multiplies b_j, and l = sum w_j / vs_j.
// So the weights that are rounded to F16 lie in [0, 256] whatever the scales are, and the cache's limits on them keep the terms of l from vanishing. Queries are scaled by a power of two per row to a maximum in [1, 2),
// which is exact, so BF16 and F32 queries of any size meet F16 codes (F32 queries are rounded to F16's 11 bits then).
//
// Bound by the rows' bytes: 2 G flops per byte of a 16-bit cache. A block of threads takes one KV head of one sequence, up to 16 rows of queries (24 of 128 values, Q8; a row
// is a (token, head of the group)) and a range of its positions; one warp brings the pages, tile by tile of 64 positions, into a ring in shared memory with bulk copies;
// two groups of four warps take the tiles in turn, a warp 16 positions of a tile against all rows. Matrix instructions (m16n8k16) with the positions, and then the values, as the
// 16 rows of the left operand and the queries as the 8 columns of the right one: S^T = K Q^T and O^T += V^T P^T, so that one query head or eight cost the same, a fragment of codes is
// widened once for all rows, and the sums of eight rows take head_dim / 4 registers. A score's row is the same in both products' registers; only the weights are transposed (movmatrix).
// Every warp has its own m, l and sums; at the end the eight warps join. Where that pays, the tiles of all sequences are shared out evenly among as many blocks as the
// device holds (PagedShare), whatever their lengths; results of cut items meet in the caller's workspace (paged_combine_kernel), in the order of the positions: no atomics.
//
// Measured: a token over 65431 positions of 5 heads of 128, F16, 167.5 MB in 35.4 us, 72% of the copy rate; a token of each of 32 sequences of 1 to 4096 positions of 4 heads of 256, Q8, 173.7 MB in
// 41.6 us, 64%. In the loop the copies run at the memory's rate; the rest is the start (places of all sequences, page numbers, the first copies: 8000 cycles), a second segment of a block, the
// join. Five tokens of each of 16 sequences, 20 rows, Q8: 35 us, 19%: 64 positions take a group of warps 4400 cycles, which are latency (scores 1150, maximum 950, weights 1000, sums 900), and
// sums for 24 rows leave registers for nine warps on a multiprocessor.
#pragma once
#include "paged_cache.cuh"
#include "tcgen05.cuh"

namespace qtb {

constexpr int kPagedTile = 64;       // positions of a tile
constexpr float kPagedLazy = 8.0f;   // growth of the maximum, in powers of two, that is waited for
constexpr float kLog2e = 1.4426950408889634f;

struct PagedAttnArgs {
    PagedView c;
    RowsView r;
    const void* q;
    size_t q_token, q_head;  // strides in elements
    int q_type, out_type;
    void* out;
    size_t o_token, o_head;
    int group;               // query heads of a KV head
    float scale;             // times log2(e); with a cap: scale / cap
    float cap;               // times log2(e); 0: none
    int window;              // 0: none
    int share;               // 0: a block of threads takes a whole item; else the items' tiles are shared out evenly among the blocks (PagedShare)
    float* part_o;           // [blocks][2][rows of a block][head_dim], where the tiles are shared out
    float2* part_ml;         // [blocks][2][rows of a block]
    int few, many;           // new tokens of the sequences that this launch serves: few <= n <= many
    unsigned int spin_limit;
};

namespace paged_detail {

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float lg2(float x) {
    float y;
    asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float rcp(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// tanh from one exponential: 1 - 2 / (1 + e^2x), off by about 2^-22 of one whatever x is; the infinities of the exponential give -1 and 1. SMALL: off by 2^-20 of itself, as a cap far above the scores asks
// for (the exponential alone spoils them by hundredths under a cap of 10^5): below 1/4 the first terms of the series, the next of which is 2^-21.5 of their sum there.
template <bool SMALL>
__device__ __forceinline__ float tanh_of(float x) {
    const float y = 1.0f - 2.0f * rcp(1.0f + ex2(x * (2.0f * kLog2e)));
    if constexpr (!SMALL) return y;
    const float t = x * x, near = fmaf(x * t, fmaf(t, fmaf(t, -17.0f / 315.0f, 2.0f / 15.0f), -1.0f / 3.0f), x);
    return fabsf(x) < 0.25f ? near : y;
}

template <bool BF16>
__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (BF16)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ void ldsm4_trans(uint32_t (&r)[4], uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ uint2 lds64(uint32_t at) {
    uint2 v;
    asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(at) : "memory");
    return v;
}
// Codes c (four bytes, two's complement) at the bytes that `low` and `high` select, as a pair of F16: 0x6400 + (c + 128) is 1024 + (c + 128) in F16.
__device__ __forceinline__ uint32_t codes_to_half2(uint32_t biased, uint32_t select) {
    uint32_t v;
    asm("prmt.b32 %0, %1, %2, %3;" : "=r"(v) : "r"(biased), "r"(0x64646464u), "r"(select));
    const __half2 h = __hsub2(*reinterpret_cast<const __half2*>(&v), __half2half2(__ushort_as_half(0x6480)));  // 1152
    return *reinterpret_cast<const uint32_t*>(&h);
}

__device__ __forceinline__ long long prefix(long long v) {  // the sum of v over the lanes up to this one
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long up = __shfl_up_sync(0xffffffffu, v, o);
        if (static_cast<int>(threadIdx.x & 31) >= o) v += up;
    }
    return v;
}

}  // namespace paged_detail

// In the place of a partial result's maximum and sum: the row is not to be written, for want of a page.
__device__ __forceinline__ float2 paged_left_out() { return make_float2(-INFINITY, -1.0f); }

template <int T> struct PagedTag { static constexpr int value = T; };

struct PagedRange {
    int begin, end;
};
// The window of a sequence's tokens: one longer than the sequence hides nothing, and the first position that a token sees is a 32-bit number with none longer.
__device__ __forceinline__ int paged_window(const PagedAttnArgs& a, const PagedSequence& q) { return min(a.window, q.length); }
// The first position that new token t of a sequence, or any behind it, sees.
__device__ __forceinline__ int paged_first_seen(const PagedAttnArgs& a, const PagedSequence& q, int t) { return a.window > 0 ? max(0, q.length - q.news + t - paged_window(a, q) + 1) : 0; }
// The positions that any new token of a sequence sees; begin is a multiple of 64.
__device__ __forceinline__ PagedRange paged_seen(const PagedAttnArgs& a, const PagedSequence& q) {
    return PagedRange{paged_first_seen(a, q, 0) & ~(kPagedTile - 1), q.length};
}

// Work shared out: the items (a sequence's KV head with all its rows) stand one after the other, sequence by sequence, each as long as its sequence's tiles and kPagedStart places in front of
// them; block b of G takes W / G of all W places, the first W % G blocks one more, whatever the lengths are. What a block has of an item is a segment: a whole item's result is written as it is,
// others go to the workspace, at most two of a block: place 0 for the segment that its places begin with, place 1 for another. Every block works the items out for itself from the lengths
// (paged_share_begin), for up to kPagedShared sequences. The places in front stand for what another segment costs a block (the end of one, the queries and the first copies of the next).
constexpr int kPagedShared = 256, kPagedStart = 5;
struct PagedShare {
    int total;
    int* before;  // [sequences + 1] in shared memory: places of the items before a sequence's
    int4* of;     // [sequences]: first token, new tokens, length, tiles of an item
};
struct PagedItem {
    int seq, kvh;
    int begin, tiles;           // the item's first place among all, its tiles
    PagedSequence q;
};
// By all threads of a block; `before` and `of` have room for kPagedShared + 1 and kPagedShared. Tiles that 32 bits do not hold, of sequences far longer
// than was announced, are not shared out: the call does nothing but report them.
__device__ __forceinline__ PagedShare paged_share_begin(const PagedAttnArgs& a, int* before, int4* of, int threads) {
    for (int s = threadIdx.x; s < a.r.sequences; s += threads) {
        const PagedSequence q = paged_sequence(a.c, a.r, s);
        const PagedRange g = paged_seen(a, q);
        const int tiles = max(1, (g.end - g.begin + kPagedTile - 1) / kPagedTile);
        before[s + 1] = q.ok && q.news >= a.few && q.news <= a.many ? static_cast<int>(min((tiles + static_cast<long long>(kPagedStart)) * a.c.kv_heads, 0x7fffffffLL)) : 0;
        of[s] = make_int4(q.first, q.news, q.length, tiles);
        if (q.news > a.r.most) atomicOr(a.c.status, kPagedBadPosition);
    }
    if (threadIdx.x == 0) before[0] = 0;
    __syncthreads();
    if (threadIdx.x < 32) {
        long long sum = 0;
        for (int s0 = 0; s0 < a.r.sequences; s0 += 32) {
            const int s = s0 + threadIdx.x;
            const long long v = sum + paged_detail::prefix(s < a.r.sequences ? before[s + 1] : 0);
            if (s < a.r.sequences) before[s + 1] = static_cast<int>(v);
            sum = __shfl_sync(0xffffffffu, v, 31);
        }
        if (sum > 0x7fffffffLL && threadIdx.x == 0) before[a.r.sequences] = 0, atomicOr(a.c.status, kPagedBadPosition);
    }
    __syncthreads();
    return PagedShare{before[a.r.sequences], before, of};
}
__device__ __forceinline__ PagedItem paged_item_at(const PagedAttnArgs& a, const PagedShare& w, int tile) {
    int lo = 0, hi = a.r.sequences - 1;  // the last sequence whose items begin at or before the tile
    while (lo < hi) {
        const int mid = (lo + hi + 1) / 2;
        if (w.before[mid] <= tile) lo = mid;
        else hi = mid - 1;
    }
    const int4 of = w.of[lo];
    const int i = (tile - w.before[lo]) / (of.w + kPagedStart);
    return PagedItem{lo, i, w.before[lo] + i * (of.w + kPagedStart), of.w, PagedSequence{of.x, of.y, of.z, true}};
}

__device__ __forceinline__ int paged_share_of(int total, int blocks, int b) { return total / blocks * b + min(b, total % blocks); }  // block b's first tile
__device__ __forceinline__ int paged_block_of(int total, int blocks, int x) {  // the block that has tile x
    const int each = total / blocks, more = total % blocks, bound = (each + 1) * more;
    return x < bound ? x / (each + 1) : more + (x - bound) / max(each, 1);
}

template <int TYPE, int BLOCKS> __host__ __device__ constexpr int paged_rows_bytes() { return kPagedTile * BLOCKS * paged_row_bytes(TYPE); }  // keys or values of a tile
template <int TYPE, int BLOCKS, int NT>  // NT: tiles of 8 rows
struct PagedFew {
    static constexpr int HD = BLOCKS * kPagedBlock, kRows = NT * 8, kThreads = 32 * 9;
    // A unit holds the keys of a tile (Q8: and the scales of keys and values) or the values. Each group has a ring of its own, so that its waits see every phase of its barriers: a wait tells
    // phases apart by their parity alone, and a group that skipped the other's phases would take an old one for its own.
    static constexpr int kUnit = paged_rows_bytes<TYPE, BLOCKS>() + (TYPE == kPagedQ8 ? 2 * kPagedTile * 4 : 0);
    static constexpr int kFit = 50 * 1024 / kUnit, kUnits = kFit > 8 ? 8 : kFit < 3 ? 3 : kFit;  // about 100 KB under way per block, two blocks per multiprocessor
    static constexpr int kPitch = HD * 2 + (TYPE == kPagedQ8 ? 32 : 16);  // bytes of a row of queries: eight rows fall into different banks
    static constexpr int kJoinPitch = HD + 4, kJoin = 8 * kRows * (kJoinPitch * 4 + 8);
    static constexpr int kBody = 2 * kUnits * kUnit > kJoin ? 2 * kUnits * kUnit : kJoin;
    static constexpr int kSmem = 1024 + kBody + kRows * kPitch + kRows * 4 + 4 * kUnits * 8 + 64;
    static constexpr int kBlocksPerSm = 2 * (kSmem + (kPagedShared + 1) * 20 + 1024 + 128) <= 228 * 1024 && (NT == 1 || NT * BLOCKS <= 2) ? 2 : 1;
};

// The pages of the tiles of [begin, end), TILE positions each, for a whole warp that asks tile after tile: 32 entries of the table at a time, one to a lane, the next 32 under way meanwhile (with a read for every tile, which
// was checked at once, a ring filled at a tile in 1700 cycles). Pieces in front of position `seen` are nobody's to look at: their pages may have been given back.
// A page that the cache does not have is reported; page 0 stands in for it, and `bad` (of the lane that asked for it) says that the results are not to be written.
template <int TILE>
struct PagedPages {
    const PagedView& c;
    const int* table;
    bool bad;
    int begin, end, seen, lane, step, per, now, next;  // step: positions of a piece, a page or 64 of it; per: pieces of a tile
    __device__ __forceinline__ PagedPages(const PagedView& c, const int* table, int begin, int end, int seen)
        : c(c), table(table), bad(false), begin(begin), end(end), seen(seen), lane(threadIdx.x & 31), step(min(1 << c.page_log2, kPagedTile)), per(TILE / step), now(0) {
        next = fetch(0);
    }
    __device__ __forceinline__ int fetch(int piece) const {
        const long long k = begin + (static_cast<long long>(piece) + lane) * step;
        return k < end && k + step > seen ? table[k >> c.page_log2] : 0;
    }
    __device__ __forceinline__ int of(int tile) {  // lane i: the page of the tile's piece i
        const int first = tile * per, at = first & 31;
        if (at == 0) {
            now = next, next = fetch(first + 32);
            if (now < 0 || now >= c.pages) {
                atomicOr(c.status, kPagedBadPage);
                bad = true, now = 0;
            }
        }
        return __shfl_sync(0xffffffffu, now, (at + lane) & 31);
    }
};

// Brings the tiles of [begin, end), of which the positions from `seen` on are looked at, of one KV head into the two rings, tile i into ring i & 1, keys and values one unit after the other; run by one
// whole warp. base0, base1: units that the rings have seen before. Returns with its own copies landed, whether a page that this lane asked for is not there.
template <int TYPE, int BLOCKS, int NT>
__device__ __forceinline__ bool paged_load_tiles(const PagedView& c, const int* table, int head, int begin, int end, int seen, uint32_t rings, uint32_t full, uint32_t empty,
                                                 int base0, int base1, volatile unsigned int* abort_flag, unsigned int limit) {
    using namespace gemm_detail;
    using F = PagedFew<TYPE, BLOCKS, NT>;
    constexpr int kRow = paged_row_bytes(TYPE), kRows = paged_rows_bytes<TYPE, BLOCKS>(), U = F::kUnits;
    const int lane = threadIdx.x & 31, P = 1 << c.page_log2, PR = min(P, kPagedTile);
    PagedPages<kPagedTile> pages_of(c, table, begin, end, seen);
    int tile = 0, asked0 = base0, asked1 = base1;  // units asked for, of either ring
    bool okay = true;
    for (int k0 = begin; k0 < end && okay; k0 += kPagedTile, ++tile) {
        const int pages = pages_of.of(tile), pieces = (min(kPagedTile, end - k0) + PR - 1) / PR;
#pragma unroll
        for (int value = 0; value < 2; ++value) {
            const int ring = tile & 1, n = (ring ? base1 : base0) + (tile >> 1) * 2 + value, slot = ring * U + n % U;
            if (!(okay = __all_sync(0xffffffffu, mbar_wait(empty + 8 * slot, ((n / U) & 1) ^ 1, abort_flag, limit)))) break;
            const uint32_t to = rings + slot * F::kUnit, bar = full + 8 * slot;
            if (lane == 0) mbar_expect_tx(bar, pieces * PR * (BLOCKS * kRow + (TYPE == kPagedQ8 && value == 0 ? 8 : 0)));
            __syncwarp();
            (ring ? asked1 : asked0) = n + 1;
            if (lane < pieces)
                bulk_load(to + lane * PR * BLOCKS * kRow, (value ? c.v : c.k) + paged_rows_at(c, TYPE, pages, head, (k0 + lane * PR) & (P - 1)), PR * BLOCKS * kRow, bar);
            if (TYPE == kPagedQ8 && value == 0 && lane < pieces) {
                const size_t from = paged_scales_at(c, pages, head) + ((k0 + lane * PR) & (P - 1));
                bulk_load(to + kRows + lane * PR * 4, c.ks + from, PR * 4, bar);
                bulk_load(to + kRows + (kPagedTile + lane * PR) * 4, c.vs + from, PR * 4, bar);
            }
        }
    }
    for (int ring = 0; ring < 2; ++ring)
        for (int asked = ring ? asked1 : asked0, n = max(ring ? base1 : base0, asked - U); n < asked; ++n) mbar_wait(full + 8 * (ring * U + n % U), (n / U) & 1, abort_flag, limit, false);
    return pages_of.bad;
}

template <int TYPE, int BLOCKS, int NT, bool FAR>  // FAR: the cap is far above the scores
__global__ void __launch_bounds__(PagedFew<TYPE, BLOCKS, NT>::kThreads, PagedFew<TYPE, BLOCKS, NT>::kBlocksPerSm) paged_few_kernel(const __grid_constant__ PagedAttnArgs a) {
    using namespace gemm_detail;
    using namespace paged_detail;
    using F = PagedFew<TYPE, BLOCKS, NT>;
    constexpr int HD = F::HD, kRow = paged_row_bytes(TYPE), kRows = paged_rows_bytes<TYPE, BLOCKS>(), U = F::kUnits, kPitch = F::kPitch, KS = HD / 16, kThreads = F::kThreads;
    constexpr bool Q8 = TYPE == kPagedQ8, BF = TYPE == kPagedBf16, kHoldQ = KS * NT <= 16 && F::kBlocksPerSm * KS <= 16;
    extern __shared__ unsigned char few_smem_raw[];
    const uint32_t ring = (smem_u32(few_smem_raw) + 1023u) & ~1023u;
    unsigned char* smem = few_smem_raw + (ring - smem_u32(few_smem_raw));
    unsigned char* s_q = smem + F::kBody;                                       // [kRows][kPitch]
    float* s_rowf = reinterpret_cast<float*>(s_q + F::kRows * kPitch);          // [kRows]: what a row's score is multiplied by
    uint64_t* bars = reinterpret_cast<uint64_t*>(s_rowf + F::kRows);
    volatile unsigned int* abort_flag = reinterpret_cast<volatile unsigned int*>(bars + 4 * U);
    __shared__ int s_before[kPagedShared + 1];
    __shared__ int4 s_of[kPagedShared];
    const uint32_t full = smem_u32(bars), empty = full + 16 * U;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

    if (tid == 0) {
        for (int s = 0; s < 2 * U; ++s) mbar_init(full + 8 * s, 1), mbar_init(empty + 8 * s, 4);
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    int at = 0, until = 1, first = 0;  // this block's tiles among all
    PagedShare shared{0, s_before, s_of};
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    if (a.share) {
        shared = paged_share_begin(a, s_before, s_of, kThreads);
        at = first = paged_share_of(shared.total, gridDim.x, blockIdx.x), until = paged_share_of(shared.total, gridDim.x, blockIdx.x + 1);
    }
    int base0 = 0, base1 = 0;  // units that the rings have seen
    while (at < until) {
    int seq, kvh, parts_place = -1;  // place of the workspace that the segment's result goes to, or none
    PagedSequence sq;
    PagedRange range;
    if (a.share) {
        const PagedItem item = paged_item_at(a, shared, at);
        seq = item.seq, kvh = item.kvh, sq = item.q;
        const int tile0 = item.begin + kPagedStart, t = max(at - tile0, 0), n = min(item.tiles, until - tile0) - t;
        if (n <= 0) break;  // (the block's places end in front of the item's tiles)
        range = paged_seen(a, sq);
        range.end = min(range.end, range.begin + (t + n) * kPagedTile), range.begin += t * kPagedTile;
        if (n < item.tiles) parts_place = static_cast<int>(blockIdx.x) * 2 + (at == first ? 0 : 1);
        at = tile0 + t + n;
    } else {
        at = until, seq = blockIdx.y, kvh = blockIdx.x;
        sq = paged_sequence(a.c, a.r, seq);
        if (!sq.ok || sq.news < a.few || sq.news > a.many) {
            if (sq.news > a.r.most && tid == 0) atomicOr(a.c.status, kPagedBadPosition);
            return;
        }
        range = paged_seen(a, sq);
    }
    const int rows = sq.news * a.group, p0 = sq.length - sq.news;
    range.end = max(range.begin, range.end);
    const int tiles = (range.end - range.begin + kPagedTile - 1) / kPagedTile;
    bool bad = false;
    __syncthreads();  // the barriers are there; the segment before has left the ring
    if (warp == 8) {
        bad = paged_load_tiles<TYPE, BLOCKS, NT>(a.c, a.r.table + static_cast<size_t>(seq) * a.r.stride, kvh, range.begin, range.end, paged_first_seen(a, sq, 0), ring, full, empty, base0, base1, abort_flag, a.spin_limit);
    } else {
        // queries: a warp takes rows warp, warp + 8, ...; a lane 8 values or none; all of them are asked for before the first is used
        auto load_rows = [&](auto of) {
            constexpr int T = decltype(of)::value;
            PagedRaw<T> raw[NT];
#pragma unroll
            for (int k = 0; k < NT; ++k) {
                const int r = min(warp + k * 8, rows - 1);
                raw[k] = paged_raw<T>(a.q, (static_cast<size_t>(sq.first) + r / a.group) * a.q_token + (kvh * a.group + r % a.group) * a.q_head + min(lane, HD / 8 - 1) * 8);
            }
#pragma unroll
            for (int k = 0; k < NT; ++k) {
                const int i = warp + k * 8;
                float x[8], f = 1.0f;
                paged_load8(raw[k].v, T, x);
#pragma unroll
                for (int e = 0; e < 8; ++e) x[e] = i < rows ? x[e] : 0.0f;
                if constexpr (Q8) {
                    float m = 0.0f;
#pragma unroll
                    for (int e = 0; e < 8; ++e) m = fmaxf(m, fabsf(x[e]));
#pragma unroll
                    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
                    const uint32_t ex = __float_as_uint(m) >> 23;  // the row's power of two, 2^(ex - 127); none for zeros, denormals and what is not finite
                    if (ex > 1 && ex < 254) {
                        f = __uint_as_float(ex << 23);
                        const float inv = __uint_as_float((254 - ex) << 23);
#pragma unroll
                        for (int e = 0; e < 8; ++e) x[e] *= inv;
                    }
                }
                if (lane < HD / 8) paged_store8(s_q + i * kPitch + lane * 16, BF ? kPagedBf16 : kPagedF16, x);
                if (lane == 0) s_rowf[i] = f * a.scale;
            }
        };
        if constexpr (TYPE != kPagedQ8) load_rows(PagedTag<TYPE>());
        else if (a.q_type == kPagedF16) load_rows(PagedTag<kPagedF16>());
        else if (a.q_type == kPagedBf16) load_rows(PagedTag<kPagedBf16>());
        else load_rows(PagedTag<kPagedF32>());
        asm volatile("bar.sync 1, 256;" ::: "memory");

        const int turn = warp >> 2, kg = warp & 3, g = lane >> 2, c4 = lane & 3;  // positions g and g + 8 of the warp's 16, rows 2 c4 and 2 c4 + 1 of a row tile
        const uint32_t q_at = smem_u32(s_q);
        // the right operand of a slice of 16 values: values 2 c, 2 c + 1 and 2 c + 8, 2 c + 9 of row g; Q8: 4 c .. 4 c + 3, as the bytes of the codes come
        auto load_q = [&](uint32_t (&r)[2], int ks, int n) {
            if constexpr (Q8) {
                const uint2 u = lds64(q_at + (n * 8 + g) * kPitch + ks * 32 + c4 * 8);
                r[0] = u.x, r[1] = u.y;
            } else {
                asm volatile("ld.shared.u32 %0, [%1];" : "=r"(r[0]) : "r"(q_at + (n * 8 + g) * kPitch + ks * 32 + c4 * 4) : "memory");
                asm volatile("ld.shared.u32 %0, [%1];" : "=r"(r[1]) : "r"(q_at + (n * 8 + g) * kPitch + ks * 32 + 16 + c4 * 4) : "memory");
            }
        };
        uint32_t qf[kHoldQ ? KS : 1][kHoldQ ? NT : 1][2];
        if constexpr (kHoldQ) {
#pragma unroll
            for (int ks = 0; ks < KS; ++ks)
#pragma unroll
                for (int n = 0; n < NT; ++n) load_q(qf[ks][n], ks, n);
        }
        float rowf[NT][2], m[NT][2], l[NT][2];
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int i = 0; i < 2; ++i) rowf[n][i] = s_rowf[n * 8 + c4 * 2 + i], m[n][i] = -INFINITY, l[n][i] = 0.0f;
        // positions that every row sees; outside of them the masks are worked out
        const int all_last = p0, all_first = a.window > 0 ? sq.length - a.window : 0;
        float o[KS][NT][4];
#pragma unroll
        for (int j = 0; j < KS; ++j)
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[j][n][e] = 0.0f;

        bool okay = true;
        int n = turn ? base1 : base0;  // units of this group's ring
        for (int k0 = range.begin + turn * kPagedTile; k0 < range.end; k0 += 2 * kPagedTile, n += 2) {
            const int key_slot = turn * U + n % U, value_slot = turn * U + (n + 1) % U, key0 = k0 + kg * 16;
            const uint32_t keys = ring + key_slot * F::kUnit, values = ring + value_slot * F::kUnit;
            const bool there = key0 < range.end;  // (what lies behind the last page was not copied)
            okay = __all_sync(0xffffffffu, mbar_wait(full + 8 * key_slot, (n / U) & 1, abort_flag, a.spin_limit));
            if (!okay) break;
            const int row = kg * 16 + (lane & 15), swz = Q8 ? (row >> 1) & 3 : row & 7;
            uint32_t pb[NT][2];
            if (there) {
                float sc[NT][4];
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e) sc[n][e] = 0.0f;
                auto score = [&](const uint32_t (&k)[4], int ks) {
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        uint32_t b[2];
                        if constexpr (kHoldQ) b[0] = qf[ks][n][0], b[1] = qf[ks][n][1];
                        else load_q(b, ks, n);
                        mma<BF>(sc[n], k, b[0], b[1]);
                    }
                };
                // (fragments are fetched a few at a time, before they are used: loads stay in their order, and one by one each would be waited for)
                constexpr int kFrags = 4;
                if constexpr (Q8) {
#pragma unroll
                    for (int k0_ = 0; k0_ < KS / 2; k0_ += kFrags < KS / 2 ? kFrags : KS / 2) {
                        constexpr int kHere = kFrags < KS / 2 ? kFrags : KS / 2;
                        uint32_t r[kHere][4];  // matrices: positions 0-7 and 8-15 of a slice, then of the next slice
#pragma unroll
                        for (int k = 0; k < kHere; ++k) {
                            const int ks = (k0_ + k) * 2;
                            ldsm4(r[k], keys + paged_row_at(TYPE, BLOCKS, ks >> 2, row) + ((((ks & 3) + (lane >> 4)) ^ swz) << 4));
                        }
#pragma unroll
                        for (int k = 0; k < kHere; ++k)
#pragma unroll
                            for (int h = 0; h < 2; ++h) {
                                const uint32_t u0 = r[k][h * 2] ^ 0x80808080u, u1 = r[k][h * 2 + 1] ^ 0x80808080u;
                                const uint32_t f[4] = {codes_to_half2(u0, 0x4140), codes_to_half2(u1, 0x4140), codes_to_half2(u0, 0x4342), codes_to_half2(u1, 0x4342)};
                                score(f, (k0_ + k) * 2 + h);
                            }
                    }
                } else {
#pragma unroll
                    for (int k0_ = 0; k0_ < KS; k0_ += kFrags) {
                        uint32_t r[kFrags][4];  // matrices: positions 0-7 and 8-15 of the slice's first 8 values, then of the others
#pragma unroll
                        for (int k = 0; k < kFrags; ++k) ldsm4(r[k], keys + paged_row_at(TYPE, BLOCKS, (k0_ + k) >> 2, row) + (((((k0_ + k) & 3) * 2 + (lane >> 4)) ^ swz) << 4));
#pragma unroll
                        for (int k = 0; k < kFrags; ++k) score(r[k], k0_ + k);
                    }
                }
                // the exponents, with masks
                float kf[2] = {1.0f, 1.0f}, lv[2] = {0.0f, 0.0f}, iv[2] = {1.0f, 1.0f};
                if constexpr (Q8) {
                    const float* f = reinterpret_cast<const float*>(smem + key_slot * F::kUnit + kRows) + kg * 16 + g;
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const float v = key0 + g + 8 * i < range.end ? f[kPagedTile + 8 * i] : 1.0f;  // (the scales behind the last page may be anything)
                        kf[i] = f[8 * i], lv[i] = lg2(v), iv[i] = rcp(v);
                    }
                }
                const bool masked = key0 + 15 > all_last || key0 + 15 >= range.end || key0 < all_first;
                float top[NT][2];
#pragma unroll
                for (int n = 0; n < NT; ++n) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        if constexpr (Q8) sc[n][e] *= kf[e >> 1];
                        sc[n][e] *= rowf[n][e & 1];
                    }
                    if (a.cap > 0.0f) {
#pragma unroll
                        for (int e = 0; e < 4; ++e) sc[n][e] = a.cap * tanh_of<FAR>(sc[n][e]);
                    }
                    if constexpr (Q8) {
#pragma unroll
                        for (int e = 0; e < 4; ++e) sc[n][e] += lv[e >> 1];
                    }
                    if (masked) {
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const int rr = n * 8 + c4 * 2 + (e & 1), p = p0 + rr / a.group, j = key0 + g + 8 * (e >> 1);
                            if (rr >= rows || j > p || j >= range.end || (a.window > 0 && j <= static_cast<int>(static_cast<unsigned int>(p) - a.window))) sc[n][e] = -INFINITY;
                        }
                    }
#pragma unroll
                    for (int i = 0; i < 2; ++i) top[n][i] = fmaxf(sc[n][i], sc[n][2 + i]);
                }
#pragma unroll
                for (int x = 4; x < 32; x <<= 1)
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int i = 0; i < 2; ++i) top[n][i] = fmaxf(top[n][i], __shfl_xor_sync(0xffffffffu, top[n][i], x));
                bool grew = false;
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int i = 0; i < 2; ++i) grew = grew || top[n][i] > m[n][i] + kPagedLazy || (m[n][i] == -INFINITY && top[n][i] > -INFINITY);
                if (__any_sync(0xffffffffu, grew)) {
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        float keep[2];
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            const bool more = top[n][i] > m[n][i] + kPagedLazy || (m[n][i] == -INFINITY && top[n][i] > -INFINITY);
                            keep[i] = more ? ex2(m[n][i] - top[n][i]) : 1.0f;  // 0 the first time
                            if (more) m[n][i] = top[n][i], l[n][i] *= keep[i];
                        }
#pragma unroll
                        for (int j = 0; j < KS; ++j)
#pragma unroll
                            for (int e = 0; e < 4; ++e) o[j][n][e] *= keep[e & 1];
                    }
                }
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    float w[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float ref = m[n][e & 1];
                        w[e] = sc[n][e] == -INFINITY ? 0.0f : ex2(sc[n][e] - ref);
                        l[n][e & 1] = fmaf(w[e], iv[e >> 1], l[n][e & 1]);
                    }
#pragma unroll
                    for (int h = 0; h < 2; ++h) {  // rows 2 c, 2 c + 1 of position g (+ 8) become positions 2 c, 2 c + 1 (+ 8) of row g
                        const uint32_t v = paged_pack2<BF ? kPagedBf16 : kPagedF16>(w[2 * h], w[2 * h + 1]);
                        asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(pb[n][h]) : "r"(v));
                    }
                }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(empty + 8 * key_slot);
            okay = __all_sync(0xffffffffu, mbar_wait(full + 8 * value_slot, ((n + 1) / U) & 1, abort_flag, a.spin_limit));
            if (!okay) break;
            if (there) {  // the weighted rows
                if constexpr (Q8) {
                    constexpr int kHere = KS / 2 < 4 ? KS / 2 : 4;
#pragma unroll
                    for (int j0 = 0; j0 < KS / 2; j0 += kHere) {
                        uint32_t r[kHere][4];  // matrices: positions 0-7 and 8-15 of slice j, then of slice j + 1; a pair of bytes is two values of a position
#pragma unroll
                        for (int k = 0; k < kHere; ++k) {
                            const int j = (j0 + k) * 2;
                            ldsm4_trans(r[k], values + paged_row_at(TYPE, BLOCKS, j >> 2, row) + ((((j & 3) + (lane >> 4)) ^ swz) << 4));
                        }
#pragma unroll
                        for (int k = 0; k < kHere; ++k)
#pragma unroll
                            for (int h = 0; h < 2; ++h) {
                                const uint32_t u0 = r[k][h * 2] ^ 0x80808080u, u1 = r[k][h * 2 + 1] ^ 0x80808080u;
                                const uint32_t v[4] = {codes_to_half2(u0, 0x4240), codes_to_half2(u0, 0x4341), codes_to_half2(u1, 0x4240), codes_to_half2(u1, 0x4341)};  // even values, odd values
#pragma unroll
                                for (int n = 0; n < NT; ++n) mma<false>(o[(j0 + k) * 2 + h][n], v, pb[n][0], pb[n][1]);
                            }
                    }
                } else {
                    const int vrow = kg * 16 + (lane & 7) + ((lane >> 4) << 3);  // matrices: (positions 0-7, values 0-7), (0-7, 8-15), (8-15, 0-7), (8-15, 8-15)
#pragma unroll
                    for (int j0 = 0; j0 < KS; j0 += 4) {
                        uint32_t r[4][4];
#pragma unroll
                        for (int k = 0; k < 4; ++k) ldsm4_trans(r[k], values + paged_row_at(TYPE, BLOCKS, (j0 + k) >> 2, vrow) + (((((j0 + k) & 3) * 2 + ((lane >> 3) & 1)) ^ (lane & 7)) << 4));
#pragma unroll
                        for (int k = 0; k < 4; ++k)
#pragma unroll
                            for (int n = 0; n < NT; ++n) mma<BF>(o[j0 + k][n], r[k], pb[n][0], pb[n][1]);
                    }
                }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(empty + 8 * value_slot);
        }
        if (!okay && lane == 0) atomicOr(a.c.status, kPagedGaveUp);
#pragma unroll
        for (int x = 4; x < 32; x <<= 1)
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int i = 0; i < 2; ++i) l[n][i] += __shfl_xor_sync(0xffffffffu, l[n][i], x);
        // every tile was read (or a wait gave up, and nothing below matters): the ring becomes the place where the warps meet
        asm volatile("bar.sync 1, 256;" ::: "memory");
        float* join = reinterpret_cast<float*>(smem) + static_cast<size_t>(warp) * F::kRows * F::kJoinPitch;
        float2* ml = reinterpret_cast<float2*>(smem + 8 * F::kRows * F::kJoinPitch * 4) + warp * F::kRows;
        if (*abort_flag == 0) {
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const int r = n * 8 + c4 * 2 + i;
                    if (g == 0) ml[r] = make_float2(m[n][i], l[n][i]);
                    float* to = join + r * F::kJoinPitch;
#pragma unroll
                    for (int j = 0; j < KS; ++j) {
                        if constexpr (Q8) {
                            *reinterpret_cast<float2*>(to + j * 16 + 2 * g) = make_float2(o[j][n][i], o[j][n][2 + i]);
                        } else {
                            to[j * 16 + g] = o[j][n][i], to[j * 16 + 8 + g] = o[j][n][2 + i];
                        }
                    }
                }
        }
    }
    const bool left_out = __syncthreads_or(bad);  // the segment's sequence has a page that is not there
    if (*abort_flag != 0) return;
    // rows out: eight values to a thread
    const float* joined = reinterpret_cast<const float*>(smem);
    const float2* mls = reinterpret_cast<const float2*>(smem + 8 * F::kRows * F::kJoinPitch * 4);
    for (int i = tid; i < rows * (HD / 8); i += kThreads) {
        const int r = i / (HD / 8), e0 = i % (HD / 8) * 8;
        float top = -INFINITY, w[8], sum = 0.0f, x[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) top = fmaxf(top, mls[k * F::kRows + r].x);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const float2 v = mls[k * F::kRows + r];
            w[k] = v.x == -INFINITY ? 0.0f : ex2(v.x - top);
            sum = fmaf(w[k], v.y, sum);
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = 0.0f;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const float* from = joined + static_cast<size_t>(k * F::kRows + r) * F::kJoinPitch + e0;
            const float4 u = *reinterpret_cast<const float4*>(from), v = *reinterpret_cast<const float4*>(from + 4);
            x[0] = fmaf(w[k], u.x, x[0]), x[1] = fmaf(w[k], u.y, x[1]), x[2] = fmaf(w[k], u.z, x[2]), x[3] = fmaf(w[k], u.w, x[3]);
            x[4] = fmaf(w[k], v.x, x[4]), x[5] = fmaf(w[k], v.y, x[5]), x[6] = fmaf(w[k], v.z, x[6]), x[7] = fmaf(w[k], v.w, x[7]);
        }
        const size_t t = static_cast<size_t>(sq.first) + r / a.group;
        const int h = kvh * a.group + r % a.group;
        if (parts_place < 0) {
            if (left_out) continue;
            const float inv = sum > 0.0f ? 1.0f / sum : sum == 0.0f ? 0.0f : sum;  // (a sum that is no number stays one)
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] *= inv;
            paged_store8(static_cast<unsigned char*>(a.out) + (t * a.o_token + h * a.o_head + e0) * paged_size_of(a.out_type), a.out_type, x);
        } else {
            const size_t row = static_cast<size_t>(parts_place) * F::kRows + r;
            paged_store8(a.part_o + row * HD + e0, kPagedF32, x);
            if (e0 == 0) a.part_ml[row] = left_out ? paged_left_out() : make_float2(top, sum);
        }
    }
    base0 += (tiles + 1) / 2 * 2, base1 += tiles / 2 * 2;
    fence_async_shared();  // the next segment's copies go where the results met
    __syncthreads();
    }
}

// Joins results: weights 2^(m_i - m) over `count` of them, the i-th in row row_of(i) of the workspace, for the values of one warp's lanes (kPer each), by the WARPS warps of a block in turn, a few results at
// a time so that their reads overlap; in the same order whenever it is asked for. The row's normalised values are the first warp's; returns whether they are to be written.
template <int HD, int WARPS, typename RowOf>
__device__ __forceinline__ bool paged_join(const float* part_o, const float2* part_ml, RowOf row_of, int count, float (&x)[HD / 32], float* shared) {
    using namespace paged_detail;
    constexpr int kPer = HD / 32;
    const int lane = threadIdx.x & 31, warp = WARPS > 1 ? threadIdx.x >> 5 : 0;
    float top = -INFINITY;
    bool left_out = false;
    for (int i = lane; i < count; i += 32) {
        const float2 v = part_ml[row_of(i)];
        top = fmaxf(top, v.x), left_out = left_out || v.y < 0.0f;
    }
    left_out = __any_sync(0xffffffffu, left_out);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    float sum = 0.0f;
#pragma unroll
    for (int e = 0; e < kPer; ++e) x[e] = 0.0f;
    constexpr int kBatch = HD > 128 ? 4 : 8;
    for (int i0 = warp; i0 < count; i0 += kBatch * WARPS) {
        float2 ml[kBatch];
        float v[kBatch][kPer];
#pragma unroll
        for (int k = 0; k < kBatch; ++k) {
            const int i = i0 + k * WARPS;
            ml[k] = i < count ? part_ml[row_of(i)] : make_float2(-INFINITY, 0.0f);
        }
#pragma unroll
        for (int k = 0; k < kBatch; ++k) {
            const bool there = !(ml[k].x == -INFINITY && ml[k].y == 0.0f);  // a range in which nothing was visible has no values
            const float* from = part_o + row_of(min(i0 + k * WARPS, count - 1)) * HD + lane * kPer;
#pragma unroll
            for (int e = 0; e < kPer; ++e) v[k][e] = there ? from[e] : 0.0f;
        }
#pragma unroll
        for (int k = 0; k < kBatch; ++k) {
            const float w = ml[k].x == -INFINITY && ml[k].y == 0.0f ? 0.0f : ex2(ml[k].x - top);
            sum = fmaf(w, ml[k].y, sum);
#pragma unroll
            for (int e = 0; e < kPer; ++e) x[e] = fmaf(w, v[k][e], x[e]);
        }
    }
    if constexpr (WARPS > 1) {
        float* mine = shared + (warp * 32 + lane) * (kPer + 1);
#pragma unroll
        for (int e = 0; e < kPer; ++e) mine[e] = x[e];
        mine[kPer] = sum;
        __syncthreads();
        if (warp != 0) return false;
#pragma unroll
        for (int w = 1; w < WARPS; ++w) {
            const float* other = shared + (w * 32 + lane) * (kPer + 1);
#pragma unroll
            for (int e = 0; e < kPer; ++e) x[e] += other[e];
            sum += other[kPer];
        }
    }
    const float inv = sum > 0.0f ? 1.0f / sum : sum == 0.0f ? 0.0f : sum;
#pragma unroll
    for (int e = 0; e < kPer; ++e) x[e] *= inv;
    return !left_out;
}
template <int PER>
__device__ __forceinline__ void paged_store_row(unsigned char* out, int type, const float (&x)[PER]) {
    if (type == kPagedF32) {
#pragma unroll
        for (int e = 0; e < PER; ++e) reinterpret_cast<float*>(out)[e] = x[e];
    } else {
#pragma unroll
        for (int e = 0; e < PER; e += 2) reinterpret_cast<uint32_t*>(out)[e / 2] = type == kPagedF16 ? paged_pack2<kPagedF16>(x[e], x[e + 1]) : paged_pack2<kPagedBf16>(x[e], x[e + 1]);
    }
}

// Joins the segments of the items that were cut. Where one block's tiles end and the next one's begin inside an item (`cuts` such places in the item), a block of this kernel stands for that place, and
// takes every cuts-th row of the item: a warp a row, or all warps a row where there are many segments. `blocks`, `block_rows`: of the launch whose tiles were shared out.
template <int BLOCKS>
__global__ void __launch_bounds__(256) paged_combine_kernel(const __grid_constant__ PagedAttnArgs a, int blocks, int block_rows) {
    constexpr int HD = BLOCKS * kPagedBlock, kPer = HD / 32;
    __shared__ float shared[8 * 32 * (kPer + 1)];
    __shared__ int before[kPagedShared + 1];
    __shared__ int4 of[kPagedShared];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, b = blockIdx.x + 1;
    const PagedShare w = paged_share_begin(a, before, of, 256);
    asm volatile("griddepcontrol.wait;" ::: "memory");  // launched while the segments are still being worked on; what was read above is input. Every block waits, so that none ends before them
    const int x = paged_share_of(w.total, blocks, b);
    if (x <= 0 || x >= w.total) return;
    const PagedItem item = paged_item_at(a, w, x);
    const int tile0 = item.begin + kPagedStart, b0 = paged_block_of(w.total, blocks, tile0), b1 = paged_block_of(w.total, blocks, tile0 + item.tiles - 1), cuts = b1 - b0;
    const int place0 = paged_share_of(w.total, blocks, b0) >= item.begin ? 0 : 1, rows = item.q.news * a.group, mine = b - b0 - 1;
    if (mine < 0 || mine >= cuts) return;  // the item's tiles are not cut here (the place is in front of them, or the block has none of its own)
    auto out = [&](int r, const float (&v)[kPer]) {
        const size_t t = static_cast<size_t>(item.q.first) + r / a.group;
        const int h = item.kvh * a.group + r % a.group;
        paged_store_row(static_cast<unsigned char*>(a.out) + (t * a.o_token + h * a.o_head + lane * kPer) * paged_size_of(a.out_type), a.out_type, v);
    };
    float v[kPer];
    if (cuts < 8) {
        for (int r = mine + cuts * warp; r < rows; r += cuts * 8) {
            if (paged_join<HD, 1>(a.part_o, a.part_ml, [&](int i) { return static_cast<size_t>((b0 + i) * 2 + (i == 0 ? place0 : 0)) * block_rows + r; }, cuts + 1, v, nullptr)) out(r, v);
        }
    } else {
        for (int r = mine; r < rows; r += cuts) {
            __syncthreads();
            if (paged_join<HD, 8>(a.part_o, a.part_ml, [&](int i) { return static_cast<size_t>((b0 + i) * 2 + (i == 0 ? place0 : 0)) * block_rows + r; }, cuts + 1, v, shared)) out(r, v);
        }
    }
}

}  // namespace qtb
