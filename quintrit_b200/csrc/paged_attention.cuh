// Attention of new tokens over a paged cache, a few rows of queries at a time.
//
// For token i of a sequence at position p and query head h with KV head h / G: z_j = scale q.k_j, or cap tanh(scale q.k_j / cap), over the visible
// positions j <= p and, with a window, j > p - window; out = sum_j exp(z_j) v_j / sum_j exp(z_j), zeros where no position is visible. One pass over the
// rows: a running maximum m, the weights exp(z_j - m) and their sum l, and the products rescaled when m grows (only when it grows by more than 2^8,
// so that weights stay below 256 and a rescale is rare). Logarithms are to base 2: log2(e) goes into the scale.
//
// Q8 rows: k_j = ks_j a_j, v_j = vs_j b_j with integer codes. The codes go into the products as they are (exact in F16), ks_j multiplies the score, and
// vs_j goes into the exponent: with y_j = z_j + log2(vs_j) the weights w_j = 2^(y_j - m), m the maximum of y, are what multiplies b_j, and l = sum w_j / vs_j.
// So the weights that are rounded to F16 lie in [0, 256] whatever the scales are. Queries are scaled by a power of two per row to a maximum in [1, 2),
// which is exact, so BF16 and F32 queries of any size meet F16 codes.
//
// Bound by the rows' bytes: 2 G flops per byte of a 16-bit cache. A block of threads takes one KV head of one sequence and a range of its positions; one
// warp brings the pages, tile by tile of 64 positions, into a ring in shared memory with bulk copies; every other warp has 16 positions of the tiles and
// 16 rows of queries (rows are (token, head of the group)), its own m, l and sums, all in registers of matrix instructions (m16n8k16); at the end
// the warps of a row tile join. Long sequences are cut into ranges for several blocks, whose results meet in the caller's workspace
// (paged_combine_kernel), in the order of the ranges: no atomics.
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
    int splits, split;       // ranges of positions per sequence, positions of a range (a multiple of the tile)
    float* part_o;           // [splits][tokens][q heads][head_dim], when splits > 1
    float2* part_ml;         // [splits][tokens][q heads]
    int few, many;           // new tokens of the sequences that this launch serves: few <= n <= many
    int most;                // new tokens of the longest chunk as announced: the grid has no rows for more
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
// tanh from one exponential: 1 - 2 / (1 + e^2x). Off by about 2^-23 of one; the infinities of the exponential give -1 and 1.
__device__ __forceinline__ float tanh_of(float x) { return 1.0f - 2.0f * rcp(1.0f + ex2(x * (2.0f * kLog2e))); }

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

}  // namespace paged_detail

// The range of positions that rows of tokens [t0, t1) of a sequence can see, cut to the range of split `i`; begin is a multiple of the tile.
struct PagedRange {
    int begin, end;
};
__device__ __forceinline__ PagedRange paged_range(const PagedAttnArgs& a, const PagedSequence& q, int t0, int t1, int split) {
    // The cuts count from the first position that any new token of the sequence sees, so that all row tiles of a sequence agree on them.
    const int p0 = q.length - q.news, low_all = a.window > 0 ? max(0, p0 - a.window + 1) & ~(kPagedTile - 1) : 0;
    const int low = a.window > 0 ? max(0, p0 + t0 - a.window + 1) & ~(kPagedTile - 1) : 0;
    PagedRange g;
    // (64 bits: a range may be as long as 2^31 positions)
    const long long cut = low_all + static_cast<long long>(split) * a.split;
    g.begin = static_cast<int>(max(static_cast<long long>(low), min(cut, static_cast<long long>(q.length))));
    g.end = split + 1 < a.splits ? static_cast<int>(min(static_cast<long long>(q.length), cut + a.split)) : q.length;
    g.end = min(g.end, max(0, p0 + t1));
    return g;
}
// Ranges of the sequence that hold anything.
__device__ __forceinline__ int paged_splits_used(const PagedAttnArgs& a, const PagedSequence& q) {
    const int p0 = q.length - q.news, low_all = a.window > 0 ? max(0, p0 - a.window + 1) & ~(kPagedTile - 1) : 0;
    return max(1, min(a.splits, static_cast<int>((static_cast<long long>(q.length) - low_all + a.split - 1) / a.split)));
}

template <int TYPE, int BLOCKS> __host__ __device__ constexpr int paged_q_pitch() { return BLOCKS * kPagedBlock * 2 + (TYPE == kPagedQ8 ? 32 : 16); }  // bytes: eight rows fall into different banks
template <int TYPE, int BLOCKS> __host__ __device__ constexpr int paged_rows_bytes() { return kPagedTile * BLOCKS * paged_row_bytes(TYPE); }  // keys or values of a tile
template <int TYPE, int BLOCKS> __host__ __device__ constexpr int paged_stage_bytes() { return 2 * paged_rows_bytes<TYPE, BLOCKS>() + (TYPE == kPagedQ8 ? 2 * kPagedTile * 4 : 0); }
template <int TYPE, int BLOCKS> __host__ __device__ constexpr int paged_stages() { return paged_stage_bytes<TYPE, BLOCKS>() > 40000 ? 3 : paged_stage_bytes<TYPE, BLOCKS>() > 20000 ? 3 : 4; }
template <int TYPE, int BLOCKS, int RT> __host__ __device__ constexpr int paged_few_smem() {
    const int ring = paged_stages<TYPE, BLOCKS>() * paged_stage_bytes<TYPE, BLOCKS>(), join = RT * 4 * 16 * (BLOCKS * kPagedBlock * 4 + 16);
    return 1024 + (ring > join ? ring : join) + RT * 16 * paged_q_pitch<TYPE, BLOCKS>() + RT * 16 * 4 + 256;
}

// Brings the tiles of [begin, end) of one KV head into the ring, in turn; run by one whole warp. The pages' numbers of the tile after are asked for
// before a wait. Returns with its own copies landed.
template <int TYPE, int BLOCKS, int STAGES>
__device__ __forceinline__ void paged_load_tiles(const PagedView& c, const int* table, int head, int begin, int end, uint32_t ring, uint32_t full, uint32_t empty,
                                                 volatile unsigned int* abort_flag, unsigned int limit) {
    using namespace gemm_detail;
    constexpr int kRow = paged_row_bytes(TYPE), kRows = paged_rows_bytes<TYPE, BLOCKS>(), kStage = paged_stage_bytes<TYPE, BLOCKS>();
    const int lane = threadIdx.x & 31, P = 1 << c.page_log2, PR = min(P, kPagedTile);
    auto page_of = [&](int k0) {  // lane i: the page of the tile's piece i
        const int k = k0 + lane * PR;
        if (lane * PR >= kPagedTile || k >= end) return 0;
        int page = table[k >> c.page_log2];
        if (page < 0 || page >= c.pages) {
            atomicOr(c.status, kPagedBadPage);
            page = 0;
        }
        return page;
    };
    int next = page_of(begin), it = 0;
    for (int k0 = begin; k0 < end; k0 += kPagedTile, ++it) {
        const int pages = next, s = it % STAGES, pieces = (min(kPagedTile, end - k0) + PR - 1) / PR;
        if (k0 + kPagedTile < end) next = page_of(k0 + kPagedTile);
        if (!__all_sync(0xffffffffu, mbar_wait(empty + 8 * s, ((it / STAGES) & 1) ^ 1, abort_flag, limit))) break;
        const uint32_t stage = ring + s * kStage, bar = full + 8 * s;
        if (lane == 0) mbar_expect_tx(bar, pieces * PR * (2 * BLOCKS * kRow + (TYPE == kPagedQ8 ? 8 : 0)));
        __syncwarp();
        for (int i0 = 0; i0 < pieces * BLOCKS * 2; i0 += 32) {  // a piece's rows of a block, keys then values
            const int i = i0 + lane, piece = i / (2 * BLOCKS), b = i % BLOCKS, value = i / BLOCKS & 1;
            const int page = __shfl_sync(0xffffffffu, pages, min(piece, 3));
            if (i < pieces * BLOCKS * 2) {
                const size_t from = paged_block_at(c, TYPE, page, head, b) + static_cast<size_t>((k0 + piece * PR) & (P - 1)) * kRow;
                bulk_load(stage + value * kRows + (b * kPagedTile + piece * PR) * kRow, (value ? c.v : c.k) + from, PR * kRow, bar);
            }
        }
        if constexpr (TYPE == kPagedQ8) {
            const int piece = lane >> 1, value = lane & 1, page = __shfl_sync(0xffffffffu, pages, min(piece, 3));
            if (piece < pieces) {
                const size_t from = paged_scales_at(c, page, head) + ((k0 + piece * PR) & (P - 1));
                bulk_load(stage + 2 * kRows + (value * kPagedTile + piece * PR) * 4, (value ? c.vs : c.ks) + from, PR * 4, bar);
            }
        }
    }
    for (int back = max(0, it - STAGES); back < it; ++back) mbar_wait(full + 8 * (back % STAGES), (back / STAGES) & 1, abort_flag, limit, false);
}

template <int TYPE, int BLOCKS, int RT>
__global__ void __launch_bounds__(32 + 128 * RT, 1) paged_few_kernel(const __grid_constant__ PagedAttnArgs a) {
    using namespace gemm_detail;
    using namespace paged_detail;
    constexpr int HD = BLOCKS * kPagedBlock, kRow = paged_row_bytes(TYPE), kRows = paged_rows_bytes<TYPE, BLOCKS>(), kStage = paged_stage_bytes<TYPE, BLOCKS>(), S = paged_stages<TYPE, BLOCKS>();
    constexpr int kPitch = paged_q_pitch<TYPE, BLOCKS>(), KS = HD / 16, kThreads = 32 + 128 * RT;
    constexpr bool Q8 = TYPE == kPagedQ8, BF = TYPE == kPagedBf16, kHoldQ = BLOCKS <= 2;
    extern __shared__ unsigned char few_smem_raw[];
    const uint32_t ring = (smem_u32(few_smem_raw) + 1023u) & ~1023u;
    unsigned char* smem = few_smem_raw + (ring - smem_u32(few_smem_raw));
    constexpr int kJoin = RT * 4 * 16 * (HD * 4 + 16), kBody = S * kStage > kJoin ? S * kStage : kJoin;
    unsigned char* s_q = smem + kBody;                                          // [RT * 16][kPitch]
    float* s_rowf = reinterpret_cast<float*>(s_q + RT * 16 * kPitch);           // [RT * 16]: what a row's score is multiplied by
    uint64_t* bars = reinterpret_cast<uint64_t*>(s_rowf + RT * 16);
    volatile unsigned int* abort_flag = reinterpret_cast<volatile unsigned int*>(bars + 2 * S);
    const uint32_t full = smem_u32(bars), empty = full + 8 * S;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

    const int seq = blockIdx.z, kvh = blockIdx.y % a.c.kv_heads, tile = blockIdx.y / a.c.kv_heads;
    const PagedSequence sq = paged_sequence(a.c, a.r, seq);
    if (!sq.ok || sq.news < a.few || sq.news > a.many) {
        if (sq.news > a.most && tid == 0) atomicOr(a.c.status, kPagedBadPosition);
        return;
    }
    const int rows = sq.news * a.group, r0 = tile * RT * 16, r1 = min(rows, r0 + RT * 16);
    if (r0 >= rows) return;
    if (static_cast<int>(blockIdx.x) >= paged_splits_used(a, sq)) return;
    const PagedRange range = paged_range(a, sq, r0 / a.group, (r1 - 1) / a.group + 1, blockIdx.x);
    const int p0 = sq.length - sq.news;

    if (tid == 0) {
        for (int s = 0; s < S; ++s) mbar_init(full + 8 * s, 1), mbar_init(empty + 8 * s, 4 * RT);
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncthreads();
    if (warp == 4 * RT) {
        paged_load_tiles<TYPE, BLOCKS, S>(a.c, a.r.table + static_cast<size_t>(seq) * a.r.stride, kvh, range.begin, range.end, ring, full, empty, abort_flag, a.spin_limit);
    } else {
        // queries: a warp takes rows warp, warp + 4 RT, ...; a lane 8 values or none
        for (int i = warp; i < RT * 16; i += 4 * RT) {
            const int r = r0 + i, t = r / a.group, h = kvh * a.group + r % a.group;
            float x[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = 0.0f;
            if (r < r1 && lane < HD / 8)
                paged_load8(static_cast<const unsigned char*>(a.q) + ((static_cast<size_t>(sq.first) + t) * a.q_token + h * a.q_head + lane * 8) * paged_size_of(a.q_type), a.q_type, x);
            float f = 1.0f;
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
        asm volatile("bar.sync 1, %0;" ::"n"(128 * RT) : "memory");

        const int rt = warp >> 2, kg = warp & 3, g = lane >> 2, c4 = lane & 3;
        const uint32_t q_at = smem_u32(s_q) + rt * 16 * kPitch;
        // a fragment of the queries: F16 / BF16 as ldmatrix gives it; Q8: values 4 c .. 4 c + 3 of a slice of 16 stand where the instruction has 2 c, 2 c + 1, 2 c + 8, 2 c + 9,
        // as the codes' bytes come
        auto load_q = [&](uint32_t (&r)[4], int ks) {
            if constexpr (Q8) {
                const uint2 u = lds64(q_at + g * kPitch + ks * 32 + c4 * 8), w = lds64(q_at + (g + 8) * kPitch + ks * 32 + c4 * 8);
                r[0] = u.x, r[1] = w.x, r[2] = u.y, r[3] = w.y;
            } else {
                ldsm4(r, q_at + (lane & 15) * kPitch + ks * 32 + (lane >> 4) * 16);
            }
        };
        uint32_t qf[kHoldQ ? KS : 1][4];
        if constexpr (kHoldQ) {
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) load_q(qf[ks], ks);
        }
        float rowf[2], m[2], l[2];
        int last[2], first[2];  // the visible positions of the two rows: first <= j <= last
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int r = r0 + rt * 16 + g + 8 * i, p = p0 + r / a.group;
            rowf[i] = s_rowf[rt * 16 + g + 8 * i], m[i] = -INFINITY, l[i] = 0.0f;
            last[i] = r < r1 ? min(p, range.end - 1) : -1;
            first[i] = a.window > 0 ? max(0, p - a.window + 1) : 0;
        }
        float o[KS][2][4];
#pragma unroll
        for (int j = 0; j < KS; ++j)
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[j][n][e] = 0.0f;

        bool okay = true;
        int it = 0;
        for (int k0 = range.begin; k0 < range.end; k0 += kPagedTile, ++it) {
            const int s = it % S, key0 = k0 + kg * 16;
            okay = __all_sync(0xffffffffu, mbar_wait(full + 8 * s, (it / S) & 1, abort_flag, a.spin_limit));
            if (!okay) break;
            const uint32_t stage = ring + s * kStage;
            if (key0 < range.end) {  // (what lies behind the last page was not copied)
                // scores of 16 rows and 16 positions
                float sc[2][4] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
                if constexpr (Q8) {
                    // four matrices: positions 0-7 and 8-15 of the first slice of 16 values, then of the second
                    const int row = kg * 16 + (lane & 15), swz = (row >> 1) & 3;
#pragma unroll
                    for (int b = 0; b < BLOCKS; ++b) {
#pragma unroll
                        for (int two = 0; two < 2; ++two) {
                            uint32_t r[4];
                            ldsm4(r, stage + (b * kPagedTile + row) * kRow + (((two * 2 + (lane >> 4)) ^ swz) << 4));
#pragma unroll
                            for (int h = 0; h < 2; ++h) {
                                const int ks = b * 4 + two * 2 + h;
                                uint32_t qa[4];
                                if constexpr (kHoldQ) {
#pragma unroll
                                    for (int e = 0; e < 4; ++e) qa[e] = qf[ks][e];
                                } else {
                                    load_q(qa, ks);
                                }
#pragma unroll
                                for (int n = 0; n < 2; ++n) {
                                    const uint32_t u = r[h * 2 + n] ^ 0x80808080u;
                                    mma<false>(sc[n], qa, codes_to_half2(u, 0x4140), codes_to_half2(u, 0x4342));
                                }
                            }
                        }
                    }
                } else {
                    const int row = kg * 16 + (lane & 7) + ((lane >> 4) << 3);
#pragma unroll
                    for (int ks = 0; ks < KS; ++ks) {
                        uint32_t r[4], qa[4];
                        ldsm4(r, stage + ((ks >> 2) * kPagedTile + row) * kRow + ((((ks & 3) * 2 + ((lane >> 3) & 1)) ^ (lane & 7)) << 4));
                        if constexpr (kHoldQ) {
#pragma unroll
                            for (int e = 0; e < 4; ++e) qa[e] = qf[ks][e];
                        } else {
                            load_q(qa, ks);
                        }
                        mma<BF>(sc[0], qa, r[0], r[1]);
                        mma<BF>(sc[1], qa, r[2], r[3]);
                    }
                }
                // the scores' exponents, with masks
                float iv[2][2];
                float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
                for (int n = 0; n < 2; ++n) {
                    float kf[2] = {1.0f, 1.0f}, lv[2] = {0.0f, 0.0f};
                    iv[n][0] = iv[n][1] = 1.0f;
                    if constexpr (Q8) {
                        const uint32_t at = stage + 2 * kRows + (kg * 16 + n * 8 + c4 * 2) * 4;
                        const uint2 ku = lds64(at), vu = lds64(at + kPagedTile * 4);
                        kf[0] = __uint_as_float(ku.x), kf[1] = __uint_as_float(ku.y);
                        lv[0] = lg2(__uint_as_float(vu.x)), lv[1] = lg2(__uint_as_float(vu.y));
                        iv[n][0] = rcp(__uint_as_float(vu.x)), iv[n][1] = rcp(__uint_as_float(vu.y));
                    }
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int i = e >> 1, j = key0 + n * 8 + c4 * 2 + (e & 1);
                        float x = sc[n][e];
                        if constexpr (Q8) x *= kf[e & 1];
                        x *= rowf[i];
                        if (a.cap > 0.0f) x = a.cap * tanh_of(x);
                        if constexpr (Q8) x += lv[e & 1];
                        x = j >= first[i] && j <= last[i] ? x : -INFINITY;
                        sc[n][e] = x;
                        top[i] = fmaxf(top[i], x);
                    }
                }
                float keep[2];
                bool grew = false;
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    top[i] = fmaxf(top[i], __shfl_xor_sync(0xffffffffu, top[i], 1));
                    top[i] = fmaxf(top[i], __shfl_xor_sync(0xffffffffu, top[i], 2));
                    keep[i] = 1.0f;
                    if (top[i] > m[i] + kPagedLazy || (m[i] == -INFINITY && top[i] > -INFINITY)) {
                        keep[i] = ex2(m[i] - top[i]);  // 0 the first time
                        m[i] = top[i];
                        l[i] *= keep[i];
                        grew = true;
                    }
                }
                if (__any_sync(0xffffffffu, grew)) {
#pragma unroll
                    for (int j = 0; j < KS; ++j)
#pragma unroll
                        for (int n = 0; n < 2; ++n)
#pragma unroll
                            for (int e = 0; e < 4; ++e) o[j][n][e] *= keep[e >> 1];
                }
                uint32_t pa[4];
#pragma unroll
                for (int n = 0; n < 2; ++n) {
                    float w[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int i = e >> 1;
                        w[e] = sc[n][e] == -INFINITY ? 0.0f : ex2(sc[n][e] - m[i]);
                        if constexpr (Q8) {
                            if (!(w[e] == 0.0f)) l[i] = fmaf(w[e], iv[n][e & 1], l[i]);  // (the scales behind the last position may be anything)
                        } else {
                            l[i] += w[e];
                        }
                    }
                    pa[n * 2] = paged_pack2(BF ? kPagedBf16 : kPagedF16, w[0], w[1]);
                    pa[n * 2 + 1] = paged_pack2(BF ? kPagedBf16 : kPagedF16, w[2], w[3]);
                }
                // the weighted rows
                const int row = kg * 16 + (lane & 15);
#pragma unroll
                for (int j = 0; j < KS; ++j) {
                    uint32_t r[4];
                    if constexpr (Q8) {
                        if ((j & 1) == 0) {  // two slices of 16 values: matrices (positions 0-7, 8-15) x (slice j, j + 1)
                            ldsm4_trans(r, stage + kRows + ((j >> 2) * kPagedTile + row) * kRow + ((((j & 3) + (lane >> 4)) ^ ((row >> 1) & 3)) << 4));
#pragma unroll
                            for (int h = 0; h < 2; ++h) {
                                const uint32_t u0 = r[h * 2] ^ 0x80808080u, u1 = r[h * 2 + 1] ^ 0x80808080u;
                                mma<false>(o[j + h][0], pa, codes_to_half2(u0, 0x4240), codes_to_half2(u1, 0x4240));  // the even values of the slice
                                mma<false>(o[j + h][1], pa, codes_to_half2(u0, 0x4341), codes_to_half2(u1, 0x4341));  // the odd ones
                            }
                        }
                    } else {
                        ldsm4_trans(r, stage + kRows + ((j >> 2) * kPagedTile + row) * kRow + ((((j & 3) * 2 + (lane >> 4)) ^ (row & 7)) << 4));
                        mma<BF>(o[j][0], pa, r[0], r[1]);
                        mma<BF>(o[j][1], pa, r[2], r[3]);
                    }
                }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(empty + 8 * s);
        }
        if (!okay && lane == 0) atomicOr(a.c.status, kPagedGaveUp);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            l[i] += __shfl_xor_sync(0xffffffffu, l[i], 1);
            l[i] += __shfl_xor_sync(0xffffffffu, l[i], 2);
        }
        // every tile was read (or a wait gave up, and nothing below matters): the ring becomes the place where the warps of a row tile meet
        asm volatile("bar.sync 1, %0;" ::"n"(128 * RT) : "memory");
        float* join = reinterpret_cast<float*>(smem) + static_cast<size_t>(warp) * 16 * HD;  // [16][HD]
        float2* ml = reinterpret_cast<float2*>(smem + static_cast<size_t>(RT) * 4 * 16 * HD * 4) + warp * 16;
        if (*abort_flag == 0) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                if (c4 == 0) ml[g + 8 * i] = make_float2(m[i], l[i]);
                float* to = join + (g + 8 * i) * HD;
#pragma unroll
                for (int j = 0; j < KS; ++j) {
                    if constexpr (Q8) {  // (slice j: the even values 4 c, 4 c + 2 and the odd ones 4 c + 1, 4 c + 3)
                        *reinterpret_cast<float4*>(to + ((j * 16 + c4 * 4) ^ (g << 2 & 12))) = make_float4(o[j][0][2 * i], o[j][1][2 * i], o[j][0][2 * i + 1], o[j][1][2 * i + 1]);
                    } else {
#pragma unroll
                        for (int n = 0; n < 2; ++n) *reinterpret_cast<float2*>(to + ((j * 16 + n * 8 + c4 * 2) ^ (g << 2 & 12))) = make_float2(o[j][n][2 * i], o[j][n][2 * i + 1]);
                    }
                }
            }
        }
    }
    __syncthreads();
    if (*abort_flag != 0) return;
    // rows out: eight values to a thread
    const float* joined = reinterpret_cast<const float*>(smem);
    const float2* mls = reinterpret_cast<const float2*>(smem + static_cast<size_t>(RT) * 4 * 16 * HD * 4);
    for (int i = tid; i < (r1 - r0) * (HD / 8); i += kThreads) {
        const int r = i / (HD / 8), e0 = i % (HD / 8) * 8, rt = r >> 4, rr = r & 15;
        float top = -INFINITY, w[4], sum = 0.0f, x[8];
#pragma unroll
        for (int k = 0; k < 4; ++k) top = fmaxf(top, mls[(rt * 4 + k) * 16 + rr].x);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const float2 v = mls[(rt * 4 + k) * 16 + rr];
            w[k] = v.x == -INFINITY ? 0.0f : ex2(v.x - top);
            sum = fmaf(w[k], v.y, sum);
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = 0.0f;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const float* from = joined + (static_cast<size_t>(rt * 4 + k) * 16 + rr) * HD;
            const float4 u = *reinterpret_cast<const float4*>(from + (e0 ^ (rr << 2 & 12))), v = *reinterpret_cast<const float4*>(from + ((e0 + 4) ^ (rr << 2 & 12)));
            x[0] = fmaf(w[k], u.x, x[0]), x[1] = fmaf(w[k], u.y, x[1]), x[2] = fmaf(w[k], u.z, x[2]), x[3] = fmaf(w[k], u.w, x[3]);
            x[4] = fmaf(w[k], v.x, x[4]), x[5] = fmaf(w[k], v.y, x[5]), x[6] = fmaf(w[k], v.z, x[6]), x[7] = fmaf(w[k], v.w, x[7]);
        }
        const size_t t = static_cast<size_t>(sq.first) + (r0 + r) / a.group;
        const int h = kvh * a.group + (r0 + r) % a.group;
        if (a.splits == 1) {
            const float inv = sum > 0.0f ? 1.0f / sum : sum == 0.0f ? 0.0f : sum;  // (a sum that is no number stays one)
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] *= inv;
            paged_store8(static_cast<unsigned char*>(a.out) + (t * a.o_token + h * a.o_head + e0) * paged_size_of(a.out_type), a.out_type, x);
        } else {
            const int heads = a.c.kv_heads * a.group;
            const size_t row = (static_cast<size_t>(blockIdx.x) * a.r.tokens + t) * heads + h;
            paged_store8(a.part_o + row * HD + e0, kPagedF32, x);
            if (e0 == 0) a.part_ml[row] = make_float2(top, sum);
        }
    }
}

// Joins the ranges of a sequence: a warp per (token, query head), in the order of the ranges.
template <int BLOCKS>
__global__ void __launch_bounds__(256) paged_combine_kernel(const __grid_constant__ PagedAttnArgs a) {
    using namespace paged_detail;
    constexpr int HD = BLOCKS * kPagedBlock, kPer = HD / 32;
    const int heads = a.c.kv_heads * a.group, lane = threadIdx.x & 31;
    const int item = blockIdx.x * 8 + (threadIdx.x >> 5), t = item / heads, h = item % heads;
    if (t >= a.r.tokens) return;
    const int s = paged_sequence_of(a.r, t);
    if (s < 0) return;
    const PagedSequence sq = paged_sequence(a.c, a.r, s);
    if (!sq.ok || t < sq.first || t >= sq.first + sq.news || sq.news < a.few || sq.news > a.many) return;
    const int used = paged_splits_used(a, sq);
    const size_t step = static_cast<size_t>(a.r.tokens) * heads, row = static_cast<size_t>(t) * heads + h;
    float top = -INFINITY;
    for (int i = lane; i < used; i += 32) top = fmaxf(top, a.part_ml[i * step + row].x);
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    float sum = 0.0f, x[kPer];
#pragma unroll
    for (int e = 0; e < kPer; ++e) x[e] = 0.0f;
    for (int i = 0; i < used; ++i) {
        const float2 v = a.part_ml[i * step + row];
        if (v.x == -INFINITY && v.y == 0.0f) continue;  // nothing visible there
        const float w = ex2(v.x - top);
        sum = fmaf(w, v.y, sum);
        const float* from = a.part_o + (i * step + row) * HD + lane * kPer;
#pragma unroll
        for (int e = 0; e < kPer; ++e) x[e] = fmaf(w, from[e], x[e]);
    }
    const float inv = sum > 0.0f ? 1.0f / sum : sum == 0.0f ? 0.0f : sum;
    unsigned char* out = static_cast<unsigned char*>(a.out) + (t * a.o_token + h * a.o_head + lane * kPer) * paged_size_of(a.out_type);
    if (a.out_type == kPagedF32) {
#pragma unroll
        for (int e = 0; e < kPer; ++e) reinterpret_cast<float*>(out)[e] = x[e] * inv;
    } else {
#pragma unroll
        for (int e = 0; e < kPer; e += 2) reinterpret_cast<uint32_t*>(out)[e / 2] = paged_pack2(a.out_type, x[e] * inv, x[e + 1] * inv);
    }
}

}  // namespace qtb
