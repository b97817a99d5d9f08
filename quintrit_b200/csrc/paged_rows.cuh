// Rows into a paged cache and out of it.
//
// Writing (paged_append_kernel): for every head x of a new token, y = x * w / sqrt(mean(x^2) + eps) where the head has norm weights, then pairs
// (x0, x1) of its first `rope` values become (x0 c - x1 s, x0 s + x1 c) with the angles' row of the token's position; value heads take neither.
// Queries are rounded to their type and written beside one another; keys and values go to their page: rounded to nearest even, or as Q8 codes
// rint(y / d) with d = max(|y|) / 127 of the row, from 2^-40 to 2^40. All arithmetic is in 32 bits; one rounding at the end.
// Reading (paged_read_kernel): the same rows back, code times scale, rounded to the output type.
//
// Writing: sixteen values to a thread, two pieces of eight half a head apart, so that the pairs of a rotation lie in one thread whether they are neighbours or halves of a head (eight
// values to a thread, the halves exchanged through shared memory: 40 us for the prompt below, now 29). Norm and maximum are exchanges within the 4 to 16 threads of a head. Reading: eight
// values to a thread. A warp takes U groups of heads of one token. Both kernels are bound by the bytes they move, small calls by
// their latency: a row's address needs four dependent reads (starts, length, page), so the heads' values are asked for before them, and where there are
// tokens enough for it, groups of heads share one address (writing: two, which keep the registers at 80; four took 36 us with the rows' way back, one 38.6, two 33.5; reading: four). Writing 4096 tokens of 32 + 2 x 4 heads of
// 128 with norm, rotation and Q8: 79.8 MB in 28.7 us, 42% of the copy rate; the multiprocessors issue in 55% of their cycles, 120 instructions for sixteen values of a warp. Reading 112000 positions
// of 4 heads of 256 values, Q8 to F16: 459 MB in 85.5 us, 82%.
#pragma once
#include "paged_cache.cuh"

namespace qtb {

constexpr int kPagedRowThreads = 256;

struct PagedAppendArgs {
    PagedView c;
    RowsView r;
    int type;            // of the cache
    int in_type, q_type; // of q, k, v and of q_out
    const void *q, *k, *v;           // [token][head][head_dim]; q may be nullptr
    size_t q_token, q_head, k_token, k_head, v_token, v_head;  // strides in elements
    void* q_out;
    size_t o_token, o_head;
    const float *q_norm, *k_norm;    // [head_dim] or nullptr
    float eps;
    const float* cos_sin;            // [positions][rope]: cos at 2 i, sin at 2 i + 1; nullptr: no rotation
    int rope, positions, neox;
    int turn;                        // PagedTurn: pairs of neighbours, rope a multiple of 8; whole heads in halves (neox); either with angles on 16-byte boundaries; else any
    int q_heads;                     // 0 where q is nullptr
};

// A token's place in the cache, by a whole warp: page < 0 where the token is behind the last sequence or something is out of range (then reported).
struct PagedPlace {
    int pos, page, row;
};
__device__ __forceinline__ PagedPlace paged_place(const PagedView& c, const RowsView& r, int t, int positions) {
    PagedPlace p{0, -1, 0};
    const int s = paged_sequence_of(r, t);
    if (s < 0) return p;
    const PagedSequence sq = paged_sequence(c, r, s);
    if (!sq.ok || t < sq.first || t >= sq.first + sq.news) return p;
    p.pos = sq.length - sq.news + (t - sq.first);
    if (p.pos < 0 || p.pos >= positions || sq.news > r.most) {
        if ((threadIdx.x & 31) == 0) atomicOr(c.status, kPagedBadPosition);
        return p;
    }
    p.row = p.pos & ((1 << c.page_log2) - 1), p.page = r.table[static_cast<size_t>(s) * r.stride + (p.pos >> c.page_log2)];
    if (p.page < 0 || p.page >= c.pages) {
        if ((threadIdx.x & 31) == 0) atomicOr(c.status, kPagedBadPage);
        p.page = -1;
    }
    return p;
}

enum PagedTurn { kPagedNoTurn, kPagedTurnPairs, kPagedTurnHalves, kPagedTurnAny };

template <int LANES, int TYPE, int U>  // threads of a head: head_dim / 16; type of q, k and v; groups of heads of a warp
__global__ void __launch_bounds__(kPagedRowThreads, 3) paged_append_kernel(const __grid_constant__ PagedAppendArgs a) {
    constexpr int kHeads = 32 / LANES, HD = LANES * 16, HALF = HD / 2;
    __shared__ __align__(16) float exchange[kPagedRowThreads / 32][kHeads][HD];  // where the values of a pair lie in two threads (kPagedTurnAny)
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, sub = lane / LANES, e0 = lane % LANES * 8;  // this thread's values: e0 .. e0 + 7 and those half a head further
    const int heads = a.q_heads + 2 * a.c.kv_heads, units = (heads + kHeads * U - 1) / (kHeads * U);
    const int item = blockIdx.x * (kPagedRowThreads / 32) + warp, t = item / units;
    if (t >= a.r.tokens) return;
    const int head0 = item % units * (kHeads * U) + sub;
    PagedRaw<TYPE> raw[U][2];
#pragma unroll
    for (int u = 0; u < U; ++u) {  // (the last head again where there are no more)
        const int h = min(head0 + u * kHeads, heads - 1), k = h - a.q_heads, v = k - a.c.kv_heads;
        const void* from = k < 0 ? a.q : v < 0 ? a.k : a.v;
        const size_t at = k < 0 ? t * a.q_token + h * a.q_head : v < 0 ? t * a.k_token + k * a.k_head : t * a.v_token + v * a.v_head;
        raw[u][0] = paged_raw<TYPE>(from, at + e0), raw[u][1] = paged_raw<TYPE>(from, at + e0 + HALF);
    }
    const PagedPlace place = paged_place(a.c, a.r, t, a.turn != kPagedNoTurn ? a.positions : 0x7fffffff);
    // (a query of a token whose page does not exist is left as it was, like its row of the cache)
    if (place.page < 0) return;
    // the angles of this thread's eight pairs: (i, i + 8) of its values, or (2 i, 2 i + 1)
    const float* angles = a.cos_sin + static_cast<size_t>(place.pos) * a.rope;
    const bool in[2] = {e0 < a.rope, e0 + HALF < a.rope};
    float cs[8], sn[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        float4 v = make_float4(1.0f, 0.0f, 1.0f, 0.0f);
        if (a.turn == kPagedTurnHalves) v = reinterpret_cast<const float4*>(angles + 2 * e0)[i];
        else if (a.turn == kPagedTurnPairs && in[i >> 1]) v = reinterpret_cast<const float4*>(angles + e0 + (i >> 1) * HALF)[i & 1];
        cs[2 * i] = v.x, sn[2 * i] = v.y, cs[2 * i + 1] = v.z, sn[2 * i + 1] = v.w;
    }
    const float most_finite = a.type == kPagedF16 ? 65504.0f : a.type == kPagedBf16 ? 3.3895313892515355e38f : 127.0f * kPagedMaxScale;
    // where the rows of this token lie in the cache, of head 0; a thread's pieces in them
    const size_t row0 = paged_rows_at(a.c, a.type, place.page, 0, 0) + paged_row_at(a.type, a.c.blocks, 0, place.row), per_head = static_cast<size_t>(a.c.blocks * paged_row_bytes(a.type)) << a.c.page_log2;
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int h = head0 + u * kHeads, k = h - a.q_heads, v = k - a.c.kv_heads;
        const bool live = h < heads, value = v >= 0;
        float x[16];
        paged_load8(raw[u][0].v, TYPE, *reinterpret_cast<float(*)[8]>(x));
        paged_load8(raw[u][1].v, TYPE, *reinterpret_cast<float(*)[8]>(x + 8));
        if (a.q_norm != nullptr || a.k_norm != nullptr) {
            const float* w = k < 0 ? a.q_norm : value ? nullptr : a.k_norm;
            float sum = 0.0f, eps = a.eps;
#pragma unroll
            for (int i = 0; i < 16; ++i) sum = fmaf(x[i], x[i], sum);
#pragma unroll
            for (int o = LANES / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
            if (w != nullptr && sum == INFINITY) {  // squares beyond 32 bits (the same for all threads of a head): of the values over 2^70 instead, beside which eps is nothing
                const unsigned int head = (0xffffffffu >> (32 - LANES)) << (sub * LANES);
                sum = 0.0f, eps = 0.0f;
#pragma unroll
                for (int i = 0; i < 16; ++i) x[i] *= 0x1p-70f, sum = fmaf(x[i], x[i], sum);
#pragma unroll
                for (int o = LANES / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(head, sum, o);
            }
            if (w != nullptr) {
                float f[16];
                paged_load8(w + e0, kPagedF32, *reinterpret_cast<float(*)[8]>(f));
                paged_load8(w + e0 + HALF, kPagedF32, *reinterpret_cast<float(*)[8]>(f + 8));
                const float inv = rsqrtf(sum * (1.0f / HD) + eps);  // (off by 2^-22 at most)
#pragma unroll
                for (int i = 0; i < 16; ++i) x[i] = x[i] * inv * f[i];
            }
        }
        if (a.turn == kPagedTurnHalves && !value) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float x0 = x[i], x1 = x[8 + i];
                x[i] = fmaf(x0, cs[i], -(x1 * sn[i])), x[8 + i] = fmaf(x1, cs[i], x0 * sn[i]);
            }
        } else if (a.turn == kPagedTurnPairs && !value) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float x0 = x[2 * i], x1 = x[2 * i + 1];
                if (in[i >> 2]) x[2 * i] = fmaf(x0, cs[i], -(x1 * sn[i])), x[2 * i + 1] = fmaf(x1, cs[i], x0 * sn[i]);
            }
        } else if (a.turn == kPagedTurnAny) {
            float* row = exchange[warp][sub];
            const int half = a.rope / 2;
            __syncwarp();
            paged_store8(row + e0, kPagedF32, *reinterpret_cast<float(*)[8]>(x));
            paged_store8(row + e0 + HALF, kPagedF32, *reinterpret_cast<float(*)[8]>(x + 8));
            __syncwarp();
            if (!value) {
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const int e = e0 + (i & 7) + (i >> 3) * HALF;
                    if (e >= a.rope) continue;
                    const bool second = a.neox ? e >= half : (e & 1) != 0;
                    const int pair = a.neox ? (second ? e - half : e) : e >> 1;
                    const float other = row[a.neox ? (second ? e - half : e + half) : e ^ 1], c = angles[2 * pair], s = angles[2 * pair + 1];
                    x[i] = fmaf(x[i], c, second ? other * s : -(other * s));
                }
            }
        }
        if (k < 0) {
            unsigned char* out = static_cast<unsigned char*>(a.q_out) + (t * a.o_token + h * a.o_head + e0) * paged_size_of(a.q_type);
            paged_store8(out, a.q_type, *reinterpret_cast<float(*)[8]>(x));
            paged_store8(out + HALF * paged_size_of(a.q_type), a.q_type, *reinterpret_cast<float(*)[8]>(x + 8));
        }
        if (__all_sync(0xffffffffu, k < 0 || !live)) continue;
        float amax = 0.0f;
        bool fits = true;
#pragma unroll
        for (int i = 0; i < 16; ++i) amax = fmaxf(amax, fabsf(x[i])), fits = fits && fabsf(x[i]) <= most_finite;
        if (!fits && k >= 0) {  // the nearest value that is finite and fits the type; zero for what is no number
            amax = 0.0f;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                if (!(fabsf(x[i]) <= most_finite)) x[i] = isnan(x[i]) ? 0.0f : copysignf(most_finite, x[i]);
                amax = fmaxf(amax, fabsf(x[i]));
            }
            if (live) atomicOr(a.c.status, kPagedSaturated);
        }
        unsigned char* row = (value ? a.c.v : a.c.k) + row0 + (value ? v : k) * per_head;
        const int block_bytes = paged_row_at(a.type, a.c.blocks, 1, 0), piece = e0 >> 3, second = piece + HALF / 8;
        if (a.type != kPagedQ8) {
            if (k < 0 || !live) continue;
            paged_store8(row + (piece >> 3) * block_bytes + paged_piece(a.type, place.row, piece & 7) * 16, a.type, *reinterpret_cast<float(*)[8]>(x));
            paged_store8(row + (second >> 3) * block_bytes + paged_piece(a.type, place.row, second & 7) * 16, a.type, *reinterpret_cast<float(*)[8]>(x + 8));
            continue;
        }
#pragma unroll
        for (int o = LANES / 2; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
        if (k < 0 || !live) continue;
        const float d = fmaxf(amax / 127.0f, kPagedMinScale), inv = 1.0f / d;
        uint32_t code[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {  // |x| / d <= 127 (1 + 2^-22), which rounds to 127. Added to 1.5 2^23 a number is rounded to its integer, in the low bits
            uint32_t q[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float v = x[4 * i + e], t = v * inv;
                q[e] = __float_as_uint(fmaf(fmaf(-t, d, v), inv, t) + 12582912.0f);  // with the remainder's part the quotient of a tie is exact, so that it goes to the even code
            }
            code[i] = __byte_perm(__byte_perm(q[0], q[1], 0x0040), __byte_perm(q[2], q[3], 0x0040), 0x5410);
        }
        *reinterpret_cast<uint2*>(row + (piece >> 3) * block_bytes + paged_piece(a.type, place.row, (piece & 7) >> 1) * 16 + (piece & 1) * 8) = make_uint2(code[0], code[1]);
        *reinterpret_cast<uint2*>(row + (second >> 3) * block_bytes + paged_piece(a.type, place.row, (second & 7) >> 1) * 16 + (second & 1) * 8) = make_uint2(code[2], code[3]);
        if (piece == 0) (value ? a.c.vs : a.c.ks)[paged_scales_at(a.c, place.page, value ? v : k) + place.row] = d;
    }
}

struct PagedReadArgs {
    PagedView c;
    RowsView r;
    int type, out_type;
    void *k, *v;  // [token][kv_heads][head_dim]; either may be nullptr
};

template <int LANES, int TYPE, int U>  // TYPE: of the cache
__global__ void __launch_bounds__(kPagedRowThreads) paged_read_kernel(const __grid_constant__ PagedReadArgs a) {
    constexpr int kHeads = 32 / LANES, HD = LANES * 8;
    const int lane = threadIdx.x & 31, sub = lane / LANES, piece = lane % LANES;
    const int heads = 2 * a.c.kv_heads, groups = (heads + U * kHeads - 1) / (U * kHeads);
    const int item = blockIdx.x * (kPagedRowThreads / 32) + (threadIdx.x >> 5), t = item / groups;
    if (t >= a.r.tokens) return;
    const int head0 = item % groups * U * kHeads + sub;
    const PagedPlace place = paged_place(a.c, a.r, t, 0x7fffffff);
    if (place.page < 0) return;
    uint4 raw[U];
    float d[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int head = min(head0 + u * kHeads, heads - 1);
        const bool value = head >= a.c.kv_heads;
        const int h = value ? head - a.c.kv_heads : head;
        const unsigned char* row = (value ? a.c.v : a.c.k) + paged_rows_at(a.c, TYPE, place.page, h, 0) + paged_row_at(TYPE, a.c.blocks, piece >> 3, place.row);
        if constexpr (TYPE == kPagedQ8) {
            const uint2 v = *reinterpret_cast<const uint2*>(row + paged_piece(TYPE, place.row, (piece & 7) >> 1) * 16 + (piece & 1) * 8);
            raw[u] = make_uint4(v.x, v.y, 0, 0);
            d[u] = (value ? a.c.vs : a.c.ks)[paged_scales_at(a.c, place.page, h) + place.row];
        } else {
            raw[u] = *reinterpret_cast<const uint4*>(row + paged_piece(TYPE, place.row, piece & 7) * 16);
        }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int head = head0 + u * kHeads;
        const bool value = head >= a.c.kv_heads;
        const int h = value ? head - a.c.kv_heads : head;
        void* out = value ? a.v : a.k;
        if (head >= heads || out == nullptr) continue;
        float x[8];
        if constexpr (TYPE == kPagedQ8) {
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = static_cast<float>(static_cast<int8_t>((i < 4 ? raw[u].x : raw[u].y) >> (8 * (i & 3)))) * d[u];
        } else {
            paged_load8(&raw[u], TYPE, x);
        }
        paged_store8(static_cast<unsigned char*>(out) + ((static_cast<size_t>(t) * a.c.kv_heads + h) * HD + piece * 8) * paged_size_of(a.out_type), a.out_type, x);
    }
}

}  // namespace qtb
