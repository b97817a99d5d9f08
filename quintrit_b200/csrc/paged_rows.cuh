// Rows into a paged cache and out of it.
//
// Writing (paged_append_kernel): for every head x of a new token, y = x * w / sqrt(mean(x^2) + eps) where the head has norm weights, then pairs
// (x0, x1) of its first `rope` values become (x0 c - x1 s, x0 s + x1 c) with the angles' row of the token's position; value heads take neither.
// Queries are rounded to their type and written beside one another; keys and values go to their page: rounded to nearest even, or as Q8 codes
// rint(y / d) with d = max(|y|) / 127 of the row. All arithmetic is in 32 bits; one rounding at the end.
// Reading (paged_read_kernel): the same rows back, code times scale, rounded to the output type.
//
// Eight values to a thread (16 bytes of a 16-bit type, 8 codes), 8 to 32 threads to a head: norm and maximum are exchanges within those threads, and a
// row of the cache is written once. A warp takes U such groups of heads of one token. Both kernels are bound by the bytes they move, small calls by
// their latency: a row's address needs four dependent reads (starts, length, page), so the heads' values are asked for before them, and where there are
// tokens enough for it, four groups of heads share one address (U = 4).
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
    int vector;                      // eight values of a thread share 16-byte pieces of an angles' row: rope a multiple of 8, with neox of 16, rows on 16-byte boundaries
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
    if (p.pos < 0 || p.pos >= positions) {
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

template <int LANES, int TYPE, int U>  // threads of a head: head_dim / 8; type of q, k and v; groups of heads of a warp
__global__ void __launch_bounds__(kPagedRowThreads, 3) paged_append_kernel(const __grid_constant__ PagedAppendArgs a) {
    constexpr int kHeads = 32 / LANES, HD = LANES * 8;  // heads of a group: all of them queries, keys or values
    __shared__ __align__(16) float exchange[kPagedRowThreads / 32][kHeads][HD];  // NEOX pairs lie half a rotation apart
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, sub = lane / LANES, piece = lane % LANES, e0 = piece * 8;
    const int q_groups = (a.q_heads + kHeads - 1) / kHeads, kv_groups = (a.c.kv_heads + kHeads - 1) / kHeads, all = q_groups + 2 * kv_groups, units = (all + U - 1) / U;
    const int item = blockIdx.x * (kPagedRowThreads / 32) + warp, t = item / units;
    if (t >= a.r.tokens) return;
    const int g0 = item % units * U;
    // group u of this warp: its kind (0 queries, 1 keys, 2 values) and this thread's head, the last one where there are no more
    auto kind_of = [&](int g) { return g < q_groups ? 0 : g < q_groups + kv_groups ? 1 : 2; };
    auto head_of = [&](int g, int kind) { return (g - (kind == 0 ? 0 : kind == 1 ? q_groups : q_groups + kv_groups)) * kHeads + sub; };
    PagedRaw<TYPE> raw[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int g = min(g0 + u, all - 1), kind = kind_of(g), h = min(head_of(g, kind), (kind == 0 ? a.q_heads : a.c.kv_heads) - 1);
        raw[u] = kind == 0 ? paged_raw<TYPE>(a.q, t * a.q_token + h * a.q_head + e0) : kind == 1 ? paged_raw<TYPE>(a.k, t * a.k_token + h * a.k_head + e0)
                                                                                               : paged_raw<TYPE>(a.v, t * a.v_token + h * a.v_head + e0);
    }
    const PagedPlace place = paged_place(a.c, a.r, t, a.cos_sin != nullptr ? a.positions : 0x7fffffff);
    // (a query of a token whose page does not exist is left as it was, like its row of the cache)
    if (place.page < 0) return;
    // this thread's factors of the rotation: x_i cos_i + partner_i sin_i
    float cs[8], sn[8];
    const int half = a.rope / 2;
    const bool turns = a.cos_sin != nullptr && g0 < q_groups + kv_groups, rotate = turns && e0 < a.rope;
    if (rotate) {
        const float* row = a.cos_sin + static_cast<size_t>(place.pos) * a.rope;
        if (a.vector && a.neox) {  // eight pairs, all first or all second values
            const bool second = e0 >= half;
            const float4* at = reinterpret_cast<const float4*>(row + 2 * (second ? e0 - half : e0));
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float4 v = at[i];
                cs[2 * i] = v.x, sn[2 * i] = second ? v.y : -v.y, cs[2 * i + 1] = v.z, sn[2 * i + 1] = second ? v.w : -v.w;
            }
        } else if (a.vector) {  // four pairs
            const float4* at = reinterpret_cast<const float4*>(row + e0);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const float4 v = at[i];
                cs[4 * i] = cs[4 * i + 1] = v.x, sn[4 * i] = -v.y, sn[4 * i + 1] = v.y, cs[4 * i + 2] = cs[4 * i + 3] = v.z, sn[4 * i + 2] = -v.w, sn[4 * i + 3] = v.w;
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int e = min(e0 + i, a.rope - 1);
                const bool second = a.neox ? e >= half : (e & 1) != 0;
                const int p = a.neox ? (second ? e - half : e) : e >> 1;
                cs[i] = row[2 * p], sn[i] = second ? row[2 * p + 1] : -row[2 * p + 1];
            }
        }
    }
    const float most_finite = a.type == kPagedF16 ? 65504.0f : a.type == kPagedBf16 ? 3.3895313892515355e38f : 8.507059173023462e37f;  // (Q8: 2^126, so that 127 d does not overflow)
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int g = g0 + u, kind = kind_of(g), h = head_of(g, kind);
        if (g >= all) break;
        const bool live = h < (kind == 0 ? a.q_heads : a.c.kv_heads);
        float x[8];
        paged_load8(raw[u].v, TYPE, x);
        const float* w = kind == 0 ? a.q_norm : kind == 1 ? a.k_norm : nullptr;
        if (w != nullptr) {
            float sum = 0.0f, f[8];
            paged_load8(w + e0, kPagedF32, f);
#pragma unroll
            for (int i = 0; i < 8; ++i) sum = fmaf(x[i], x[i], sum);
#pragma unroll
            for (int o = LANES / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
            const float inv = rsqrtf(sum * (1.0f / HD) + a.eps);  // (off by 2^-22 at most)
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = x[i] * inv * f[i];
        }
        if (turns && kind != 2) {
            float y[8];  // the other one of each pair
            if (a.neox) {
                float* row = exchange[warp][sub];
                __syncwarp();
                paged_store8(row + e0, kPagedF32, x);
                __syncwarp();
                if (a.vector) {
                    if (rotate) paged_load8(row + (e0 >= half ? e0 - half : e0 + half), kPagedF32, y);
                } else {
#pragma unroll
                    for (int i = 0; i < 8; ++i) y[i] = row[e0 + i >= a.rope ? e0 + i : e0 + i >= half ? e0 + i - half : e0 + i + half];
                }
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) y[i] = x[i ^ 1];
            }
            if (rotate && a.vector) {
#pragma unroll
                for (int i = 0; i < 8; ++i) y[i] = fmaf(x[i], cs[i], y[i] * sn[i]);
#pragma unroll
                for (int i = 0; i < 8; ++i) x[i] = y[i];
            } else if (rotate) {
#pragma unroll
                for (int i = 0; i < 8; ++i) y[i] = e0 + i < a.rope ? fmaf(x[i], cs[i], y[i] * sn[i]) : x[i];
#pragma unroll
                for (int i = 0; i < 8; ++i) x[i] = y[i];
            }
        }
        if (kind == 0) {
            if (live) paged_store8(static_cast<unsigned char*>(a.q_out) + (t * a.o_token + h * a.o_head + e0) * paged_size_of(a.q_type), a.q_type, x);
            continue;
        }
        float amax = 0.0f;
        bool fits = true;
#pragma unroll
        for (int i = 0; i < 8; ++i) amax = fmaxf(amax, fabsf(x[i])), fits = fits && fabsf(x[i]) <= most_finite;
        if (!fits) {  // the nearest value that is finite and fits the type; zero for what is no number
            amax = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                if (!(fabsf(x[i]) <= most_finite)) x[i] = isnan(x[i]) ? 0.0f : copysignf(most_finite, x[i]);
                amax = fmaxf(amax, fabsf(x[i]));
            }
            if (live) atomicOr(a.c.status, kPagedSaturated);
        }
        unsigned char* row = (kind == 1 ? a.c.k : a.c.v) + paged_rows_at(a.c, a.type, place.page, h, 0) + paged_row_at(a.type, a.c.blocks, piece >> 3, place.row);
        if (a.type != kPagedQ8) {
            if (live) paged_store8(row + paged_piece(a.type, place.row, piece & 7) * 16, a.type, x);
            continue;
        }
#pragma unroll
        for (int o = LANES / 2; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
        if (!live) continue;
        const float d = fmaxf(amax / 127.0f, kPagedMinScale), inv = __fdividef(1.0f, d);
        uint32_t code[2] = {0u, 0u};
#pragma unroll
        for (int i = 0; i < 8; ++i) {  // (|x| / d <= 127 (1 + 2^-22), which rounds to 127; x (1 / d) is off x / d by 2^-16 of a step at most)
            const int q = __float2int_rn(x[i] * inv);
            code[i >> 2] |= static_cast<uint32_t>(q & 0xff) << (8 * (i & 3));
        }
        *reinterpret_cast<uint2*>(row + paged_piece(a.type, place.row, (piece & 7) >> 1) * 16 + (piece & 1) * 8) = make_uint2(code[0], code[1]);
        if (piece == 0) (kind == 1 ? a.c.ks : a.c.vs)[paged_scales_at(a.c, place.page, h) + place.row] = d;
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
