// Rows into a paged cache and out of it.
//
// Writing (paged_append_kernel): for every head x of a new token, y = x * w / sqrt(mean(x^2) + eps) where the head has norm weights, then pairs
// (x0, x1) of its first `rope` values become (x0 c - x1 s, x0 s + x1 c) with the angles' row of the token's position; value heads take neither.
// Queries are rounded to their type and written beside one another; keys and values go to their page: rounded to nearest even, or as Q8 codes
// rint(y / d) with d = max(|y|) / 127 of the row. All arithmetic is in 32 bits; one rounding at the end.
// Reading (paged_read_kernel): the same rows back, code times scale, rounded to the output type.
//
// Eight values to a thread (16 bytes of a 16-bit type, 8 codes), 8 to 32 threads to a head: norm and maximum are exchanges within those threads, and a
// row of the cache is written once. Both are bound by the bytes they move, small calls by their latency: the addresses need four dependent reads
// (starts, length, page, row), behind which the head's values are already on their way.
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
    int q_heads;                     // 0 where q is nullptr
};

template <int LANES>  // threads of a head: head_dim / 8
__global__ void __launch_bounds__(kPagedRowThreads) paged_append_kernel(const __grid_constant__ PagedAppendArgs a) {
    constexpr int kHeads = 32 / LANES, HD = LANES * 8;  // heads of a warp
    __shared__ float exchange[kPagedRowThreads / 32][kHeads][HD];  // NEOX pairs lie half a rotation apart
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, sub = lane / LANES, piece = lane % LANES;
    const int heads = a.q_heads + 2 * a.c.kv_heads, groups = (heads + kHeads - 1) / kHeads;
    const int item = blockIdx.x * (kPagedRowThreads / 32) + warp, t = item / groups;
    if (t >= a.r.tokens) return;
    const int head = item % groups * kHeads + sub, kind = head < a.q_heads ? 0 : head < a.q_heads + a.c.kv_heads ? 1 : 2;  // query, key, value
    const bool live = head < heads;
    const int h = kind == 0 ? head : kind == 1 ? head - a.q_heads : head - a.q_heads - a.c.kv_heads;
    float x[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = 0.0f;
    if (live) {
        const size_t at = kind == 0 ? t * a.q_token + h * a.q_head : kind == 1 ? t * a.k_token + h * a.k_head : t * a.v_token + h * a.v_head;
        const void* base = kind == 0 ? a.q : kind == 1 ? a.k : a.v;
        paged_load8(static_cast<const unsigned char*>(base) + (at + piece * 8) * paged_size_of(a.in_type), a.in_type, x);
    }
    const int s = paged_sequence_of(a.r, t);
    if (s < 0) return;  // a row behind the last sequence is left as it was
    const PagedSequence sq = paged_sequence(a.c, a.r, s);
    if (!sq.ok || t < sq.first || t >= sq.first + sq.news) return;
    const int pos = sq.length - sq.news + (t - sq.first);
    if (pos < 0 || (a.cos_sin != nullptr && pos >= a.positions)) {
        if (lane == 0) atomicOr(a.c.status, kPagedBadPosition);
        return;
    }
    const float* w = kind == 0 ? a.q_norm : kind == 1 ? a.k_norm : nullptr;
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) sum = fmaf(x[i], x[i], sum);
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (w != nullptr) {
        const float inv = 1.0f / sqrtf(sum / HD + a.eps);
        float g[8];
        paged_load8(w + piece * 8, kPagedF32, g);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = x[i] * inv * g[i];
    }
    if (a.cos_sin != nullptr) {
        const float* cs = a.cos_sin + static_cast<size_t>(pos) * a.rope;
        if (!a.neox) {
            if (kind != 2) {
#pragma unroll
                for (int i = 0; i < 8; i += 2)
                    if (piece * 8 + i < a.rope) {
                        const float c = cs[piece * 8 + i], sn = cs[piece * 8 + i + 1], x0 = x[i], x1 = x[i + 1];
                        x[i] = x0 * c - x1 * sn, x[i + 1] = x0 * sn + x1 * c;
                    }
            }
        } else {
            float* row = exchange[warp][sub];
#pragma unroll
            for (int i = 0; i < 8; ++i) row[piece * 8 + i] = x[i];
            __syncwarp();
            if (kind != 2) {
                const int half = a.rope / 2;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const int e = piece * 8 + i;
                    if (e >= a.rope) continue;
                    const bool second = e >= half;
                    const int p = second ? e - half : e;
                    const float c = cs[2 * p], sn = cs[2 * p + 1], other = row[second ? p : p + half];
                    x[i] = second ? other * sn + x[i] * c : x[i] * c - other * sn;
                }
            }
        }
    }
    if (live && kind == 0) {
        paged_store8(static_cast<unsigned char*>(a.q_out) + (t * a.o_token + h * a.o_head + piece * 8) * paged_size_of(a.q_type), a.q_type, x);
        if (a.type != kPagedQ8) return;  // (the exchanges below are for whole warps)
    }
    if (a.type != kPagedQ8 && !live) return;
    // what is not finite, or does not fit the type, becomes the nearest value that does, and a value that is none becomes zero
    const float most_finite = a.type == kPagedF16 ? 65504.0f : a.type == kPagedBf16 ? 3.3895313892515355e38f : 8.507059173023462e37f;  // (Q8: 2^126, so that 127 d does not overflow)
    bool odd = false;
    float amax = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        if (!(fabsf(x[i]) <= most_finite)) odd = true, x[i] = isnan(x[i]) ? 0.0f : copysignf(most_finite, x[i]);
        amax = fmaxf(amax, fabsf(x[i]));
    }
    if (odd && live && kind != 0) atomicOr(a.c.status, kPagedSaturated);
    const int row = pos & ((1 << a.c.page_log2) - 1), page = a.r.table[static_cast<size_t>(s) * a.r.stride + (pos >> a.c.page_log2)];
    const bool there = page >= 0 && page < a.c.pages;
    if (!there && lane == 0) atomicOr(a.c.status, kPagedBadPage);
    unsigned char* store = kind == 1 ? a.c.k : a.c.v;
    if (a.type != kPagedQ8) {
        if (there)
            paged_store8(store + paged_block_at(a.c, a.type, page, h, piece >> 3) + row * 128 + paged_piece(a.type, row, piece & 7) * 16, a.type, x);
        return;
    }
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    if (!live || kind == 0 || !there) return;
    const float d = fmaxf(amax / 127.0f, kPagedMinScale);
    uint32_t code[2] = {0u, 0u};
#pragma unroll
    for (int i = 0; i < 8; ++i) {  // (127 / d rounds to 127 at most, as d is at least the rounded amax / 127: |x| / d <= 127 (1 + 2^-23), and rint gives 127)
        const int q = max(-127, min(127, __float2int_rn(x[i] / d)));
        code[i >> 2] |= static_cast<uint32_t>(q & 0xff) << (8 * (i & 3));
    }
    *reinterpret_cast<uint2*>(store + paged_block_at(a.c, a.type, page, h, piece >> 3) + row * 64 + paged_piece(a.type, row, (piece & 7) >> 1) * 16 + (piece & 1) * 8) =
        make_uint2(code[0], code[1]);
    if (piece == 0) (kind == 1 ? a.c.ks : a.c.vs)[paged_scales_at(a.c, page, h) + row] = d;
}

struct PagedReadArgs {
    PagedView c;
    RowsView r;
    int type, out_type;
    void *k, *v;  // [token][kv_heads][head_dim]; either may be nullptr
};

template <int LANES>
__global__ void __launch_bounds__(kPagedRowThreads) paged_read_kernel(const __grid_constant__ PagedReadArgs a) {
    constexpr int kHeads = 32 / LANES, HD = LANES * 8;
    const int lane = threadIdx.x & 31, sub = lane / LANES, piece = lane % LANES;
    const int heads = 2 * a.c.kv_heads, groups = (heads + kHeads - 1) / kHeads;
    const int item = blockIdx.x * (kPagedRowThreads / 32) + (threadIdx.x >> 5), t = item / groups;
    if (t >= a.r.tokens) return;
    const int head = item % groups * kHeads + sub;
    const bool value = head >= a.c.kv_heads;
    const int h = value ? head - a.c.kv_heads : head;
    const int s = paged_sequence_of(a.r, t);
    if (s < 0) return;
    const PagedSequence sq = paged_sequence(a.c, a.r, s);
    if (!sq.ok || t < sq.first || t >= sq.first + sq.news) return;
    const int pos = sq.length - sq.news + (t - sq.first);
    if (pos < 0) {
        if (lane == 0) atomicOr(a.c.status, kPagedBadPosition);
        return;
    }
    const int row = pos & ((1 << a.c.page_log2) - 1), page = a.r.table[static_cast<size_t>(s) * a.r.stride + (pos >> a.c.page_log2)];
    if (page < 0 || page >= a.c.pages) {
        if (lane == 0) atomicOr(a.c.status, kPagedBadPage);
        return;
    }
    void* out = value ? a.v : a.k;
    if (head >= heads || out == nullptr) return;
    const unsigned char* store = (value ? a.c.v : a.c.k) + paged_block_at(a.c, a.type, page, h, piece >> 3);
    float x[8];
    if (a.type == kPagedQ8) {
        const uint2 code = *reinterpret_cast<const uint2*>(store + row * 64 + paged_piece(a.type, row, (piece & 7) >> 1) * 16 + (piece & 1) * 8);
        const float d = (value ? a.c.vs : a.c.ks)[paged_scales_at(a.c, page, h) + row];
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = static_cast<float>(static_cast<int8_t>((i < 4 ? code.x : code.y) >> (8 * (i & 3)))) * d;
    } else {
        paged_load8(store + row * 128 + paged_piece(a.type, row, piece & 7) * 16, a.type, x);
    }
    paged_store8(static_cast<unsigned char*>(out) + ((static_cast<size_t>(t) * a.c.kv_heads + h) * HD + piece * 8) * paged_size_of(a.out_type), a.out_type, x);
}

}  // namespace qtb
