// A key / value cache in pages: what its kernels share.
//
// A cache holds `pages` pages of P positions for every layer. A page of a layer keeps, per KV head, the rows of P positions, eight positions together, cut into blocks of 64
// values: [page][head][P / 8][block][8 positions][64 values], keys and values apart. So any run of whole eights of a page and head is contiguous, and comes to shared memory by one bulk copy, without a
// tensor map, whatever the page table says. Rows lie in it the way matrix instructions want them in shared memory: groups of eight rows a constant distance apart, the 16-byte pieces of a
// row permuted, so that eight rows of one piece fall into eight different banks:
//   F16, BF16: rows of 128 bytes, piece c of row r at c ^ (r & 7) (the 128-byte swizzle of the tensor cores' operands);
//   Q8:        rows of 64 bytes,  piece c of row r at c ^ ((r >> 1) & 3), and one F32 scale per row and head, [page][head][position].
//
// What the cache holds is finite: the writer saturates. A place that a mask hides enters a product as weight zero times a finite value, whatever was
// written there, and pages that were used before need no clearing (a new cache is zeros).
//
// Row sets (RowsView): the new tokens of a call, packed; sequence s has tokens starts[s] .. starts[s + 1] - 1, of which the last one is at position
// lengths[s] - 1, and its position p lies in page table[s][p / P], row p % P. All three live in device memory, so that a captured launch serves
// whatever they hold when it is replayed; what is out of range there is skipped and raises a bit of the cache's status word.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>

namespace qtb {

enum PagedType : int { kPagedF32 = 0, kPagedF16 = 1, kPagedBf16 = 2, kPagedQ8 = 3 };  // element types; a cache holds one of the last three
enum PagedStatus : unsigned int {
    kPagedBadPage = 1,      // a page table names a page that the cache does not have
    kPagedBadPosition = 2,  // a token or a length outside the page table, the table of angles or the packed rows
    kPagedSaturated = 4,    // a value was not finite, or too large for the stored type
    kPagedGaveUp = 8,       // a wait inside a kernel ran out
};
constexpr int kPagedBlock = 64;  // values of a block
constexpr int kPagedLongest = 0x7fff0000;  // positions of a sequence at most: a tile, or a few for each of a launch's ranges, beyond its end is still a 32-bit number
// The scales of Q8 rows: 2^-40 (rows of values below it by half are zeros) to 2^40 (larger values are saturated). Attention takes a position's part of a sum as 2^(score + log2 scale - maximum)
// / scale, and 32 bits end at 2^-126: within these 80 powers no position is lost whose part is 2^-46 of the largest or more (with rows of zeros at 2^-100 they fell out of the sum beside values of 2^33).
constexpr float kPagedMinScale = 9.094947017729282e-13f, kPagedMaxScale = 1099511627776.0f;
constexpr int kPagedFreshScale = 0x2C;  // the bytes of a scale that no row has set: 0x2C2C2C2C is about 2^-39, a row of zeros as if it had been written

struct PagedView {  // one layer of a cache
    unsigned char *k, *v;
    float *ks, *vs;  // Q8: scales
    int pages, page_log2, kv_heads, blocks;
    unsigned int* status;
};
struct RowsView {
    const int *starts, *lengths, *table;
    int sequences, tokens, stride, room;  // of the table: from row to row, and entries of a row
    int most;                             // new tokens of a sequence, as announced
};

__host__ __device__ constexpr int paged_row_bytes(int type) { return type == kPagedQ8 ? kPagedBlock : kPagedBlock * 2; }
__device__ __forceinline__ int paged_piece(int type, int row, int piece) { return type == kPagedQ8 ? piece ^ ((row >> 1) & 3) : piece ^ (row & 7); }
// Where row r of a block lies in a run of rows that begins with a whole eight: in shared memory as in a page.
__host__ __device__ constexpr int paged_row_at(int type, int blocks, int block, int r) { return (((r >> 3) * blocks + block) * 8 + (r & 7)) * paged_row_bytes(type); }
// The first byte of a page's rows of a head, from row r on (a multiple of 8); the page's scales of a head.
__device__ __forceinline__ size_t paged_rows_at(const PagedView& c, int type, int page, int head, int r) {
    return (((static_cast<size_t>(page) * c.kv_heads + head) << c.page_log2) + r) * (c.blocks * paged_row_bytes(type));
}
__device__ __forceinline__ size_t paged_scales_at(const PagedView& c, int page, int head) { return (static_cast<size_t>(page) * c.kv_heads + head) << c.page_log2; }

// The sequence that packed token t belongs to, or -1 (behind the last one): the last s with starts[s] <= t. All lanes of a warp ask for the same token.
__device__ __forceinline__ int paged_sequence_of(const RowsView& r, int t) {
    const int lane = threadIdx.x & 31;
    int n = 0;
    for (int s0 = 0; s0 <= r.sequences; s0 += 32) n += __popc(__ballot_sync(0xffffffffu, s0 + lane <= r.sequences && r.starts[min(s0 + lane, r.sequences)] <= t));
    return n - 1 < r.sequences ? n - 1 : -1;
}
// A sequence's new tokens and cached positions. `ok` false: it has no new tokens, or numbers that make no sense, and nothing is done for it.
struct PagedSequence {
    int first, news, length;
    bool ok;
};
__device__ __forceinline__ PagedSequence paged_sequence(const PagedView& c, const RowsView& r, int s) {
    PagedSequence q;
    const int end = r.starts[s + 1];
    q.first = r.starts[s], q.length = r.lengths[s];
    const bool fits = q.first >= 0 && q.first <= end && end <= r.tokens && q.length >= 0 && q.length <= min(static_cast<long long>(r.room) << c.page_log2, static_cast<long long>(kPagedLongest));
    q.news = fits ? end - q.first : 0;
    q.ok = q.news > 0;
    if (!fits) atomicOr(c.status, kPagedBadPosition);
    return q;
}

// Eight values of element type T (kPagedF32, kPagedF16 or kPagedBf16) at p, 16-byte aligned.
__device__ __forceinline__ void paged_load8(const void* p, int type, float (&x)[8]) {
    if (type == kPagedF32) {
        const float4 a = static_cast<const float4*>(p)[0], b = static_cast<const float4*>(p)[1];
        x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
        return;
    }
    const uint4 w = *static_cast<const uint4*>(p);
    const uint32_t v[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (type == kPagedF16) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&v[i]));
            x[2 * i] = f.x, x[2 * i + 1] = f.y;
        } else {
            x[2 * i] = __uint_as_float(v[i] << 16), x[2 * i + 1] = __uint_as_float(v[i] & 0xffff0000u);
        }
    }
}
template <int TYPE>
__device__ __forceinline__ uint32_t paged_pack2(float a, float b) {
    if constexpr (TYPE == kPagedF16) {
        const __half2 h = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ void paged_store8(void* p, int type, const float (&x)[8]) {
    if (type == kPagedF32) {
        static_cast<float4*>(p)[0] = make_float4(x[0], x[1], x[2], x[3]);
        static_cast<float4*>(p)[1] = make_float4(x[4], x[5], x[6], x[7]);
    } else if (type == kPagedF16) {  // (one branch for all eight values)
        *static_cast<uint4*>(p) = make_uint4(paged_pack2<kPagedF16>(x[0], x[1]), paged_pack2<kPagedF16>(x[2], x[3]), paged_pack2<kPagedF16>(x[4], x[5]), paged_pack2<kPagedF16>(x[6], x[7]));
    } else {
        *static_cast<uint4*>(p) = make_uint4(paged_pack2<kPagedBf16>(x[0], x[1]), paged_pack2<kPagedBf16>(x[2], x[3]), paged_pack2<kPagedBf16>(x[4], x[5]), paged_pack2<kPagedBf16>(x[6], x[7]));
    }
}
__host__ __device__ constexpr int paged_size_of(int type) { return type == kPagedF32 ? 4 : type == kPagedQ8 ? 1 : 2; }

// Eight values of a head as they lie in memory, and as 32-bit values.
template <int TYPE> struct PagedRaw { uint4 v[TYPE == kPagedF32 ? 2 : 1]; };
template <int TYPE>
__device__ __forceinline__ PagedRaw<TYPE> paged_raw(const void* base, size_t element) {
    PagedRaw<TYPE> r;
    const uint4* p = reinterpret_cast<const uint4*>(static_cast<const unsigned char*>(base) + element * paged_size_of(TYPE));
    r.v[0] = *p;
    if constexpr (TYPE == kPagedF32) r.v[1] = p[1];
    return r;
}

}  // namespace qtb
