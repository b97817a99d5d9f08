// C ABI of the paged key / value cache (declared in include/quintrit_b200.h): handles, checks of arguments, launches.
#include <algorithm>
#include <atomic>
#include <cmath>
#include <cstddef>
#include <initializer_list>
#include <type_traits>

#include "capi_common.cuh"
#include "paged.hpp"
#include "paged_attention.cuh"
#include "paged_attention_tc.cuh"
#include "paged_rows.cuh"

using namespace qtb;

namespace {

constexpr uint32_t kMagicPaged = 0x51545047u;  // "QTPG"
// A cap below the first leaves all scores as good as equal, and none above the last touches a score of 16-bit keys and queries; between them, with a scale of up to 2^30, scale / cap and its products with
// the scales of Q8 rows are ordinary 32-bit numbers.
constexpr float kPagedLeastCap = 9.31322574615478515625e-10f, kPagedMostCap = 3.777893186295716e22f, kPagedMostScale = 1073741824.0f;  // 2^-30, 2^75, 2^30
constexpr unsigned int kPagedSpin = 1u << 17;  // tries of a wait (up to 20 us each) before it gives up

int check_cache(const quintrit_b200_paged_cache* c) {
    if (c == nullptr || c->magic != kMagicPaged) return fail(QUINTRIT_ERR_INVALID_HANDLE, "paged cache handle is NULL, freed or of the wrong type");
    return QUINTRIT_OK;
}
int check_layer(const quintrit_b200_paged_cache* c, uint32_t layer) {
    if (layer >= c->layers) return fail(QUINTRIT_ERR_INVALID_ARGUMENT, "layer %u of %u", layer, c->layers);
    return QUINTRIT_OK;
}
uint32_t table_pages_of(const quintrit_b200_paged_rows_t* r) {
    const uint32_t pages = r->struct_size < offsetof(quintrit_b200_paged_rows_t, table_pages) + sizeof r->table_pages ? 0 : r->table_pages;
    return pages != 0 ? pages : r->table_stride;
}
int check_rows(const quintrit_b200_paged_cache*, const quintrit_b200_paged_rows_t* r, bool pointers) {
    if (r == nullptr) return fail(QUINTRIT_ERR_NULL_POINTER, "rows is NULL");
    if (r->struct_size < offsetof(quintrit_b200_paged_rows_t, table_pages)) return fail(QUINTRIT_ERR_INVALID_ARGUMENT, "rows.struct_size %u is too small", r->struct_size);
    if (r->sequences == 0 || r->sequences > 65535) return fail(QUINTRIT_ERR_INVALID_ARGUMENT, "sequences must be in [1, 65535], got %u", r->sequences);
    if (r->tokens > (1u << 24)) return fail(QUINTRIT_ERR_INVALID_ARGUMENT, "at most 2^24 tokens, got %u", r->tokens);
    if (r->table_stride == 0 || r->table_stride > (1u << 24)) return fail(QUINTRIT_ERR_INVALID_ARGUMENT, "table_stride must be in [1, 2^24], got %u", r->table_stride);
    if (table_pages_of(r) > r->table_stride) return fail(QUINTRIT_ERR_INVALID_ARGUMENT, "table_pages %u is more than table_stride = %u", r->table_pages, r->table_stride);
    if (r->tokens != 0 && (r->max_new == 0 || r->max_new > r->tokens)) return fail(QUINTRIT_ERR_INVALID_ARGUMENT, "max_new %u must be in [1, tokens = %u]", r->max_new, r->tokens);
    if (r->max_length > kPagedLongest) return fail(QUINTRIT_ERR_INVALID_ARGUMENT, "max_length %u is too large", r->max_length);
    if (pointers && (r->d_starts == nullptr || r->d_lengths == nullptr || r->d_table == nullptr)) return fail(QUINTRIT_ERR_NULL_POINTER, "rows.d_starts, d_lengths or d_table is NULL");
    if (pointers && (reinterpret_cast<uintptr_t>(r->d_starts) % 4 != 0 || reinterpret_cast<uintptr_t>(r->d_lengths) % 4 != 0 || reinterpret_cast<uintptr_t>(r->d_table) % 4 != 0))
        return fail(QUINTRIT_ERR_INVALID_ARGUMENT, "rows.d_starts, d_lengths and d_table must be 4-byte aligned");
    return QUINTRIT_OK;
}
// What calls have reported so far, taken out in one step, so that a call that reports at the same time is heard now or the next time.
__global__ void paged_take_status_kernel(unsigned int* status) { status[1] = atomicExch(status, 0u); }
bool dense_type(int32_t t) { return t == kPagedF32 || t == kPagedF16 || t == kPagedBf16; }
int check_array(const char* name, const void* p, int32_t type, std::initializer_list<size_t> strides) {
    if (p == nullptr) return fail(QUINTRIT_ERR_NULL_POINTER, "%s is NULL", name);
    if (reinterpret_cast<uintptr_t>(p) % 16 != 0) return fail(QUINTRIT_ERR_INVALID_ARGUMENT, "%s must be 16-byte aligned", name);
    for (size_t s : strides)
        if (s * paged_size_of(type) % 16 != 0) return fail(QUINTRIT_ERR_INVALID_ARGUMENT, "%s: a stride of %zu elements is not a multiple of 16 bytes", name, s);
    return QUINTRIT_OK;
}

PagedView view_of(const quintrit_b200_paged_cache* c, uint32_t layer) {
    PagedView v{};
    v.k = c->k + layer * c->layer_bytes, v.v = c->v + layer * c->layer_bytes;
    if (c->type == kPagedQ8) v.ks = c->ks + layer * c->layer_scales, v.vs = c->vs + layer * c->layer_scales;
    int log2 = 0;
    while ((1u << log2) < c->page_tokens) ++log2;
    v.pages = static_cast<int>(c->pages), v.page_log2 = log2, v.kv_heads = static_cast<int>(c->kv_heads), v.blocks = static_cast<int>(c->head_dim) / kPagedBlock;
    v.status = c->status;
    return v;
}
RowsView view_of(const quintrit_b200_paged_rows_t* r) {
    RowsView v{};
    v.starts = r->d_starts, v.lengths = r->d_lengths, v.table = r->d_table;
    v.sequences = static_cast<int>(r->sequences), v.tokens = static_cast<int>(r->tokens), v.stride = static_cast<int>(r->table_stride);
    v.room = static_cast<int>(table_pages_of(r)), v.most = static_cast<int>(r->max_new);
    return v;
}
void destroy(quintrit_b200_paged_cache* c) {
    if (c == nullptr) return;
    DeviceGuard g(c->device);
    cudaFree(c->k);
    cudaFree(c->v);
    cudaFree(c->ks);
    cudaFree(c->vs);
    cudaFree(c->status);
    c->magic = 0;
    delete c;
}

struct AppendKernel {
    static constexpr int kValues = 16;  // of a thread
    static int heads(const PagedAppendArgs& a) { return a.q_heads + 2 * a.c.kv_heads; }
    template <int LANES, int TYPE, int U> static constexpr auto of() { return paged_append_kernel<LANES, TYPE, U>; }
};
struct ReadKernel {
    static constexpr int kValues = 8;
    static int heads(const PagedReadArgs& a) { return 2 * a.c.kv_heads; }
    template <int LANES, int TYPE, int U> static constexpr auto of() { return paged_read_kernel<LANES, TYPE, U>; }
};
// A warp takes several groups of heads where that leaves a few warps for every place of the device, else one.
template <typename Kernel, int HD, int TYPE, typename Args>
int launch_rows_of(const Args& a, uint32_t tokens, int sm_count, void* stream) {
    constexpr int LANES = HD / Kernel::kValues, kHeads = 32 / LANES, kWarps = kPagedRowThreads / 32, U = Kernel::kValues == 16 ? 2 : 4;
    const int groups = (Kernel::heads(a) + kHeads - 1) / kHeads;
    const long long one = static_cast<long long>(tokens) * groups, more = static_cast<long long>(tokens) * ((groups + U - 1) / U);
    if (one > 0x7fffff00LL) return fail(QUINTRIT_ERR_INVALID_SHAPE, "%u tokens of %d heads are too many for one call", tokens, Kernel::heads(a));
    const bool many = more >= 64LL * sm_count;
    auto kernel = many ? Kernel::template of<LANES, TYPE, U>() : Kernel::template of<LANES, TYPE, 1>();
    kernel<<<static_cast<unsigned int>(((many ? more : one) + kWarps - 1) / kWarps), kPagedRowThreads, 0, static_cast<cudaStream_t>(stream)>>>(a);
    QTB_LAUNCH_CHECK();
    return QUINTRIT_OK;
}

// Whether the kernel for few rows shares its tiles out, and among how many blocks: all that the device holds, as long as each gets four tiles or so; sequences of a few tiles each, or very many
// sequences, go one item to a block. (By the longest sequence: shorter ones leave the blocks less.)
int few_blocks(const quintrit_b200_paged_cache* c, const quintrit_b200_paged_rows_t* r, uint32_t window, int places) {
    long long span = std::max<uint32_t>(r->max_length, 1);
    if (window > 0) span = std::min<long long>(span, static_cast<long long>(window) + r->max_new + kPagedTile);
    const long long tiles = (span + kPagedTile - 1) / kPagedTile, items = static_cast<long long>(r->sequences) * c->kv_heads, all = tiles * items;
    if (r->sequences > kPagedShared || tiles < 6 || all + items * kPagedStart > 0x7fffffffLL || items > 8LL * places) return 0;
    return static_cast<int>(std::min<long long>(places, std::max<long long>(all / 4, 1)));
}

// The shared memory a kernel may ask for, raised once per device (`done`: a bit per device; two threads at once set the same).
template <typename Kernel>
int allow_smem(Kernel kernel, int bytes, int device, std::atomic<uint64_t>& done) {
    const uint64_t bit = uint64_t(1) << (device & 63);
    if (device < 64 && (done.load(std::memory_order_acquire) & bit) != 0) return QUINTRIT_OK;
    QTB_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
    done.fetch_or(bit, std::memory_order_release);
    return QUINTRIT_OK;
}

template <int TYPE, int BLOCKS, int NT, bool FAR>
int launch_few(const PagedAttnArgs& a, int device, dim3 grid, cudaStream_t s) {
    using F = PagedFew<TYPE, BLOCKS, NT>;
    static_assert(F::kSmem <= 227 * 1024, "the ring does not fit");
    static std::atomic<uint64_t> done{0};
    const int rc = allow_smem(paged_few_kernel<TYPE, BLOCKS, NT, FAR>, F::kSmem, device, done);
    if (rc != QUINTRIT_OK) return rc;
    paged_few_kernel<TYPE, BLOCKS, NT, FAR><<<grid, F::kThreads, F::kSmem, s>>>(a);
    QTB_LAUNCH_CHECK();
    return QUINTRIT_OK;
}
template <int TYPE, int BLOCKS, bool FAR>
int launch_few_rows(const PagedAttnArgs& a, int device, int nt, dim3 grid, cudaStream_t s) {
    if (nt == 1) return launch_few<TYPE, BLOCKS, 1, FAR>(a, device, grid, s);
    if constexpr (TYPE == kPagedQ8 && BLOCKS == 2)
        if (nt == 3) return launch_few<TYPE, BLOCKS, 3, FAR>(a, device, grid, s);
    return launch_few<TYPE, BLOCKS, 2, FAR>(a, device, grid, s);
}
template <int TYPE, bool FAR>
int launch_few_type(const PagedAttnArgs& a, int device, int nt, dim3 grid, cudaStream_t s) {
    return a.c.blocks == 1 ? launch_few_rows<TYPE, 1, FAR>(a, device, nt, grid, s) : a.c.blocks == 2 ? launch_few_rows<TYPE, 2, FAR>(a, device, nt, grid, s) : launch_few_rows<TYPE, 4, FAR>(a, device, nt, grid, s);
}
// Blocks of the kernel for few rows on all multiprocessors, by tiles of 8 rows.
template <int TYPE>
int blocks_per_sm(int head_dim, int nt) {
    if constexpr (TYPE == kPagedQ8)
        if (nt == 3) return PagedFew<TYPE, 2, 3>::kBlocksPerSm;
    return head_dim == 64 ? (nt == 1 ? PagedFew<TYPE, 1, 1>::kBlocksPerSm : PagedFew<TYPE, 1, 2>::kBlocksPerSm)
         : head_dim == 128 ? (nt == 1 ? PagedFew<TYPE, 2, 1>::kBlocksPerSm : PagedFew<TYPE, 2, 2>::kBlocksPerSm)
                           : (nt == 1 ? PagedFew<TYPE, 4, 1>::kBlocksPerSm : PagedFew<TYPE, 4, 2>::kBlocksPerSm);
}
int places_of(const quintrit_b200_paged_cache* c, int nt) {
    return c->sm_count * (c->type == kPagedQ8 ? blocks_per_sm<kPagedQ8>(static_cast<int>(c->head_dim), nt) : blocks_per_sm<kPagedF16>(static_cast<int>(c->head_dim), nt));
}

// The schedule of the kernel for many rows (PagedSchedule), and the rows of results that it takes of the workspace, at most `limit`. A block of threads costs its tiles, and for its start and
// end about 11000 cycles; ranges cost their results' way through memory and one more launch, about 15000 more. A tile is 4300 cycles of two row tiles, 1900 of one. (1024 new tokens of 12 heads of 256 values:
// whole row blocks 26.8 us, in ranges of 9 tiles 34; 257 tokens of 32 heads of 128, windowed, next to seven single tokens: whole 64 us, in ranges of 3 tiles 47.) `few`: the new tokens of sequences that it leaves out. Where the sequences' chunks differ,
// the row blocks are not known here: about as many as the tokens fill, at most one more for every sequence that may be among them.
size_t schedule_of(const quintrit_b200_paged_cache* c, const quintrit_b200_paged_rows_t* r, uint32_t group, uint32_t window, int few, int rows, size_t limit, PagedSchedule* g) {
    const double start = rows == 256 ? 2.5 : 6.0, join = rows == 256 ? 3.5 : 8.0;
    const int tile = c->head_dim == 256 ? 64 : 128, sms = c->sm_count;
    const long long most = static_cast<long long>(r->max_new) * group, longest_blocks = (most + rows - 1) / rows, all = static_cast<long long>(r->tokens) * group;
    const bool even = static_cast<long long>(r->max_new) * r->sequences == r->tokens;
    const long long m = even ? static_cast<long long>(c->kv_heads) * r->sequences : c->kv_heads;
    const long long blocks = even ? longest_blocks : (all + rows - 1) / rows, bound = even ? blocks : all / rows + std::min<long long>(r->sequences, r->tokens / (few + 1u));
    // tiles that the row block of an order sees, if its sequence has the length that was announced
    auto tiles_of = [&](long long order) -> long long {
        if (!even) order = 0;
        const long long first = (longest_blocks - 1 - order) * rows / group, last = std::min<long long>(((longest_blocks - order) * rows - 1) / group, r->max_new - 1),
                        before = static_cast<long long>(r->max_length) - r->max_new;
        const long long high = std::max<long long>(before + last + 1, 1), low = window > 0 ? std::max<long long>(before + first - window + 1, 0) : 0;
        return std::max<long long>(1, (high - low + tile - 1) / tile);
    };
    g->m = static_cast<int>(m), g->even = even, g->orders = static_cast<int>(bound), g->mapped = 0, g->whole = static_cast<int>(bound), g->cut = 1;
    if (blocks * m < sms) {
        // Ranges of at most `length` tiles, the shortest for which they are there at once.
        const size_t per_range = static_cast<size_t>(all) * c->kv_heads;
        const long long longest = tiles_of(0);
        auto fits = [&](long long length) {  // longer ranges are fewer
            long long parts = 0, mapped = 0;
            for (long long o = 0; o < bound && mapped <= kPagedMapped; ++o) {
                const long long n = (tiles_of(o) + length - 1) / length;
                mapped += n;
                if (o < blocks) parts += n;
            }
            return parts * m <= sms && mapped <= kPagedMapped && static_cast<size_t>((longest + length - 1) / length) * per_range <= limit;
        };
        long long best = longest;
        for (long long low = 2; low < best;) {
            const long long mid = (low + best) / 2;
            if (fits(mid)) best = mid;
            else low = mid + 1;
        }
        if (static_cast<double>(best) + join >= static_cast<double>(longest)) return 0;
        int x = 0;
        for (long long o = 0; o < bound; ++o) {
            const int ranges = static_cast<int>((tiles_of(o) + best - 1) / best);
            g->at[o] = static_cast<unsigned char>(x);
            for (int i = 0; i < ranges; ++i, ++x) g->order[x] = static_cast<unsigned char>(o), g->range[x] = static_cast<unsigned char>(i), g->ranges[x] = static_cast<unsigned char>(ranges);
        }
        g->mapped = x, g->whole = 0;
        return static_cast<size_t>((longest + best - 1) / best) * per_range;
    }
    const long long whole = blocks * m / sms * sms / m, left = blocks - whole;  // row blocks that fill whole waves, and those that do not
    if (left == 0) return 0;
    const double tiles = static_cast<double>(tiles_of(whole));
    const long long room = sms + (blocks * m / sms * sms - whole * m);
    auto slots = [&](int s) { return static_cast<size_t>(bound - whole) * m * s * rows; };
    int best = 1;
    double least = 1e30;
    for (int s = 1; s <= 24 && (s == 1 || (slots(s) <= limit && tiles / s >= 2.0)); ++s) {
        const double cost = static_cast<double>((left * m * s + room - 1) / room) * (std::ceil(tiles / s) + start) + (s > 1 ? join : 0.0);
        if (cost < least * 0.97) best = s, least = cost;
    }
    if (best == 1) return 0;
    g->whole = static_cast<int>(whole), g->cut = best;
    return slots(best);
}
template <int TYPE, int BLOCKS, int NT, bool FAR>
int launch_many_of(const PagedAttnArgs& a, const PagedSchedule& g, int device, unsigned grid, cudaStream_t s) {
    using M = PagedMany<TYPE, BLOCKS, NT>;
    static_assert(M::kSmem <= 227 * 1024, "the rings do not fit");
    static std::atomic<uint64_t> done{0};
    const int rc = allow_smem(paged_many_kernel<TYPE, BLOCKS, NT, FAR>, M::kSmem, device, done);
    if (rc != QUINTRIT_OK) return rc;
    paged_many_kernel<TYPE, BLOCKS, NT, FAR><<<grid, M::kThreads, M::kSmem, s>>>(a, g);
    QTB_LAUNCH_CHECK();
    return QUINTRIT_OK;
}
template <int TYPE, bool FAR>
int launch_many_type(const PagedAttnArgs& a, const PagedSchedule& g, int device, int rows, unsigned grid, cudaStream_t s) {
    if (a.c.blocks == 4) return launch_many_of<TYPE, 4, 1, FAR>(a, g, device, grid, s);
    if (rows == 128) return a.c.blocks == 1 ? launch_many_of<TYPE, 1, 1, FAR>(a, g, device, grid, s) : launch_many_of<TYPE, 2, 1, FAR>(a, g, device, grid, s);
    return a.c.blocks == 1 ? launch_many_of<TYPE, 1, 2, FAR>(a, g, device, grid, s) : launch_many_of<TYPE, 2, 2, FAR>(a, g, device, grid, s);
}
// By the cache's type and the cap. Up to a cap of 64 one exponential's error of 2^-22 of the cap is 2^-16 of a weight and below its rounding; in the same kernels the series took 52.5 us of a mixed batch
// under a cap of 30 instead of 49.6, and, not even called, 421 us of 2048 tokens over Q8 instead of 410.
constexpr float kPagedNearCap = 64.0f;
template <typename Launch>
int by_type(const PagedAttnArgs& a, int32_t type, Launch launch) {
    auto with = [&](auto far) {
        constexpr bool FAR = decltype(far)::value;
        return type == kPagedF16 ? launch(std::integral_constant<int, kPagedF16>(), std::bool_constant<FAR>()) : type == kPagedBf16 ? launch(std::integral_constant<int, kPagedBf16>(), std::bool_constant<FAR>())
                                                                                                                           : launch(std::integral_constant<int, kPagedQ8>(), std::bool_constant<FAR>());
    };
    return a.cap > kPagedNearCap * kLog2e ? with(std::true_type()) : with(std::false_type());
}

// Launches a kernel that joins results, 256 threads to a block: it comes up while the one before it in the stream still runs, and waits for that one's end itself.
template <typename Kernel, typename... Args>
int launch_behind(Kernel kernel, unsigned grid, cudaStream_t s, const Args&... args) {
    cudaLaunchConfig_t cfg{};
    cudaLaunchAttribute dependent{};
    dependent.id = cudaLaunchAttributeProgrammaticStreamSerialization, dependent.val.programmaticStreamSerializationAllowed = 1;
    cfg.gridDim = dim3(grid), cfg.blockDim = dim3(256), cfg.stream = s, cfg.attrs = &dependent, cfg.numAttrs = 1;
    QTB_CUDA(cudaLaunchKernelEx(&cfg, kernel, args...));
    ++g_launches;
    return QUINTRIT_OK;
}

// How a call is served: sequences of up to `few_new` new tokens by the kernel for few rows, the others by the one for many; either may have nothing to do.
struct PagedPlan {
    int few_new;             // 0: all by the kernel for many rows
    bool many;
    int nt;                  // few: tiles of 8 rows of a block, blocks that the tiles are shared out among (0: an item a block)
    int few_share;
    PagedSchedule schedule;  // many: which blocks, their number, slots of the workspace
    int many_rows;           // rows of a block of threads
    long long many_blocks;
    size_t part_rows;
    size_t few_bytes, many_bytes;  // of the workspace
};
// Rows of a KV head up to which the kernel for few rows takes a sequence: two row tiles of 8, three where their sums' registers are there. With it and with the many rows' kernel, us, 16 sequences of 3000, 4 KV heads,
// 8, 12 and 16 rows: F16, heads of 64: 22, 24, 25 and 32, 32, 32; of 128: 29, 31, 31 and 38, 38, 39; of 256: 45, 54, 55 and 54, 57, 56; Q8, heads of 64: 21, 23, 23 and 43, 43, 44; of 128: 22, 29, 30 and 46, 47, 46
// (20 and 24 rows: 36, 37 and 47, 47); of 256: 35, 43, 45 and 62, 65, 66.
inline int few_rows(const quintrit_b200_paged_cache* c) { return c->type == kPagedQ8 && c->head_dim == 128 ? 24 : 16; }
constexpr size_t up16(size_t n) { return (n + 15) / 16 * 16; }
void plan_of(const quintrit_b200_paged_cache* c, const quintrit_b200_paged_rows_t* r, uint32_t q_heads, uint32_t window, PagedPlan* p) {
    const long long group = q_heads / c->kv_heads, most = r->max_new * group, limit = few_rows(c);
    p->many = most > limit;
    p->few_new = static_cast<int>(!p->many ? r->max_new : r->sequences == 1 ? 0 : std::min<long long>(std::max<long long>(8 / group, group <= limit ? 1 : 0), r->max_new - 1));  // (a sequence alone is the longest)
    p->few_share = 0, p->part_rows = 0, p->few_bytes = p->many_bytes = 0, p->many_blocks = 0;
    const size_t row_bytes = c->head_dim * sizeof(float) + sizeof(float2);
    if (p->few_new > 0) {
        p->nt = static_cast<int>((p->few_new * group + 7) / 8);
        const int places = places_of(c, p->nt), share = few_blocks(c, r, 0, places);
        p->few_share = window > 0 ? std::min(share, few_blocks(c, r, window, places)) : share;  // (no window takes more of the workspace than none)
        p->few_bytes = up16(static_cast<size_t>(share) * 2 * 8 * p->nt * row_bytes);
    }
    if (p->many) {
        const int rows = c->head_dim == 256 || most <= 128 ? 128 : 256;
        p->many_rows = rows;
        // (up to four results for every row of a block of threads on every multiprocessor, about 80 MB; no window takes more than none)
        p->part_rows = schedule_of(c, r, static_cast<uint32_t>(group), 0, p->few_new, rows, static_cast<size_t>(4) * c->sm_count * rows, &p->schedule);
        if (window > 0) p->part_rows = schedule_of(c, r, static_cast<uint32_t>(group), window, p->few_new, rows, p->part_rows, &p->schedule);
        p->many_bytes = up16(p->part_rows * row_bytes);
        const PagedSchedule& g = p->schedule;
        p->many_blocks = (g.mapped ? g.mapped : g.whole + static_cast<long long>(g.orders - g.whole) * g.cut) * g.m;
    }
}
}  // namespace

void qtb::paged_cache_destroy(quintrit_b200_paged_cache* cache) { destroy(cache); }

extern "C" int quintrit_b200_paged_cache_create(uint32_t device_index, uint32_t layers, uint32_t pages, uint32_t page_tokens, uint32_t kv_heads, uint32_t head_dim, int32_t type,
                                                quintrit_b200_paged_cache_t** out_cache) {
    return guard([&]() -> int {
        if (out_cache == nullptr) return fail(QUINTRIT_ERR_NULL_POINTER, "out_cache is NULL");
        *out_cache = nullptr;
        if (layers == 0 || layers > 4096) return fail(QUINTRIT_ERR_INVALID_SHAPE, "layers must be in [1, 4096], got %u", layers);
        if (pages == 0 || pages > (1u << 24)) return fail(QUINTRIT_ERR_INVALID_SHAPE, "pages must be in [1, 2^24], got %u", pages);
        if (page_tokens < 16 || page_tokens > 256 || (page_tokens & (page_tokens - 1)) != 0) return fail(QUINTRIT_ERR_INVALID_SHAPE, "page_tokens must be 16, 32, 64, 128 or 256, got %u", page_tokens);
        if (kv_heads == 0 || kv_heads > 1024) return fail(QUINTRIT_ERR_INVALID_SHAPE, "kv_heads must be in [1, 1024], got %u", kv_heads);
        if (head_dim != 64 && head_dim != 128 && head_dim != 256) return fail(QUINTRIT_ERR_UNSUPPORTED, "head_dim must be 64, 128 or 256, got %u", head_dim);
        if (type != kPagedF16 && type != kPagedBf16 && type != kPagedQ8) return fail(QUINTRIT_ERR_INVALID_ARGUMENT, "cache type %d: F16, BF16 or Q8", type);
        cudaDeviceProp prop;
        int rc = require_b200(static_cast<int>(device_index), &prop);
        if (rc != QUINTRIT_OK) return rc;
        DeviceGuard g(static_cast<int>(device_index));
        quintrit_b200_paged_cache* c = new quintrit_b200_paged_cache();
        c->magic = kMagicPaged, c->device = static_cast<int>(device_index), c->sm_count = prop.multiProcessorCount;
        c->layers = layers, c->pages = pages, c->page_tokens = page_tokens, c->kv_heads = kv_heads, c->head_dim = head_dim, c->type = type;
        c->layer_scales = static_cast<size_t>(pages) * kv_heads * page_tokens;
        c->layer_bytes = c->layer_scales * head_dim * paged_size_of(type);
        auto alloc = [&](void** p, size_t bytes, int fill = 0) -> cudaError_t {
            cudaError_t e = cudaMalloc(p, bytes);
            if (e == cudaSuccess) e = cudaMemset(*p, fill, bytes);
            c->device_bytes += bytes;
            return e;
        };
        cudaError_t e = alloc(reinterpret_cast<void**>(&c->k), layers * c->layer_bytes);
        if (e == cudaSuccess) e = alloc(reinterpret_cast<void**>(&c->v), layers * c->layer_bytes);
        if (e == cudaSuccess && type == kPagedQ8) e = alloc(reinterpret_cast<void**>(&c->ks), layers * c->layer_scales * sizeof(float), kPagedFreshScale);
        if (e == cudaSuccess && type == kPagedQ8) e = alloc(reinterpret_cast<void**>(&c->vs), layers * c->layer_scales * sizeof(float), kPagedFreshScale);
        if (e == cudaSuccess) e = alloc(reinterpret_cast<void**>(&c->status), 16);
        if (e == cudaSuccess) e = cudaStreamSynchronize(nullptr);  // the zeros are there before a call on any stream
        if (e != cudaSuccess) {
            cudaGetLastError();
            destroy(c);
            return cuda_fail(e, "cudaMalloc(paged cache)");
        }
        *out_cache = c;
        return ok();
    });
}

extern "C" int quintrit_b200_paged_cache_free(quintrit_b200_paged_cache_t* cache) {
    return guard([&]() -> int {
        if (cache == nullptr) return ok();
        const int rc = check_cache(cache);
        if (rc != QUINTRIT_OK) return rc;
        destroy(cache);
        return ok();
    });
}

extern "C" int quintrit_b200_paged_cache_info(const quintrit_b200_paged_cache_t* cache, size_t* out_device_bytes, uint32_t* out_device) {
    return guard([&]() -> int {
        const int rc = check_cache(cache);
        if (rc != QUINTRIT_OK) return rc;
        if (out_device_bytes) *out_device_bytes = cache->device_bytes;
        if (out_device) *out_device = static_cast<uint32_t>(cache->device);
        return ok();
    });
}

extern "C" int quintrit_b200_paged_cache_status(quintrit_b200_paged_cache_t* cache) {
    return guard([&]() -> int {
        const int rc = check_cache(cache);
        if (rc != QUINTRIT_OK) return rc;
        DeviceGuard g(cache->device);
        std::lock_guard<std::mutex> one(cache->report);
        unsigned int bits = 0;
        paged_take_status_kernel<<<1, 1>>>(cache->status);
        QTB_LAUNCH_CHECK();
        QTB_CUDA(cudaMemcpy(&bits, cache->status + 1, sizeof bits, cudaMemcpyDeviceToHost));
        if (bits == 0) return ok();
        std::string said;
        auto add = [&](unsigned int bit, const std::string& text) {
            if (bits & bit) said += (said.empty() ? "" : "; ") + text;
        };
        add(kPagedGaveUp, "the paged attention kernel on the CUDA device gave up waiting for its copies");
        add(kPagedBadPage, "a page table named a page that the cache does not have (" + std::to_string(cache->pages) + " pages)");
        add(kPagedBadPosition, "a token or length lay outside the page table, the angles or the packed rows, or a chunk was longer than announced");
        add(kPagedSaturated, "a key or value was not finite or too large for the cache's type");
        return fail(bits & kPagedGaveUp ? QUINTRIT_ERR_DEVICE : QUINTRIT_ERR_INVALID_VALUE, "%s", said.c_str());
    });
}

extern "C" int quintrit_b200_paged_append_device(quintrit_b200_paged_cache_t* cache, uint32_t layer, const quintrit_b200_paged_rows_t* rows, const quintrit_b200_paged_append_t* args,
                                                 void* stream) {
    return guard([&]() -> int {
        int rc = check_cache(cache);
        if (rc != QUINTRIT_OK || (rc = check_layer(cache, layer)) != QUINTRIT_OK || (rc = check_rows(cache, rows, true)) != QUINTRIT_OK) return rc;
        if (args == nullptr) return fail(QUINTRIT_ERR_NULL_POINTER, "args is NULL");
        if (args->struct_size < sizeof(quintrit_b200_paged_append_t)) return fail(QUINTRIT_ERR_INVALID_ARGUMENT, "args.struct_size %u is too small", args->struct_size);
        if (!dense_type(args->type)) return fail(QUINTRIT_ERR_INVALID_ARGUMENT, "type %d: F32, F16 or BF16", args->type);
        if (rows->tokens == 0) return ok();
        PagedAppendArgs a{};
        if (args->d_q != nullptr) {
            if (!dense_type(args->q_out_type)) return fail(QUINTRIT_ERR_INVALID_ARGUMENT, "q_out_type %d: F32, F16 or BF16", args->q_out_type);
            if (args->q_heads == 0 || args->q_heads > 65536) return fail(QUINTRIT_ERR_INVALID_SHAPE, "q_heads must be in [1, 65536], got %u", args->q_heads);
            if ((rc = check_array("d_q", args->d_q, args->type, {args->q_token_stride, args->q_head_stride})) != QUINTRIT_OK ||
                (rc = check_array("d_q_out", args->d_q_out, args->q_out_type, {args->out_token_stride, args->out_head_stride})) != QUINTRIT_OK)
                return rc;
            if (args->d_q == args->d_q_out && (args->type != args->q_out_type || args->q_token_stride != args->out_token_stride || args->q_head_stride != args->out_head_stride))
                return fail(QUINTRIT_ERR_INVALID_ARGUMENT, "d_q_out may be d_q only with the same type and strides");
            a.q_heads = static_cast<int>(args->q_heads);
        }
        if ((rc = check_array("d_k", args->d_k, args->type, {args->k_token_stride, args->k_head_stride})) != QUINTRIT_OK ||
            (rc = check_array("d_v", args->d_v, args->type, {args->v_token_stride, args->v_head_stride})) != QUINTRIT_OK)
            return rc;
        for (const float* w : {args->d_q_norm, args->d_k_norm})
            if (reinterpret_cast<uintptr_t>(w) % 16 != 0) return fail(QUINTRIT_ERR_INVALID_ARGUMENT, "d_q_norm and d_k_norm must be 16-byte aligned");
        if ((args->d_q_norm != nullptr || args->d_k_norm != nullptr) && !(args->norm_eps >= 0.0f && std::isfinite(args->norm_eps)))
            return fail(QUINTRIT_ERR_INVALID_ARGUMENT, "norm_eps must be finite and not negative");
        if (args->d_cos_sin != nullptr) {
            if (args->rope_dims < 2 || args->rope_dims % 2 != 0 || args->rope_dims > cache->head_dim)
                return fail(QUINTRIT_ERR_INVALID_ARGUMENT, "rope_dims must be even and in [2, head_dim = %u], got %u", cache->head_dim, args->rope_dims);
            if (args->positions == 0 || args->positions > 0x7fffffffu) return fail(QUINTRIT_ERR_INVALID_ARGUMENT, "positions must be in [1, 2^31 - 1], got %u", args->positions);
            if (reinterpret_cast<uintptr_t>(args->d_cos_sin) % 4 != 0) return fail(QUINTRIT_ERR_INVALID_ARGUMENT, "d_cos_sin must be 4-byte aligned");
        }
        DeviceGuard g(cache->device);
        a.c = view_of(cache, layer), a.r = view_of(rows);
        a.type = cache->type, a.in_type = args->type, a.q_type = args->q_out_type;
        a.q = args->d_q, a.k = args->d_k, a.v = args->d_v, a.q_out = args->d_q_out;
        a.q_token = args->q_token_stride, a.q_head = args->q_head_stride, a.k_token = args->k_token_stride, a.k_head = args->k_head_stride, a.v_token = args->v_token_stride,
        a.v_head = args->v_head_stride, a.o_token = args->out_token_stride, a.o_head = args->out_head_stride;
        a.q_norm = args->d_q_norm, a.k_norm = args->d_k_norm, a.eps = args->norm_eps;
        a.cos_sin = args->d_cos_sin, a.rope = static_cast<int>(args->rope_dims), a.positions = static_cast<int>(args->positions), a.neox = args->neox != 0;
        const bool pieces = reinterpret_cast<uintptr_t>(a.cos_sin) % 16 == 0 && a.rope % 8 == 0;
        a.turn = a.cos_sin == nullptr ? kPagedNoTurn : pieces && !a.neox ? kPagedTurnPairs : pieces && a.rope == static_cast<int>(cache->head_dim) ? kPagedTurnHalves : kPagedTurnAny;
        auto launch = [&](auto type) {
            constexpr int T = decltype(type)::value;
            return cache->head_dim == 64 ? launch_rows_of<AppendKernel, 64, T>(a, rows->tokens, cache->sm_count, stream)
                 : cache->head_dim == 128 ? launch_rows_of<AppendKernel, 128, T>(a, rows->tokens, cache->sm_count, stream)
                                          : launch_rows_of<AppendKernel, 256, T>(a, rows->tokens, cache->sm_count, stream);
        };
        rc = args->type == kPagedF32 ? launch(std::integral_constant<int, kPagedF32>()) : args->type == kPagedF16 ? launch(std::integral_constant<int, kPagedF16>())
                                                                                                                  : launch(std::integral_constant<int, kPagedBf16>());
        if (rc != QUINTRIT_OK) return rc;
        return ok();
    });
}

extern "C" int quintrit_b200_paged_read_device(quintrit_b200_paged_cache_t* cache, uint32_t layer, const quintrit_b200_paged_rows_t* rows, int32_t type, void* d_k, void* d_v, void* stream) {
    return guard([&]() -> int {
        int rc = check_cache(cache);
        if (rc != QUINTRIT_OK || (rc = check_layer(cache, layer)) != QUINTRIT_OK || (rc = check_rows(cache, rows, true)) != QUINTRIT_OK) return rc;
        if (!dense_type(type)) return fail(QUINTRIT_ERR_INVALID_ARGUMENT, "type %d: F32, F16 or BF16", type);
        if (rows->tokens == 0) return ok();
        if (d_k == nullptr && d_v == nullptr) return fail(QUINTRIT_ERR_NULL_POINTER, "d_k and d_v are NULL");
        if ((d_k != nullptr && (rc = check_array("d_k", d_k, type, {})) != QUINTRIT_OK) || (d_v != nullptr && (rc = check_array("d_v", d_v, type, {})) != QUINTRIT_OK)) return rc;
        DeviceGuard g(cache->device);
        PagedReadArgs a{};
        a.c = view_of(cache, layer), a.r = view_of(rows), a.type = cache->type, a.out_type = type, a.k = d_k, a.v = d_v;
        auto launch = [&](auto of) {
            constexpr int T = decltype(of)::value;
            return cache->head_dim == 64 ? launch_rows_of<ReadKernel, 64, T>(a, rows->tokens, cache->sm_count, stream)
                 : cache->head_dim == 128 ? launch_rows_of<ReadKernel, 128, T>(a, rows->tokens, cache->sm_count, stream)
                                          : launch_rows_of<ReadKernel, 256, T>(a, rows->tokens, cache->sm_count, stream);
        };
        rc = cache->type == kPagedF16 ? launch(std::integral_constant<int, kPagedF16>()) : cache->type == kPagedBf16 ? launch(std::integral_constant<int, kPagedBf16>())
                                                                                                                     : launch(std::integral_constant<int, kPagedQ8>());
        if (rc != QUINTRIT_OK) return rc;
        return ok();
    });
}

namespace {
int check_heads(const quintrit_b200_paged_cache* c, uint32_t q_heads) {
    if (q_heads == 0 || q_heads % c->kv_heads != 0 || q_heads > 65536) return fail(QUINTRIT_ERR_INVALID_SHAPE, "q_heads %u must be a multiple of kv_heads = %u", q_heads, c->kv_heads);
    return QUINTRIT_OK;
}
}  // namespace

extern "C" int quintrit_b200_paged_attention_workspace(const quintrit_b200_paged_cache_t* cache, const quintrit_b200_paged_rows_t* rows, uint32_t q_heads, size_t* out_bytes) {
    return guard([&]() -> int {
        int rc = check_cache(cache);
        if (rc != QUINTRIT_OK) return rc;
        if (out_bytes == nullptr) return fail(QUINTRIT_ERR_NULL_POINTER, "out_bytes is NULL");
        *out_bytes = 0;
        if ((rc = check_rows(cache, rows, false)) != QUINTRIT_OK || (rc = check_heads(cache, q_heads)) != QUINTRIT_OK) return rc;
        if (rows->tokens == 0) return ok();
        PagedPlan plan;
        plan_of(cache, rows, q_heads, 0, &plan);
        *out_bytes = plan.few_bytes + plan.many_bytes;
        return ok();
    });
}

extern "C" int quintrit_b200_paged_attention_device(quintrit_b200_paged_cache_t* cache, uint32_t layer, const quintrit_b200_paged_rows_t* rows, const quintrit_b200_paged_attention_t* args,
                                                    void* stream) {
    return guard([&]() -> int {
        int rc = check_cache(cache);
        if (rc != QUINTRIT_OK || (rc = check_layer(cache, layer)) != QUINTRIT_OK || (rc = check_rows(cache, rows, true)) != QUINTRIT_OK) return rc;
        if (args == nullptr) return fail(QUINTRIT_ERR_NULL_POINTER, "args is NULL");
        if (args->struct_size < sizeof(quintrit_b200_paged_attention_t)) return fail(QUINTRIT_ERR_INVALID_ARGUMENT, "args.struct_size %u is too small", args->struct_size);
        if (!dense_type(args->q_type) || (cache->type != kPagedQ8 && args->q_type != cache->type))
            return fail(QUINTRIT_ERR_INVALID_ARGUMENT, "q_type %d: the cache's type, or F32, F16 or BF16 over a Q8 cache", args->q_type);
        if (!dense_type(args->out_type)) return fail(QUINTRIT_ERR_INVALID_ARGUMENT, "out_type %d: F32, F16 or BF16", args->out_type);
        if ((rc = check_heads(cache, args->q_heads)) != QUINTRIT_OK) return rc;
        if (!(std::fabs(args->scale) <= kPagedMostScale)) return fail(QUINTRIT_ERR_INVALID_ARGUMENT, "scale must be in [-2^30, 2^30]");
        if (!(args->cap >= 0.0f) || !std::isfinite(args->cap)) return fail(QUINTRIT_ERR_INVALID_ARGUMENT, "cap must be finite and not negative (0: none)");
        if (args->window > 0x7fffffffu) return fail(QUINTRIT_ERR_INVALID_ARGUMENT, "window %u is too large", args->window);
        if (rows->tokens == 0) return ok();
        if ((rc = check_array("d_q", args->d_q, args->q_type, {args->q_token_stride, args->q_head_stride})) != QUINTRIT_OK ||
            (rc = check_array("d_out", args->d_out, args->out_type, {args->out_token_stride, args->out_head_stride})) != QUINTRIT_OK)
            return rc;
        const int group = static_cast<int>(args->q_heads / cache->kv_heads);
        PagedPlan plan;
        plan_of(cache, rows, args->q_heads, args->window, &plan);
        if (plan.many_blocks > 0x7fffffffLL || static_cast<long long>(rows->tokens) * args->q_heads > 0x7fff0000LL)  // (rows are counted in 32 bits, up to whole row blocks)
            return fail(QUINTRIT_ERR_INVALID_SHAPE, "%u new tokens of %u query heads are too many for one call", rows->max_new, args->q_heads);
        const size_t need = plan.few_bytes + plan.many_bytes;
        if (need > 0 && args->d_workspace == nullptr) return fail(QUINTRIT_ERR_NULL_POINTER, "d_workspace is NULL, %zu bytes are needed", need);
        if (need > args->workspace_bytes) return fail(QUINTRIT_ERR_BUFFER_TOO_SMALL, "the workspace holds %zu bytes, %zu are needed", args->workspace_bytes, need);
        if (need > 0 && reinterpret_cast<uintptr_t>(args->d_workspace) % 16 != 0) return fail(QUINTRIT_ERR_INVALID_ARGUMENT, "d_workspace must be 16-byte aligned");
        DeviceGuard g(cache->device);
        cudaStream_t s = static_cast<cudaStream_t>(stream);
        PagedAttnArgs a{};
        a.c = view_of(cache, layer), a.r = view_of(rows);
        a.q = args->d_q, a.q_token = args->q_token_stride, a.q_head = args->q_head_stride, a.q_type = args->q_type;
        a.out = args->d_out, a.o_token = args->out_token_stride, a.o_head = args->out_head_stride, a.out_type = args->out_type;
        a.group = group;
        const bool level = args->cap > 0.0f && args->cap < kPagedLeastCap, capped = !level && args->cap > 0.0f && args->cap <= kPagedMostCap;
        a.scale = level ? 0.0f : capped ? args->scale / args->cap : args->scale * kLog2e;
        a.cap = capped ? args->cap * kLog2e : 0.0f;
        a.window = static_cast<int>(args->window);
        a.spin_limit = kPagedSpin;
        const int device = cache->device;
        unsigned char* workspace = static_cast<unsigned char*>(args->d_workspace);
        if (plan.many) {
            a.few = plan.few_new + 1, a.many = a.r.most;
            PagedSchedule& g = plan.schedule;
            g.part_o = reinterpret_cast<float*>(workspace + plan.few_bytes), g.part_ml = reinterpret_cast<float2*>(g.part_o + plan.part_rows * cache->head_dim);
            const unsigned grid = static_cast<unsigned>(plan.many_blocks);
            rc = by_type(a, cache->type, [&](auto type, auto far) { return launch_many_type<decltype(type)::value, decltype(far)::value>(a, g, device, plan.many_rows, grid, s); });
            if (rc != QUINTRIT_OK) return rc;
            if (plan.part_rows > 0) {
                auto kernel = a.c.blocks == 1 ? paged_join_kernel<1> : a.c.blocks == 2 ? paged_join_kernel<2> : paged_join_kernel<4>;
                rc = launch_behind(kernel, static_cast<unsigned>((static_cast<long long>(rows->tokens) * ((args->q_heads + kPagedJoinRows - 1) / kPagedJoinRows) + 7) / 8), s, a, g, plan.many_rows);
                if (rc != QUINTRIT_OK) return rc;
            }
        }
        if (plan.few_new > 0) {
            a.few = 1, a.many = plan.few_new, a.share = plan.few_share;
            const int block_rows = 8 * plan.nt;
            a.part_o = reinterpret_cast<float*>(workspace);
            a.part_ml = reinterpret_cast<float2*>(a.part_o + static_cast<size_t>(plan.few_share) * 2 * block_rows * cache->head_dim);
            const dim3 grid = plan.few_share > 0 ? dim3(static_cast<unsigned>(plan.few_share)) : dim3(cache->kv_heads, rows->sequences);
            rc = by_type(a, cache->type, [&](auto type, auto far) { return launch_few_type<decltype(type)::value, decltype(far)::value>(a, device, plan.nt, grid, s); });
            if (rc != QUINTRIT_OK) return rc;
            if (plan.few_share > 1) {
                auto kernel = a.c.blocks == 1 ? paged_combine_kernel<1> : a.c.blocks == 2 ? paged_combine_kernel<2> : paged_combine_kernel<4>;
                rc = launch_behind(kernel, static_cast<unsigned>(plan.few_share - 1), s, a, plan.few_share, block_rows);
                if (rc != QUINTRIT_OK) return rc;
            }
        }
        return ok();
    });
}
