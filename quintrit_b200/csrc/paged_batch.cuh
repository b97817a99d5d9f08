// A batch whose sequences share one paged cache: the pages' bookkeeping on the host, and a layer's attention by way of the paged operators.
#pragma once
#include "decode.cuh"
#include "paged.hpp"

namespace qtb {

// The query, key and value rows of a token's projections as floats, from the integer sums (the arithmetic of rope_kv_kernel). Grid (values / 1024, 1, tokens).
__global__ void __launch_bounds__(256) paged_sums_kernel(const __grid_constant__ RopeKvArgs a, float* __restrict__ out) {
    const int qkv = a.q_dim + 2 * a.kv_dim, i0 = (blockIdx.x * 256 + threadIdx.x) * 4;
    if (i0 >= qkv) return;
    const size_t z = blockIdx.z;
    const float s = a.act_scale[z];
    const bool live = s > 0.0f;
    const float post = live ? __fdiv_rn(i0 < a.q_dim ? a.ws_q : i0 < a.q_dim + a.kv_dim ? a.ws_k : a.ws_v, s) : 0.0f;
    float v[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const int i = i0 + e;
        const int32_t sum = a.v_q.base == nullptr ? a.acc[z * a.b_acc + i] : rope_acc(a, i);
        v[e] = live ? __fmul_rn(static_cast<float>(sum), post) : 0.0f;
    }
    *reinterpret_cast<float4*>(out + z * qkv + i0) = make_float4(v[0], v[1], v[2], v[3]);
}

// Attention's output rows to the codes of the output projection: sub-norm, where the model has one, and quantisation (the arithmetic of attn_finish_kernel). Grid (1, 1, tokens).
__global__ void __launch_bounds__(kRowThreads) paged_finish_kernel(const float* __restrict__ rows, int n, const float* __restrict__ sub_norm_w, float eps, int8_t* q_out, float* scale_out) {
    __shared__ double sh_d[32];
    __shared__ float sh_f[32];
    extern __shared__ float y_s[];  // n floats
    const int tid = threadIdx.x;
    const float* x = rows + static_cast<size_t>(blockIdx.z) * n;
    double sum = 0.0;
    for (int i = tid; i < n; i += kRowThreads) {
        const float v = x[i];
        y_s[i] = v;
        sum += static_cast<double>(__fmul_rn(v, v));
    }
    if (sub_norm_w != nullptr) {
        sum = block_sum_f64(sum, sh_d);
        const float mean = __double2float_rn(sum / static_cast<double>(n));
        const float inv = __fdiv_rn(1.0f, __fsqrt_rn(__fadd_rn(mean, eps)));
        for (int i = tid; i < n; i += kRowThreads) y_s[i] = __fmul_rn(__fmul_rn(y_s[i], inv), sub_norm_w[i]);
    }
    float amax = 0.0f;
    for (int i = tid; i < n; i += kRowThreads) amax = fmaxf(amax, fabsf(y_s[i]));
    __syncthreads();
    quantize_vector(y_s, n, amax, q_out + static_cast<size_t>(blockIdx.z) * n, scale_out + blockIdx.z, nullptr, sh_f);
}

// The rows of a step, one new token for each of its sequences (a block each): their lengths, and their rows of the page table one after the other. `page` has the page of every new position.
struct PagedStep {
    int32_t page[kReportTokens];
};
__global__ void __launch_bounds__(128) paged_step_kernel(const __grid_constant__ PagedStep step, const uint32_t* __restrict__ slot, const uint32_t* __restrict__ pos, int32_t* __restrict__ table, int stride,
                                                         int page_tokens, int32_t* __restrict__ rows_table, int32_t* __restrict__ starts, int32_t* __restrict__ lengths) {
    const int k = blockIdx.x;
    int32_t* from = table + static_cast<size_t>(slot[k]) * stride;
    const uint32_t at = pos[slot[k]];
    const int last = static_cast<int>(at / page_tokens);
    for (int i = threadIdx.x; i <= last; i += 128) rows_table[static_cast<size_t>(k) * stride + i] = i == last ? step.page[k] : from[i];
    if (threadIdx.x == 0) {
        from[last] = step.page[k];
        lengths[k] = static_cast<int32_t>(at) + 1;
        starts[k] = k;
        if (k == static_cast<int>(gridDim.x) - 1) starts[k + 1] = k + 1;
    }
}
__global__ void paged_chunk_kernel(int32_t* rows, int n, int length) { rows[0] = 0, rows[1] = n, rows[2] = length; }
__global__ void paged_report_kernel(const unsigned int* status, volatile unsigned int* host) {
    *host = *status;
    __threadfence_system();
}

struct PagedBatch {
    quintrit_b200_paged_cache_t* cache = nullptr;
    uint32_t stride = 0;                      // pages that a sequence's row of the table has room for
    std::vector<std::vector<int32_t>> pages;  // of every sequence, in order
    std::vector<int32_t> free;
    int32_t *d_table = nullptr, *d_rows_table = nullptr, *d_starts = nullptr, *d_lengths = nullptr, *d_chunk = nullptr;  // d_chunk: starts[2] and length of a prompt's chunk
    void *step_space = nullptr, *chunk_space = nullptr;  // workspaces of the attention: of steps (captured into graphs: it stays), of prompts' chunks (it grows)
    size_t step_bytes = 0, chunk_bytes = 0;
    unsigned int* host_status = nullptr;      // pinned: the cache's status word as of the last step

    size_t pages_for(size_t tokens) const { return (tokens + cache->page_tokens - 1) / cache->page_tokens; }
    void trim(size_t sequence, size_t tokens) {  // pages behind the first `tokens` positions go back
        std::vector<int32_t>& own = pages[sequence];
        for (const size_t keep = pages_for(tokens); own.size() > keep; own.pop_back()) free.push_back(own.back());
    }
    void grow(size_t sequence, size_t tokens) {  // (the caller has seen that there are enough)
        std::vector<int32_t>& own = pages[sequence];
        for (const size_t need = pages_for(tokens); own.size() < need; free.pop_back()) own.push_back(free.back());
    }
    size_t missing(size_t sequence, size_t tokens) const { return std::max(pages_for(tokens), pages[sequence].size()) - pages[sequence].size(); }
};

}  // namespace qtb
