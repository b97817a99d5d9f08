// The paged cache as the rest of the library sees it (paged.cu).
#pragma once
#include <cuda_runtime.h>

#include <mutex>

#include "../../include/quintrit_b200.h"

struct quintrit_b200_paged_cache {
    uint32_t magic;
    int device, sm_count;
    uint32_t layers, pages, page_tokens, kv_heads, head_dim;
    int32_t type;
    unsigned char *k = nullptr, *v = nullptr;  // [layers] of the layout of paged_cache.cuh
    float *ks = nullptr, *vs = nullptr;        // Q8: scales
    unsigned int* status = nullptr;            // the calls' word, and what a report last took out of it
    size_t layer_bytes = 0, layer_scales = 0, device_bytes = 0;
    std::mutex report;                         // one report at a time
};

namespace qtb {
void paged_cache_destroy(quintrit_b200_paged_cache* cache);  // quintrit_b200_paged_cache_free that leaves the thread's last error as it is
}
