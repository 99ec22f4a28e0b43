// prefix.cuh -- the handle of a shared prefix kept as XKV blobs (made in api.cu, read in batch.cu).
#pragma once

#include <vector>

#include "paged.cuh"

struct kvx_prefix_s {
    int n_kv_heads = 0, dim = 0, seq = 0, device = 0;
    kvx::XkvDev dev{};
    std::vector<void *> owned;   // device arrays
    ~kvx_prefix_s() {
        for (void *p : owned) cudaFree(p);
    }
};
