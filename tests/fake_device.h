// fake_device.h -- one recorded launch of the stand-in for the CUDA runtime (fake_device.cpp).
#pragma once

#include <cstdint>

enum { ROTATE, PREFIX, STREAM, COMBINE, OTHER };

struct Launch {
    int32_t kind, device, grid, threads, smem, allowed;   // allowed: bytes the kernel may take on this device
    int32_t counter;                                       // of shared runs, before the launch
    int32_t prefix_tiles, n_split, split_tiles, row_groups, stream_ctas, stream_runs, shared_runs, rows;
};

// What an attention kernel's arguments say (fake_device.cu); does to the counter of runs what the kernel does.
extern "C" void fake_paged(const void *args, Launch *l);
