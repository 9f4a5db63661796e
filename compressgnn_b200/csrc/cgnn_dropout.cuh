// A dropout as the row operators take it.
#pragma once

#include <algorithm>

#include "cgnn_philox.cuh"

namespace cgnn {

// An element is dropped when its 32-bit random word is below `threshold`; the survivors are multiplied by `scale`.
// The key is a number, or lies in device memory, where a captured graph finds another one at every replay.
struct Drop {
    uint32_t threshold = 0;  // 0: nothing is dropped
    double scale = 1.0;
    uint64_t seed = 0;
    const int64_t *device_seed = nullptr;

    static Drop of(double p, uint64_t seed, const int64_t *device_seed) {
        Drop d;
        d.threshold = drop_threshold_of(p);
        if (d.threshold) d.scale = 1.0 / (1.0 - p);
        d.seed = seed;
        d.device_seed = device_seed;
        return d;
    }
    __device__ __forceinline__ uint64_t key() const { return device_seed ? (uint64_t)*device_seed : seed; }
};

}  // namespace cgnn
