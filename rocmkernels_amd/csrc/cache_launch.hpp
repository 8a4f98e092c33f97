// Host-side launch interface between the cache's C entry points (cache_abi.hip) and its kernels (cache_append.hip,
// cache_attention.hip). Arguments are already validated when the launchers are called.
#pragma once

#include <hip/hip_runtime.h>

#include <rocmkernels_cache.h>

#include <stdint.h>

#include "cache_plan.hpp"

namespace rk {

constexpr int kScaleLow = -100;    // exponents a scale may take: 448 * 2^120 is the largest FP32 magnitude
constexpr int kScaleHigh = 120;

struct CacheView {
    uint8_t *keys, *values;
    float *scales;
    int pages, page_size, heads;
};

struct AppendArgs {
    const void *k, *v, *q;
    const float *cos, *sin;
    void *oq;
    CacheView cache;
    SequenceView seqs;
    int query_heads, positions;
    rocmkernels_strides ks, vs, qs, os, cs, ss;
    int dtype;
};

struct CacheForwardArgs {
    const void *q;
    CacheView cache;
    SequenceView seqs;
    void *output;
    float *lse;
    int query_heads, max_keys, radius, causal;
    rocmkernels_strides qs, os;
    int dtype;
    void *workspace;
};

hipError_t launch_cache_append(int width, const AppendArgs &a, hipStream_t stream);
hipError_t launch_cache_forward(int width, const CacheForwardArgs &a, const ForwardPlan &plan, hipStream_t stream);

} // namespace rk
