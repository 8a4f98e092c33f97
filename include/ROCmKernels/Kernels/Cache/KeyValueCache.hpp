#pragma once

// Throwing C++ wrappers over the paged 8-bit key/value cache's C entry points (no reference counterpart). The cache's layout, the
// packed sequences and every argument are described in rocmkernels_cache.h; each wrapper throws ROCmKernels::HipError when the
// entry point returns a non-zero hipError_t.

#include <ROCmKernels/Common/Error.hpp>
#include <ROCmKernels/Kernels/DType.hpp>
#include <ROCmKernels/Kernels/Strides.hpp>

#include <rocmkernels_cache.h>

#include <cstddef>

namespace ROCmKernels::Kernels {
    using KeyValueCache = rocmkernels_cache;
    using CacheSequences = rocmkernels_sequences;

    /// Quantises the rows of k and v into the cache, K rotated by position with cos and sin (both or neither); with q and oq the
    /// query rows are rotated too.
    inline void CacheAppend(const void *k, const void *v, const void *q, const float *cos, const float *sin, void *oq,
            const KeyValueCache &cache, const CacheSequences &sequences, const int queryHeads, const int positions, const Strides &ks,
            const Strides &vs, const Strides &qs, const Strides &os, const Strides &cs, const Strides &ss, const DType dtype,
            hipStream_t stream = nullptr) {
        ROCMKERNELS_HIP_CHECK(attention_cache_append(k, v, q, cos, sin, oq, cache, sequences, queryHeads, positions, ks, vs, qs, os, cs, ss,
                static_cast<rocmkernels_dtype>(dtype), stream));
    }

    /// Attention of the query rows over the cached keys of their sequence; flags as in AttentionForwardFlashEx.
    inline void CacheForward(const void *q, const KeyValueCache &cache, const CacheSequences &sequences, void *output, float *lse,
            const int queryHeads, const int maxKeys, const int radius, const int flags, const Strides &qs, const Strides &os,
            const DType dtype, void *workspace, const std::size_t workspaceBytes, hipStream_t stream = nullptr) {
        ROCMKERNELS_HIP_CHECK(attention_cache_forward(q, cache, sequences, output, lse, queryHeads, maxKeys, radius, flags, qs, os,
                static_cast<rocmkernels_dtype>(dtype), workspace, workspaceBytes, stream));
    }

    /// Bytes of CacheForward's workspace for these sizes (no pointer is read).
    inline std::size_t CacheWorkspace(const KeyValueCache &cache, const CacheSequences &sequences, const int queryHeads,
            const int maxKeys, const DType dtype) {
        std::size_t bytes = 0;
        ROCMKERNELS_HIP_CHECK(
                attention_cache_workspace(cache, sequences, queryHeads, maxKeys, static_cast<rocmkernels_dtype>(dtype), &bytes));
        return bytes;
    }
} // namespace ROCmKernels::Kernels
