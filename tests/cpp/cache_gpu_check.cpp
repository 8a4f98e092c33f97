// GPU run of the paged cache's C++ wrappers (include/ROCmKernels/Kernels/Cache/KeyValueCache.hpp), built as a small shared library:
// tests/test_cache_gpu.py calls it in its own process on tensors of its own and compares the results bit for bit with the
// same step through the C entry points, so a wrapper that swapped or dropped an argument fails.
//
// int cache_step(...): appends k and v with the rotation, rotates q into oq and attends with it; returns the workspace bytes of the
// attention call, or -1 where a wrapper threw (its message on stderr). workspace has to hold what CacheWorkspace reports.
#include <ROCmKernels/Kernels/Cache/KeyValueCache.hpp>

#include <cstdio>

extern "C" __attribute__((visibility("default"))) long long cache_step(const void *k, const void *v, const void *q, const float *cos,
        const float *sin, void *oq, void *output, float *lse, const rocmkernels_cache cache, const rocmkernels_sequences sequences,
        const int queryHeads, const int positions, const int maxKeys, const int radius, const int flags, const rocmkernels_strides ks,
        const rocmkernels_strides vs, const rocmkernels_strides qs, const rocmkernels_strides os, const rocmkernels_strides cs,
        const rocmkernels_strides ss, const unsigned char dtype, void *workspace, const unsigned long long workspaceBytes, hipStream_t stream) {
    using namespace ROCmKernels::Kernels;
    try {
        const auto type = static_cast<DType>(dtype);
        const std::size_t need = CacheWorkspace(cache, sequences, queryHeads, maxKeys, type);
        CacheAppend(k, v, q, cos, sin, oq, cache, sequences, queryHeads, positions, ks, vs, qs, os, cs, ss, type, stream);
        CacheForward(oq, cache, sequences, output, lse, queryHeads, maxKeys, radius, flags, os, os, type, workspace, workspaceBytes, stream);
        return static_cast<long long>(need);
    } catch (const ROCmKernels::HipError &error) {
        std::fprintf(stderr, "%s\n", error.what());
        return -1;
    }
}
