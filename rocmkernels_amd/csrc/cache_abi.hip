// C entry points of the paged 8-bit cache: argument validation, then one launch path for each.
#include <rocmkernels_cache.h>

#include "cache_launch.hpp"

namespace {

constexpr int kInvalid = hipErrorInvalidValue;
constexpr long long kIntLimit = 1ll << 31;
constexpr int kPositionLimit = 1 << 30;

// Sizes of the cache and the sequences, without their pointers.
bool bad_sizes(const rocmkernels_cache &c, const rocmkernels_sequences &s) {
    if (c.pages <= 0 || c.heads <= 0 || (c.width != 32 && c.width != 64 && c.width != 128)) return true;
    if (c.page_size < rk::kBlockTokens || c.page_size > rk::kMaxPage || c.page_size % rk::kBlockTokens != 0) return true;
    if (s.batch <= 0 || s.tokens < 0 || s.tokens >= kPositionLimit || s.columns <= 0 || s.table_stride < s.columns) return true;
    // Positions and 16-token blocks are numbered with 32 bits.
    if (static_cast<long long>(s.columns) * c.page_size > kPositionLimit) return true;
    if (static_cast<long long>(c.pages) * c.heads >= kIntLimit / (c.page_size / rk::kBlockTokens)) return true;
    // So is what a sequence's rows are found by: tokens + batch * (2 * page_size - 2) + page_size.
    return s.tokens + static_cast<long long>(s.batch) * (2 * c.page_size) + c.page_size >= kIntLimit;
}

bool misaligned(const void *p, const uintptr_t mask) { return (reinterpret_cast<uintptr_t>(p) & mask) != 0; }

bool bad_pointers(const rocmkernels_cache &c, const rocmkernels_sequences &s) {
    return !c.keys || !c.values || !c.scales || misaligned(c.keys, 15) || misaligned(c.values, 15) || misaligned(c.scales, 7) ||
            !s.starts || !s.lengths || !s.table;
}

bool bad_dtype(const rocmkernels_dtype dtype) { return dtype > ROCMKERNELS_DTYPE_BFLOAT16; }

bool bad_query_heads(const rocmkernels_cache &c, const rocmkernels_sequences &s, const int query_heads) {
    if (query_heads <= 0 || query_heads % c.heads != 0) return true;
    const long long group = query_heads / c.heads;
    // Rows of a sequence times the heads of a group, and a tile for each sequence, are counted with 31 bits.
    return s.tokens * group + static_cast<long long>(s.batch) * rk::kMaxRows + rk::kMaxRows >= kIntLimit;
}

rk::CacheView view(const rocmkernels_cache &c) {
    return {static_cast<uint8_t *>(c.keys), static_cast<uint8_t *>(c.values), c.scales, c.pages, c.page_size, c.heads};
}
rk::SequenceView view(const rocmkernels_sequences &s) {
    return {s.starts, s.lengths, s.table, s.batch, s.tokens, s.columns, s.table_stride};
}

// Keys that a launch is shaped for: max_keys within the table's positions; negative for a bad argument.
int key_limit(const rocmkernels_cache &c, const rocmkernels_sequences &s, const int max_keys) {
    const int most = s.columns * c.page_size;
    return max_keys < 0 ? -1 : max_keys == 0 || max_keys > most ? most : max_keys;
}

} // namespace

extern "C" {

int attention_cache_append(const void *k, const void *v, const void *q, const float *cos, const float *sin, void *oq,
        rocmkernels_cache cache, rocmkernels_sequences sequences, int query_heads, int positions, rocmkernels_strides ks,
        rocmkernels_strides vs, rocmkernels_strides qs, rocmkernels_strides os, rocmkernels_strides cs, rocmkernels_strides ss,
        rocmkernels_dtype dtype, hipStream_t stream) {
    if (!k || !v || bad_sizes(cache, sequences) || bad_pointers(cache, sequences) || bad_dtype(dtype)) return kInvalid;
    if (!cos != !sin || !q != !oq || (q && !cos)) return kInvalid;
    if (q && bad_query_heads(cache, sequences, query_heads)) return kInvalid;
    if (cos && positions <= 0) return kInvalid;
    const int capacity = sequences.columns * cache.page_size;
    const rk::AppendArgs a{k, v, q, cos, sin, oq, view(cache), view(sequences), query_heads,
            cos && positions < capacity ? positions : capacity, ks, vs, qs, os, cs, ss, dtype};
    if (sequences.tokens == 0) return hipSuccess;
    return rk::launch_cache_append(cache.width, a, stream);
}

int attention_cache_forward(const void *q, rocmkernels_cache cache, rocmkernels_sequences sequences, void *output, float *lse,
        int query_heads, int max_keys, int radius, int flags, rocmkernels_strides qs, rocmkernels_strides os, rocmkernels_dtype dtype,
        void *workspace, size_t workspace_bytes, hipStream_t stream) {
    if (!q || !output || bad_sizes(cache, sequences) || bad_pointers(cache, sequences) || bad_dtype(dtype)) return kInvalid;
    if (bad_query_heads(cache, sequences, query_heads) || radius < -1 || (flags & ~ROCMKERNELS_ATTENTION_CAUSAL) != 0) return kInvalid;
    const int keys = key_limit(cache, sequences, max_keys);
    if (keys < 0) return kInvalid;
    if (sequences.tokens == 0) return hipSuccess;
    const int window = radius >= kPositionLimit ? -1 : radius;
    const rk::CacheForwardArgs a{q, view(cache), view(sequences), output, lse, query_heads, keys, window,
            flags & ROCMKERNELS_ATTENTION_CAUSAL, qs, os, dtype, workspace};
    const rk::ForwardPlan plan = rk::plan_cache_forward(cache.width, a.seqs, cache.heads, query_heads, keys, window, a.causal != 0);
    if (plan.workspace > 0 && (!workspace || misaligned(workspace, 15) || workspace_bytes < plan.workspace)) return kInvalid;
    return rk::launch_cache_forward(cache.width, a, plan, stream);
}

int attention_cache_workspace(rocmkernels_cache cache, rocmkernels_sequences sequences, int query_heads, int max_keys,
        rocmkernels_dtype dtype, size_t *bytes) {
    if (!bytes || bad_sizes(cache, sequences) || bad_dtype(dtype) || bad_query_heads(cache, sequences, query_heads)) return kInvalid;
    const int keys = key_limit(cache, sequences, max_keys);
    if (keys < 0) return kInvalid;
    *bytes = sequences.tokens == 0 ? 0
                                   : rk::plan_cache_forward(cache.width, view(sequences), cache.heads, query_heads, keys, -1, false)
                                             .workspace_most;
    return hipSuccess;
}

} // extern "C"
