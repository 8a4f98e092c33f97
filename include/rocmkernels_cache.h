/*
 * C ABI of the paged 8-bit key/value cache of libROCmKernels.Kernels.Shared.so (MI355X, gfx950): appending keys and values
 * with the position rotation applied on the way, and attention over what the cache holds.
 *
 * The cache. A page holds page_size tokens of one sequence for every K/V head. Keys and values are OCP e4m3 bytes, with one
 * scale per page and head for the keys and one for the values; a scale is a power of two between 2^-100 and 2^120 (only its
 * exponent is read, clamped to that range), and a byte stands for its e4m3 value times its scale.
 *   keys    [page][head][page_size / 16][16 tokens][width]
 *   values  [page][head][page_size / 16][width][16 tokens]   (each 16-token block transposed: the matrix operand's order)
 *   scales  [page][head][2] = {keys, values}, float
 * page_size is a multiple of 16 from 16 to 128, width 32, 64 or 128. keys and values are 16-byte aligned, scales 8-byte.
 *
 * The sequences. The new rows of all sequences are packed: sequence b owns rows starts[b] .. starts[b + 1] - 1 of every
 * [token][head][width] tensor, and lengths[b] counts its keys INCLUDING these rows, so row i of its n rows stands at position
 * lengths[b] - n + i. table[b * table_stride + p] is the page of positions p * page_size .. (p + 1) * page_size - 1, for
 * p < columns. One scheduler state therefore serves both calls of a step: append, then forward. starts (ascending, batch + 1
 * values), lengths and table are device memory. Sequences may have no rows.
 *   - Rows at or behind starts[batch] are left as they were in every output.
 *   - A page id outside 0 .. pages - 1 is no page: nothing is written there, and its keys are not visible.
 *   - A row at a negative position (fewer keys than rows) or at one that has no column is not written to the cache.
 *
 * Conventions, as in rocmkernels_attention.h: strides are element strides of [token][head][width] tensors with contiguous
 * features (the batch entry is not used); the softmax scale is 1/sqrt(width); lse is packed [token][query head][2] = {row
 * maximum of the scaled scores, sum of exp(score - maximum)}, and a row with no visible key gets output 0 and lse {-inf, 0};
 * dtype is the type of q, k, v and the outputs: ROCMKERNELS_DTYPE_FLOAT32, _FLOAT16 or _BFLOAT16. Query head i reads K/V head
 * i / (query_heads / cache.heads). Calls are asynchronous on `stream`; nothing is allocated, freed or synchronised; the return
 * value is a hipError_t as int, hipErrorInvalidValue for invalid arguments, found before any HIP call.
 */
#ifndef ROCMKERNELS_CACHE_H
#define ROCMKERNELS_CACHE_H

#include <rocmkernels_attention.h>

#include <stddef.h>

#ifdef __cplusplus
extern "C" {
#endif

typedef struct rocmkernels_cache {
    void *keys;
    void *values;
    float *scales;
    int pages;
    int page_size;
    int heads;
    int width;
} rocmkernels_cache;

typedef struct rocmkernels_sequences {
    const int *starts;
    const int *lengths;
    const int *table;
    int batch;
    int tokens; /* rows of the packed tensors; starts are clamped to it */
    int columns;
    int table_stride;
} rocmkernels_sequences;

/*
 * Appends the rows of k and v to the cache. With cos and sin (both or neither) k is rotated first, in the convention of
 * rotary_fp32: column c < width / 2 pairs with c + width / 2, out[c] = x[c] cos[c] - x[c + w/2] sin[c] and out[c + w/2] =
 * x[c + w/2] cos[c + w/2] + x[c] sin[c + w/2], each product rounded to FP32 before the sum. cos and sin hold `width` floats for
 * each of `positions` positions (row stride: the token entry of cs and ss), shared by heads and sequences; a row at a position
 * behind them is neither rotated nor written. With q and oq (both or neither; they need cos and sin) the query rows are rotated
 * too and written to oq, which may be q; query_heads is not read without them.
 *
 * For each page and head touched: a = the largest finite magnitude among the new rows (after rotation) and e the smallest
 * exponent with a <= 448 * 2^e. A page whose first token is among the new rows takes the scale 2^e; a page that held tokens
 * before keeps the larger of its scale and 2^e, and where it grows the rows before the first new one are requantised from their
 * stored values (exact but for values that fall into e4m3's subnormals). Rows behind the last new one are left alone. Values
 * are rounded to nearest even; infinities and NaN become e4m3's NaN and touch no scale.
 *
 * A page that receives rows belongs to one sequence: where two sequences append to one page in a call, what it holds afterwards
 * is not defined. Appending the same rows again at the same positions is allowed (drafted tokens that were rejected).
 */
ROCMKERNELS_EXPORT int attention_cache_append(const void *k, const void *v, const void *q, const float *cos, const float *sin, void *oq,
        rocmkernels_cache cache, rocmkernels_sequences sequences, int query_heads, int positions, rocmkernels_strides ks,
        rocmkernels_strides vs, rocmkernels_strides qs, rocmkernels_strides os, rocmkernels_strides cs, rocmkernels_strides ss,
        rocmkernels_dtype dtype, hipStream_t stream);

/*
 * Attention of the query rows over the cached keys of their sequence. Keys at positions lengths[b] and behind are not visible;
 * with ROCMKERNELS_ATTENTION_CAUSAL in flags a row sees keys at its own position and before; with radius >= 0 it sees keys with
 * |row position - key position| <= radius. A key that a row does not see contributes nothing to it, whatever it holds.
 * lse may be NULL. max_keys is a number of keys that no sequence exceeds (at most columns * page_size; 0: that): it shapes the
 * launch, and keys behind it are not visible.
 * Scores, softmax statistics and sums are FP32. FP32 rows are formed from two fp16 terms of each operand (22 bits or more), 16-bit
 * rows from one (weights keep 11 bits).
 * workspace: 16-byte aligned device memory of at least the bytes that attention_cache_workspace reports for the same sizes (NULL
 * where it reports 0). Its contents on entry do not matter; calls that may run at the same time need one each.
 * Results are the same bits from run to run.
 */
ROCMKERNELS_EXPORT int attention_cache_forward(const void *q, rocmkernels_cache cache, rocmkernels_sequences sequences, void *output,
        float *lse, int query_heads, int max_keys, int radius, int flags, rocmkernels_strides qs, rocmkernels_strides os,
        rocmkernels_dtype dtype, void *workspace, size_t workspace_bytes, hipStream_t stream);

/* Workspace bytes of attention_cache_forward for any radius and flags; only cache's and sequences' sizes are read, not their pointers. */
ROCMKERNELS_EXPORT int attention_cache_workspace(rocmkernels_cache cache, rocmkernels_sequences sequences, int query_heads,
        int max_keys, rocmkernels_dtype dtype, size_t *bytes);

#ifdef __cplusplus
} /* extern "C" */
#endif

#endif /* ROCMKERNELS_CACHE_H */
