// Attention over the paged 8-bit cache for single tokens, drafted tokens and prompts (MI355X, gfx950).
//
// With K = 2^ek k8 and V = 2^ev v8 (k8, v8 the e4m3 values, ek and ev the exponents of the key's page and head) and everything in
// the exponent of 2:  s = (q . k8) 2^ek log2(e) / sqrt(D),  O = sum 2^s 2^ev v8 / sum 2^s.
//   * e4m3 values are fp16 values, so both products run on v_mfma_f32_16x16x32_f16 with k8 and v8 converted exactly (two to a
//     v_cvt_scalef32_pk_f16_fp8). The only operands that are rounded are q and the weights: fp16 rows as they are, bf16 and FP32
//     rows scaled by a power of two that brings the row's maximum to [2^14, 2^15); FP32 rows and their weights in two terms
//     x = hi + lo, 22 bits and more.
//   * The V scale is part of the softmax reference instead of a product per value: w = 2^(s + ev - M), with M the running maximum
//     of s + ev over the row, weighs v8 directly and stays in fp16's range whatever the scales are; the sum of 2^s is kept as
//     sum w 2^-ev in the same units, so O = acc / l. Weights are held 2^7 higher (w <= 2^7 at the reference): they keep all
//     11 bits down to 2^-21 of it. The reference moves only when a score passes it by more than 2^8 (w <= 2^15).
//   * S^T = K Q^T and O^T = V^T P^T: a lane holds the scores of one query row (column lane % 16), so the softmax needs no
//     exchange but the maximum over the four lanes of a column. A wave takes 64 keys a step, as 4 tiles of 16. Row r of tile t is
//     token 16 (r / 4) + 4 t + r % 4, which leaves lane (column, g) with the scores of the 16 tokens of block g, in the order
//     in which V's block g lies in memory: weights and V meet with no exchange. Each 16-token block has a page and scales of its
//     own, so any page size is a matter of addresses.
//   * A row of K is 16 contiguous bytes a lane (the features of both operands in the same permuted order), a feature of V's block too:
//     every load is 16 bytes wide and covers whole lines.
// Rows of a sequence are flattened to (row, query head of the group), so that grouped heads share a read of K and V. Four
// waves of a workgroup take alternate steps and are merged through LDS; where there are few rows, the keys are also cut into
// chunks for several workgroups, merged in order by a second kernel.
#include "cache_device.hpp"
#include "cache_launch.hpp"

namespace rk {

namespace {

constexpr float kWeightShift = 7.0f;   // weights are 2^7 at the reference
constexpr float kLazyRange = 8.0f;     // and reach 2^15 before it moves

__device__ __forceinline__ f32x4 mfma_16(const f16x8 a, const f16x8 b, const f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

// 8 e4m3 bytes as fp16, exactly.
__device__ __forceinline__ f16x8 widen(const uint32_t lo, const uint32_t hi) {
    const f16x2 a = __builtin_bit_cast(f16x2, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.0f, false));
    const f16x2 b = __builtin_bit_cast(f16x2, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.0f, true));
    const f16x2 c = __builtin_bit_cast(f16x2, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.0f, false));
    const f16x2 d = __builtin_bit_cast(f16x2, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.0f, true));
    return f16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// 0xff in the bytes of w that hold NaN (0x7f or 0xff).
__device__ __forceinline__ uint32_t nan_bytes(const uint32_t w) {
    const uint32_t x = (w & 0x7f7f7f7fu) + 0x01010101u; // bit 7 set exactly where the low 7 bits are all ones
    return ((x & 0x80808080u) >> 7) * 0xffu;
}

// Byte mask of a dword of 4 tokens from the low 4 bits of `bits`.
__device__ __forceinline__ uint32_t byte_mask(const uint32_t bits) {
    return ((bits & 1u) | ((bits & 2u) << 7) | ((bits & 4u) << 14) | ((bits & 8u) << 21)) * 0xffu;
}

// Keys that the rows of a tile see: row i of the sequence sees [low(i), high(i)).
struct Visibility {
    int length, radius, causal;
    __device__ __forceinline__ int low(const int position) const { return radius >= 0 ? max(0, position - radius) : 0; }
    __device__ __forceinline__ int high(const int position) const {
        int h = length;
        if (radius >= 0) h = min(h, position + radius + 1); // both below 2^30
        if (causal) h = min(h, position + 1);
        return max(h, 0);
    }
};

// A workgroup's rows and keys.
struct Tile {
    Sequence s;
    Visibility vis;
    int row0, rows;            // flattened rows row0 .. row0 + rows - 1 of the sequence; rows <= 0: nothing to do
    int step0, steps, chunks;  // steps of 64 keys that any of them sees, and the chunks they are cut into
};

__device__ __forceinline__ Tile tile_of(const CacheForwardArgs &a, const ForwardPlan &plan, const uint32_t unit, const int group) {
    Tile t;
    t.s = find_sequence(a.seqs, unit, group, plan.rows - 1, plan.rows);
    const uint32_t index = unit - t.s.base;
    const uint32_t flat = static_cast<uint32_t>(t.s.count) * group;
    t.row0 = static_cast<int>(index * plan.rows);
    t.rows = index < (flat + plan.rows - 1) / plan.rows ? min(plan.rows, static_cast<int>(flat) - t.row0) : 0;
    t.vis = Visibility{min(t.s.length, a.max_keys), a.radius, a.causal};
    const int first = t.s.first + t.row0 / group, last = t.s.first + (t.row0 + t.rows - 1) / group;
    const int low = t.vis.low(first), high = t.vis.high(last);
    t.step0 = low / kStep;
    t.steps = t.rows > 0 && high > low ? (high + kStep - 1) / kStep - t.step0 : 0;
    t.chunks = (t.steps + plan.chunk_steps - 1) / plan.chunk_steps;
    return t;
}

// Writes one row's output from its sums: acc over N features, l, the reference M (s + ev) and the maximum m of s (all base 2).
template<int T, bool VEC, int N>
__device__ __forceinline__ void finish_row(const CacheForwardArgs &a, const int64_t token, const int head, const int feature,
        const float (&acc)[N], const float l, const float reference, const float m, const bool writes_lse) {
    const bool nan_row = isnan(l), has_keys = l > 0.0f;
    const float factor = has_keys ? 1.0f / l : (nan_row ? NAN : 0.0f);
    float o[N];
#pragma unroll
    for (int i = 0; i < N; ++i) o[i] = has_keys ? acc[i] * factor : factor;
    store_row<T, VEC>(a.output, token * a.os.token + static_cast<int64_t>(head) * a.os.head + feature, o);
    if (writes_lse && a.lse) {
        float *const p = a.lse + 2 * (token * a.query_heads + head);
        p[0] = has_keys ? m / kLog2e : (nan_row ? NAN : -INFINITY);
        p[1] = has_keys ? l * exp2_fast(reference - m - kWeightShift) : (nan_row ? NAN : 0.0f);
    }
}

// Workspace: [slot][rows][D] partial sums, then [slot][rows][4] = {M, l, m, unused}; slot = (unit * heads + head) * chunks + chunk.
struct Partial {
    float *acc, *stats;
};
template<int D>
__device__ __forceinline__ Partial partial_of(const CacheForwardArgs &a, const ForwardPlan &plan, const int64_t slot, const int row) {
    float *const base = static_cast<float *>(a.workspace);
    const int64_t slots = static_cast<int64_t>(plan.units) * a.cache.heads * plan.chunks, r = slot * plan.rows + row;
    return {base + r * D, base + slots * plan.rows * D + r * 4};
}

// The two terms of 8 values that are already scaled into fp16's range.
template<bool TWO>
__device__ __forceinline__ void split_terms(f16x8 &hi, f16x8 &lo, const float (&x)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        hi[i] = static_cast<_Float16>(x[i]);
        if constexpr (TWO) lo[i] = static_cast<_Float16>(x[i] - static_cast<float>(hi[i]));
    }
}

// NQ tiles of 16 rows a workgroup.
template<int T, int D, int NQ, bool VEC>
__global__ __launch_bounds__(kThreads) __attribute__((amdgpu_waves_per_eu(2))) void cache_attention_kernel(const CacheForwardArgs a,
        const ForwardPlan plan) {
    constexpr bool TWO = T == kFloat32;
    constexpr int KC = D / 32;                   // MFMAs of a score tile
    constexpr int KL = D >= 64 ? D / 64 : 1;     // loads of a K row tile
    constexpr int DT = D / 16;                   // output tiles
    constexpr int ROWS = 16 * NQ;
    constexpr int STRIDE = D + 4;
    __shared__ float merged[kWaves][ROWS][STRIDE];
    __shared__ float stats[kWaves][ROWS][4];

    const int lane = threadIdx.x & (kWave - 1), col = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int heads = a.cache.heads, group = a.query_heads / heads;
    const uint32_t slot = blockIdx.x, pair = slot / plan.chunks;
    const int chunk = static_cast<int>(slot - pair * plan.chunks);
    const uint32_t unit = pair / heads;
    const int head = static_cast<int>(pair - unit * heads);

    const Tile t = tile_of(a, plan, unit, group);
    if (t.rows <= 0 || chunk >= max(t.chunks, 1)) return;
    const int step_begin = t.step0 + chunk * plan.chunk_steps;
    const int step_end = t.step0 + min(t.steps, (chunk + 1) * plan.chunk_steps);

    // This lane's rows: q in operand order, the factor of its scores, and the keys it sees.
    f16x8 qh[NQ][KC], ql[TWO ? NQ : 1][TWO ? KC : 1];
    float c2[NQ];
    int low[NQ], high[NQ];
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
        const int r = 16 * n + col;
        const bool used = r < t.rows;
        const int flat = t.row0 + (used ? r : 0), i = flat / group, query_head = head * group + (flat - i * group);
        const int64_t row = static_cast<int64_t>(t.s.row0 + i) * a.qs.token + static_cast<int64_t>(query_head) * a.qs.head;
        const int position = t.s.first + i;
        low[n] = t.vis.low(position);
        high[n] = t.vis.high(position);
        float x[KC][8];
#pragma unroll
        for (int k = 0; k < KC; ++k) {
            const int f = D >= 64 ? 64 * (k / 2) + 16 * g + 8 * (k % 2) : 8 * g;
            load8<T, VEC>(x[k], a.q, row + f);
        }
        float scale = 1.0f, back = 1.0f;
        if constexpr (T != kFloat16) {
            float most = 0.0f;
#pragma unroll
            for (int k = 0; k < KC; ++k) {
#pragma unroll
                for (int j = 0; j < 8; ++j) most = fmaxf(most, fabsf(x[k][j]));
            }
            most = fmaxf(most, __shfl_xor(most, 16));
            most = fmaxf(most, __shfl_xor(most, 32));
            const int e = clamped(static_cast<int>(__float_as_uint(most) >> 23) - 127, -100, 127);
            scale = power(14 - e);
            back = power(e - 14);
        }
        c2[n] = back * (kLog2e / sqrtf(static_cast<float>(D)));
#pragma unroll
        for (int k = 0; k < KC; ++k) {
#pragma unroll
            for (int j = 0; j < 8; ++j) x[k][j] *= scale;
            split_terms<TWO>(qh[n][k], ql[TWO ? n : 0][TWO ? k : 0], x[k]);
        }
    }
    // Keys that every row sees: between the last row's first key and the first row's end.
    const int all_low = t.vis.low(t.s.first + (t.row0 + t.rows - 1) / group), all_high = t.vis.high(t.s.first + t.row0 / group);

    float M[NQ], l[NQ], m[NQ];
    f32x4 acc[NQ][DT];
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
        M[n] = -INFINITY;
        m[n] = -INFINITY;
        l[n] = 0.0f;
#pragma unroll
        for (int d = 0; d < DT; ++d) acc[n][d] = f32x4{};
    }

    // The 64 blocks of this wave's next 16 steps, one a lane: the block's place in the cache (-1: none) and its exponents.
    const int blocks = a.cache.page_size / kBlockTokens;
    int place = -1, exponents = 0;
    uint64_t absent = 0;
    auto look_up = [&](const int step) __attribute__((always_inline)) {
        const int s = step + kWaves * (lane / 4), position = kStep * s + kBlockTokens * (lane % 4);
        place = -1;
        exponents = 0;
        if (s < step_end && position < t.vis.length) {
            const int index = position / a.cache.page_size;
            const int page = a.seqs.table[static_cast<int64_t>(t.s.b) * a.seqs.table_stride + index];
            if (page >= 0 && page < a.cache.pages) {
                const int cell = page * heads + head;
                place = cell * blocks + (position - index * a.cache.page_size) / kBlockTokens;
                exponents = (scale_exponent(a.cache.scales[2 * static_cast<int64_t>(cell)]) & 0xffff) |
                        (scale_exponent(a.cache.scales[2 * static_cast<int64_t>(cell) + 1]) << 16);
            }
        }
        absent = __ballot(place < 0);
    };

    struct Keys {
        u32x4 k[4][KL]; // D = 32: 8 bytes of each
        u32x4 v[DT];
    };
    auto load_keys = [&](Keys &x, const int turn) __attribute__((always_inline)) {
        // Blocks that are not there read block 0 of the cache, which is; their keys are hidden.
        const int64_t kb = max(__shfl(place, 4 * turn + (col >> 2)), 0), vb = max(__shfl(place, 4 * turn + g), 0);
        const uint8_t *const k = a.cache.keys + kb * (kBlockTokens * D) + (col & 3) * D;
        const uint8_t *const v = a.cache.values + vb * (kBlockTokens * D) + col * 16;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (D >= 64) {
#pragma unroll
                for (int j = 0; j < KL; ++j) x.k[i][j] = *reinterpret_cast<const u32x4 *>(k + 4 * i * D + 64 * j + 16 * g);
            } else {
                const u32x2 w = *reinterpret_cast<const u32x2 *>(k + 4 * i * D + 8 * g);
                x.k[i][0] = u32x4{w[0], w[1], 0u, 0u};
            }
        }
#pragma unroll
        for (int d = 0; d < DT; ++d) x.v[d] = *reinterpret_cast<const u32x4 *>(v + d * 256);
    };

    auto compute = [&](Keys &x, const int turn, const int step) __attribute__((always_inline)) {
        const int exps = __shfl(exponents, 4 * turn + g);
        const int ek = static_cast<int16_t>(exps & 0xffff), ev = exps >> 16;
        const float fev = static_cast<float>(ev), inverse = power(-ev), kscale = power(ek);
        f32x4 sc[NQ][4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
#pragma unroll
            for (int n = 0; n < NQ; ++n) sc[n][i] = f32x4{};
#pragma unroll
            for (int k = 0; k < KC; ++k) {
                const f16x8 w = widen(x.k[i][k / 2][2 * (k % 2)], x.k[i][k / 2][2 * (k % 2) + 1]);
#pragma unroll
                for (int n = 0; n < NQ; ++n) {
                    sc[n][i] = mfma_16(w, qh[n][k], sc[n][i]);
                    if constexpr (TWO) sc[n][i] = mfma_16(w, ql[n][k], sc[n][i]);
                }
            }
        }
        const int key0 = kStep * step, base = key0 + 16 * g;
        const bool full = key0 >= all_low && key0 + kStep <= all_high && ((absent >> (4 * turn)) & 15u) == 0;
        uint32_t visible[NQ];
        bool any_nan = false;
        if (!full) {
            const bool here = !((absent >> (4 * turn + g)) & 1u);
#pragma unroll
            for (int n = 0; n < NQ; ++n) {
                visible[n] = here ? bit_range(low[n] - base, high[n] - base - 1) & 0xffffu : 0u;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) sc[n][i][j] = (visible[n] >> (4 * i + j)) & 1u ? sc[n][i][j] : -INFINITY;
                }
            }
            // Bytes behind the sequence's end may hold anything, and 0 times NaN is no 0.
            const uint32_t held = here ? bit_range(0, t.vis.length - base - 1) & 0xffffu : 0u;
            uint32_t nans = 0;
#pragma unroll
            for (int d = 0; d < DT; ++d) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    x.v[d][i] &= byte_mask(held >> (4 * i));
                    nans |= nan_bytes(x.v[d][i]);
                }
            }
            any_nan = __ballot(nans != 0) != 0;
        }
#pragma unroll
        for (int n = 0; n < NQ; ++n) {
            const float c = fmaxf(c2[n] * kscale, 1.17549435e-38f); // > 0, so that hidden scores stay -inf
            float most = sc[n][0][0];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
#pragma unroll
                for (int j = 0; j < 4; ++j) most = fmaxf(most, sc[n][i][j]);
            }
            most *= c;
            m[n] = fmaxf(m[n], most);
            const float candidate = most + fev;
            if (__ballot(candidate > M[n] + kLazyRange)) {
                float raised = fmaxf(M[n], candidate);
                raised = fmaxf(raised, __shfl_xor(raised, 16));
                raised = fmaxf(raised, __shfl_xor(raised, 32));
                const float alpha = M[n] == raised ? 1.0f : exp2_fast(M[n] - raised);
                M[n] = raised;
                l[n] *= alpha;
#pragma unroll
                for (int d = 0; d < DT; ++d) acc[n][d] *= alpha;
            }
            const float r = (M[n] == -INFINITY ? 0.0f : M[n]) - fev - kWeightShift;
            float sum = 0.0f;
            f16x8 wh[2], wl[2];
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                float w[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    w[j] = exp2_fast(fmaf(sc[n][2 * u + j / 4][j % 4], c, -r));
                    sum += w[j];
                }
                split_terms<TWO>(wh[u], wl[u], w);
            }
            l[n] = fmaf(sum, inverse, l[n]);
#pragma unroll
            for (int d = 0; d < DT; ++d) {
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    u32x2 bytes{x.v[d][2 * u], x.v[d][2 * u + 1]};
                    if (any_nan) {
                        bytes[0] &= ~nan_bytes(bytes[0]);
                        bytes[1] &= ~nan_bytes(bytes[1]);
                    }
                    const f16x8 v = widen(bytes[0], bytes[1]);
                    acc[n][d] = mfma_16(v, wh[u], acc[n][d]);
                    if constexpr (TWO) acc[n][d] = mfma_16(v, wl[u], acc[n][d]);
                }
            }
            if (any_nan) {
                // NaN in V reaches the rows that see its key and no other: count them with a product of ones.
                f16x8 sees[2];
#pragma unroll
                for (int u = 0; u < 2; ++u) {
#pragma unroll
                    for (int j = 0; j < 8; ++j) sees[u][j] = static_cast<_Float16>((visible[n] >> (8 * u + j)) & 1u ? 1.0f : 0.0f);
                }
#pragma unroll
                for (int d = 0; d < DT; ++d) {
                    f32x4 hits{};
#pragma unroll
                    for (int u = 0; u < 2; ++u) // 0x38 is 1.0 in e4m3
                        hits = mfma_16(widen(nan_bytes(x.v[d][2 * u]) & 0x38383838u, nan_bytes(x.v[d][2 * u + 1]) & 0x38383838u), sees[u], hits);
#pragma unroll
                    for (int j = 0; j < 4; ++j) acc[n][d][j] = hits[j] > 0.0f ? NAN : acc[n][d][j];
                }
            }
        }
    };

    const int steps = step_end - step_begin - wave;
    const int mine = steps > 0 ? (steps + kWaves - 1) / kWaves : 0;
    for (int i = 0; i < mine; ++i) {
        const int step = step_begin + wave + kWaves * i, turn = i % 16;
        if (turn == 0) look_up(step);
        Keys x;
        load_keys(x, turn);
        compute(x, turn, step);
    }

    // Merge: each wave's sums over the lanes of a column, then the four waves.
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
        l[n] += __shfl_xor(l[n], 16);
        l[n] += __shfl_xor(l[n], 32);
        m[n] = fmaxf(m[n], __shfl_xor(m[n], 16));
        m[n] = fmaxf(m[n], __shfl_xor(m[n], 32));
        const int r = 16 * n + col;
        if (g == 0) {
            stats[wave][r][0] = M[n];
            stats[wave][r][1] = l[n];
            stats[wave][r][2] = m[n];
        }
#pragma unroll
        for (int d = 0; d < DT; ++d) *reinterpret_cast<f32x4 *>(&merged[wave][r][16 * d + 4 * g]) = acc[n][d];
    }
    __syncthreads();
    constexpr int SPAN = 8;
    for (int i = threadIdx.x; i < ROWS * (D / SPAN); i += kThreads) {
        const int r = i / (D / SPAN), f = i % (D / SPAN) * SPAN;
        if (r >= t.rows) continue;
        float reference = -INFINITY, most = -INFINITY, sum = 0.0f, o[SPAN] = {};
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            reference = fmaxf(reference, stats[w][r][0]);
            most = fmaxf(most, stats[w][r][2]);
        }
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            const float alpha = stats[w][r][0] == reference ? 1.0f : exp2_fast(stats[w][r][0] - reference);
            sum = fmaf(stats[w][r][1], alpha, sum);
#pragma unroll
            for (int j = 0; j < SPAN; ++j) o[j] = fmaf(merged[w][r][f + j], alpha, o[j]);
        }
        if (t.chunks <= 1) {
            const int flat = t.row0 + r, token = flat / group;
            finish_row<T, VEC>(a, t.s.row0 + token, head * group + flat - token * group, f, o, sum, reference, most, f == 0);
        } else {
            const Partial p = partial_of<D>(a, plan, slot, r);
#pragma unroll
            for (int j = 0; j < SPAN; j += 4) *reinterpret_cast<f32x4 *>(p.acc + f + j) = f32x4{o[j], o[j + 1], o[j + 2], o[j + 3]};
            if (f == 0) *reinterpret_cast<f32x4 *>(p.stats) = f32x4{reference, sum, most, 0.0f};
        }
    }
}

// Joins the chunks of a tile, in their order.
template<int T, int D, bool VEC>
__global__ __launch_bounds__(kThreads) void cache_join_kernel(const CacheForwardArgs a, const ForwardPlan plan) {
    const int heads = a.cache.heads, group = a.query_heads / heads;
    const uint32_t pair = blockIdx.x, unit = pair / heads;
    const int head = static_cast<int>(pair - unit * heads);
    const Tile t = tile_of(a, plan, unit, group);
    if (t.rows <= 0 || t.chunks <= 1) return;
    constexpr int SPAN = 8;
    const int64_t slot = static_cast<int64_t>(pair) * plan.chunks;
    for (int i = threadIdx.x; i < t.rows * (D / SPAN); i += kThreads) {
        const int r = i / (D / SPAN), f = i % (D / SPAN) * SPAN;
        float reference = -INFINITY, most = -INFINITY, sum = 0.0f, o[SPAN] = {};
        for (int c = 0; c < t.chunks; ++c) {
            const f32x4 s = *reinterpret_cast<const f32x4 *>(partial_of<D>(a, plan, slot + c, r).stats);
            reference = fmaxf(reference, s[0]);
            most = fmaxf(most, s[2]);
        }
        for (int c = 0; c < t.chunks; ++c) {
            const Partial p = partial_of<D>(a, plan, slot + c, r);
            const f32x4 s = *reinterpret_cast<const f32x4 *>(p.stats);
            const float alpha = s[0] == reference ? 1.0f : exp2_fast(s[0] - reference);
            sum = fmaf(s[1], alpha, sum);
#pragma unroll
            for (int j = 0; j < SPAN; j += 4) {
                const f32x4 x = *reinterpret_cast<const f32x4 *>(p.acc + f + j);
#pragma unroll
                for (int k = 0; k < 4; ++k) o[j + k] = fmaf(x[k], alpha, o[j + k]);
            }
        }
        const int flat = t.row0 + r, token = flat / group;
        finish_row<T, VEC>(a, t.s.row0 + token, head * group + flat - token * group, f, o, sum, reference, most, f == 0);
    }
}

template<int T, int D, int NQ, bool VEC>
void launch(const CacheForwardArgs &a, const ForwardPlan &plan, hipStream_t stream) {
    const uint32_t pairs = static_cast<uint32_t>(plan.units) * a.cache.heads;
    hipLaunchKernelGGL((cache_attention_kernel<T, D, NQ, VEC>), dim3(pairs * plan.chunks), dim3(kThreads), 0, stream, a, plan);
    if (plan.chunks > 1) hipLaunchKernelGGL((cache_join_kernel<T, D, VEC>), dim3(pairs), dim3(kThreads), 0, stream, a, plan);
}

template<int T, int D>
void dispatch(const CacheForwardArgs &a, const ForwardPlan &plan, const bool vec, hipStream_t stream) {
    if (plan.rows == 16) {
        if (vec) launch<T, D, 1, true>(a, plan, stream);
        else launch<T, D, 1, false>(a, plan, stream);
    } else {
        if (vec) launch<T, D, 2, true>(a, plan, stream);
        else launch<T, D, 2, false>(a, plan, stream);
    }
}

template<int T>
void dispatch(const int width, const CacheForwardArgs &a, const ForwardPlan &plan, const bool vec, hipStream_t stream) {
    if (width == 32) dispatch<T, 32>(a, plan, vec, stream);
    else if (width == 64) dispatch<T, 64>(a, plan, vec, stream);
    else dispatch<T, 128>(a, plan, vec, stream);
}

} // namespace

hipError_t launch_cache_forward(const int width, const CacheForwardArgs &a, const ForwardPlan &plan, hipStream_t stream) {
    if (plan.units == 0) return hipSuccess;
    if (static_cast<long long>(plan.units) * a.cache.heads * plan.chunks >= (1ll << 32) / kThreads) return hipErrorInvalidValue;
    const int unit = a.dtype == kFloat32 ? 4 : 8;
    auto fits = [&](const void *p, const rocmkernels_strides &s) {
        return (reinterpret_cast<uintptr_t>(p) & 15u) == 0 && (s.head % unit) == 0 && (s.token % unit) == 0;
    };
    const bool vec = fits(a.q, a.qs) && fits(a.output, a.os);
    if (a.dtype == kFloat32) dispatch<kFloat32>(width, a, plan, vec, stream);
    else if (a.dtype == kFloat16) dispatch<kFloat16>(width, a, plan, vec, stream);
    else dispatch<kBFloat16>(width, a, plan, vec, stream);
    return hipGetLastError();
}

} // namespace rk
