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
//     l = sum w 2^-ev in the same units, so O = acc / l. Weights are held 2^7 higher (w <= 2^7 at the reference): they keep all
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

#include <algorithm>

namespace rk {

namespace {

constexpr float kWeightShift = 7.0f;   // weights are 2^7 at the reference
constexpr float kLazyRange = 8.0f;     // and reach 2^15 before it moves
// Sums of weights are held 2^12 lower: with a scale of 2^-100 (V all zero) 2^25 weights of 2^15 then add up within FP32's range, and
// with one of 2^120 a weight of 2^7 is still no less than 2^-125.
constexpr float kSumShift = 12.0f;
constexpr float kSumScale = 0x1p-12f;

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

__device__ __forceinline__ Tile tile_of(const CacheForwardArgs &a, const ForwardPart &part, const uint32_t unit, const int group) {
    Tile t;
    uint32_t index;
    if (part.direct) {
        t.s = sequence_at(a.seqs, static_cast<int>(unit / part.direct));
        index = unit % part.direct;
    } else {
        t.s = find_sequence(a.seqs, unit, group, part.rows - 1, part.rows);
        index = unit - t.s.base;
    }
    const uint32_t flat = static_cast<uint32_t>(t.s.count) * group;
    const bool taken = flat >= static_cast<uint32_t>(part.least) && flat <= static_cast<uint32_t>(part.most) &&
            index < (flat + part.rows - 1) / part.rows;
    t.row0 = taken ? static_cast<int>(index * part.rows) : 0;
    t.rows = taken ? min(part.rows, static_cast<int>(flat) - t.row0) : 0;
    t.vis = Visibility{min(t.s.length, a.max_keys), a.radius, a.causal};
    const int low = t.vis.low(t.s.first + t.row0 / group), high = t.vis.high(t.s.first + max(t.row0 + t.rows - 1, 0) / group);
    t.step0 = low / kStep;
    t.steps = t.rows > 0 && high > low ? (high + kStep - 1) / kStep - t.step0 : 0;
    t.chunks = (t.steps + part.chunk_steps - 1) / part.chunk_steps;
    return t;
}

// Writes one row's output from its sums: acc over N features, l, the reference M (s + ev) and the maximum m of s (all base 2).
template<int T, bool VEC, int N>
__device__ __forceinline__ void finish_row(const CacheForwardArgs &a, const int64_t token, const int head, const int feature,
        const float (&acc)[N], const float l, const float reference, const float m, const bool writes_lse) {
    const bool nan_row = isnan(l), has_keys = l > 0.0f;
    const float factor = has_keys ? kSumScale / l : (nan_row ? NAN : 0.0f);
    float o[N];
#pragma unroll
    for (int i = 0; i < N; ++i) o[i] = has_keys ? acc[i] * factor : factor;
    store_row<T, VEC>(a.output, token * a.os.token + static_cast<int64_t>(head) * a.os.head + feature, o);
    if (writes_lse && a.lse) {
        float *const p = a.lse + 2 * (token * a.query_heads + head);
        p[0] = has_keys ? m / kLog2e : (nan_row ? NAN : -INFINITY);
        p[1] = has_keys ? l * exp2_fast(reference - m - kWeightShift + kSumShift) : (nan_row ? NAN : 0.0f);
    }
}

// Workspace: [slot][rows][D] partial sums, then [slot][rows][4] = {M, l, m, unused}; slot = (unit * heads + head) * chunks + chunk.
struct Partial {
    float *acc, *stats;
};
template<int D>
__device__ __forceinline__ Partial partial_of(const CacheForwardArgs &a, const ForwardPart &part, const int64_t slot, const int row) {
    float *const base = reinterpret_cast<float *>(static_cast<char *>(a.workspace) + part.workspace_at);
    const int64_t slots = static_cast<int64_t>(part.units) * a.cache.heads * part.chunks, r = slot * part.rows + row;
    return {base + r * D, base + slots * part.rows * D + r * 4};
}

// The two terms of 8 values that are already scaled into fp16's range: a pair is rounded by one packed conversion, and what is left
// of each value by one mixed-precision FMA that reads the fp16 term and writes fp16 (the empty asm keeps the compiler from
// taking the pair apart again).
template<bool TWO>
__device__ __forceinline__ void split_terms(f16x8 &hi, f16x8 &lo, const float (&x)[8]) {
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
        f16x2 pair{static_cast<_Float16>(x[i]), static_cast<_Float16>(x[i + 1])};
        if constexpr (TWO) {
            uint32_t bits = __builtin_bit_cast(uint32_t, pair);
            __asm__("" : "+v"(bits));
            pair = __builtin_bit_cast(f16x2, bits);
            lo[i] = static_cast<_Float16>(fmaf(x[i], 1.0f, -static_cast<float>(pair[0])));
            lo[i + 1] = static_cast<_Float16>(fmaf(x[i + 1], 1.0f, -static_cast<float>(pair[1])));
        }
        hi[i] = pair[0];
        hi[i + 1] = pair[1];
    }
}

// A tile of 16 rows: each of the WAVES waves of the workgroup streams keys of its own, and they are merged through LDS.
template<int D, int WAVES>
constexpr int kSmallShared = WAVES * 16 * (D + 4) * 4 + WAVES * 16 * 4 * 4; // bytes

template<int T, int D, bool VEC, int WAVES>
__device__ __forceinline__ void small_tile(const CacheForwardArgs &a, const ForwardPart &part, const uint32_t number, uint8_t *shared) {
    constexpr bool TWO = T == kFloat32;
    constexpr int KC = D / 32;                   // MFMAs of a score tile
    constexpr int KL = D >= 64 ? D / 64 : 1;     // loads of a K row tile
    constexpr int DT = D / 16;                   // output tiles
    constexpr int ROWS = 16;
    auto merged = reinterpret_cast<float(*)[ROWS][D + 4]>(shared);
    auto stats = reinterpret_cast<float(*)[ROWS][4]>(shared + WAVES * ROWS * (D + 4) * 4);

    const int lane = threadIdx.x & (kWave - 1), col = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int heads = a.cache.heads, group = a.query_heads / heads;
    // First chunks first: every sequence has one, and the short ends of sequences come last, when the chip runs empty.
    const uint32_t pairs = static_cast<uint32_t>(part.units) * heads, pair = number % pairs, unit = pair / heads;
    const int chunk = static_cast<int>(number / pairs), head = static_cast<int>(pair - unit * heads);
    const int64_t slot = static_cast<int64_t>(pair) * part.chunks + chunk;

    const Tile t = tile_of(a, part, unit, group);
    if (t.rows <= 0 || chunk >= max(t.chunks, 1)) return;
    const int step_begin = t.step0 + chunk * part.chunk_steps;
    const int step_end = t.step0 + min(t.steps, (chunk + 1) * part.chunk_steps);

    // This lane's row: q in operand order, the factor of its scores, and the keys it sees. Lanes past the last row repeat the first.
    f16x8 qh[KC], ql[TWO ? KC : 1];
    float c2;
    int low, high;
    {
        const int flat = t.row0 + (col < t.rows ? col : 0), i = flat / group, query_head = head * group + (flat - i * group);
        const int64_t row = static_cast<int64_t>(t.s.row0 + i) * a.qs.token + static_cast<int64_t>(query_head) * a.qs.head;
        const int position = t.s.first + i;
        low = t.vis.low(position);
        high = t.vis.high(position);
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
        c2 = back * (kLog2e / sqrtf(static_cast<float>(D)));
#pragma unroll
        for (int k = 0; k < KC; ++k) {
#pragma unroll
            for (int j = 0; j < 8; ++j) x[k][j] *= scale;
            split_terms<TWO>(qh[k], ql[TWO ? k : 0], x[k]);
        }
    }
    // Keys that every row sees: between the last row's first key and the first row's end.
    const int all_low = t.vis.low(t.s.first + (t.row0 + t.rows - 1) / group), all_high = t.vis.high(t.s.first + t.row0 / group);

    float M = -INFINITY, l = 0.0f, m = -INFINITY;
    f32x4 acc[DT];
#pragma unroll
    for (int d = 0; d < DT; ++d) acc[d] = f32x4{};

    // The 64 blocks of this wave's next 16 steps, one a lane: the block's place in the cache (-1: none) and its exponents.
    const int blocks = a.cache.page_size / kBlockTokens;
    int place = -1, exponents = 0;
    uint64_t absent = 0;
    auto look_up = [&](const int step) __attribute__((always_inline)) {
        const int s = step + WAVES * (lane / 4), position = kStep * s + kBlockTokens * (lane % 4);
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
        f32x4 sc[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            sc[i] = f32x4{};
#pragma unroll
            for (int k = 0; k < KC; ++k) {
                const f16x8 w = widen(x.k[i][k / 2][2 * (k % 2)], x.k[i][k / 2][2 * (k % 2) + 1]);
                sc[i] = mfma_16(w, qh[k], sc[i]);
                if constexpr (TWO) sc[i] = mfma_16(w, ql[k], sc[i]);
            }
        }
        const int key0 = kStep * step, base = key0 + 16 * g;
        const bool full = key0 >= all_low && key0 + kStep <= all_high && ((absent >> (4 * turn)) & 15u) == 0;
        uint32_t visible = 0, held = 0;
        bool any_nan = false;
        if (!full) {
            const bool here = !((absent >> (4 * turn + g)) & 1u);
            visible = here ? bit_range(low - base, high - base - 1) & 0xffffu : 0u;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
#pragma unroll
                for (int j = 0; j < 4; ++j) sc[i][j] = (visible >> (4 * i + j)) & 1u ? sc[i][j] : -INFINITY;
            }
            // Bytes behind the sequence's end may hold anything, and 0 times NaN is no 0: NaN counts for the rows that see its key.
            held = here ? bit_range(0, t.vis.length - base - 1) & 0xffffu : 0u;
            uint32_t nans = 0;
#pragma unroll
            for (int d = 0; d < DT; ++d) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const uint32_t w = x.v[d][i] & byte_mask(held >> (4 * i)), bad = nan_bytes(w);
                    x.v[d][i] = w & ~bad;
                    nans |= bad;
                }
            }
            any_nan = __ballot(nans != 0) != 0;
        }
        const float c = fmaxf(c2 * kscale, 1.17549435e-38f); // > 0, so that hidden scores stay -inf
        float most = sc[0][0];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
#pragma unroll
            for (int j = 0; j < 4; ++j) most = fmaxf(most, sc[i][j]);
        }
        most *= c;
        m = fmaxf(m, most);
        const float candidate = most + fev;
        if (__ballot(candidate > M + kLazyRange)) {
            float raised = fmaxf(M, candidate);
            raised = fmaxf(raised, __shfl_xor(raised, 16));
            raised = fmaxf(raised, __shfl_xor(raised, 32));
            const float alpha = M == raised ? 1.0f : exp2_fast(M - raised);
            M = raised;
            l *= alpha;
#pragma unroll
            for (int d = 0; d < DT; ++d) acc[d] *= alpha;
        }
        const float r = (M == -INFINITY ? 0.0f : M) - fev - kWeightShift;
        float sum = 0.0f;
        f16x8 wh[2], wl[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            float w[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) w[j] = exp2_fast(fmaf(sc[2 * u + j / 4][j % 4], c, -r));
#pragma unroll
            for (int j = 0; j < 8; ++j) sum += w[j];
            split_terms<TWO>(wh[u], wl[u], w);
        }
        l = fmaf(sum * kSumScale, inverse, l);
#pragma unroll
        for (int d = 0; d < DT; ++d) {
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const f16x8 v = widen(x.v[d][2 * u], x.v[d][2 * u + 1]);
                acc[d] = mfma_16(v, wh[u], acc[d]);
                if constexpr (TWO) acc[d] = mfma_16(v, wl[u], acc[d]);
            }
        }
        if (__builtin_expect(any_nan, 0)) {
            // Count the NaN values that each row sees with a product of ones (0x38 is 1.0 in e4m3); V's bytes are read again.
            const int64_t vb = max(__shfl(place, 4 * turn + g), 0);
            const uint8_t *const v = a.cache.values + vb * (kBlockTokens * D) + col * 16;
            f16x8 sees[2];
#pragma unroll
            for (int u = 0; u < 2; ++u) {
#pragma unroll
                for (int j = 0; j < 8; ++j) sees[u][j] = static_cast<_Float16>((visible >> (8 * u + j)) & 1u ? 1.0f : 0.0f);
            }
#pragma unroll
            for (int d = 0; d < DT; ++d) {
                const u32x4 y = *reinterpret_cast<const u32x4 *>(v + d * 256);
                f32x4 hits{};
#pragma unroll
                for (int u = 0; u < 2; ++u)
                    hits = mfma_16(widen(nan_bytes(y[2 * u] & byte_mask(held >> (8 * u))) & 0x38383838u,
                                           nan_bytes(y[2 * u + 1] & byte_mask(held >> (8 * u + 4))) & 0x38383838u),
                            sees[u], hits);
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[d][j] = hits[j] > 0.0f ? NAN : acc[d][j];
            }
        }
    };

    const int steps = step_end - step_begin - wave;
    const int mine = steps > 0 ? (steps + WAVES - 1) / WAVES : 0;
    for (int i = 0; i < mine; ++i) {
        const int step = step_begin + wave + WAVES * i, turn = i % 16;
        if (turn == 0) look_up(step);
        Keys x;
        load_keys(x, turn);
        compute(x, turn, step);
    }

    // Merge: each wave's sums over the lanes of a column, then the waves.
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
    m = fmaxf(m, __shfl_xor(m, 16));
    m = fmaxf(m, __shfl_xor(m, 32));
    if (g == 0) {
        stats[wave][col][0] = M;
        stats[wave][col][1] = l;
        stats[wave][col][2] = m;
    }
#pragma unroll
    for (int d = 0; d < DT; ++d) *reinterpret_cast<f32x4 *>(&merged[wave][col][16 * d + 4 * g]) = acc[d];
    __syncthreads();
    constexpr int SPAN = 8;
    for (int i = threadIdx.x; i < ROWS * (D / SPAN); i += WAVES * kWave) {
        const int r = i / (D / SPAN), f = i % (D / SPAN) * SPAN;
        if (r >= t.rows) continue;
        float reference = -INFINITY, most = -INFINITY, sum = 0.0f, o[SPAN] = {};
#pragma unroll
        for (int w = 0; w < WAVES; ++w) {
            reference = fmaxf(reference, stats[w][r][0]);
            most = fmaxf(most, stats[w][r][2]);
        }
#pragma unroll
        for (int w = 0; w < WAVES; ++w) {
            const float alpha = stats[w][r][0] == reference ? 1.0f : exp2_fast(stats[w][r][0] - reference);
            sum = fmaf(stats[w][r][1], alpha, sum);
#pragma unroll
            for (int j = 0; j < SPAN; ++j) o[j] = fmaf(merged[w][r][f + j], alpha, o[j]);
        }
        if (t.chunks <= 1) {
            const int flat = t.row0 + r, token = flat / group;
            finish_row<T, VEC>(a, t.s.row0 + token, head * group + flat - token * group, f, o, sum, reference, most, f == 0);
        } else {
            const Partial p = partial_of<D>(a, part, slot, r);
#pragma unroll
            for (int j = 0; j < SPAN; j += 4) *reinterpret_cast<f32x4 *>(p.acc + f + j) = f32x4{o[j], o[j + 1], o[j + 2], o[j + 3]};
            if (f == 0) *reinterpret_cast<f32x4 *>(p.stats) = f32x4{reference, sum, most, 0.0f};
        }
    }
}

// Tiles of 128 rows, 32 a wave, that share the keys: each step's 64 keys are read once, widened to fp16 and staged in LDS for the
// four waves (double-buffered, one barrier a step), so a byte of the cache is converted once for 128 rows. Products are on
// v_mfma_f32_32x32x16_f16, S^T = K Q^T and O^T = V^T P^T as above: accumulator register v of a lane in half h holds token 8 (v / 4)
// + 4 h + v % 4 of a 32-key tile. Registers 8 u .. 8 u + 7 then hold eight tokens of the 16-token block u: one page's scales, and,
// with V's tokens staged in the order 0-3, 8-11 and 4-7, 12-15 for the two halves, one operand of V.
// Staged layouts: K [8-feature chunk][token] and V [block][half][feature] of 16 bytes, so operand reads cover 512 contiguous bytes a
// half-wave; a K chunk is padded by 16 * 128 / D bytes, which puts the writes of 16 neighbouring lanes on distinct banks.
// While a wave weighs scores it has the priority over the one that only issues products: 323 against 335 us for a prompt of 2048 rows
// (32 heads on 8, 128-wide fp16) behind 8192 keys.
//
// GROUPS: groups of a step's keys that share their scales, one where pages are multiples of 64 tokens, else a group for each block.
// TEAMS: of four waves. A step takes a wave about 2 us whether it has its SIMD for itself or not (products, softmax and staging wait
// for one another), so where there are fewer tiles than would fill the chip two teams share one, each with stages of its own, and
// take turns with its steps; that halves the steps in a row and needs no partial results in memory. 768 rows behind 3328 keys: 91 ->
// 73 us, against 89 with twice the chunks.
template<int D>
constexpr int kChunkBytes = kStep * 16 + 16 * 128 / D; // a staged 8-feature chunk of K
template<int D>
constexpr int kLargeShared = 2 * (D / 8 * kChunkBytes<D> + kStep * D * 2) + 2 * kWaves * 4; // bytes

template<int T, int D, bool VEC, int GROUPS, int TEAMS>
__device__ __forceinline__ void large_tile(const CacheForwardArgs &a, const ForwardPart &part, const uint32_t number, uint8_t *shared) {
    constexpr bool TWO = T == kFloat32;
    constexpr int KC = D / 16;                       // MFMAs of a 32-key score tile
    constexpr int DT = D / 32;                       // output tiles
    constexpr int K_CHUNK = kChunkBytes<D>;
    constexpr int K_BYTES = D / 8 * K_CHUNK, V_BYTES = kStep * D * 2;
    constexpr int LOADS = (kStep * D / 16 + kThreads - 1) / kThreads; // 16-byte loads of K, and of V, of a thread
    constexpr bool ALL = kStep * D / 16 >= kThreads; // D = 32: half the threads load
    const int lane = threadIdx.x & (kWave - 1), col = lane & 31, h = lane >> 5, thread = threadIdx.x % kThreads; // of the team
    const int team = TEAMS > 1 ? __builtin_amdgcn_readfirstlane(threadIdx.x / kThreads) : 0;
    const int wave = __builtin_amdgcn_readfirstlane(thread / kWave);
    auto staged = reinterpret_cast<uint8_t(*)[K_BYTES + V_BYTES]>(shared + team * kLargeShared<D>);
    auto nan_flags = reinterpret_cast<int(*)[kWaves]>(shared + team * kLargeShared<D> + 2 * (K_BYTES + V_BYTES));
    const int heads = a.cache.heads, group = a.query_heads / heads;
    // Workgroups go round the 8 XCDs: give each XCD whole heads, whose keys then stay in its L2, and of a head the last tiles
    // (under a causal mask the longest) first.
    const uint32_t pairs = static_cast<uint32_t>(part.units) * heads, total = pairs * part.chunks;
    const uint32_t xcd = number % 8, place_in_order = xcd * (total / 8) + min(xcd, total % 8) + number / 8;
    const int head = static_cast<int>(place_in_order / (part.units * part.chunks));
    const uint32_t rest = place_in_order - static_cast<uint32_t>(head) * part.units * part.chunks;
    const uint32_t unit = part.units - 1 - rest / part.chunks;
    const int chunk = static_cast<int>(rest % part.chunks);
    const int64_t slot = (static_cast<int64_t>(unit) * heads + head) * part.chunks + chunk;

    const Tile t = tile_of(a, part, unit, group);
    if (t.rows <= 0 || chunk >= max(t.chunks, 1)) return;
    // The teams take the chunk's steps in turns: `rounds` of them, of which this one has `steps`.
    const int first_step = t.step0 + chunk * part.chunk_steps + team;
    const int chunk_steps = max(min(t.steps, (chunk + 1) * part.chunk_steps) - chunk * part.chunk_steps, 0);
    const int rounds = (chunk_steps + TEAMS - 1) / TEAMS, steps = (chunk_steps - team + TEAMS - 1) / TEAMS;
    auto first_key = [&](const int index) __attribute__((always_inline)) { return kStep * (first_step + TEAMS * index); };

    // This wave's rows; a wave past the tile's last row only loads.
    const int wave_row0 = 32 * wave, wave_rows = min(32, t.rows - wave_row0);
    const int r = wave_row0 + col;
    const bool used = r < t.rows;
    const int flat = t.row0 + (used ? r : 0), i = flat / group, query_head = head * group + (flat - i * group);
    const int low = t.vis.low(t.s.first + i), high = t.vis.high(t.s.first + i);
    const int wave_first = t.s.first + (t.row0 + min(wave_row0, t.rows - 1)) / group;
    const int wave_last = t.s.first + (t.row0 + min(wave_row0 + 31, t.rows - 1)) / group;
    const int any_low = t.vis.low(wave_first), any_high = t.vis.high(wave_last);  // keys that some row of the wave sees
    const int all_low = t.vis.low(wave_last), all_high = t.vis.high(wave_first);  // and keys that every one sees
    const int tile_low = t.vis.low(t.s.first + (t.row0 + t.rows - 1) / group), tile_high = t.vis.high(t.s.first + t.row0 / group);

    f16x8 qh[KC], ql[TWO ? KC : 1];
    float c2;
    {
        const int64_t row = static_cast<int64_t>(t.s.row0 + i) * a.qs.token + static_cast<int64_t>(query_head) * a.qs.head;
        float x[KC][8];
#pragma unroll
        for (int k = 0; k < KC; ++k) load8<T, VEC>(x[k], a.q, row + 16 * k + 8 * h);
        float scale = 1.0f, back = 1.0f;
        if constexpr (T != kFloat16) {
            float most = 0.0f;
#pragma unroll
            for (int k = 0; k < KC; ++k) {
#pragma unroll
                for (int j = 0; j < 8; ++j) most = fmaxf(most, fabsf(x[k][j]));
            }
            const int e = clamped(static_cast<int>(__float_as_uint(halves_max(most)) >> 23) - 127, -100, 127);
            scale = power(14 - e);
            back = power(e - 14);
        }
        c2 = back * (kLog2e / sqrtf(static_cast<float>(D)));
#pragma unroll
        for (int k = 0; k < KC; ++k) {
#pragma unroll
            for (int j = 0; j < 8; ++j) x[k][j] *= scale;
            split_terms<TWO>(qh[k], ql[TWO ? k : 0], x[k]);
        }
    }

    float M = -INFINITY, l = 0.0f, m = -INFINITY;
    f32x16 acc[DT];
#pragma unroll
    for (int d = 0; d < DT; ++d) acc[d] = f32x16{};

    // The 64 blocks of the next 16 steps, one a lane: the block's place in the cache (-1: none) and its exponents, as bytes.
    const int blocks = a.cache.page_size / kBlockTokens;
    int place = -1, exponents = 0;
    auto look_up = [&](const int index) __attribute__((always_inline)) {
        const int s = index + lane / 4, position = first_key(s) + kBlockTokens * (lane % 4);
        place = -1;
        exponents = 0;
        if (s < steps && position < t.vis.length) {
            const int column = position / a.cache.page_size;
            const int page = a.seqs.table[static_cast<int64_t>(t.s.b) * a.seqs.table_stride + column];
            if (page >= 0 && page < a.cache.pages) {
                const int cell = page * heads + head;
                place = cell * blocks + (position - column * a.cache.page_size) / kBlockTokens;
                exponents = (scale_exponent(a.cache.scales[2 * static_cast<int64_t>(cell)]) & 255) |
                        ((scale_exponent(a.cache.scales[2 * static_cast<int64_t>(cell) + 1]) & 255) << 8);
            }
        }
    };
    // A step's bytes on their way to LDS, and the exponents of its four blocks (as bytes, in scalar registers).
    u32x4 raw_k[LOADS], raw_v[LOADS];
    struct Scales {
        int exps[4], places[4];
        uint32_t absent;
    };
    auto load = [&](Scales &e, const int index) __attribute__((always_inline)) {
        const int turn = index % 16;
        if (turn == 0) look_up(index);
#pragma unroll
        for (int b = 0; b < 4; ++b) {
            e.exps[b] = __builtin_amdgcn_readlane(exponents, 4 * turn + b);
            e.places[b] = __builtin_amdgcn_readlane(place, 4 * turn + b);
        }
        e.absent = static_cast<uint32_t>(__ballot(place < 0) >> (4 * turn)) & 15u;
#pragma unroll
        for (int n = 0; n < LOADS; ++n) {
            // K: token x / (D / 16), 16 of its features; V: block x / D, feature x % D, with x = thread + n * kThreads. From D = 64 on a
            // wave's 64 chunks of either lie in one block, at D = 32 in two. Blocks that are not there read the cache's first.
            constexpr int SHARE = D / 64; // waves that share a block
            int64_t at;
            if constexpr (D >= 64) at = max(__builtin_amdgcn_readlane(place, 4 * turn + wave / SHARE + n * (kWaves / SHARE)), 0);
            else at = max(__shfl(place, 4 * turn + (2 * wave + h) % 4), 0);
            if (ALL || wave < 2) {
                const uint32_t token = (static_cast<uint32_t>(thread) / (D / 16)) % 16;
                raw_k[n] = *reinterpret_cast<const u32x4 *>(a.cache.keys + at * (kBlockTokens * D) + (token * D + thread % (D / 16) * 16));
                raw_v[n] = *reinterpret_cast<const u32x4 *>(a.cache.values + at * (kBlockTokens * D) + thread % D * 16);
            }
        }
    };
    // Whether every row of the tile sees every key of a step.
    auto no_key_hidden = [&](const int key0, const uint32_t absent) __attribute__((always_inline)) {
        return key0 >= tile_low && key0 + kStep <= tile_high && absent == 0;
    };
    auto stage = [&](const int index, const uint32_t absent) __attribute__((always_inline)) {
        uint8_t *const k = staged[index & 1], *const v = k + K_BYTES;
        const int key0 = first_key(index);
        const bool full = no_key_hidden(key0, absent);
        uint32_t nans = 0;
#pragma unroll
        for (int n = 0; n < LOADS; ++n) {
            const int x = thread + n * kThreads, token = x / (D / 16), block = x / D;
            if (!ALL && x >= kStep * D / 16) continue;
            if (!full) {
                // Bytes behind the sequence's end may hold anything, and 0 times NaN is no 0: NaN counts for the rows that see its key.
                const uint32_t held = (absent >> block) & 1u ? 0u : bit_range(0, t.vis.length - key0 - 16 * block - 1) & 0xffffu;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const uint32_t w = raw_v[n][j] & byte_mask(held >> (4 * j)), bad = nan_bytes(w);
                    raw_v[n][j] = w & ~bad;
                    nans |= bad;
                }
            }
            uint8_t *const to = k + (x % (D / 16)) * (2 * K_CHUNK) + token * 16;
            *reinterpret_cast<f16x8 *>(to) = widen(raw_k[n][0], raw_k[n][1]);
            *reinterpret_cast<f16x8 *>(to + K_CHUNK) = widen(raw_k[n][2], raw_k[n][3]);
            uint8_t *const tv = v + (2 * block * D + x % D) * 16;
            *reinterpret_cast<f16x8 *>(tv) = widen(raw_v[n][0], raw_v[n][2]);
            *reinterpret_cast<f16x8 *>(tv + D * 16) = widen(raw_v[n][1], raw_v[n][3]);
        }
        const bool any = __ballot(nans != 0) != 0;
        if (lane == 0) nan_flags[index & 1][wave] = any;
    };
    auto compute = [&](const int index, const Scales &e) __attribute__((always_inline)) {
        const int key0 = first_key(index);
        if (wave_rows <= 0 || key0 >= any_high || key0 + kStep <= any_low) return;
        const uint8_t *const k = staged[index & 1] + col * 16 + h * K_CHUNK;
        const uint8_t *const v = staged[index & 1] + K_BYTES + (h * D + col) * 16;
        // LDS answers after several products' time, so operands are asked for well ahead: all of the first tile's K, then the second
        // tile's as the first's are used, V's first block before the softmax, and each next block before the one at hand is weighed.
        f32x16 sc[2] = {f32x16{}, f32x16{}};
        constexpr bool AHEAD = !(TWO && D == 128); // V's operands, where registers allow
        f16x8 kx[KC], vx[AHEAD ? 2 : 1][DT];
#pragma unroll
        for (int c = 0; c < KC; ++c) kx[c] = *reinterpret_cast<const f16x8 *>(k + c * (2 * K_CHUNK));
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int n = 0; n < 2; ++n) {
#pragma unroll
            for (int c = 0; c < KC; ++c) {
                sc[n] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kx[c], qh[c], sc[n], 0, 0, 0);
                if constexpr (TWO) sc[n] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kx[c], ql[c], sc[n], 0, 0, 0);
                if (n == 0) kx[c] = *reinterpret_cast<const f16x8 *>(k + c * (2 * K_CHUNK) + 512);
                else if (AHEAD && c < DT) vx[0][c] = *reinterpret_cast<const f16x8 *>(v + 32 * c * 16);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        const bool full = key0 >= all_low && key0 + kStep <= all_high && e.absent == 0;
        bool any_nan = false;
        if (!full) {
#pragma unroll
            for (int b = 0; b < 4; ++b) {
                const int base = key0 + 16 * b + 4 * h;
                const uint32_t visible = (e.absent >> b) & 1u ? 0u : bit_range(low - base, high - base - 1);
#pragma unroll
                for (int j = 0; j < 8; ++j) sc[b / 2][8 * (b % 2) + j] = (visible >> (8 * (j >> 2) + (j & 3))) & 1u ? sc[b / 2][8 * (b % 2) + j] : -INFINITY;
            }
        }
        if (!no_key_hidden(key0, e.absent)) { // staged without its NaN, also for the waves that see every key
#pragma unroll
            for (int w = 0; w < kWaves; ++w) any_nan |= nan_flags[index & 1][w] != 0;
        }
        constexpr int BLOCKS = 4 / GROUPS;
        __builtin_amdgcn_s_setprio(1);
        float c[GROUPS], ev[GROUPS], candidate = -INFINITY;
#pragma unroll
        for (int b = 0; b < GROUPS; ++b) {
            c[b] = fmaxf(c2 * power(static_cast<int8_t>(e.exps[b])), 1.17549435e-38f); // > 0, so that hidden scores stay -inf
            ev[b] = static_cast<float>(static_cast<int8_t>(e.exps[b] >> 8));
            float most = sc[b / 2][8 * (b % 2)];
#pragma unroll
            for (int j = 1; j < 8 * BLOCKS; ++j) most = fmaxf(most, sc[(b * BLOCKS + j / 8) / 2][8 * ((b * BLOCKS + j / 8) % 2) + j % 8]);
            most *= c[b];
            m = fmaxf(m, most);
            candidate = fmaxf(candidate, most + ev[b]);
        }
        if (__ballot(candidate > M + kLazyRange)) {
            const float raised = halves_max(fmaxf(M, candidate));
            const float alpha = M == raised ? 1.0f : exp2_fast(M - raised);
            M = raised;
            l *= alpha;
#pragma unroll
            for (int d = 0; d < DT; ++d) acc[d] *= alpha;
        }
        const float reference = (M == -INFINITY ? 0.0f : M) - kWeightShift;
        float sum = 0.0f;
#pragma unroll
        for (int b = 0; b < 4; ++b) {
            const int of = b / BLOCKS;
            const float r = reference - ev[of];
            if (AHEAD && b < 3) {
#pragma unroll
                for (int d = 0; d < DT; ++d) vx[AHEAD ? (b + 1) % 2 : 0][d] = *reinterpret_cast<const f16x8 *>(v + (2 * (b + 1) * D + 32 * d) * 16);
                __builtin_amdgcn_sched_barrier(0);
            }
            float w[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) w[j] = exp2_fast(fmaf(sc[b / 2][8 * (b % 2) + j], c[of], -r));
            f16x8 wh, wl;
#pragma unroll
            for (int j = 0; j < 8; ++j) sum += w[j];
            split_terms<TWO>(wh, wl, w);
            if (b % BLOCKS == BLOCKS - 1) {
                l = fmaf(sum * kSumScale, power(-static_cast<int8_t>(e.exps[of] >> 8)), l);
                sum = 0.0f;
            }
#pragma unroll
            for (int d = 0; d < DT; ++d) {
                const f16x8 x = AHEAD ? vx[AHEAD ? b % 2 : 0][d] : *reinterpret_cast<const f16x8 *>(v + (2 * b * D + 32 * d) * 16);
                acc[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(x, wh, acc[d], 0, 0, 0);
                if constexpr (TWO) acc[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(x, wl, acc[d], 0, 0, 0);
            }
            __asm__ volatile("" : "+v"(l), "+v"(sum)); // the sums are formed here, not sunk behind the step: that kept all weights alive
        }
        __builtin_amdgcn_s_setprio(0);
        if (__builtin_expect(any_nan, 0)) {
            // Count the NaN values that each row sees with a product of ones (0x38 is 1.0 in e4m3); V's bytes are read again.
#pragma unroll 1
            for (int b = 0; b < 4; ++b) {
                const int base = key0 + 16 * b + 4 * h;
                const bool here = !((e.absent >> b) & 1u);
                const uint32_t seen = here ? bit_range(low - base, high - base - 1) : 0u, held = here ? bit_range(0, t.vis.length - base - 1) : 0u;
                f16x8 sees;
#pragma unroll
                for (int j = 0; j < 8; ++j) sees[j] = static_cast<_Float16>((seen >> (8 * (j >> 2) + (j & 3))) & 1u ? 1.0f : 0.0f);
                const int64_t vb = max(b == 0 ? e.places[0] : b == 1 ? e.places[1] : b == 2 ? e.places[2] : e.places[3], 0);
                const uint32_t *const words = reinterpret_cast<const uint32_t *>(a.cache.values + vb * (kBlockTokens * D) + col * 16);
#pragma unroll
                for (int d = 0; d < DT; ++d) {
                    const uint32_t lo = words[32 * d * 4 + h], hi = words[32 * d * 4 + 2 + h];
                    const f32x16 hits = __builtin_amdgcn_mfma_f32_32x32x16_f16(widen(nan_bytes(lo & byte_mask(held)) & 0x38383838u,
                            nan_bytes(hi & byte_mask(held >> 8)) & 0x38383838u), sees, f32x16{}, 0, 0, 0);
#pragma unroll
                    for (int j = 0; j < 16; ++j) acc[d][j] = hits[j] > 0.0f ? NAN : acc[d][j];
                    __builtin_amdgcn_sched_barrier(0); // one tile of counts at a time
                }
            }
        }
    };

    // The rows of q are here before the first step is asked for: a wait for them inside the loop would be one for the newest loads.
    __builtin_amdgcn_s_waitcnt(0x0f70); // vmcnt 0
    Scales now{}, next{}, after{};
    if (steps > 0) {
        load(now, 0);
        stage(0, now.absent);
        if (steps > 1) load(next, 1);
    }
    __syncthreads();
    for (int index = 0; index < rounds; ++index) {
        if (index + 1 < steps) stage(index + 1, next.absent);
        if (index + 2 < steps) load(after, index + 2);
        if (TEAMS == 1 || index < steps) compute(index, now);
        __syncthreads();
        now = next;
        next = after;
    }

    l = halves_sum(l);
    m = halves_max(m);
    if constexpr (TEAMS == 2) {
        // The second team hands over its state, register by register, through the stages, which nobody reads any more.
        static_assert((4 * DT + 1) * kThreads * 16 <= TEAMS * kLargeShared<D>, "the state fits the stages");
        auto state = reinterpret_cast<f32x4(*)[kThreads]>(shared);
        if (team == 1) {
#pragma unroll
            for (int q = 0; q < 4 * DT; ++q)
                state[q][thread] = f32x4{acc[q / 4][4 * (q % 4)], acc[q / 4][4 * (q % 4) + 1], acc[q / 4][4 * (q % 4) + 2], acc[q / 4][4 * (q % 4) + 3]};
            state[4 * DT][thread] = f32x4{M, l, m, 0.0f};
        }
        __syncthreads();
        if (team == 1) return;
        const f32x4 other = state[4 * DT][thread];
        const float raised = fmaxf(M, other[0]);
        const float mine = M == raised ? 1.0f : exp2_fast(M - raised), theirs = other[0] == raised ? 1.0f : exp2_fast(other[0] - raised);
        M = raised;
        l = l * mine + other[1] * theirs;
        m = fmaxf(m, other[2]);
#pragma unroll
        for (int q = 0; q < 4 * DT; ++q) {
            const f32x4 x = state[q][thread];
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[q / 4][4 * (q % 4) + j] = acc[q / 4][4 * (q % 4) + j] * mine + x[j] * theirs;
        }
    }
    if (!used) return;
#pragma unroll
    for (int d = 0; d < DT; ++d) {
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int f = 32 * d + 8 * u + 4 * h;
            const float o[4] = {acc[d][4 * u], acc[d][4 * u + 1], acc[d][4 * u + 2], acc[d][4 * u + 3]};
            if (t.chunks <= 1) {
                finish_row<T, VEC>(a, t.s.row0 + i, query_head, f, o, l, M, m, f == 0);
            } else {
                const Partial p = partial_of<D>(a, part, slot, r);
                *reinterpret_cast<f32x4 *>(p.acc + f) = f32x4{o[0], o[1], o[2], o[3]};
                if (f == 0) *reinterpret_cast<f32x4 *>(p.stats) = f32x4{M, l, m, 0.0f};
            }
        }
    }
}

template<int T, int D, bool VEC, int WAVES>
__global__ __launch_bounds__(WAVES * kWave) __attribute__((amdgpu_waves_per_eu(WAVES > 8 ? 4 : 2))) void cache_attention_small_kernel(
        const CacheForwardArgs a, const ForwardPart part) {
    __shared__ __align__(16) uint8_t shared[kSmallShared<D, WAVES>];
    small_tile<T, D, VEC, WAVES>(a, part, blockIdx.x, shared);
}

// Large tiles and, in the workgroups behind theirs, small ones: in a batch that mixes prompts with single tokens the matrix
// work of the first and the memory traffic of the second run side by side.
template<int T, int D, bool VEC, int GROUPS, int TEAMS>
__global__ __launch_bounds__(TEAMS * kThreads) __attribute__((amdgpu_waves_per_eu(2))) void cache_attention_kernel(const CacheForwardArgs a,
        const ForwardPart large, const ForwardPart small, const uint32_t large_groups) {
    __shared__ __align__(16) uint8_t shared[std::max(kSmallShared<D, TEAMS * kWaves>, TEAMS * kLargeShared<D>)];
    if (blockIdx.x < large_groups) large_tile<T, D, VEC, GROUPS, TEAMS>(a, large, blockIdx.x, shared);
    else small_tile<T, D, VEC, TEAMS * kWaves>(a, small, blockIdx.x - large_groups, shared);
}

// Joins the chunks of a tile, in an order that their number fixes. D / 4 lanes hold a row's features; the other lanes of a wave,
// and for many chunks the other waves of the workgroup, take chunks of their own with a running reference and are merged at the end.
constexpr int kJoinTogether = 8; // up to this many chunks a wave joins rows by itself; with more the four waves share one
constexpr int kJoinRows = 16;    // rows that a workgroup then has under way, four a wave

struct Joined {
    float reference = -INFINITY, most = -INFINITY, sum = 0.0f, o[4] = {};
    __device__ __forceinline__ void add(const float other_reference, const float other_most, const float other_sum, const float (&x)[4]) {
        const float raised = fmaxf(reference, other_reference);
        const float mine = reference == raised ? 1.0f : exp2_fast(reference - raised),
                    theirs = other_reference == raised ? 1.0f : exp2_fast(other_reference - raised);
        reference = raised;
        most = fmaxf(most, other_most);
        sum = sum * mine + other_sum * theirs; // a sum of two products: the same for both lanes of an exchange
#pragma unroll
        for (int j = 0; j < 4; ++j) o[j] = o[j] * mine + x[j] * theirs;
    }
};

// Rows of a workgroup: two rounds for the large tiles (3584 workgroups of one round took 15.6 us where 2048 took 12.0).
__host__ __device__ inline int join_rows(const ForwardPart &part) { return part.chunks > kJoinTogether ? 1 : std::min(part.rows, 2 * kJoinRows); }
inline uint32_t join_groups(const ForwardPart &part, const int heads) {
    return part.chunks > 1 ? static_cast<uint32_t>(part.units) * heads * (part.rows / join_rows(part)) : 0;
}

template<int T, int D, bool VEC>
__global__ __launch_bounds__(kThreads) void cache_join_kernel(const CacheForwardArgs a, const ForwardPart large, const ForwardPart small,
        const uint32_t large_groups) {
    constexpr int LANES = D / 4, SIDE = kWave / LANES; // chunks side by side in a wave
    __shared__ float merged[kWaves][4 * LANES + 4];
    const bool of_large = blockIdx.x < large_groups;
    const ForwardPart part = of_large ? large : small;
    const uint32_t number = of_large ? blockIdx.x : blockIdx.x - large_groups;
    const int rows = join_rows(part);
    const int heads = a.cache.heads, group = a.query_heads / heads;
    const uint32_t row_groups = part.rows / rows, pair = number / row_groups, unit = pair / heads;
    const int head = static_cast<int>(pair - unit * heads);
    const Tile t = tile_of(a, part, unit, group);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), lane = threadIdx.x & (kWave - 1);
    const int first_row = static_cast<int>(number - pair * row_groups) * rows, f = 4 * (lane % LANES);
    const int64_t slot = static_cast<int64_t>(pair) * part.chunks;
    if (t.chunks <= 1 || first_row >= t.rows) return;
    // Lanes side by side hold different chunks of a row.
    auto gather = [&](Joined &row, const int r, const int first, const int stride) __attribute__((always_inline)) {
#pragma unroll 4
        for (int c = first + lane / LANES; c < t.chunks; c += stride) {
            const Partial p = partial_of<D>(a, part, slot + c, r);
            const f32x4 s = *reinterpret_cast<const f32x4 *>(p.stats), y = *reinterpret_cast<const f32x4 *>(p.acc + f);
            const float x[4] = {y[0], y[1], y[2], y[3]};
            row.add(s[0], s[2], s[1], x);
        }
    };
    auto across = [&](Joined &row) __attribute__((always_inline)) {
#pragma unroll
        for (int m = LANES; m < kWave; m <<= 1) {
            float x[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) x[j] = __shfl_xor(row.o[j], m);
            row.add(__shfl_xor(row.reference, m), __shfl_xor(row.most, m), __shfl_xor(row.sum, m), x);
        }
    };
    auto finish = [&](const Joined &row, const int r) __attribute__((always_inline)) {
        if (lane >= LANES || r >= t.rows) return;
        const int flat = t.row0 + r, token = flat / group;
        finish_row<T, VEC>(a, t.s.row0 + token, head * group + flat - token * group, f, row.o, row.sum, row.reference, row.most, f == 0);
    };
    if (part.chunks > kJoinTogether) {
        Joined row;
        gather(row, first_row, wave * SIDE, kWaves * SIDE);
        across(row);
        if (lane < LANES) {
            *reinterpret_cast<f32x4 *>(&merged[wave][f]) = f32x4{row.o[0], row.o[1], row.o[2], row.o[3]};
            if (f == 0) *reinterpret_cast<f32x4 *>(&merged[wave][4 * LANES]) = f32x4{row.reference, row.most, row.sum, 0.0f};
        }
        __syncthreads();
        if (wave != 0) return;
#pragma unroll
        for (int w = 1; w < kWaves; ++w) {
            const f32x4 s = *reinterpret_cast<const f32x4 *>(&merged[w][4 * LANES]), y = *reinterpret_cast<const f32x4 *>(&merged[w][f]);
            const float x[4] = {y[0], y[1], y[2], y[3]};
            row.add(s[0], s[1], s[2], x);
        }
        finish(row, first_row);
    } else {
        for (int base = first_row; base < min(first_row + rows, t.rows); base += kJoinRows) {
            Joined row[kJoinRows / kWaves]; // a wave's rows side by side: their reads are under way together
#pragma unroll
            for (int i = 0; i < kJoinRows / kWaves; ++i) gather(row[i], min(base + wave + kWaves * i, t.rows - 1), 0, SIDE);
#pragma unroll
            for (int i = 0; i < kJoinRows / kWaves; ++i) {
                across(row[i]);
                finish(row[i], base + wave + kWaves * i);
            }
        }
    }
}

uint32_t attention_groups(const ForwardPart &part, const int heads) { return static_cast<uint32_t>(part.units) * heads * part.chunks; }

template<int T, int D, bool VEC, int GROUPS>
void launch_tiles(const CacheForwardArgs &a, const ForwardPlan &plan, const uint32_t large, const uint32_t small, hipStream_t stream) {
    if (plan.large.waves == 2 * kWaves)
        hipLaunchKernelGGL((cache_attention_kernel<T, D, VEC, GROUPS, 2>), dim3(large + small), dim3(2 * kThreads), 0, stream, a, plan.large,
                plan.small, large);
    else
        hipLaunchKernelGGL((cache_attention_kernel<T, D, VEC, GROUPS, 1>), dim3(large + small), dim3(kThreads), 0, stream, a, plan.large,
                plan.small, large);
}

template<int T, int D, bool VEC>
void launch(const CacheForwardArgs &a, const ForwardPlan &plan, hipStream_t stream) {
    const int heads = a.cache.heads;
    const uint32_t large = attention_groups(plan.large, heads), small = attention_groups(plan.small, heads);
    if (large == 0 && plan.small.waves == 16) {
        if constexpr (D < 128) // (never asked for otherwise)
            hipLaunchKernelGGL((cache_attention_small_kernel<T, D, VEC, 16>), dim3(small), dim3(16 * kWave), 0, stream, a, plan.small);
    } else if (large == 0 && plan.small.waves == 8)
        hipLaunchKernelGGL((cache_attention_small_kernel<T, D, VEC, 8>), dim3(small), dim3(8 * kWave), 0, stream, a, plan.small);
    else if (large == 0)
        hipLaunchKernelGGL((cache_attention_small_kernel<T, D, VEC, kWaves>), dim3(small), dim3(kThreads), 0, stream, a, plan.small);
    else if (a.cache.page_size % kStep == 0) launch_tiles<T, D, VEC, 1>(a, plan, large, small, stream);
    else launch_tiles<T, D, VEC, 4>(a, plan, large, small, stream);
    const uint32_t large_joins = join_groups(plan.large, heads), joins = large_joins + join_groups(plan.small, heads);
    if (joins > 0)
        hipLaunchKernelGGL((cache_join_kernel<T, D, VEC>), dim3(joins), dim3(kThreads), 0, stream, a, plan.large, plan.small, large_joins);
}

template<int T, int D>
void dispatch(const CacheForwardArgs &a, const ForwardPlan &plan, const bool vec, hipStream_t stream) {
    if (vec) launch<T, D, true>(a, plan, stream);
    else launch<T, D, false>(a, plan, stream);
}

template<int T>
void dispatch(const int width, const CacheForwardArgs &a, const ForwardPlan &plan, const bool vec, hipStream_t stream) {
    if (width == 32) dispatch<T, 32>(a, plan, vec, stream);
    else if (width == 64) dispatch<T, 64>(a, plan, vec, stream);
    else dispatch<T, 128>(a, plan, vec, stream);
}

} // namespace

hipError_t launch_cache_forward(const int width, const CacheForwardArgs &a, const ForwardPlan &plan, hipStream_t stream) {
    long long groups = 0; // of the kernel, or of the join if that has more
    for (const ForwardPart *part : {&plan.small, &plan.large})
        groups += static_cast<long long>(part->units) * a.cache.heads * std::max(part->chunks, part->chunks > 1 ? part->rows / join_rows(*part) : 1);
    if (groups >= (1ll << 32) / (kWave * std::max({kWaves, plan.small.waves, plan.large.waves}))) return hipErrorInvalidValue; // threads of a launch
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
