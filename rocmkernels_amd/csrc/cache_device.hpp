// Device-side building blocks of the paged 8-bit cache's kernels: rows of the three storage types, scales as exponents, e4m3
// conversions, and the search for the sequence that a workgroup works on.
#pragma once

#include <hip/hip_runtime.h>

#include <stdint.h>

#include "attention_device.hpp"
#include "cache_launch.hpp"

namespace rk {

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));

enum Storage { kFloat32 = 0, kFloat16 = 1, kBFloat16 = 2 }; // the rocmkernels_dtype codes

template<int T>
constexpr int kSize = T == kFloat32 ? 4 : 2;

__device__ __forceinline__ float from_bf16(const uint32_t bits) { return __uint_as_float(bits << 16); }

// Round to nearest even; NaN stays NaN.
__device__ __forceinline__ uint32_t to_bf16(const float x) {
    const uint32_t u = __float_as_uint(x);
    const uint32_t rounded = (u + 0x7fffu + ((u >> 16) & 1u)) >> 16;
    return isnan(x) ? ((u >> 16) | 0x40u) : rounded;
}

// 8 contiguous elements as floats. VEC: 16-byte aligned.
template<int T, bool VEC>
__device__ __forceinline__ void load8(float (&x)[8], const void *base, const int64_t element) {
    if constexpr (T == kFloat32) {
        const float *p = static_cast<const float *>(base) + element;
        if constexpr (VEC) {
            const f32x4 a = *reinterpret_cast<const f32x4 *>(p), b = *reinterpret_cast<const f32x4 *>(p + 4);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                x[i] = a[i];
                x[4 + i] = b[i];
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = p[i];
        }
    } else {
        const uint16_t *p = static_cast<const uint16_t *>(base) + element;
        uint32_t w[4];
        if constexpr (VEC) {
            const u32x4 a = *reinterpret_cast<const u32x4 *>(p);
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = a[i];
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = p[2 * i] | (static_cast<uint32_t>(p[2 * i + 1]) << 16);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (T == kFloat16) {
                const f16x2 h = __builtin_bit_cast(f16x2, w[i]);
                x[2 * i] = static_cast<float>(h[0]);
                x[2 * i + 1] = static_cast<float>(h[1]);
            } else {
                x[2 * i] = from_bf16(w[i] & 0xffffu);
                x[2 * i + 1] = from_bf16(w[i] >> 16);
            }
        }
    }
}

// Two floats rounded to a 16-bit type, packed.
template<int T>
__device__ __forceinline__ uint32_t pack2(const float a, const float b) {
    static_assert(T != kFloat32);
    if constexpr (T == kFloat16) return __builtin_bit_cast(uint32_t, f16x2{static_cast<_Float16>(a), static_cast<_Float16>(b)});
    else return to_bf16(a) | (to_bf16(b) << 16);
}

// N (a multiple of 4) contiguous elements rounded to the storage type. VEC: 16-byte aligned for N = 8, else 4 elements aligned.
template<int T, bool VEC, int N>
__device__ __forceinline__ void store_row(void *base, const int64_t element, const float (&x)[N]) {
    static_assert(N % 4 == 0);
    if constexpr (T == kFloat32) {
        float *p = static_cast<float *>(base) + element;
#pragma unroll
        for (int i = 0; i < N; i += 4) {
            if constexpr (VEC) {
                *reinterpret_cast<f32x4 *>(p + i) = f32x4{x[i], x[i + 1], x[i + 2], x[i + 3]};
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j) p[i + j] = x[i + j];
            }
        }
    } else {
        uint16_t *p = static_cast<uint16_t *>(base) + element;
        uint32_t w[N / 2];
#pragma unroll
        for (int i = 0; i < N / 2; ++i) w[i] = pack2<T>(x[2 * i], x[2 * i + 1]);
        if constexpr (VEC && N % 8 == 0) {
#pragma unroll
            for (int i = 0; i < N / 8; ++i)
                *reinterpret_cast<u32x4 *>(p + 8 * i) = u32x4{w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]};
        } else if constexpr (VEC) {
#pragma unroll
            for (int i = 0; i < N / 4; ++i) *reinterpret_cast<u32x2 *>(p + 4 * i) = u32x2{w[2 * i], w[2 * i + 1]};
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) p[i] = static_cast<uint16_t>(w[i / 2] >> (16 * (i & 1)));
        }
    }
}

// ---- scales -----------------------------------------------------------------------------------------------
// 2^e for -126 <= e <= 127.
__device__ __forceinline__ float power(const int e) { return __uint_as_float(static_cast<uint32_t>(e + 127) << 23); }

// Exponent of a stored scale. Whatever the float holds (0 in a fresh cache), the result is an exponent that a scale may take.
__device__ __forceinline__ int scale_exponent(const float scale) {
    const int e = static_cast<int>((__float_as_uint(scale) >> 23) & 255u) - 127;
    return min(max(e, kScaleLow), kScaleHigh);
}

// Smallest e with most <= 448 * 2^e (448 = 1.75 * 2^8), clamped; most is finite and not negative.
__device__ __forceinline__ int exponent_for(const float most) {
    const uint32_t u = __float_as_uint(most);
    const int e = static_cast<int>(u >> 23) - 127 - 8 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);
    return min(max(e, kScaleLow), kScaleHigh);
}

// ---- e4m3 -------------------------------------------------------------------------------------------------
// Four values to e4m3 bytes (nearest even), infinities as NaN. The finite ones are within 448.
__device__ __forceinline__ uint32_t to_e4m3(const float a, const float b, const float c, const float d) {
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(isinf(a) ? NAN : a, isinf(b) ? NAN : b, 0, false);
    w = __builtin_amdgcn_cvt_pk_fp8_f32(isinf(c) ? NAN : c, isinf(d) ? NAN : d, w, true);
    return static_cast<uint32_t>(w);
}

// Four bytes requantised by a factor that does not enlarge them.
__device__ __forceinline__ uint32_t requantise(const uint32_t bytes, const float factor) {
    const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(bytes), false);
    const auto hi = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(bytes), true);
    return to_e4m3(lo[0] * factor, lo[1] * factor, hi[0] * factor, hi[1] * factor);
}

// ---- sequences --------------------------------------------------------------------------------------------
__device__ __forceinline__ int clamped(const int x, const int low, const int high) { return min(max(x, low), high); }

constexpr int kLengthLimit = 1 << 30; // lengths are clamped to it, so positions fit 32 bits whatever the array holds

struct Sequence {
    int b, row0, count; // its rows row0 .. row0 + count - 1
    int length, first;  // its keys, and the position of its first row (may be negative)
    uint32_t base;      // the first unit that belongs to it
};

__device__ __forceinline__ Sequence make_sequence(const int b, const int row0, const int end, const int length) {
    Sequence r;
    r.b = b;
    r.row0 = row0;
    r.count = max(0, end - row0);
    r.length = clamped(length, 0, kLengthLimit);
    r.first = r.length - r.count;
    r.base = 0;
    return r;
}

__device__ __forceinline__ Sequence sequence_at(const SequenceView &s, const int b) {
    return make_sequence(b, clamped(s.starts[b], 0, s.tokens), clamped(s.starts[b + 1], 0, s.tokens), s.lengths[b]);
}

// The sequence that unit `unit` belongs to (cache_plan.hpp). A sequence's first unit ascends with b, so each lane of the wave tests
// one of 64 spaced sequences and a ballot gives the last whose base is not past the unit: one load per lane and round, two rounds
// for up to 4096 sequences (a binary search has a dependent load for each bit). The last round's lanes hold neighbouring sequences,
// with all that is known of them, so what it finds needs no further load.
__device__ __forceinline__ Sequence find_sequence(const SequenceView &s, const uint32_t unit, const uint32_t mul, const uint32_t add,
        const uint32_t div) {
    const int lane = threadIdx.x & (kWave - 1);
    int low = 0, span = s.batch;
    while (span > kWave) {
        const int step = search_step(span);
        const int b = low + lane * step;
        const bool in = lane * step < span;
        const uint64_t reached = __ballot(in && reaches(clamped(s.starts[in ? b : low], 0, s.tokens), b, unit, mul, add, div));
        const int hit = reached ? 63 - __builtin_clzll(reached) : 0;
        low += hit * step;
        span = min(step, span - hit * step);
    }
    const bool in = lane < span;
    const int b = in ? low + lane : low;
    const int start = clamped(s.starts[b], 0, s.tokens), end = clamped(s.starts[b + 1], 0, s.tokens), length = s.lengths[b];
    const uint64_t reached = __ballot(in && reaches(start, b, unit, mul, add, div));
    const int hit = reached ? 63 - __builtin_clzll(reached) : 0;
    Sequence r = make_sequence(low + hit, __builtin_amdgcn_readlane(start, hit), __builtin_amdgcn_readlane(end, hit),
            __builtin_amdgcn_readlane(length, hit));
    r.base = unit_base(r.row0, r.b, mul, add, div);
    return r;
}

} // namespace rk
