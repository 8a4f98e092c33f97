// Appending keys and values to the paged 8-bit cache, with the position rotation on the way (MI355X, gfx950).
//
// Per (page, head) that receives rows, for K and for V: a = max |x| over the new finite values (K after rotation), e the smallest
// exponent with a <= 448 * 2^e, at least the page's own where earlier rows stay; byte = e4m3(x * 2^-e). A power-of-two scale
// costs e4m3 nothing, as a float's relative step does not depend on the scale, and makes every step exact but the one rounding: x * 2^-e
// is exact, and earlier rows keep their values when the scale grows (but for subnormals).
//
// One job per (page, head, K or V), because the scale needs all the new rows of the page before the first byte is written: a wave
// (four jobs to a workgroup) where sequences bring a few rows or the page fits a wave's registers, four waves otherwise. A job
// holds its rotated values in registers between the two passes (rows beyond what fits are read again, from L2). Query rows are
// rotated by further workgroups of the same launch, so that all reads of a call are in flight together.
#include "cache_device.hpp"
#include "cache_launch.hpp"

namespace rk {

namespace {

// Sixteen values of a row: columns c .. c + 7 and their partners c + D / 2 .. c + D / 2 + 7.
struct Pairs {
    float lo[8], hi[8];
};
template<int T, int D, bool VEC>
__device__ __forceinline__ Pairs load_pairs(const void *x, const int64_t element) {
    Pairs p;
    load8<T, VEC>(p.lo, x, element);
    load8<T, VEC>(p.hi, x, element + D / 2);
    return p;
}

// Rotated by a row of the tables. Each product is rounded before the sum, as rotary.hip does (the library is built with
// -ffp-contract=off).
__device__ __forceinline__ Pairs turned(const Pairs &x, const Pairs &cos, const Pairs &sin) {
    Pairs y;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        y.lo[i] = x.lo[i] * cos.lo[i] - x.hi[i] * sin.lo[i];
        y.hi[i] = x.hi[i] * cos.hi[i] + x.lo[i] * sin.hi[i];
    }
    return y;
}

__device__ __forceinline__ float largest(float most, const float (&x)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) most = fmaxf(most, isfinite(x[i]) ? fabsf(x[i]) : 0.0f);
    return most;
}

// The largest value of a job's threads, for all of them.
template<int W>
__device__ __forceinline__ float job_max(float x, float *shared) {
#pragma unroll
    for (int m = 1; m < kWave; m <<= 1) x = fmaxf(x, __shfl_xor(x, m));
    if constexpr (W > 1) {
        if ((threadIdx.x & (kWave - 1)) == 0) shared[threadIdx.x / kWave] = x;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < W; ++i) x = fmaxf(x, shared[i]);
    }
    return x;
}

// Ends the writes of earlier rows before those of the new ones: all of them come from this job's threads.
template<int W>
__device__ __forceinline__ void job_sync() {
    if constexpr (W > 1) __syncthreads();
    else wave_lds_sync();
}

// The rows of one sequence that land on one page. Nothing of it depends on the page's number, so the rows are on their way before the
// table has answered.
struct PageRows {
    int slot0, count;  // new rows take slots slot0 .. slot0 + count - 1
    int64_t row;       // packed row of slot 0 (counted back from the first new row)
    int64_t position;  // position of slot 0
    int64_t cell;      // page * heads + head; negative: no page
};

// New scale exponent of the page for one of its halves; writes it.
__device__ __forceinline__ int settle_scale(const AppendArgs &a, const PageRows &p, const int which, const float most, const int before,
        const int thread) {
    int e = exponent_for(most);
    if (p.slot0 > 0) e = max(e, before);
    if (thread == 0) a.cache.scales[2 * p.cell + which] = power(e);
    return e;
}

template<int T, int D, bool VEC, int W>
__device__ __forceinline__ void append_keys(const AppendArgs &a, const PageRows &p, const int head, const int thread, float *shared) {
    constexpr int CG = D / 16;          // threads of a row
    constexpr int THREADS = W * kWave;
    constexpr int KEPT = 4;             // a page of 128 tokens at D = 128 with four waves, 4096 values with one
    const int items = p.count * CG;
    auto load = [&](const int item) __attribute__((always_inline)) {
        const int slot = p.slot0 + item / CG, c = 8 * (item % CG);
        const int64_t at = p.position + slot;
        const Pairs x = load_pairs<T, D, VEC>(a.k, (p.row + slot) * a.ks.token + static_cast<int64_t>(head) * a.ks.head + c);
        if (!a.cos) return x;
        return turned(x, load_pairs<kFloat32, D, VEC>(a.cos, at * a.cs.token + c), load_pairs<kFloat32, D, VEC>(a.sin, at * a.ss.token + c));
    };
    Pairs kept[KEPT];
    float most = 0.0f;
#pragma unroll
    for (int i = 0; i < KEPT; ++i) {
        const int item = thread + i * THREADS;
        if (item < items) {
            kept[i] = load(item);
            most = largest(largest(most, kept[i].lo), kept[i].hi);
        }
    }
    for (int item = thread + KEPT * THREADS; item < items; item += THREADS) {
        const Pairs y = load(item);
        most = largest(largest(most, y.lo), y.hi);
    }
    if (p.cell < 0) return;
    const int before = scale_exponent(a.cache.scales[2 * p.cell]);
    const int e = settle_scale(a, p, 0, job_max<W>(most, shared), before, thread);
    uint8_t *const page = a.cache.keys + p.cell * a.cache.page_size * D;
    if (p.slot0 > 0 && e > before) { // rows in front of the new ones: whole rows, so none shares a byte with them
        const float factor = power(max(before - e, -126));
        for (int i = thread; i < p.slot0 * (D / 16); i += THREADS) {
            u32x4 *const q = reinterpret_cast<u32x4 *>(page) + i;
            const u32x4 x = *q;
            *q = u32x4{requantise(x[0], factor), requantise(x[1], factor), requantise(x[2], factor), requantise(x[3], factor)};
        }
    }
    const float factor = power(-e);
    auto store = [&](const Pairs &y, const int item) __attribute__((always_inline)) {
        uint8_t *const row = page + (p.slot0 + item / CG) * D + 8 * (item % CG);
        auto bytes = [&](const float (&x)[8]) __attribute__((always_inline)) {
            return u32x2{to_e4m3(x[0] * factor, x[1] * factor, x[2] * factor, x[3] * factor),
                    to_e4m3(x[4] * factor, x[5] * factor, x[6] * factor, x[7] * factor)};
        };
        *reinterpret_cast<u32x2 *>(row) = bytes(y.lo);
        *reinterpret_cast<u32x2 *>(row + D / 2) = bytes(y.hi);
    };
#pragma unroll
    for (int i = 0; i < KEPT; ++i) {
        const int item = thread + i * THREADS;
        if (item < items) store(kept[i], item);
    }
    for (int item = thread + KEPT * THREADS; item < items; item += THREADS) store(load(item), item);
}

// V is stored with the 16 tokens of a block side by side for each feature, so a thread takes 4 tokens (slots 4q .. 4q + 3) by 8
// features and packs the 4 bytes of a feature into one dword. Whole new blocks then pass through LDS and leave as 16-byte stores;
// the quads of a block that is not all new are stored from registers, byte by byte where a quad is not all new either.
template<int D>
constexpr int kBlockStride = D * 16 + D / 8 * 16; // LDS bytes of a block: 16 bytes of padding per 8 features keep the writes on distinct banks
constexpr int kWavePage = 4096;                   // values of a page that one wave holds in registers, and stages
constexpr int kStaged = kWaves * (kWavePage + kWavePage / 8); // four waves' pages, or one workgroup's of 128 tokens at D = 128

template<int T, int D, bool VEC, int W>
__device__ __forceinline__ void append_values(const AppendArgs &a, const PageRows &p, const int head, const int thread, float *shared,
        uint8_t *staged) {
    constexpr int CG = D / 8;
    constexpr int THREADS = W * kWave;
    constexpr int KEPT = 2;
    const int end = p.slot0 + p.count;
    const int quad0 = p.slot0 / 4;
    const int items = ((end + 3) / 4 - quad0) * CG;
    auto load = [&](float (&y)[4][8], const int item) __attribute__((always_inline)) {
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            const int slot = 4 * (quad0 + item / CG) + t;
            if (slot >= p.slot0 && slot < end) {
                load8<T, VEC>(y[t], a.v, (p.row + slot) * a.vs.token + static_cast<int64_t>(head) * a.vs.head + 8 * (item % CG));
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) y[t][i] = 0.0f;
            }
        }
    };
    float kept[KEPT][4][8];
    float most = 0.0f;
#pragma unroll
    for (int i = 0; i < KEPT; ++i) {
        const int item = thread + i * THREADS;
        if (item < items) {
            load(kept[i], item);
#pragma unroll
            for (int t = 0; t < 4; ++t) most = largest(most, kept[i][t]);
        }
    }
    for (int item = thread + KEPT * THREADS; item < items; item += THREADS) {
        float y[4][8];
        load(y, item);
#pragma unroll
        for (int t = 0; t < 4; ++t) most = largest(most, y[t]);
    }
    if (p.cell < 0) return;
    const int before = scale_exponent(a.cache.scales[2 * p.cell + 1]);
    const int e = settle_scale(a, p, 1, job_max<W>(most, shared), before, thread);
    uint8_t *const page = a.cache.values + p.cell * a.cache.page_size * D;
    if (p.slot0 > 0 && e > before) {
        // Dwords of 4 tokens; the last one may hold new slots too, whose bytes pass through and are written below.
        const float factor = power(max(before - e, -126));
        for (int i = thread; i < (p.slot0 + 3) / 4 * D; i += THREADS) {
            const int quad = i / D, stay = p.slot0 - 4 * quad;
            uint32_t *const q = reinterpret_cast<uint32_t *>(page + (quad / 4) * (16 * D) + (i % D) * 16 + (quad % 4) * 4);
            const uint32_t x = *q, y = requantise(x, factor), mask = stay >= 4 ? 0xffffffffu : (1u << (8 * stay)) - 1u;
            *q = (y & mask) | (x & ~mask);
        }
        job_sync<W>();
    }
    const float factor = power(-e);
    const bool staging = W > 1 || a.cache.page_size * D <= kWavePage;
    auto store = [&](const float (&y)[4][8], const int item) __attribute__((always_inline)) {
        const int quad = quad0 + item / CG, block = quad / 4, d0 = 8 * (item % CG);
        const bool whole = staging && 16 * block >= p.slot0 && 16 * block + 16 <= end;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const uint32_t w = to_e4m3(y[0][i] * factor, y[1][i] * factor, y[2][i] * factor, y[3][i] * factor);
            if (whole) {
                *reinterpret_cast<uint32_t *>(staged + block * kBlockStride<D> + (d0 + i) * 16 + (d0 / 8) * 16 + (quad % 4) * 4) = w;
            } else {
                uint8_t *const q = page + block * (16 * D) + (d0 + i) * 16 + (quad % 4) * 4;
                if (4 * quad >= p.slot0 && 4 * quad + 4 <= end) {
                    *reinterpret_cast<uint32_t *>(q) = w;
                } else {
#pragma unroll
                    for (int t = 0; t < 4; ++t)
                        if (4 * quad + t >= p.slot0 && 4 * quad + t < end) q[t] = static_cast<uint8_t>(w >> (8 * t));
                }
            }
        }
    };
#pragma unroll
    for (int i = 0; i < KEPT; ++i) {
        const int item = thread + i * THREADS;
        if (item < items) store(kept[i], item);
    }
    for (int item = thread + KEPT * THREADS; item < items; item += THREADS) {
        float y[4][8];
        load(y, item);
        store(y, item);
    }
    if (!staging) return;
    job_sync<W>();
    const int block0 = (p.slot0 + 15) / 16, blocks = end / 16 - block0;
    for (int i = thread; i < blocks * D; i += THREADS) {
        const int block = block0 + i / D, d = i % D;
        *reinterpret_cast<u32x4 *>(page + block * (16 * D) + d * 16) =
                *reinterpret_cast<const u32x4 *>(staged + block * kBlockStride<D> + d * 16 + (d / 8) * 16);
    }
}

// One token a wave (several tokens in turn a wave are slower: 48 against 43 us for 8192 tokens of 32 + 8 heads, 128-wide fp16).
template<int T, int D, bool VEC>
__device__ __forceinline__ void rotate_queries(const AppendArgs &a, const int token) {
    constexpr int CG = D / 16;
    if (token >= a.seqs.tokens) return;
    const Sequence s = find_sequence(a.seqs, static_cast<uint32_t>(token), 1, 0, 1);
    const int i = token - s.row0, position = s.first + i;
    if (i < 0 || i >= s.count || position < 0 || position >= a.positions) return;
    const int lane = threadIdx.x & (kWave - 1), c = 8 * (lane % CG);
    const Pairs cos = load_pairs<kFloat32, D, VEC>(a.cos, static_cast<int64_t>(position) * a.cs.token + c);
    const Pairs sin = load_pairs<kFloat32, D, VEC>(a.sin, static_cast<int64_t>(position) * a.ss.token + c);
    constexpr int TOGETHER = T == kFloat32 ? 2 : 4, SIDE = kWave / CG; // heads a lane has under way, heads side by side
    for (int head0 = lane / CG; head0 < a.query_heads; head0 += TOGETHER * SIDE) {
        Pairs x[TOGETHER];
#pragma unroll
        for (int j = 0; j < TOGETHER; ++j) {
            const int head = min(head0 + j * SIDE, a.query_heads - 1);
            x[j] = load_pairs<T, D, VEC>(a.q, static_cast<int64_t>(token) * a.qs.token + static_cast<int64_t>(head) * a.qs.head + c);
        }
#pragma unroll
        for (int j = 0; j < TOGETHER; ++j) {
            const int head = head0 + j * SIDE;
            if (head >= a.query_heads) break;
            const Pairs y = turned(x[j], cos, sin);
            const int64_t to = static_cast<int64_t>(token) * a.os.token + static_cast<int64_t>(head) * a.os.head + c;
            store_row<T, VEC>(a.oq, to, y.lo);
            store_row<T, VEC>(a.oq, to + D / 2, y.hi);
        }
    }
}

template<int T, int D, bool VEC, int W>
__global__ __launch_bounds__(kThreads) __attribute__((amdgpu_waves_per_eu(4))) void cache_append_kernel(const AppendArgs a, const uint32_t jobs, const uint32_t job_groups) {
    __shared__ float shared[kWaves];
    __shared__ __align__(16) uint8_t staged[kStaged];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    if (blockIdx.x >= job_groups) {
        rotate_queries<T, D, VEC>(a, static_cast<int>(blockIdx.x - job_groups) * kWaves + wave);
        return;
    }
    const uint32_t job = W > 1 ? blockIdx.x : blockIdx.x * kWaves + wave;
    if (job >= jobs) return;
    const int thread = W > 1 ? threadIdx.x : threadIdx.x & (kWave - 1);
    const uint32_t heads = a.cache.heads, unit = job / (2 * heads), rest = job - unit * 2 * heads;
    const int head = static_cast<int>(rest >> 1), size = a.cache.page_size;
    const Sequence s = find_sequence(a.seqs, unit, 1, 2 * size - 2, size);
    const int page_index = max(s.first, 0) / size + static_cast<int>(min(unit - s.base, 1u << 24));
    if (page_index >= a.seqs.columns) return;
    const int low = max(max(s.first, 0), page_index * size), high = min(min(s.length, (page_index + 1) * size), a.positions);
    if (low >= high) return;
    const int page = a.seqs.table[static_cast<int64_t>(s.b) * a.seqs.table_stride + page_index];
    PageRows p;
    p.slot0 = low - page_index * size;
    p.count = high - low;
    p.position = static_cast<int64_t>(page_index) * size;
    p.row = s.row0 + (p.position - s.first);
    p.cell = page < 0 || page >= a.cache.pages ? -1 : static_cast<int64_t>(page) * a.cache.heads + head;
    uint8_t *const own = staged + (W > 1 ? 0 : wave * (kStaged / kWaves));
    if (rest & 1) append_values<T, D, VEC, W>(a, p, head, thread, shared, own);
    else append_keys<T, D, VEC, W>(a, p, head, thread, shared);
}

bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// Few rows a sequence, or a page that a wave holds in registers: a wave for each job.
bool wave_jobs(const int width, const AppendArgs &a) {
    return a.seqs.tokens <= 8ll * a.seqs.batch || a.cache.page_size * width <= kWavePage;
}
long long job_groups_for(const int width, const AppendArgs &a, const long long jobs) {
    return wave_jobs(width, a) ? (jobs + kWaves - 1) / kWaves : jobs;
}

template<int T, int D, bool VEC, int W>
void launch(const AppendArgs &a, const uint32_t jobs, hipStream_t stream) {
    const uint32_t job_groups = static_cast<uint32_t>(job_groups_for(D, a, jobs));
    const uint32_t query_groups = a.q ? static_cast<uint32_t>((static_cast<int64_t>(a.seqs.tokens) + kWaves - 1) / kWaves) : 0;
    hipLaunchKernelGGL((cache_append_kernel<T, D, VEC, W>), dim3(job_groups + query_groups), dim3(kThreads), 0, stream, a, jobs, job_groups);
}

template<int T, int D>
void dispatch(const AppendArgs &a, const bool vec, const uint32_t jobs, hipStream_t stream) {
    if (wave_jobs(D, a)) {
        if (vec) launch<T, D, true, 1>(a, jobs, stream);
        else launch<T, D, false, 1>(a, jobs, stream);
    } else {
        if (vec) launch<T, D, true, kWaves>(a, jobs, stream);
        else launch<T, D, false, kWaves>(a, jobs, stream);
    }
}

template<int T>
void dispatch(const int width, const AppendArgs &a, const bool vec, const uint32_t jobs, hipStream_t stream) {
    if (width == 32) dispatch<T, 32>(a, vec, jobs, stream);
    else if (width == 64) dispatch<T, 64>(a, vec, jobs, stream);
    else dispatch<T, 128>(a, vec, jobs, stream);
}

} // namespace

hipError_t launch_cache_append(const int width, const AppendArgs &a, hipStream_t stream) {
    const int unit = a.dtype == kFloat32 ? 4 : 8; // elements in 16 bytes
    auto fits = [&](const void *p, const rocmkernels_strides &s) { return aligned16(p) && (s.head % unit) == 0 && (s.token % unit) == 0; };
    auto table_fits = [&](const void *p, const rocmkernels_strides &s) { return aligned16(p) && (s.token % 4) == 0; };
    const bool vec = fits(a.k, a.ks) && fits(a.v, a.vs) && (!a.q || (fits(a.q, a.qs) && fits(a.oq, a.os))) &&
            (!a.cos || (table_fits(a.cos, a.cs) && table_fits(a.sin, a.ss)));
    const int size = a.cache.page_size;
    const long long jobs = page_units(a.seqs.tokens, a.seqs.batch, size) * a.cache.heads * 2;
    if (jobs >= 0xffffffffll || job_groups_for(width, a, jobs) + a.seqs.tokens / kWaves >= (1ll << 32) / kThreads - 1)
        return hipErrorInvalidValue; // threads of a launch
    const uint32_t n = static_cast<uint32_t>(jobs);
    if (a.dtype == kFloat32) dispatch<kFloat32>(width, a, vec, n, stream);
    else if (a.dtype == kFloat16) dispatch<kFloat16>(width, a, vec, n, stream);
    else dispatch<kBFloat16>(width, a, vec, n, stream);
    return hipGetLastError();
}

} // namespace rk
