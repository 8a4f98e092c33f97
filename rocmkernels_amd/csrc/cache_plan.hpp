// How a cache call is cut into workgroups: host and device arithmetic without any HIP call (tests/cpp/cache_plan_check.cpp runs it on
// the CPU).
//
// starts, the division of the packed rows over sequences, is device memory, so the host sizes a launch from tokens and batch
// alone: sequence b owns the units from floor((starts[b] * mul + b * add) / div) up to the next sequence's first. For tiles of `rows`
// flattened rows (mul = heads of a group, add = rows - 1, div = rows) these are at least ceil(n / rows) units for n rows, and
// exactly one for each sequence of a decoding batch; for pages of `size` tokens (mul = 1, add = 2 size - 2, div = size) at least
// floor((n + 2 size - 2) / size), the most pages that n rows touch.
#pragma once

#include <hip/hip_runtime.h>

#include <stddef.h>
#include <stdint.h>

#include <algorithm>

namespace rk {

constexpr int kBlockTokens = 16;   // tokens of one block of a page: K rows [16][D], V columns [D][16]
constexpr int kMaxPage = 128;
constexpr int kMaxRows = 256;      // no tile of the attention kernels has more rows
constexpr int kStep = 64;          // keys of a step of the attention kernels

struct SequenceView {
    const int *starts, *lengths, *table;
    int batch, tokens, columns, table_stride;
};

__host__ __device__ inline uint32_t unit_base(const int start, const int b, const uint32_t mul, const uint32_t add, const uint32_t div) {
    return (static_cast<uint32_t>(start) * mul + static_cast<uint32_t>(b) * add) / div;
}

// Whether sequence b's first unit is not past `unit`: floor(x / div) <= unit exactly where x < (unit + 1) * div.
__host__ __device__ inline bool reaches(const int start, const int b, const uint32_t unit, const uint32_t mul, const uint32_t add,
        const uint32_t div) {
    return static_cast<uint32_t>(start) * mul + static_cast<uint32_t>(b) * add < (unit + 1) * div;
}

// The search's rounds: 64 lanes test sequences `search_step` apart.
__host__ __device__ inline int search_step(const int span) { return (span + 63) / 64; }

inline long long row_units(const long long flat_rows, const int batch, const int rows) {
    return (flat_rows + static_cast<long long>(batch) * (rows - 1)) / rows;
}

inline long long page_units(const int tokens, const int batch, const int size) {
    return (tokens + static_cast<long long>(batch) * (2 * size - 2)) / size;
}

// One launch of the attention kernels. Rows of a sequence are flattened to (row, query head of the group) and cut into tiles of
// `rows`; the keys a tile sees are cut into chunks of `chunk_steps` steps, `chunks` at most. A part takes the sequences that have
// between `least` and `most` flattened rows; with `direct` every sequence has that many units, otherwise they are searched.
struct ForwardPart {
    int rows, units, direct, least, most, chunk_steps, chunks;
    int waves;           // of a workgroup; the waves of a small tile take turns with the steps
    size_t workspace;   // bytes: one partial result for each chunk of each tile
    size_t workspace_at; // where they start
};

// A call: tiles of few rows stream the keys for themselves (`small`), tiles of many rows share them (`large`).
struct ForwardPlan {
    ForwardPart small, large;
    size_t workspace;      // bytes this call needs
    size_t workspace_most; // and with any smaller window
};

constexpr int kSmallRows = 32;  // sequences of up to this many flattened rows are small work where both kinds may be
constexpr int kLargeTile = 128; // rows of a large tile

// How many workgroups the large tiles are to make, and the waves of one: four, or two teams of four that take turns with a tile's steps
// and merge in LDS, which needs no join but gives a compute unit to one tile. `filled` tiles of all heads together, about; `steps`
// of the keys that a tile may see. Fewer of them never mean more workspace: where they change the waves, the smaller number makes fewer
// chunks.
// us with four waves, then with two teams; fp16 and bf16 32 heads on 8, 128-wide, but where a width is given:
//   one sequence, 768 rows x 4096 keys 91, 73; 1024 x 4096 94, 77; 300 x 32768 268, 199; 64-wide 1500 x 1500 31.6, 25.0; but 1536 x 4096
//     (384 tiles) 118, 118; 64 x 2000 (16 tiles) 35, 37
//   several, 256 x 2048 twice to four times 54, 44; 128 x 3000 six times 76, 60; 64-wide FP32 2 x 1500 x 1500 (281 tiles) 49, 47, ragged
//     4 x 1500 50, 55
//   one prompt beside 31 tokens, 384 x 2048 53, 43; 512 x 4096 84, 80; but 512 x 8192 136, 167; 256 x 4096 (64 tiles) 62, 79; 1024
//     x 4096 beside 63 (264 tiles) 136, 172: the tokens' streams then wait for the tiles
// Where several sequences have many keys, the longest one's steps in a row count: three chunks a tile (ragged 4 x 256 x 8192 145 -> 107,
// 8 x 128 x 8192 186 -> 109, 64-wide FP32 2 x 1500 x 6000 179 -> 152, ragged 148 -> 107).
inline int large_waves(const int batch, const long long flat, const long long filled, const long long steps, long long &workgroups) {
    const bool prompts = batch == 1 || flat >= static_cast<long long>(kLargeTile) * batch; // not: mostly single tokens
    // Beside the tokens of a mixed batch, with four waves: 128 workgroups take 108 us, 256 90, 384 90, 512 106.
    workgroups = batch > 1 ? 256 : 512;
    if (steps < 8 || filled <= (batch > 1 ? 85 : 64)) return 4;
    if (batch > 1 && prompts && steps >= 90 && filled < 512) {
        workgroups = 3 * filled;
        return 4;
    }
    if (filled > (prompts ? 256 : 128) || (!prompts && steps >= 80)) return 4;
    workgroups = prompts ? 256 / filled * filled : filled;
    return 8;
}

inline ForwardPlan plan_cache_forward(const int width, const SequenceView &s, const int heads, const int query_heads, const int max_keys,
        const int radius, const bool causal) {
    const int group = query_heads / heads;
    const long long flat = static_cast<long long>(s.tokens) * group;
    ForwardPlan p{};
    size_t most = 0;
    // Batches whose sequences have a few rows on average are small work throughout, whatever a single sequence has.
    const bool small_only = flat <= 16ll * s.batch || flat <= kSmallRows;
    // The steps of the keys that a tile of `rows` rows may see: all, or its window.
    auto span_steps = [&](const int rows) {
        long long span = max_keys;
        if (radius >= 0) span = std::min(span, (causal ? 1ll : 2ll) * radius + 1 + (rows + group - 1) / group + kStep);
        return (span + kStep - 1) / kStep;
    };
    long long large_groups = 0;
    const int waves = small_only ? 4 : large_waves(s.batch, flat, std::max(flat / kLargeTile, 1ll) * heads, span_steps(kLargeTile), large_groups);
    // `tiles`: about how many of the units have rows, which the division over sequences leaves open.
    auto cut = [&](ForwardPart &part, const long long tiles, const long long workgroups, const int least_steps) {
        const long long steps = span_steps(part.rows);
        const long long pairs = static_cast<long long>(part.units) * heads, filled = std::max(tiles * heads, 1ll);
        const long long wanted = std::max((workgroups + filled / 2) / filled, 1ll);
        const long long chunks = std::min(wanted, std::max(1ll, steps / least_steps)); // grows with the keys and the window
        const size_t chunk_bytes = static_cast<size_t>(pairs) * part.rows * (width + 4) * sizeof(float);
        most += chunks > 1 ? chunk_bytes * chunks : 0;
        bool single = false;
        part.waves = waves;
        if (&part == &p.small && small_only) {
            // More waves a workgroup where the chip has room for them and one chunk then holds the keys in four steps a wave: that saves
            // the join (16 x 5 drafted rows x 4001 keys, 64-wide: 19.5 -> 14.2 us; 8 waves for several chunks of 1 x 32768: no change).
            const long long room = (width == 128 ? 8 : 16) * 256ll; // waves at the kernels' registers
            for (int more = width == 128 ? 8 : 16; more > 4; more /= 2) {
                if (steps > 4ll * more || steps <= more / 2 || filled * more > room) continue;
                part.waves = more;
                single = true;
                break;
            }
        }
        part.chunk_steps = static_cast<int>(single ? steps : ((steps + chunks - 1) / chunks + 3) / 4 * 4); // whole turns of four waves
        part.chunks = static_cast<int>((steps + part.chunk_steps - 1) / part.chunk_steps);
        part.workspace = part.chunks > 1 ? chunk_bytes * part.chunks : 0;
        part.workspace_at = p.workspace;
        p.workspace += part.workspace;
    };
    if (!small_only) {
        p.large.rows = kLargeTile;
        p.large.units = static_cast<int>(row_units(flat, s.batch, kLargeTile));
        p.large.least = s.batch > 1 ? kSmallRows + 1 : 1;
        p.large.most = 0x7fffffff;
        cut(p.large, flat / kLargeTile, large_groups, waves == 8 ? 16 : 8);
    }
    if (small_only || s.batch > 1) {
        p.small.rows = 16;
        p.small.direct = small_only ? 0 : kSmallRows / 16;
        p.small.units = small_only ? static_cast<int>(row_units(flat, s.batch, 16)) : s.batch * p.small.direct;
        p.small.least = 1;
        p.small.most = small_only ? 0x7fffffff : kSmallRows;
        // 64 sequences of up to 8192 keys, 8 heads: 512 workgroups 132 us, 1024 137, 2048 133. Beside large tiles, which hold half
        // the chip for longer, few chunks: 512 84 us, 1024 86, 2048 90 (32 sequences of up to 4096 keys, one with 512 new rows).
        cut(p.small, small_only ? std::max(flat / 16, static_cast<long long>(std::min(s.batch, s.tokens))) : s.batch, small_only ? 2048 : 2048 / waves, 16);
    }
    p.workspace_most = most;
    return p;
}

} // namespace rk
