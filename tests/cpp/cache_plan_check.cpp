// Host check of the arithmetic that maps workgroups to sequences (cache_plan.hpp): for random divisions of rows over sequences,
// every tile of rows and every page that receives rows has exactly one unit, units of one sequence never reach into the next
// one's, and the search finds the sequence of a unit. Random plans stay within their limits, and a smaller window never needs more
// workspace than the largest.
#include "cache_plan.hpp"

#include <cstdio>
#include <random>
#include <vector>

namespace {
int failures = 0;
void check(const bool ok, const char *what) {
    if (!ok && ++failures < 20) std::printf("FAIL %s\n", what);
}

// The device's search, one lane after the other.
int search(const std::vector<int> &starts, const int batch, const int tokens, const uint32_t unit, const uint32_t mul, const uint32_t add,
        const uint32_t div) {
    int low = 0, span = batch;
    for (bool last = false; !last;) {
        last = span <= 64;
        const int step = rk::search_step(span); // 1 in the last round
        int hit = 0;
        for (int lane = 0; lane < 64; ++lane) {
            const int b = low + lane * step;
            if (lane * step < span && rk::reaches(std::min(std::max(starts[b], 0), tokens), b, unit, mul, add, div)) hit = lane;
        }
        low += hit * step;
        span = std::min(step, span - hit * step);
    }
    return low;
}
} // namespace

int main() {
    std::mt19937 rng(7);
    auto pick = [&](const int low, const int high) { return low + static_cast<int>(rng() % (high - low + 1)); };
    for (int round = 0; round < 4000; ++round) {
        const int batch = round % 50 == 0 ? pick(1000, 9000) : pick(1, 200), most = pick(0, 3) == 0 ? 400 : 3;
        std::vector<int> starts(batch + 1, 0);
        for (int b = 0; b < batch; ++b) starts[b + 1] = starts[b] + (pick(0, 3) == 0 ? 0 : pick(0, most));
        const int tokens = starts[batch] + pick(0, 2), group = pick(1, 9);
        // Row tiles.
        for (const int rows : {16, 32, 128}) {
            const uint32_t mul = group, add = rows - 1, div = rows;
            const long long units = rk::row_units(static_cast<long long>(tokens) * group, batch, rows);
            for (int b = 0; b < batch; ++b) {
                const uint32_t base = rk::unit_base(starts[b], b, mul, add, div), next = rk::unit_base(starts[b + 1], b + 1, mul, add, div);
                const uint32_t tiles = (static_cast<uint32_t>(starts[b + 1] - starts[b]) * group + rows - 1) / rows;
                check(base + tiles <= next && next <= static_cast<uint32_t>(units), "row tiles reach into the next sequence");
                if (b % 7 == 0 || batch < 300)
                    for (uint32_t t = 0; t < tiles; t += std::max(1u, tiles / 3))
                        check(search(starts, batch, tokens, base + t, mul, add, div) == b, "search for a row tile");
            }
        }
        // Pages.
        const int size = 16 * pick(1, 8);
        const uint32_t add = 2 * size - 2;
        const long long units = rk::page_units(tokens, batch, size);
        for (int b = 0; b < batch; ++b) {
            const int count = starts[b + 1] - starts[b], first = pick(0, 500);
            const uint32_t pages = count ? (first + count - 1) / size - first / size + 1 : 0;
            const uint32_t base = rk::unit_base(starts[b], b, 1, add, size);
            check(base + pages <= rk::unit_base(starts[b + 1], b + 1, 1, add, size), "pages reach into the next sequence");
            check(base + pages <= static_cast<uint32_t>(units), "more pages than units");
            if (pages && (b % 7 == 0 || batch < 300)) check(search(starts, batch, tokens, base + pages - 1, 1, add, size) == b, "search for a page");
        }
        // Tokens.
        for (int b = 0; b < batch; b += 1 + batch / 50)
            if (starts[b + 1] > starts[b]) check(search(starts, batch, tokens, starts[b + 1] - 1, 1, 0, 1) == b, "search for a token");
        // Plans.
        const rk::SequenceView s{nullptr, nullptr, nullptr, batch, tokens, 1, 1};
        const int heads = pick(1, 12), keys = pick(0, 2) ? pick(1, 5000) : pick(1, 200000), width = 32 << pick(0, 2);
        const size_t whole = rk::plan_cache_forward(width, s, heads, heads * group, keys, -1, false).workspace_most;
        for (const int radius : {-1, 0, 1, 100, 777, 5000, 100000}) {
            const rk::ForwardPlan p = rk::plan_cache_forward(width, s, heads, heads * group, keys, radius, round % 2 == 0);
            check(p.workspace <= whole, "a window needs more workspace than the whole");
            check(p.small.workspace + p.large.workspace == p.workspace, "parts of the workspace");
            for (const rk::ForwardPart *part : {&p.small, &p.large}) {
                if (part->units == 0) continue;
                check(part->waves >= 4 && part->waves <= (width == 128 ? 8 : 16) && part->rows > 0 && part->rows <= rk::kMaxRows && part->chunks >= 1 && part->chunk_steps >= 1, "part");
                check(part->workspace_at + part->workspace <= p.workspace, "a part lies behind the workspace");
                // The steps of any tile fit the chunks: rows of neighbouring tokens anywhere, against their window.
                for (int trial = 0; trial < 5; ++trial) {
                    const bool causal = round % 2 == 0;
                    const int row0 = pick(0, 300), rows = pick(1, part->rows), position = pick(-100, keys);
                    const int from = position + row0 / group, to = position + (row0 + rows - 1) / group;
                    long long low = 0, high = keys;
                    if (radius >= 0) {
                        low = std::max(0, from - radius);
                        high = std::min<long long>(high, static_cast<long long>(to) + radius + 1);
                    }
                    if (causal) high = std::min<long long>(high, to + 1);
                    const long long steps = high > low ? (high + rk::kStep - 1) / rk::kStep - low / rk::kStep : 0;
                    check(steps <= static_cast<long long>(part->chunks) * part->chunk_steps, "a tile has more steps than its chunks");
                }
                if (radius < 0) check(static_cast<long long>(part->chunks) * part->chunk_steps * rk::kStep >= keys, "chunks do not cover the keys");
            }
            // Every number of rows belongs to exactly one part, and a part with one unit a sequence holds all its rows.
            for (int b = 0; b < batch; b += 1 + batch / 20) {
                const int rows = (starts[b + 1] - starts[b]) * group;
                if (rows == 0) continue;
                int parts = 0;
                for (const rk::ForwardPart *part : {&p.small, &p.large}) {
                    const bool takes = part->units > 0 && rows >= part->least && rows <= part->most;
                    parts += takes;
                    if (takes && part->direct) check(rows <= part->direct * part->rows, "a direct part leaves rows out");
                }
                check(parts == 1, "rows of no part or of two");
            }
        }
    }
    // Large tiles of eight waves, as tests/test_cache_gpu.py expects them: batch, tokens, heads, group, keys, radius, waves.
    for (const auto &c : {std::vector<int>{1, 131, 13, 5, 704, -1, 8}, {1, 131, 13, 5, 704, 500, 8}, {1, 131, 13, 5, 2240, -1, 8},
                 {4, 251, 13, 5, 704, -1, 8}, {11, 161, 16, 5, 912, -1, 8}, {1, 130, 13, 5, 1008, -1, 8}, {1, 130, 13, 5, 1008, 100, 4},
                 {1, 20, 13, 5, 1008, -1, 4}}) {
        const rk::SequenceView s{nullptr, nullptr, nullptr, c[0], c[1], 1, 1};
        const rk::ForwardPlan p = rk::plan_cache_forward(64, s, c[2], c[2] * c[3], c[4], c[5], true);
        check(p.large.waves == c[6] && (p.small.units == 0 || p.small.waves == c[6]), "waves of a large tile");
    }
    std::printf("%d failure(s)\n", failures);
    return failures != 0;
}
