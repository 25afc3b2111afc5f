// Walks the index arithmetic of the paged cache's kernels on the host: every
// key, page and LDS slot that they would touch lies in its bounds, the splits
// cover what is seen exactly once, and an eviction keeps what it says.
#include <cstdio>
#include <cstdlib>
#include <random>
#include <vector>

#define HIP_INCLUDE_HIP_HIP_EXT_H  // launches, which only hipcc compiles
#include "../franken_ocr_amd/csrc/k_paged_index.hpp"

using namespace focr;

static void require(bool ok, const char* what, unsigned long long at) {
    if (ok) return;
    std::printf("FAILED: %s (case %llu)\n", what, at);
    std::exit(1);
}

int main() {
    std::mt19937_64 rng(5);
    const auto pick = [&](uint64_t lo, uint64_t hi) { return lo + rng() % (hi - lo + 1); };
    for (unsigned long long at = 0; at < 20000; ++at) {
        const int shift = static_cast<int>(pick(0, 10));
        const size_t max_pages = pick(1, std::max<uint64_t>(1, (at % 8 == 0 ? 40000 : 3000) >> shift));
        const uint32_t held = static_cast<uint32_t>(max_pages << shift);
        const uint32_t max_len = at % 3 == 0 ? held : static_cast<uint32_t>(pick(1, held));
        uint32_t len = static_cast<uint32_t>(pick(0, max_len + 2));  // past it too: cut
        if (at % 17 == 0) len = kPagedNone;
        if (at % 19 == 0) len = kPagedNone - 1;
        const uint32_t prefix = static_cast<uint32_t>(at % 5 == 0 ? kPagedNone : pick(0, max_len + 1));
        const uint32_t window = at % 2 ? static_cast<uint32_t>(pick(1, max_len + 1)) : 0;
        const bool step = at % 4 < 2, with_prefix = at % 7 != 0;
        const size_t n_seqs = pick(1, 200), heads = pick(1, 16);
        const int group = static_cast<int>(pick(1, 64));
        std::vector<uint32_t> table(max_pages, 0);
        const PagedTables t{table.data(), &len, 1, max_pages, max_len};
        const Seen e = seen_of(t, with_prefix ? &prefix : nullptr, window, step, 0);
        require(e.none == (len == kPagedNone), "none", at);
        if (e.none) continue;
        require(e.n <= max_len && e.nvis <= e.n && e.p <= e.nvis, "counts", at);
        require(e.own == (step && len < max_len), "own", at);
        const uint32_t seen = window && !with_prefix ? std::min(max_len, window) : max_len;
        require(e.nvis <= seen, "the call is sized for what is seen", at);
        const PagedSplits splits = pick_splits(n_seqs, heads, group, seen, window != 0, 256);
        const int nsplit = splits.count;
        require(nsplit >= 1, "splits", at);
        const uint32_t chunk = split_keys(e.nvis, nsplit, splits.least);
        require(chunk <= static_cast<uint32_t>(kPagedChunkMax) && chunk % kPagedChunkUnit == 0, "a split fits LDS", at);
        std::vector<uint8_t> hit(max_pages << shift, 0);
        uint32_t covered = 0;
        const uint32_t parts = (e.nvis + chunk - 1) / chunk;
        require(parts <= static_cast<uint32_t>(nsplit), "parts", at);
        for (int z = 0; z < nsplit; ++z) {
            const uint32_t b0 = static_cast<uint32_t>(z) * chunk;
            if (b0 >= e.nvis) {
                require(static_cast<uint32_t>(z) >= parts, "an empty split is past the joined ones", at);
                continue;
            }
            const uint32_t cnt = std::min(chunk, e.nvis - b0);
            for (int tile : {4, 8, 16, 32, 64})
                require((cnt + tile - 1) / tile * tile <= static_cast<uint32_t>(kPagedChunkMax), "a padded split fits", at);
            for (uint32_t j = 0; j < cnt; ++j) {
                const uint32_t key = b0 + j < e.p ? b0 + j : b0 + j + e.shift;
                require(key < e.n && (key >> shift) < max_pages, "a key is in the table", at);
                require(!hit[key], "a key is seen once", at);
                hit[key] = 1;
                ++covered;
            }
        }
        require(covered == e.nvis, "all that is seen is split", at);
        for (uint32_t key = 0; key < e.n; ++key) {
            const uint32_t first = with_prefix ? std::min(prefix, e.n) : 0;
            const bool want = window == 0 || key < first || static_cast<uint64_t>(key) + window >= e.n;
            require(hit[key] == want, "the keys seen are the documented ones", at);
        }
        if (e.own) require(hit[len] && len == e.n - 1, "a step sees its own key, the last", at);

        PagedEvict ev{};
        ev.t = t;
        ev.budget = static_cast<uint32_t>(pick(1, max_len + 3));
        ev.sinks = static_cast<uint32_t>(pick(0, ev.budget));
        ev.recent = static_cast<uint32_t>(pick(0, ev.budget - ev.sinks));
        const Cut c = cut_of(ev, 0);
        require(c.n == std::min(len, max_len) && c.lo <= c.hi && c.hi <= c.n, "the cut's bounds", at);
        const uint32_t stay = c.lo + c.want + (c.n - c.hi);
        require(c.want <= c.hi - c.lo && stay == std::min(c.n, ev.budget), "the cut keeps its budget", at);

        const PoolGeom g{nullptr, nullptr, 1u + static_cast<uint32_t>(pick(0, 1000)), shift, static_cast<uint32_t>(heads)};
        table[0] = static_cast<uint32_t>(pick(0, 1200));
        for (uint32_t hk = 0; hk < heads; ++hk) {
            const uint32_t off = static_cast<uint32_t>(pick(0, (1u << shift) - 1));
            const uint32_t row = row_of(t, g, 0, hk, off);
            if (table[0] >= g.n_pages)
                require(row == kBadRow, "a page that is none has no row", at);
            else
                require(row < static_cast<uint64_t>(g.n_pages) * heads << shift && row != kBadRow, "a row is in the pool", at);
        }
    }
    std::printf("ok\n");
    return 0;
}
