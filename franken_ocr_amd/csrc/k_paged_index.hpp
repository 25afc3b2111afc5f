// k_paged_index.hpp — which keys a call on the paged cache sees, how they are
// split, where their rows lie, and what an eviction keeps. Plain integer
// arithmetic, compiled for the device by k_paged.hip and for the host by the
// test that walks its bounds.
#pragma once

#include <algorithm>
#include <cstddef>
#include <cstdint>

#include "focr_internal.hpp"

#ifdef __HIP__
#define FOCR_INDEX __device__ __forceinline__
#else
#define FOCR_INDEX inline
#endif

namespace focr {
namespace {

constexpr uint32_t kBadRow = 0xFFFFFFFFu;  // no key (past the end, or a page that is none)

FOCR_INDEX uint32_t umin32(uint32_t a, uint32_t b) { return a < b ? a : b; }
FOCR_INDEX uint32_t umax32(uint32_t a, uint32_t b) { return a > b ? a : b; }

struct PoolGeom {
    void* k;
    void* v;
    uint32_t n_pages;
    int page_shift;
    uint32_t kv_heads;
};

// What sequence s's token sees: keys [0, p) and [p + shift, n), nvis of them.
// own: the key that a step writes (the last one seen), or none.
struct Seen {
    uint32_t n, p, shift, nvis;
    bool none, own;
};

FOCR_INDEX Seen seen_of(const PagedTables& t, const uint32_t* prefix, uint32_t window, bool step, int s) {
    Seen e{};
    const uint32_t len = t.lens[s];
    e.none = len == kPagedNone;
    if (e.none) return e;
    e.own = step && len < t.max_len;
    e.n = umin32(len, t.max_len) + (e.own ? 1u : 0u);
    e.p = e.n;
    e.nvis = e.n;
    if (window != 0u && window < e.n) {
        e.p = prefix ? umin32(prefix[s], e.n) : 0u;
        const uint32_t w0 = umax32(e.n - window, e.p);
        e.shift = w0 - e.p;
        e.nvis = e.p + (e.n - w0);
    }
    return e;
}

// Keys of one split: at least `least`, and enough for the visible ones to make
// at most nsplit splits, in whole units.
FOCR_INDEX uint32_t split_keys(uint32_t nvis, int nsplit, uint32_t least) {
    const uint32_t each = (nvis + nsplit - 1) / nsplit;
    return umax32((each + kPagedChunkUnit - 1) / kPagedChunkUnit * kPagedChunkUnit, least);
}

// Splits of a call whose sequences see up to max_seen keys: as many as give
// every CU twelve blocks were all that long, of at most kPagedChunkMax keys.
// Sequences that are shorter get fewer splits of the same length, so that
// blocks are alike (equal counts of unequal splits left CUs idle a quarter of
// the time where lengths are ragged); but where a window hides most of what
// max_seen counts, what is seen is divided by the count. Blocks a CU at 6 / 12 /
// 32, us: 16 sequences x 10 heads of up to 4096 keys 53 / 49 / 51; 2 x 8 heads
// of up to 131071 171 / 171 / 184; 24 x 10 windowed 27 / 28 / 32. At most 2048 /
// 512 / 256 keys: 128 x 2 heads of up to 16384 keys 132 / 119 / 127.
inline PagedSplits pick_splits(size_t n_seqs, size_t kv_heads, int group, uint32_t max_seen, bool window, int cu_count) {
    const uint64_t rows = n_seqs * kv_heads * static_cast<uint64_t>((group + 15) / 16);
    const uint64_t unit = kPagedChunkUnit;
    const uint64_t even = (rows * max_seen + 12 * static_cast<uint64_t>(cu_count) - 1) / (12 * static_cast<uint64_t>(cu_count));
    const uint64_t keys = std::min<uint64_t>(std::max<uint64_t>((even + unit - 1) / unit, 1) * unit, kPagedChunkMax);
    const uint64_t count = std::max<uint64_t>((max_seen + keys - 1) / keys, 1);
    return PagedSplits{static_cast<int>(count), static_cast<uint32_t>(window ? unit : keys)};
}

// The row (of head_dim elements) of key `key` of sequence s and head hk.
FOCR_INDEX uint32_t row_of(const PagedTables& t, const PoolGeom& g, int s, uint32_t hk, uint32_t key) {
    const uint32_t page = t.tables[static_cast<size_t>(s) * t.max_pages + (key >> g.page_shift)];
    if (page >= g.n_pages) return kBadRow;
    return ((page * g.kv_heads + hk) << g.page_shift) + (key & ((1u << g.page_shift) - 1u));
}

struct Cut {
    uint32_t n, lo, hi, want;  // of the slots [lo, hi) the `want` heaviest stay, and all outside
    bool none, whole;
};

FOCR_INDEX Cut cut_of(const PagedEvict& a, int s) {
    Cut c{};
    const uint32_t len = a.t.lens[s];
    c.none = len == kPagedNone;
    if (c.none) return c;
    c.n = umin32(len, a.t.max_len);
    c.whole = c.n <= a.budget;
    c.lo = umin32(a.sinks, c.n);
    c.hi = c.n - umin32(a.recent, c.n - c.lo);
    c.want = c.whole ? c.hi - c.lo : a.budget - c.lo - (c.n - c.hi);
    return c;
}

}  // namespace
}  // namespace focr
