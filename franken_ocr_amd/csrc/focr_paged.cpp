// focr_paged.cpp — the C ABI of the paged key-value cache (write, attention,
// step, eviction) and of beam search (selection, reordering of the states).
// Argument checks on the host; with check = 1 also of what the device arrays
// hold, before anything is launched that reads or writes by it.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdarg>
#include <cstdio>
#include <limits>
#include <memory>
#include <mutex>
#include <new>
#include <string>

#include "focr_internal.hpp"

using namespace focr;

namespace {

std::string fmt(const char* f, ...) {
    char buf[512];
    va_list ap;
    va_start(ap, f);
    vsnprintf(buf, sizeof(buf), f, ap);
    va_end(ap);
    return buf;
}

// A C entry: the context's lock and device, and no exception past it.
template <typename F>
int32_t entry(focr_hip_ctx* ctx, F body) noexcept {
    try {
        if (!ctx) return fail(FOCR_HIP_E_BAD_HANDLE, "null focr_hip_ctx");
        std::lock_guard<std::mutex> lock(ctx->mu);
        clear_error();
        FOCR_HIP_TRY(ctx->bind(), "hipSetDevice");
        return body();
    } catch (const std::exception&) {
        return FOCR_HIP_E_OOM;
    }
}

constexpr size_t kMaxLen = size_t(1) << 26;  // keeps every grid within 2^32 threads
constexpr size_t kI32Max = static_cast<size_t>(std::numeric_limits<int32_t>::max());

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

bool overlap(const void* a, const void* b, size_t a_bytes, size_t b_bytes) {
    const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
    return x < y ? y - x < a_bytes : x - y < b_bytes;
}

// Whether two caches' pools have memory in common.
bool overlap(const focr_hip_paged* a, const focr_hip_paged* b) {
    const size_t na = a->n_pages * a->page_bytes(), nb = b->n_pages * b->page_bytes();
    return overlap(a->k, b->k, na, nb) || overlap(a->k, b->v, na, nb) || overlap(a->v, b->k, na, nb) || overlap(a->v, b->v, na, nb);
}

// Status of a scratch request that came back empty: out of memory, or a capture that cannot allocate.
int32_t no_scratch(focr_hip_ctx* ctx) { return ctx->captures() ? FOCR_HIP_E_STATE : FOCR_HIP_E_OOM; }

int32_t cache_ok(const char* who, const focr_hip_ctx* ctx, const focr_hip_paged* c) {
    if (!c) return fail(FOCR_HIP_E_BAD_HANDLE, fmt("%s: null paged cache", who));
    if (c->device != ctx->device)
        return fail(FOCR_HIP_E_ARG, fmt("%s: the cache is on device %d, the context on %d", who, c->device, ctx->device));
    return FOCR_HIP_OK;
}

int32_t tables_ok(const char* who, const focr_hip_paged* c, const uint32_t* tables, const uint32_t* lens, size_t n_seqs,
                  size_t max_pages, size_t max_len, PagedTables* t) {
    if (!tables || !lens) return fail(FOCR_HIP_E_ARG, fmt("%s: null device pointer", who));
    if (n_seqs > 65535) return fail(FOCR_HIP_E_SHAPE, fmt("%s: n_seqs %zu exceeds the gfx950 tier limit of 65535", who, n_seqs));
    if (max_pages == 0 || max_pages > (kI32Max >> c->page_shift))
        return fail(FOCR_HIP_E_SHAPE, fmt("%s: max_pages %zu is outside 1 .. %zu", who, max_pages, kI32Max >> c->page_shift));
    if (max_len > (max_pages << c->page_shift))
        return fail(FOCR_HIP_E_SHAPE, fmt("%s: max_len %zu exceeds max_pages * page_size %zu", who, max_len,
                                          max_pages << c->page_shift));
    if (max_len > kMaxLen)
        return fail(FOCR_HIP_E_SHAPE, fmt("%s: max_len %zu exceeds the gfx950 tier limit of %zu", who, max_len, kMaxLen));
    *t = PagedTables{tables, lens, static_cast<int>(n_seqs), max_pages, static_cast<uint32_t>(max_len)};
    return FOCR_HIP_OK;
}

// The checks on the device: one word, the first fault or all ones.
struct Check {
    focr_hip_ctx* ctx;
    unsigned long long* err = nullptr;
    int32_t begin(const char* who) {
        if (ctx->captures()) return fail(FOCR_HIP_E_STATE, fmt("%s: check = 1 waits for the stream and cannot be captured", who));
        err = static_cast<unsigned long long*>(ctx->scratch_get(kScrCheck, sizeof(*err)));
        if (!err) return FOCR_HIP_E_OOM;
        const unsigned long long none = ~0ull;
        FOCR_HIP_TRY(hipMemcpyAsync(err, &none, sizeof(none), hipMemcpyHostToDevice, ctx->stream), "H2D check");
        FOCR_HIP_TRY(hipStreamSynchronize(ctx->stream), "hipStreamSynchronize");
        return FOCR_HIP_OK;
    }
    int32_t end(const char* who, const char* row_name) {
        unsigned long long e = 0;
        FOCR_HIP_TRY(hipMemcpyAsync(&e, err, sizeof(e), hipMemcpyDeviceToHost, ctx->stream), "D2H check");
        FOCR_HIP_TRY(hipStreamSynchronize(ctx->stream), "hipStreamSynchronize");
        if (e == ~0ull) return FOCR_HIP_OK;
        const unsigned long long row = e >> 8;
        const auto say = [&](int32_t status, const char* what) {
            return fail(status, fmt("%s: %s %llu: %s", who, row_name, row, what));
        };
        switch (static_cast<int>(e & 255u)) {
            case kFaultLen: return say(FOCR_HIP_E_STATE, "its length is more than the tables (or max_len) hold");
            case kFaultPage: return say(FOCR_HIP_E_SHAPE, "its table names a page that the cache does not have");
            case kFaultSeq: return say(FOCR_HIP_E_SHAPE, "its sequence is not below n_seqs");
            case kFaultDstPage: return say(FOCR_HIP_E_SHAPE, "its dst_tables name a page that the cache does not have");
            case kFaultDstShared:
                return say(FOCR_HIP_E_SHAPE, "its dst_tables name a page that is read, or written twice");
            case kFaultParent: return say(FOCR_HIP_E_SHAPE, "its parent is not below beams");
            case kFaultGroupLen: return say(FOCR_HIP_E_STATE, "its length is not its group's");
            case kFaultTail: return say(FOCR_HIP_E_STATE, "its page in progress is another beam's too");
            default: return say(FOCR_HIP_E_STATE, "its history is full");
        }
    }
};

// The attention's workspace in one scratch slot; seen_most: keys that a row sees at most.
int32_t carve(focr_hip_ctx* ctx, const char* who, const focr_hip_paged* c, PagedAttend* a, bool scores, size_t seen_most) {
    const size_t n = a->t.n_seqs, heads = c->n_kv_heads * a->group, parts = n * heads * a->nsplit;
    const size_t seen = (n * sizeof(uint4) + 255) & ~size_t(255);
    const size_t acc = (parts * c->head_dim * sizeof(float) + 255) & ~size_t(255);
    const size_t ml = (parts * sizeof(float2) + 255) & ~size_t(255);
    a->score_ld = scores ? seen_most : 0;
    char* p = static_cast<char*>(
        ctx->scratch_get_capturable(kScrPaged, seen + acc + ml + n * heads * a->score_ld * sizeof(float), who));
    if (!p) return no_scratch(ctx);
    a->seen = reinterpret_cast<uint4*>(p);
    a->part_acc = reinterpret_cast<float*>(p + seen);
    a->part_ml = reinterpret_cast<float2*>(p + seen + acc);
    a->scores = scores ? reinterpret_cast<float*>(p + seen + acc + ml) : nullptr;
    return FOCR_HIP_OK;
}

int32_t attend(focr_hip_ctx* ctx, const char* who, const focr_hip_paged* c, const float* q, size_t ldq, size_t n_heads,
               const float* k_steps, const float* v_steps, size_t ldkv, bool step, const uint32_t* tables, size_t n_seqs,
               size_t max_pages, uint32_t* lens, size_t max_len, const uint32_t* prefix, size_t window, float scale,
               float* out, size_t ldo, float* weights, size_t ldw, bool advance, int32_t check) {
    int32_t st = cache_ok(who, ctx, c);
    if (st) return st;
    if (n_seqs == 0) return FOCR_HIP_OK;
    PagedAttend a{};
    if ((st = tables_ok(who, c, tables, lens, n_seqs, max_pages, max_len, &a.t))) return st;
    if (!q || !out || (step && (!k_steps || !v_steps))) return fail(FOCR_HIP_E_ARG, fmt("%s: null device pointer", who));
    if (n_heads == 0 || n_heads % c->n_kv_heads || n_heads / c->n_kv_heads > 64)
        return fail(FOCR_HIP_E_SHAPE, fmt("%s: n_heads %zu is not 1 .. 64 times n_kv_heads %zu", who, n_heads, c->n_kv_heads));
    if (n_heads > 65535) return fail(FOCR_HIP_E_SHAPE, fmt("%s: n_heads %zu exceeds the gfx950 tier limit", who, n_heads));
    if (ldq < n_heads * c->head_dim || ldo < n_heads * c->head_dim || (step && ldkv < c->n_kv_heads * c->head_dim))
        return fail(FOCR_HIP_E_SHAPE, fmt("%s: a row stride is shorter than the row", who));
    // the join's grid: a block of up to 1024 threads to a head, and to 512 keys of a key head
    if (weights && c->n_kv_heads * (max_len / 512 + 65) > (size_t(1) << 22) - 1)
        return fail(FOCR_HIP_E_SHAPE, fmt("%s: max_len %zu of %zu key heads exceeds the gfx950 tier limit with weights", who, max_len,
                                          c->n_kv_heads));
    if (weights && ldw < max_len) return fail(FOCR_HIP_E_SHAPE, fmt("%s: ldw %zu is less than max_len %zu", who, ldw, max_len));
    if (step && max_len == 0) return fail(FOCR_HIP_E_SHAPE, fmt("%s: max_len is 0", who));
    if (!(scale >= 0.0f) || std::isinf(scale)) return fail(FOCR_HIP_E_ARG, fmt("%s: scale is not a positive number", who));
    a.prefix = prefix;
    a.window = static_cast<uint32_t>(std::min<size_t>(window, 0xFFFFFFFEu));
    a.q = q;
    a.ldq = ldq;
    a.group = static_cast<int>(n_heads / c->n_kv_heads);
    a.scale = scale == 0.0f ? 1.0f / std::sqrt(static_cast<float>(c->head_dim)) : scale;
    a.k_steps = step ? k_steps : nullptr;
    a.v_steps = v_steps;
    a.ldkv = ldkv;
    a.lens_advance = advance ? lens : nullptr;
    a.out = out;
    a.ldo = ldo;
    a.weights = weights;
    a.ldw = ldw;
    const size_t seen = window && !prefix ? std::min(max_len, window) : max_len;
    const PagedSplits splits = paged_pick_splits(n_seqs, c->n_kv_heads, a.group, static_cast<uint32_t>(seen), window != 0,
                                                 ctx->cu_count);
    a.nsplit = splits.count;
    a.split_least = splits.least;
    if (check) {
        Check k{ctx};
        if ((st = k.begin(who))) return st;
        FOCR_HIP_TRY(launch_paged_check(ctx->stream, c, a.t, step ? 1 : 0, prefix, a.window, k.err), "check launch");
        if ((st = k.end(who, "sequence"))) return st;
    }
    if ((st = carve(ctx, who, c, &a, weights != nullptr, seen))) return st;
    FOCR_HIP_TRY(launch_paged_attend(ctx->stream, c, a, ctx), "paged attention launch");
    return FOCR_HIP_OK;
}

}  // namespace

extern "C" {

int32_t focr_hip_paged_create(focr_hip_ctx* ctx, size_t n_pages, size_t page_size, size_t n_kv_heads, size_t head_dim,
                              int32_t dtype, void* k_pool, void* v_pool, focr_hip_paged** out) {
    return entry(ctx, [&]() -> int32_t {
        if (!out) return fail(FOCR_HIP_E_ARG, "paged_create: null out");
        *out = nullptr;
        if (dtype != FOCR_HIP_DT_F32 && dtype != FOCR_HIP_DT_F16 && dtype != FOCR_HIP_DT_BF16)
            return fail(FOCR_HIP_E_ARG, fmt("paged_create: dtype %d is not F32, F16 or BF16", dtype));
        if (head_dim != 64 && head_dim != 128 && head_dim != 256)
            return fail(FOCR_HIP_E_SHAPE, fmt("paged_create: head_dim %zu is not 64, 128 or 256", head_dim));
        if (page_size == 0 || page_size > 1024 || (page_size & (page_size - 1)))
            return fail(FOCR_HIP_E_SHAPE, fmt("paged_create: page_size %zu is not a power of two up to 1024", page_size));
        if (n_pages == 0 || n_kv_heads == 0 || n_kv_heads > 1024)
            return fail(FOCR_HIP_E_SHAPE, "paged_create: n_pages and n_kv_heads (at most 1024) must be positive");
        // rows are numbered in 32 bits, all ones meaning none
        if (n_pages > 0xFFFFFFFEull / (page_size * n_kv_heads))
            return fail(FOCR_HIP_E_SHAPE, "paged_create: n_pages * n_kv_heads * page_size exceeds 2^32 - 2");
        if (!k_pool != !v_pool) return fail(FOCR_HIP_E_ARG, "paged_create: one pool of two given");
        if (!aligned16(k_pool) || !aligned16(v_pool))
            return fail(FOCR_HIP_E_ARG, "paged_create: the pools must be 16-byte aligned");
        std::unique_ptr<focr_hip_paged> c(new focr_hip_paged());
        c->device = ctx->device;
        c->n_pages = n_pages;
        c->n_kv_heads = n_kv_heads;
        c->head_dim = head_dim;
        while ((size_t(1) << c->page_shift) < page_size) ++c->page_shift;
        c->dtype = dtype;
        c->k = k_pool;
        c->v = v_pool;
        const size_t bytes = n_pages * c->page_bytes();
        if (k_pool && overlap(k_pool, v_pool, bytes, bytes)) return fail(FOCR_HIP_E_ARG, "paged_create: the pools overlap");
        if (!k_pool) {
            FOCR_HIP_TRY(hipMalloc(&c->k, bytes), "hipMalloc paged K");
            hipError_t e = hipMalloc(&c->v, bytes);
            if (e == hipSuccess) e = hipMemsetAsync(c->k, 0, bytes, ctx->stream);
            if (e == hipSuccess) e = hipMemsetAsync(c->v, 0, bytes, ctx->stream);
            if (e == hipSuccess) e = hipStreamSynchronize(ctx->stream);
            if (e != hipSuccess) {
                hipFree(c->k);
                if (c->v) hipFree(c->v);
                return hip_fail(e, "paged pools");
            }
            c->owned = true;
        }
        *out = c.release();
        return FOCR_HIP_OK;
    });
}

int32_t focr_hip_paged_free(focr_hip_paged* c) {
    if (!c) return FOCR_HIP_OK;
    if (c->owned) {
        hipSetDevice(c->device);
        hipDeviceSynchronize();  // calls of any context may be using them
        hipFree(c->k);
        hipFree(c->v);
    }
    delete c;
    return FOCR_HIP_OK;
}

int32_t focr_hip_paged_regions(const focr_hip_paged* c, void** k_pool, void** v_pool) {
    if (!c) return fail(FOCR_HIP_E_BAD_HANDLE, "null paged cache");
    if (k_pool) *k_pool = c->k;
    if (v_pool) *v_pool = c->v;
    return FOCR_HIP_OK;
}

int32_t focr_hip_paged_write(focr_hip_ctx* ctx, focr_hip_paged* c, const float* k, const float* v, size_t ld, size_t rows,
                             const uint32_t* seq, const uint32_t* pos, const uint32_t* tables, size_t n_seqs,
                             size_t max_pages, int32_t check) {
    return entry(ctx, [&]() -> int32_t {
        const char* who = "paged_write";
        int32_t st = cache_ok(who, ctx, c);
        if (st) return st;
        if (rows == 0) return FOCR_HIP_OK;
        PagedTables t;
        if ((st = tables_ok(who, c, tables, pos, n_seqs, max_pages, 0, &t))) return st;
        if (!k || !v) return fail(FOCR_HIP_E_ARG, "paged_write: null device pointer");
        if (ld < c->n_kv_heads * c->head_dim) return fail(FOCR_HIP_E_SHAPE, "paged_write: a row stride is shorter than the row");
        if (!seq && rows > n_seqs)
            return fail(FOCR_HIP_E_SHAPE, fmt("paged_write: %zu rows for %zu sequences", rows, n_seqs));
        if (rows > kI32Max / (c->n_kv_heads * c->head_dim * c->esize() / 16))
            return fail(FOCR_HIP_E_SHAPE, "paged_write: rows exceed the gfx950 tier limit");
        if (check) {
            Check kk{ctx};
            if ((st = kk.begin(who))) return st;
            FOCR_HIP_TRY(launch_paged_check_rows(ctx->stream, c, rows, seq, pos, tables, t.n_seqs, max_pages, kk.err),
                         "check launch");
            if ((st = kk.end(who, "row"))) return st;
        }
        ProfScope ps(ctx, "paged_write");
        FOCR_HIP_TRY(launch_paged_write(ctx->stream, c, k, v, ld, rows, seq, pos, tables, t.n_seqs, max_pages),
                     "paged write launch");
        return FOCR_HIP_OK;
    });
}

int32_t focr_hip_paged_attention(focr_hip_ctx* ctx, const focr_hip_paged* c, const float* q, size_t ldq, size_t n_heads,
                                 const uint32_t* tables, size_t n_seqs, size_t max_pages, const uint32_t* lens,
                                 size_t max_len, const uint32_t* prefix, size_t window, float scale, float* out,
                                 size_t ldo, float* weights, size_t ldw, int32_t check) {
    return entry(ctx, [&]() -> int32_t {
        return attend(ctx, "paged_attention", c, q, ldq, n_heads, nullptr, nullptr, 0, false, tables, n_seqs, max_pages,
                      const_cast<uint32_t*>(lens), max_len, prefix, window, scale, out, ldo, weights, ldw, false, check);
    });
}

int32_t focr_hip_paged_step(focr_hip_ctx* ctx, focr_hip_paged* c, const float* q, size_t ldq, size_t n_heads,
                            const float* k_steps, const float* v_steps, size_t ldkv, const uint32_t* tables,
                            size_t n_seqs, size_t max_pages, uint32_t* lens, size_t max_len, const uint32_t* prefix,
                            size_t window, float scale, float* out, size_t ldo, float* weights, size_t ldw,
                            int32_t advance, int32_t check) {
    return entry(ctx, [&]() -> int32_t {
        return attend(ctx, "paged_step", c, q, ldq, n_heads, k_steps, v_steps, ldkv, true, tables, n_seqs, max_pages, lens,
                      max_len, prefix, window, scale, out, ldo, weights, ldw, advance != 0, check);
    });
}

int32_t focr_hip_paged_evict(focr_hip_ctx* ctx, focr_hip_paged* c, const uint32_t* tables, size_t n_seqs,
                             size_t max_pages, const uint32_t* lens, size_t max_len, const float* weights, size_t ldw,
                             size_t budget, size_t sinks, size_t recent, const uint32_t* dst_tables,
                             size_t dst_max_pages, uint32_t* dst_lens, float* dst_weights, size_t dst_ldw,
                             uint32_t* kept, int32_t check) {
    return entry(ctx, [&]() -> int32_t {
        const char* who = "paged_evict";
        int32_t st = cache_ok(who, ctx, c);
        if (st) return st;
        if (n_seqs == 0) return FOCR_HIP_OK;
        PagedEvict a{};
        if ((st = tables_ok(who, c, tables, lens, n_seqs, max_pages, max_len, &a.t))) return st;
        if (!weights || !dst_tables || !dst_lens || !dst_weights) return fail(FOCR_HIP_E_ARG, "paged_evict: null device pointer");
        if (dst_weights == weights || dst_tables == tables)
            return fail(FOCR_HIP_E_ARG, "paged_evict: what stays goes to other pages and weights than it comes from");
        if (budget == 0 || budget > kI32Max) return fail(FOCR_HIP_E_SHAPE, fmt("paged_evict: budget %zu is outside 1 .. 2^31 - 1", budget));
        if (sinks > budget || recent > budget - sinks)
            return fail(FOCR_HIP_E_SHAPE, fmt("paged_evict: sinks %zu and recent %zu exceed the budget %zu", sinks, recent, budget));
        const size_t most = std::min(budget, max_len);
        if (dst_max_pages > (kI32Max >> c->page_shift) || (dst_max_pages << c->page_shift) < most)
            return fail(FOCR_HIP_E_SHAPE, fmt("paged_evict: dst_max_pages %zu do not hold %zu slots", dst_max_pages, most));
        if (ldw < max_len || dst_ldw < most) return fail(FOCR_HIP_E_SHAPE, "paged_evict: a row of weights is shorter than its slots");
        a.weights = weights;
        a.ldw = ldw;
        a.budget = static_cast<uint32_t>(budget);
        a.sinks = static_cast<uint32_t>(sinks);
        a.recent = static_cast<uint32_t>(recent);
        a.dst_tables = dst_tables;
        a.dst_max_pages = dst_max_pages;
        a.dst_lens = dst_lens;
        a.dst_weights = dst_weights;
        a.dst_ldw = dst_ldw;
        if (check) {
            Check k{ctx};
            if ((st = k.begin(who))) return st;
            FOCR_HIP_TRY(launch_paged_check(ctx->stream, c, a.t, 0, nullptr, 0, k.err), "check launch");
            if ((st = k.end(who, "sequence"))) return st;
            uint32_t* marks = static_cast<uint32_t*>(ctx->scratch_get(kScrEvict, (c->n_pages + 31) / 32 * 4));
            if (!marks) return FOCR_HIP_E_OOM;
            FOCR_HIP_TRY(launch_paged_check_dst(ctx->stream, c, a, marks, k.err), "check launch");
            if ((st = k.end(who, "sequence"))) return st;
        }
        const size_t hist = paged_evict_hist_words(n_seqs * c->n_kv_heads, a.t.max_len, ctx->cu_count);
        if (!kept) a.budget = static_cast<uint32_t>(std::max<size_t>(most, 1));  // more than max_len keeps no more
        const size_t words = hist + (kept ? 0 : n_seqs * c->n_kv_heads * a.budget);
        a.kept = kept;
        if (words) {
            uint32_t* p = static_cast<uint32_t*>(ctx->scratch_get_capturable(kScrEvict, words * sizeof(uint32_t), who));
            if (!p) return no_scratch(ctx);
            a.hist = hist ? p : nullptr;
            if (!kept) a.kept = p + hist;
        }
        FOCR_HIP_TRY(launch_paged_evict(ctx->stream, c, a, ctx), "paged eviction launch");
        return FOCR_HIP_OK;
    });
}

int32_t focr_hip_beam_select(focr_hip_ctx* ctx, const float* logits, size_t ld, size_t groups, size_t beams, size_t vocab,
                             const float* scores, const uint8_t* done, uint32_t eos_token_id, const uint32_t* history,
                             size_t history_cap, const uint32_t* history_len, size_t ngram_size, size_t window,
                             const uint32_t* whitelist, size_t n_whitelist, uint32_t* parents, uint32_t* tokens,
                             float* new_scores, uint8_t* new_done, int32_t check) {
    return entry(ctx, [&]() -> int32_t {
        const char* who = "beam_select";
        if (groups == 0) return FOCR_HIP_OK;
        if (!logits || !scores || !parents || !tokens || !new_scores) return fail(FOCR_HIP_E_ARG, "beam_select: null device pointer");
        if (beams == 0 || beams > static_cast<size_t>(kBeamMax))
            return fail(FOCR_HIP_E_SHAPE, fmt("beam_select: beams %zu is outside 1 .. %d", beams, kBeamMax));
        if (vocab == 0) return fail(FOCR_HIP_E_SHAPE, "sampler::argmax_row: empty logits row");
        if (ld < vocab) return fail(FOCR_HIP_E_SHAPE, "beam_select: a row stride is shorter than the row");
        if (vocab > (size_t(1) << 19) || groups > 65535 / beams)
            return fail(FOCR_HIP_E_SHAPE, "beam_select: shape exceeds the gfx950 tier limit (2^19 tokens, 65535 rows)");
        if (history_cap > kI32Max || ngram_size > kI32Max || window > kI32Max || n_whitelist > 4096)
            return fail(FOCR_HIP_E_SHAPE, "beam_select: history_cap / ngram_size / window / whitelist exceed the gfx950 tier limits");
        if (ngram_size && (!history || !history_len || history_cap == 0))
            return fail(FOCR_HIP_E_ARG, "beam_select: the no-repeat-ngram ban needs history, history_len and a positive history_cap");
        if (n_whitelist && !whitelist) return fail(FOCR_HIP_E_ARG, "beam_select: null whitelist");
        const size_t rows = groups * beams;
        BeamSelect a{};
        a.logits = logits;
        a.ld = ld;
        a.groups = static_cast<int>(groups);
        a.beams = static_cast<int>(beams);
        a.vocab = static_cast<int>(vocab);
        a.scores = scores;
        a.done = done;
        a.eos = eos_token_id;
        a.parents = parents;
        a.tokens = tokens;
        a.new_scores = new_scores;
        a.new_done = new_done;
        a.nparts = beam_parts(a.vocab);
        a.part = ctx->scratch_get_capturable(kScrBeam, beam_part_bytes(static_cast<int>(rows), a.beams, a.nparts), who);
        if (!a.part) return no_scratch(ctx);
        // what the ban looks at; a thread a token finds it inside the scan (check = 1 needs the flags of the launch before)
        const size_t span = window ? std::min(window, history_cap) : history_cap;
        if (ngram_size && span <= static_cast<size_t>(kBeamBanSpan) && !check) {
            a.history = history;
            a.history_len = history_len;
            a.cap = static_cast<int>(history_cap);
            a.ngram = static_cast<int>(ngram_size);
            a.window = static_cast<int>(window);
            a.whitelist = whitelist;
            a.n_white = static_cast<int>(n_whitelist);
        } else if (ngram_size) {
            const size_t words = (vocab + 31) / 32;
            SamplerArgs p{};
            p.history = history;
            p.history_len = const_cast<uint32_t*>(history_len);
            p.cap = static_cast<int>(history_cap);
            p.ngram = static_cast<int>(ngram_size);
            p.window = static_cast<int>(window);
            p.whitelist = whitelist;
            p.n_white = static_cast<int>(n_whitelist);
            p.vocab = a.vocab;
            p.ban_words = static_cast<int>(words);
            p.ban_bits = static_cast<uint32_t*>(ctx->scratch_get_capturable(kScrBeamBan, rows * words * sizeof(uint32_t), who));
            p.err = static_cast<int*>(ctx->scratch_get_capturable(kScrBeamFlag, rows * sizeof(int), who));
            if (!p.ban_bits || !p.err) return no_scratch(ctx);
            if (check && ctx->captures())
                return fail(FOCR_HIP_E_STATE, "beam_select: check = 1 waits for the stream and cannot be captured");
            ProfScope ps(ctx, "sampler_prep");
            FOCR_HIP_TRY(launch_sampler_prep(ctx->stream, static_cast<int>(rows), nullptr, 0, nullptr, nullptr, p),
                         "sampler_prep launch");
            if (check) {
                std::unique_ptr<int[]> flags(new int[rows]);
                FOCR_HIP_TRY(hipMemcpyAsync(flags.get(), p.err, rows * sizeof(int), hipMemcpyDeviceToHost, ctx->stream),
                             "D2H sampler flags");
                FOCR_HIP_TRY(hipStreamSynchronize(ctx->stream), "hipStreamSynchronize");
                for (size_t r = 0; r < rows; ++r)
                    if (flags[r])
                        return fail(FOCR_HIP_E_SHAPE, fmt("sampler: history_len of row %zu exceeds history_cap %zu", r, history_cap));
            }
            a.ban_bits = p.ban_bits;
            a.ban_words = p.ban_words;
        }
        FOCR_HIP_TRY(launch_beam_select(ctx->stream, a, ctx), "beam selection launch");
        return FOCR_HIP_OK;
    });
}

int32_t focr_hip_beam_reorder(focr_hip_ctx* ctx, size_t groups, size_t beams, const uint32_t* parents,
                              const uint32_t* tokens, uint32_t* history, size_t history_cap, uint32_t* history_len,
                              int32_t advance, focr_hip_paged* const* caches, size_t n_caches, uint32_t* tables,
                              size_t max_pages, const uint32_t* lens, focr_hip_rswa* const* rings, size_t n_rings,
                              int32_t check) {
    return focr_hip_beam_reorder_weighted(ctx, groups, beams, parents, tokens, history, history_cap, history_len, advance,
                                          caches, n_caches, tables, max_pages, lens, nullptr, 0, rings, n_rings, check);
}

int32_t focr_hip_beam_reorder_weighted(focr_hip_ctx* ctx, size_t groups, size_t beams, const uint32_t* parents,
                                       const uint32_t* tokens, uint32_t* history, size_t history_cap,
                                       uint32_t* history_len, int32_t advance, focr_hip_paged* const* caches,
                                       size_t n_caches, uint32_t* tables, size_t max_pages, const uint32_t* lens,
                                       float* const* weights, size_t ldw, focr_hip_rswa* const* rings, size_t n_rings,
                                       int32_t check) {
    return entry(ctx, [&]() -> int32_t {
        const char* who = "beam_reorder";
        if (groups == 0) return FOCR_HIP_OK;
        if (!parents) return fail(FOCR_HIP_E_ARG, "beam_reorder: null device pointer");
        if (beams == 0 || beams > static_cast<size_t>(kBeamMax))
            return fail(FOCR_HIP_E_SHAPE, fmt("beam_reorder: beams %zu is outside 1 .. %d", beams, kBeamMax));
        if (groups > 65535 / beams) return fail(FOCR_HIP_E_SHAPE, "beam_reorder: more than 65535 rows");
        if (history && (!history_len || history_cap == 0 || history_cap > kI32Max))
            return fail(FOCR_HIP_E_ARG, "beam_reorder: a history needs history_len and a history_cap of 1 .. 2^31 - 1");
        if ((n_caches && !caches) || (n_rings && !rings)) return fail(FOCR_HIP_E_ARG, "beam_reorder: null handles");
        if (tables && !n_caches)
            return fail(FOCR_HIP_E_ARG, "beam_reorder: tables move with the caches that share them, and none is given");
        const size_t rows = groups * beams;
        int32_t st;
        BeamReorder a{};
        a.groups = static_cast<int>(groups);
        a.beams = static_cast<int>(beams);
        a.parents = parents;
        a.tokens = tokens;
        a.history = history;
        a.cap = history_cap;
        a.history_len = history_len;
        a.advance = advance != 0;
        for (size_t i = 0; i < n_caches; ++i) {
            if ((st = cache_ok(who, ctx, caches[i]))) return st;
            for (size_t j = 0; j < i; ++j)
                if (overlap(caches[i], caches[j]))
                    return fail(FOCR_HIP_E_ARG, fmt("beam_reorder: caches %zu and %zu are the same, or their pools overlap", j, i));
            if (caches[i]->page_shift != caches[0]->page_shift)
                return fail(FOCR_HIP_E_SHAPE, "beam_reorder: caches of different page sizes share no tables");
            if (!weights || !weights[i]) continue;
            if (ldw == 0 || ldw > kMaxLen)
                return fail(FOCR_HIP_E_SHAPE, fmt("beam_reorder: ldw %zu is outside 1 .. %zu", ldw, kMaxLen));
            for (size_t j = 0; j < i; ++j)
                if (weights[i] == weights[j])
                    return fail(FOCR_HIP_E_ARG, fmt("beam_reorder: the weights of caches %zu and %zu are the same", j, i));
        }
        if (n_caches) {
            PagedTables t;
            if ((st = tables_ok(who, caches[0], tables, lens, rows, max_pages, 0, &t))) return st;
            a.tables = tables;
            a.max_pages = max_pages;
            a.lens = lens;
            a.page_shift = caches[0]->page_shift;
            a.permute = 1;
        }
        uint32_t ring_rows = 0;
        for (size_t i = 0; i < n_rings; ++i) {
            const focr_hip_rswa* c = rings[i];
            if (!c) return fail(FOCR_HIP_E_BAD_HANDLE, "null rswa cache");
            for (size_t j = 0; j < i; ++j)
                if (rings[j] == c) return fail(FOCR_HIP_E_ARG, fmt("beam_reorder: rings %zu and %zu are the same", j, i));
            if (c->ctx->device != ctx->device) return fail(FOCR_HIP_E_ARG, "beam_reorder: a ring cache of another device");
            if (c->n_streams != rows)
                return fail(FOCR_HIP_E_SHAPE, fmt("beam_reorder: %zu streams for %zu rows", c->n_streams, rows));
            for (size_t s = 0; s < rows; ++s) {
                const size_t f = s / beams * beams;
                if (c->prefill_len[s] < 0) return fail(FOCR_HIP_E_STATE, "rswa: beam_reorder before record_prefill");
                if (c->prefill_len[s] != c->prefill_len[f] || c->ring_len[s] != c->ring_len[f] || c->ring_pos[s] != c->ring_pos[f])
                    return fail(FOCR_HIP_E_STATE, fmt("beam_reorder: stream %zu is not where its group is", s));
                ring_rows = std::max(ring_rows, c->ring_len[s]);
            }
        }
        // a graph's replays find the rings further on than the capture did: whole windows follow
        if (n_rings && ctx->captures()) ring_rows = kRingWindow;
        if (check) {
            Check k{ctx};
            if ((st = k.begin(who))) return st;
            FOCR_HIP_TRY(launch_beam_check(ctx->stream, a, k.err), "check launch");
            if ((st = k.end(who, "row"))) return st;
            for (size_t i = 0; i < n_caches; ++i) {
                const PagedTables t{tables, lens, static_cast<int>(rows), max_pages,
                                    static_cast<uint32_t>(max_pages << a.page_shift)};
                FOCR_HIP_TRY(launch_paged_check(ctx->stream, caches[i], t, 0, nullptr, 0, k.err), "check launch");
            }
            if (n_caches && (st = k.end(who, "row"))) return st;
        }
        ProfScope ps(ctx, "beam_reorder");
        if (weights)
            FOCR_HIP_TRY(launch_beam_weights(ctx->stream, a, caches, weights, n_caches, ldw), "beam weights launch");
        FOCR_HIP_TRY(launch_beam_reorder(ctx->stream, a, caches, n_caches, rings, n_rings, ring_rows), "beam reorder launch");
        return FOCR_HIP_OK;
    });
}

}  // extern "C"
