// k_beam.hip — one step of beam search over given logits, and the states of
// the chosen beams put where their slots are.
//
// Of a group's beams b with scores S_b and logits x_bv, the candidates are
//   c_bv = S_b + (x_bv - L_b),  L_b = log sum_v exp(x_bv),
// and the first W of the order (c descending, beam ascending, logit
// descending, token ascending) become the new beams. L and c are f64: an f32
// sum over 10^5 tokens would decide between beams by its rounding. Within a
// beam the order is the logits' own, so a chunk of a row keeps its W best by
// logit alone, and the beams meet only at the end.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "focr_internal.hpp"
#include "k_common.hpp"

namespace focr {
namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;
constexpr int kPer = 16;                // logits of a thread
constexpr int kChunk = kThreads * kPer;  // logits of a block
constexpr int kList = 256;               // candidates of a chunk that are sorted at once

// The chunks' results: max and f64 sum of exp(x - max) per chunk, and its W
// best keys (argmax_key order), descending, 0 where there are fewer.
struct Parts {
    double* sum;    // [rows][nparts]
    uint64_t* key;  // [rows][nparts][W]
    float* max;     // [rows][nparts]
};

__host__ __device__ inline Parts parts_of(void* p, int rows, int beams, int nparts) {
    Parts q;
    const size_t n = static_cast<size_t>(rows) * nparts;
    q.sum = static_cast<double*>(p);
    q.key = reinterpret_cast<uint64_t*>(q.sum + n);
    q.max = reinterpret_cast<float*>(q.key + n * beams);
    return q;
}

// exp(d) for d <= 0: d = n ln 2 + r with |r| <= ln 2 / 2, the Taylor series of
// exp(r) to r^10 (its rest is below 3e-13 of the value, n's multiple of the
// rounded ln 2 adds less), times 2^n. Below -700 as at -700, which adds
// nothing to a sum that is at least 1.
__device__ __forceinline__ double exp_below(double d) {
    d = fmax(d, -700.0);
    const double n = rint(d * 1.4426950408889634);
    const double r = fma(n, -0.6931471805599453, d);
    double p = 1.0 / 3628800.0;
    p = fma(p, r, 1.0 / 362880.0);
    p = fma(p, r, 1.0 / 40320.0);
    p = fma(p, r, 1.0 / 5040.0);
    p = fma(p, r, 1.0 / 720.0);
    p = fma(p, r, 1.0 / 120.0);
    p = fma(p, r, 1.0 / 24.0);
    p = fma(p, r, 1.0 / 6.0);
    p = fma(p, r, 0.5);
    p = fma(p, r, 1.0);
    p = fma(p, r, 1.0);
    return ldexp(p, static_cast<int>(n));
}

// What lanes of this wave wrote to LDS is there for its other lanes.
__device__ __forceinline__ void wave_lds_fence() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// A float's place in the order of floats, as a whole number (NaN: 0), -0 as +0.
__device__ __forceinline__ uint32_t float_order(float v) { return static_cast<uint32_t>(argmax_key(v, 0u) >> 32); }

// A number that at least W of a wave's lanes reach with theirs: the leading
// bits of the W-th greatest, a ballot a bit; 0 where fewer than W have one.
__device__ __forceinline__ uint32_t wave_bound(uint32_t mine, int W) {
    uint32_t bound = 0u;
#pragma unroll
    for (int bit = 31; bit >= 16; --bit) {
        const uint32_t t = bound | (1u << bit);
        if (__popcll(__ballot(mine >= t)) >= W) bound = t;
    }
    return bound;
}

// The no-repeat-ngram ban of the row's history (the sampler's: a position whose
// n - 1 tokens are the last n - 1 bans the token behind it) as bits of the chunk
// from token t0 on, by the scan's own blocks: a window of up to a thread a token
// lies in LDS. A launch that finds the ban beforehand takes 4 us and the wait
// here 1.6 to 3.2: a step of 1 x 4 beams 19.9 -> 16.8 us, of 8 x 8 103 and 104.
// Returns how many tokens the ban looked at.
__device__ __forceinline__ int ban_chunk(const BeamSelect& a, int row, uint32_t raw_len, int t0, uint32_t* s_seq, uint32_t* s_ban) {
    const int L = raw_len > static_cast<uint32_t>(a.cap) ? a.cap : static_cast<int>(raw_len);
    const int start = a.window != 0 && L > a.window ? L - a.window : 0;
    const int span = L - start, n = a.ngram;
    if (span < n) return 0;  // uniform
    const int i = threadIdx.x;
    if (i < kChunk / 32) s_ban[i] = 0u;
    if (i < span) s_seq[i] = a.history[static_cast<size_t>(row) * a.cap + start + i];
    __syncthreads();
    if (i < span - n + 1) {
        bool match = true;
        for (int j = 0; match && j < n - 1; j += 8) {  // eight at a time: one at a time waits for each pair in turn
            uint32_t differ = 0u;
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const int jj = min(j + k, n - 2);  // past the end: the last pair again
                differ |= s_seq[i + jj] ^ s_seq[span - (n - 1) + jj];
            }
            match = differ == 0u;
        }
        if (match) {
            const uint32_t banned = s_seq[i + n - 1], off = banned - static_cast<uint32_t>(t0);
            bool white = false;
            for (int j = 0; j < a.n_white; ++j) white |= a.whitelist[j] == banned;
            if (!white && off < static_cast<uint32_t>(kChunk)) atomicOr(&s_ban[off >> 5], 1u << (off & 31));
        }
    }
    __syncthreads();
    return span;
}

// Grid (chunk, row): one pass over the chunk's logits, held in registers. Its W
// best: at least W of a wave's lanes have a logit that reaches the wave's
// bound, so only logits that reach the greatest of the four waves' bounds can
// be among them. They are few; they are listed and each counts the greater
// ones. Where the list does not hold them (long runs of equal logits), the
// maximum is taken W times instead. 64 rows of 129280 logits for W = 8 take 16
// us (33 MB) with the ban found beforehand: issue of vector instructions, 595 a
// wave (a tenth of the rows done), the sixteen f64 exponentials nearly half of
// them. Taking the maximum W times took 36 us.
__global__ __launch_bounds__(kThreads) void beam_scan_kernel(BeamSelect a, Parts q) {
    __shared__ float s_max[kWaves];
    __shared__ double s_sum[kWaves];
    __shared__ uint32_t s_bound[kWaves];
    __shared__ uint64_t s_list[kList];
    __shared__ uint64_t s_key[2][kWaves];
    __shared__ int s_n;
    __shared__ uint32_t s_seq[kBeamBanSpan], s_ban[kChunk / 32];
    const int part = blockIdx.x;
    const int row = blockIdx.y;
    const uint32_t raw_len = a.ngram ? a.history_len[row] : 0u;
    if (a.done && a.done[row]) return;  // its one candidate needs no logits
    const int W = a.beams;
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const float* x = a.logits + static_cast<size_t>(row) * a.ld;
    const uint32_t* ban = a.ban_bits ? a.ban_bits + static_cast<size_t>(row) * a.ban_words : nullptr;
    const float none = __uint_as_float(0x7FC00000u);  // NaN: no logit
    float v[kPer];
    const int t0 = part * kChunk + static_cast<int>(threadIdx.x);
    if ((part + 1) * kChunk <= a.vocab) {  // uniform
#pragma unroll
        for (int i = 0; i < kPer; ++i) v[i] = x[t0 + i * kThreads];
    } else {
#pragma unroll
        for (int i = 0; i < kPer; ++i) v[i] = t0 + i * kThreads < a.vocab ? x[t0 + i * kThreads] : none;
    }
    // the wave's words of the ban, one a lane: word 2 i + h is that of the tokens of v[i] in half h of the wave
    uint32_t ban_word = 0u;
    if (a.ngram) {
        const int span = ban_chunk(a, row, raw_len, part * kChunk, s_seq, s_ban);
        if (span && lane < 2 * kPer) ban_word = s_ban[(lane >> 1) * (kThreads / 32) + wave * 2 + (lane & 1)];
    }
    if (ban && lane < 2 * kPer) {
        const int word = (part * kChunk + (lane >> 1) * kThreads + wave * 64 + (lane & 1) * 32) >> 5;
        if (word < a.ban_words) ban_word = ban[word];
    }
    if (threadIdx.x == 0) s_n = 0;
    float most = -INFINITY;
#pragma unroll
    for (int i = 0; i < kPer; ++i) most = fmaxf(most, v[i]);  // a NaN is skipped
    const float m = wave_max_f_full(most);
    // each wave sums relative to its own maximum, and they meet at the end; a
    // NaN's difference counts as -700, which adds nothing beside the maximum's 1
    double sum = 0.0;
    if (m > -INFINITY && m < INFINITY) {
        const double dm = static_cast<double>(m);
#pragma unroll
        for (int i = 0; i < kPer; ++i) sum += exp_below(static_cast<double>(v[i]) - dm);
    } else if (m == INFINITY) {
#pragma unroll
        for (int i = 0; i < kPer; ++i) sum += v[i] == m ? 1.0 : 0.0;
    }
    sum = wave_sum_d_full(sum);
    if (__any(ban_word != 0u)) {
        most = -INFINITY;
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            const uint32_t w = __shfl(ban_word, 2 * i + (lane >> 5), 64);
            v[i] = w >> (lane & 31) & 1u ? none : v[i];
            most = fmaxf(most, v[i]);
        }
    }
    // a lane without a logit above -inf counts as having none for the bound alone
    const uint32_t bound = wave_bound(most > -INFINITY ? float_order(most) : 0u, W);
    if (lane == 0) {
        s_max[wave] = m;
        s_sum[wave] = sum;
        s_bound[wave] = bound;
    }
    __syncthreads();
    const uint32_t top = max(max(s_bound[0], s_bound[1]), max(s_bound[2], s_bound[3]));
    const float least = top ? key_value(static_cast<uint64_t>(top) << 32) : -INFINITY;
    int n = 0;
    uint64_t in[kPer];
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        in[i] = __ballot(v[i] >= least);
        n += __popcll(in[i]);
    }
    int at = 0;
    if (n) {
        if (lane == 0) at = atomicAdd(&s_n, n);
        at = __builtin_amdgcn_readfirstlane(at);
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            if (in[i]) {
                const int to = at + __popcll(in[i] & ((1ull << lane) - 1));
                if ((in[i] >> lane & 1u) && to < kList) s_list[to] = argmax_key(v[i], static_cast<uint32_t>(t0 + i * kThreads));
                at += __popcll(in[i]);
            }
        }
    }
    __syncthreads();
    n = s_n;
    const size_t to = static_cast<size_t>(row) * a.nparts + part;
    uint64_t* out = q.key + to * W;
    if (n <= kList) {
        for (int j = threadIdx.x; j < n; j += kThreads) {
            const uint64_t k = s_list[j];
            int place = 0;
#pragma unroll 8
            for (int o = 0; o < n; ++o) place += s_list[o] > k ? 1 : 0;
            if (place < W) out[place] = k;
        }
        for (int j = n + threadIdx.x; j < W; j += kThreads) out[j] = 0ull;
    } else {
        uint64_t key[kPer], best = 0ull;
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            key[i] = argmax_key(v[i], static_cast<uint32_t>(t0 + i * kThreads));
            best = umax64(best, key[i]);
        }
        for (int w = 0; w < W; ++w) {
            const uint64_t mine = wave_max_u64_full(best);
            if (lane == 0) s_key[w & 1][wave] = mine;
            __syncthreads();
            const uint64_t* k = s_key[w & 1];
            const uint64_t now = umax64(umax64(k[0], k[1]), umax64(k[2], k[3]));
            if (threadIdx.x == 0) out[w] = now;
            if (now == best) {
                best = 0ull;
#pragma unroll
                for (int i = 0; i < kPer; ++i) {
                    if (key[i] == now) key[i] = 0ull;
                    best = umax64(best, key[i]);
                }
            }
        }
    }
    if (wave == kWaves - 1) {  // a lane a wave's sum
        const float mx = fmaxf(fmaxf(s_max[0], s_max[1]), fmaxf(s_max[2], s_max[3]));
        const float mw = s_max[lane & (kWaves - 1)];
        const double d = mw == mx ? 0.0 : static_cast<double>(mw) - static_cast<double>(mx);
        const double mine = mw > -INFINITY ? s_sum[lane & (kWaves - 1)] * exp_below(d) : 0.0;
        const double total = (readlane_d(mine, 0) + readlane_d(mine, 1)) + (readlane_d(mine, 2) + readlane_d(mine, 3));
        if (lane == 0) {
            q.max[to] = mx;
            q.sum[to] = total;
        }
    }
}

// Grid (group). A wave takes a row at a time: L from the chunks, and the W
// best keys by merging the chunks' lists, which lie in LDS (a lane has the
// heads of its lists; the greatest goes and its list moves up). Then a thread
// has a candidate, whose place among the group's is the number before it in
// its own beam's list and, by bisection, in the others'. One chain of latencies:
// 9 us for eight groups of eight beams, 6 us for one of four.
__global__ __launch_bounds__(1024) void beam_pick_kernel(BeamSelect a, Parts q, int waves) {
    extern __shared__ uint64_t s_keys[];  // [waves][nparts * W]
    __shared__ double s_c[kBeamMax * kBeamMax];
    __shared__ uint64_t s_k[kBeamMax * kBeamMax];
    __shared__ int s_n[kBeamMax];  // candidates of a beam
    __shared__ uint8_t s_done[kBeamMax];
    const int W = a.beams;
    const int t = threadIdx.x;
    const int wave = t >> 6, lane = t & 63;
    const size_t row0 = static_cast<size_t>(blockIdx.x) * W;
    if (t < W) s_done[t] = a.done ? a.done[row0 + t] : 0;
    for (int i = t; i < W * W; i += blockDim.x) s_k[i] = 0ull;
    __syncthreads();
    for (int b = wave; wave < waves && b < W; b += waves) {
        const size_t at = (row0 + b) * a.nparts;
        uint64_t* keys = s_keys + static_cast<size_t>(wave) * a.nparts * W;
        constexpr int kHeads = kBeamParts / 64;
        // everything the row needs is requested before anything of it is used
        const double score = static_cast<double>(a.scores[row0 + b]);
        float mp[kHeads];
        double sp[kHeads];
#pragma unroll
        for (int h = 0; h < kHeads; ++h) {
            const int p = lane + 64 * h;
            mp[h] = p < a.nparts ? q.max[at + p] : -INFINITY;
            sp[h] = p < a.nparts ? q.sum[at + p] : 0.0;
        }
#pragma unroll 4
        for (int i = lane; i < a.nparts * W; i += 64) keys[i] = q.key[at * W + i];
        if (s_done[b]) {
            if (lane == 0) {
                s_k[b * W] = (1ull << 32) | (0xFFFFFFFFull - a.eos);
                s_c[b * W] = score == score ? score : -INFINITY;
                s_n[b] = 1;
            }
            continue;
        }
        float m = -INFINITY;
#pragma unroll
        for (int h = 0; h < kHeads; ++h) m = fmaxf(m, mp[h]);
        m = wave_max_f_full(m);
        double sum = 0.0;
#pragma unroll
        for (int h = 0; h < kHeads; ++h) {
            const double d = mp[h] == m ? 0.0 : static_cast<double>(mp[h]) - static_cast<double>(m);
            sum += mp[h] > -INFINITY ? sp[h] * exp_below(d) : 0.0;
        }
        sum = wave_sum_d_full(sum);
        const double total = static_cast<double>(m) + log(sum);
        wave_lds_fence();
        uint64_t head[kHeads];
        int left[kHeads];  // what a list holds behind its head
        uint64_t best = 0ull;
#pragma unroll
        for (int h = 0; h < kHeads; ++h) {
            const int p = lane + 64 * h;
            head[h] = p < a.nparts ? keys[p * W] : 0ull;
            left[h] = W - 1;
            best = umax64(best, head[h]);
        }
        int n = 0;
        uint64_t mine = 0ull;  // lane w keeps the w-th best
        for (; n < W; ++n) {
            const uint64_t k = wave_max_u64_full(best);
            if (k == 0ull) break;
            if (lane == n) mine = k;
            if (k == best) {
                best = 0ull;
#pragma unroll
                for (int h = 0; h < kHeads; ++h) {
                    if (head[h] == k) {
                        head[h] = left[h] > 0 ? keys[(lane + 64 * h) * W + W - left[h]] : 0ull;
                        --left[h];
                    }
                    best = umax64(best, head[h]);
                }
            }
        }
        if (lane < n) {
            const double c = score + (static_cast<double>(key_value(mine)) - total);
            s_k[b * W + lane] = mine;
            s_c[b * W + lane] = c == c ? c : -INFINITY;
        }
        if (lane == 0) s_n[b] = n;
    }
    __syncthreads();
    const int b = t / W, i = t - b * W;
    if (t < W * W && i < s_n[b]) {
        const double c = s_c[t];
        int place = i;
        for (int o = 0; o < W && place < W; ++o) {
            if (o == b) continue;
            int lo = 0, hi = s_n[o];
            while (lo < hi) {
                const int mid = (lo + hi) >> 1;
                const double d = s_c[o * W + mid];
                if (d > c || (o < b && d == c))
                    lo = mid + 1;
                else
                    hi = mid;
            }
            place += lo;
        }
        if (place < W) {
            const uint32_t tok = argmax_key_index(s_k[t]);
            a.parents[row0 + place] = static_cast<uint32_t>(b);
            a.tokens[row0 + place] = tok;
            a.new_scores[row0 + place] = static_cast<float>(c);
            if (a.new_done) a.new_done[row0 + place] = s_done[b] || tok == a.eos ? 1 : 0;
        }
    }
    if (t < W) {  // fewer candidates than slots: the rest end here
        int n = 0;
        for (int o = 0; o < W; ++o) n += s_n[o];
        if (t >= n) {
            a.parents[row0 + t] = static_cast<uint32_t>(t);
            a.tokens[row0 + t] = a.eos;
            a.new_scores[row0 + t] = -INFINITY;
            if (a.new_done) a.new_done[row0 + t] = 1;
        }
    }
}

// ---- the states ------------------------------------------------------------------

constexpr int kStores = 32;  // caches and rings of one launch

struct Store {
    char* k;
    char* v;
    size_t stride;       // bytes from one page's (stream's) head 0 to the next's
    size_t head_stride;  // bytes from one head to the next
    uint32_t n_pages;    // 0: a ring, whose "page" is its stream
    uint32_t heads;
    uint32_t slot_bytes;
};

struct Stores {
    Store s[kStores];
    int n;
    uint32_t ring_rows;
    uint32_t pieces;  // blocks to a head's rows
};

typedef uint32_t u4 __attribute__((ext_vector_type(4)));

// The beams of group `grp` as slots: parent (a number out of range: itself),
// and the common length of their caches.
struct Group {
    uint32_t len;
    bool ok;  // a common length, its page in the tables
};

__device__ __forceinline__ uint32_t parent_of(const BeamReorder& a, int grp, int b) {
    const uint32_t p = a.parents[static_cast<size_t>(grp) * a.beams + b];
    return p < static_cast<uint32_t>(a.beams) ? p : static_cast<uint32_t>(b);
}

__device__ __forceinline__ Group group_of(const BeamReorder& a, int grp) {
    Group g{};
    const uint32_t* lens = a.lens + static_cast<size_t>(grp) * a.beams;
    g.len = lens[0];
    g.ok = g.len != kPagedNone;
    for (int b = 1; b < a.beams; ++b) g.ok = g.ok && lens[b] == g.len;
    const uint32_t rest = g.len & ((1u << a.page_shift) - 1u);
    g.ok = g.ok && (g.len >> a.page_shift) + (rest ? 1u : 0u) <= a.max_pages;
    return g;
}

// Rows b of [W][n] take rows parent[b], in place: a thread reads its column of
// every row, then writes it, so nothing is overwritten before it is read.
template <int WB, typename V, typename At>
__device__ __forceinline__ void permute_columns(const uint32_t* parent, int W, size_t n, size_t first, size_t step, At at) {
    for (size_t i = first; i < n; i += step) {
        V v[WB];
#pragma unroll
        for (int b = 0; b < WB; ++b)
            if (b < W && parent[b] != static_cast<uint32_t>(b)) v[b] = *at(parent[b], i);
#pragma unroll
        for (int b = 0; b < WB; ++b)
            if (b < W && parent[b] != static_cast<uint32_t>(b)) __builtin_nontemporal_store(v[b], at(b, i));
    }
}

// Grid (head x piece, group, store x {K, V} then one for histories and tables).
// A table's entries before the page in progress follow the parents; the page in
// progress and those after it stay with the slot, and the page's rows follow, a
// block to 256 columns of 16 bytes and every `pieces`-th after them: eight
// groups of eight beams, 12 layers, 31 slots of 512 bytes in progress took 90 us
// with a block to a head's four pieces and 70 us with a block to each.
template <int WB>
__global__ __launch_bounds__(256) void beam_reorder_kernel(BeamReorder a, Stores st) {
    __shared__ uint32_t s_parent[WB], s_page[WB], s_len[WB];
    const int grp = blockIdx.y;
    const int W = a.beams;
    const size_t row0 = static_cast<size_t>(grp) * W;
    if (static_cast<int>(blockIdx.z) == 2 * st.n) {
        if (blockIdx.x == 0 && a.history) {
            if (threadIdx.x < W) {
                s_parent[threadIdx.x] = parent_of(a, grp, threadIdx.x);
                s_len[threadIdx.x] = static_cast<uint32_t>(min(static_cast<size_t>(a.history_len[row0 + threadIdx.x]), a.cap));
            }
            __syncthreads();
            uint32_t longest = 0;
            for (int b = 0; b < W; ++b) longest = max(longest, s_len[b]);
            uint32_t* h = a.history + row0 * a.cap;
            permute_columns<WB, uint32_t>(s_parent, W, longest, threadIdx.x, 256,
                                          [&](uint32_t b, size_t i) { return h + b * a.cap + i; });
            __syncthreads();  // every history is in place before a token is written behind it
            if (threadIdx.x < W) {
                const uint32_t len = s_len[s_parent[threadIdx.x]];
                const bool room = a.tokens && len < a.cap;
                if (room) h[threadIdx.x * a.cap + len] = a.tokens[row0 + threadIdx.x];
                a.history_len[row0 + threadIdx.x] = len + (room && a.advance ? 1u : 0u);
            }
        }
        if (blockIdx.x == 1 && a.tables && a.permute) {
            if (threadIdx.x < W) s_parent[threadIdx.x] = parent_of(a, grp, threadIdx.x);
            __syncthreads();
            const Group g = group_of(a, grp);
            uint32_t* t = a.tables + row0 * a.max_pages;
            if (g.ok)
                permute_columns<WB, uint32_t>(s_parent, W, g.len >> a.page_shift, threadIdx.x, 256,
                                              [&](uint32_t b, size_t i) { return t + b * a.max_pages + i; });
        }
        return;
    }
    const Store& s = st.s[blockIdx.z >> 1];
    const uint32_t head = blockIdx.x / st.pieces;
    const size_t first = (blockIdx.x - head * st.pieces) * 256u;
    if (head >= s.heads) return;
    const uint32_t rows = s.n_pages ? a.lens[row0] & ((1u << a.page_shift) - 1u) : st.ring_rows;
    const size_t n = static_cast<size_t>(rows) * s.slot_bytes / 16;
    if (first >= n) return;
    if (threadIdx.x < W) {
        s_parent[threadIdx.x] = parent_of(a, grp, threadIdx.x);
        s_page[threadIdx.x] = static_cast<uint32_t>(row0 + threadIdx.x);
    }
    if (s.n_pages) {
        const Group g = group_of(a, grp);
        if (!g.ok) return;
        if (threadIdx.x < W) s_page[threadIdx.x] = a.tables[(row0 + threadIdx.x) * a.max_pages + (g.len >> a.page_shift)];
    }
    __syncthreads();
    if (s.n_pages)
        for (int b = 0; b < W; ++b)
            if (s_page[b] >= s.n_pages) return;
    char* base = (blockIdx.z & 1 ? s.v : s.k) + head * s.head_stride;
    permute_columns<WB, u4>(s_parent, W, n, first + threadIdx.x, 256 * st.pieces, [&](uint32_t b, size_t i) {
        return reinterpret_cast<u4*>(base + s_page[b] * s.stride) + i;
    });
}

// The weights that attention gathered for the keys of each slot's cache, of up
// to kStores caches: [rows][heads][ld] each.
struct Gathered {
    float* w[kStores];
    uint32_t heads[kStores];
    int n;
    size_t ld;
    uint32_t pieces;  // blocks to a head's row
};

// Grid (head x piece, group, cache): a thread a key of every slot. Bound by HBM:
// eight groups of eight beams, 12 layers of 10 key heads and 1151 keys, 65 MB
// read and written, take 20 us behind the reorder's 63.
template <int WB>
__global__ __launch_bounds__(256) void beam_weights_kernel(BeamReorder a, Gathered w) {
    __shared__ uint32_t s_parent[WB];
    const int grp = blockIdx.y;
    const uint32_t head = blockIdx.x / w.pieces;
    const size_t first = (blockIdx.x - head * w.pieces) * 256u;
    const size_t heads = w.heads[blockIdx.z];
    if (head >= heads) return;
    const Group g = group_of(a, grp);
    const size_t n = min(static_cast<size_t>(g.len), w.ld);
    if (!g.ok || first >= n) return;
    if (threadIdx.x < a.beams) s_parent[threadIdx.x] = parent_of(a, grp, threadIdx.x);
    __syncthreads();
    uint32_t* base = reinterpret_cast<uint32_t*>(w.w[blockIdx.z]) + (static_cast<size_t>(grp) * a.beams * heads + head) * w.ld;
    permute_columns<WB, uint32_t>(s_parent, a.beams, n, first + threadIdx.x, 256 * w.pieces,
                                  [&](uint32_t b, size_t i) { return base + b * heads * w.ld + i; });
}

__global__ void beam_check_kernel(BeamReorder a, unsigned long long* err) {
    const int grp = blockIdx.x;
    const size_t row0 = static_cast<size_t>(grp) * a.beams;
    const auto fault = [&](int b, int code) {
        atomicMin(err, (static_cast<unsigned long long>(row0 + b) << 8) | static_cast<unsigned long long>(code));
    };
    const int b = threadIdx.x;
    if (b >= a.beams) return;
    if (a.parents[row0 + b] >= static_cast<uint32_t>(a.beams)) fault(b, kFaultParent);
    if (a.history && static_cast<size_t>(a.history_len[row0 + b]) + (a.tokens ? 1 : 0) > a.cap) fault(b, kFaultHistory);
    if (!a.tables) return;
    const uint32_t len = a.lens[row0 + b];
    if (len != a.lens[row0]) return fault(b, kFaultGroupLen);
    if (len == kPagedNone) return;
    const uint32_t rest = len & ((1u << a.page_shift) - 1u), at = len >> a.page_shift;
    if (at + (rest ? 1u : 0u) > a.max_pages) return fault(b, kFaultLen);
    if (!rest) return;
    for (int o = 0; o < b; ++o)
        if (a.tables[(row0 + o) * a.max_pages + at] == a.tables[(row0 + b) * a.max_pages + at]) fault(b, kFaultTail);
}

}  // namespace

int beam_parts(int vocab) { return (vocab + kChunk - 1) / kChunk; }

size_t beam_part_bytes(int rows, int beams, int nparts) {
    const size_t n = static_cast<size_t>(rows) * nparts;
    return n * (sizeof(double) + sizeof(float) + beams * sizeof(uint64_t));
}

hipError_t launch_beam_select(hipStream_t s, const BeamSelect& a, focr_hip_ctx* ctx) {
    const int rows = a.groups * a.beams;
    const Parts q = parts_of(a.part, rows, a.beams, a.nparts);
    ProfScope ps(ctx, "beam_select");
    FOCR_LAUNCH(beam_scan_kernel, dim3(a.nparts, rows), dim3(kThreads), 0, s, a, q);
    // a row's lists in LDS for as many rows at once as 128 KB hold (one: nparts * beams <= 4096 keys, 32 KB)
    const size_t row_bytes = static_cast<size_t>(a.nparts) * a.beams * sizeof(uint64_t);
    const int waves = static_cast<int>(std::min<size_t>({16, static_cast<size_t>(a.beams), (size_t(128) << 10) / row_bytes}));
    const size_t lds = waves * row_bytes;
    const int threads = std::max(64 * waves, (a.beams * a.beams + 63) / 64 * 64);
    FOCR_LAUNCH(beam_pick_kernel, dim3(a.groups), dim3(threads), lds, s, a, q, waves);
    return hipGetLastError();
}

hipError_t launch_beam_reorder(hipStream_t s, const BeamReorder& a, const focr_hip_paged* const* caches,
                               size_t n_caches, const focr_hip_rswa* const* rings, size_t n_rings,
                               uint32_t ring_rows) {
    const size_t total = n_caches + (ring_rows ? n_rings : 0);
    BeamReorder now = a;
    for (size_t i = 0; i == 0 || i < total; i += kStores) {
        Stores st{};
        st.n = static_cast<int>(std::min<size_t>(kStores, total - i));
        st.ring_rows = ring_rows;
        uint32_t heads = 1;
        size_t most = 0;  // bytes of a head's rows at most
        for (int j = 0; j < st.n; ++j) {
            Store& o = st.s[j];
            if (i + j < n_caches) {
                const focr_hip_paged* c = caches[i + j];
                o.slot_bytes = static_cast<uint32_t>(c->head_dim * c->esize());
                o.head_stride = static_cast<size_t>(o.slot_bytes) << c->page_shift;
                o.stride = c->page_bytes();
                o.heads = static_cast<uint32_t>(c->n_kv_heads);
                o.n_pages = static_cast<uint32_t>(c->n_pages);
                o.k = static_cast<char*>(c->k);
                most = std::max(most, (o.head_stride - o.slot_bytes));
                o.v = static_cast<char*>(c->v);
            } else {
                const focr_hip_rswa* c = rings[i + j - n_caches];
                o.slot_bytes = kHeadDim * sizeof(float);
                o.head_stride = static_cast<size_t>(kRingWindow) * o.slot_bytes;
                o.stride = c->stream_floats() * sizeof(float);
                o.heads = kNumHeads;
                o.n_pages = 0;
                o.k = reinterpret_cast<char*>(c->ring_k(0));
                most = std::max(most, static_cast<size_t>(ring_rows) * o.slot_bytes);
                o.v = reinterpret_cast<char*>(c->ring_v(0));
            }
            heads = std::max(heads, o.heads);
        }
        st.pieces = static_cast<uint32_t>(std::min<size_t>(std::max<size_t>((most + 4095) / 4096, 1), 8));
        const dim3 grid(std::max(heads * st.pieces, 2u), a.groups, 2 * st.n + 1);
        if (a.beams <= 4)
            FOCR_LAUNCH(beam_reorder_kernel<4>, grid, dim3(256), 0, s, now, st);
        else if (a.beams <= 8)
            FOCR_LAUNCH(beam_reorder_kernel<8>, grid, dim3(256), 0, s, now, st);
        else if (a.beams <= 16)
            FOCR_LAUNCH(beam_reorder_kernel<16>, grid, dim3(256), 0, s, now, st);
        else
            FOCR_LAUNCH(beam_reorder_kernel<32>, grid, dim3(256), 0, s, now, st);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
        now.history = nullptr;  // once; and the tables too, whose entries of the pages in progress stay as they are
        now.permute = 0;
    }
    return hipSuccess;
}

hipError_t launch_beam_weights(hipStream_t s, const BeamReorder& a, const focr_hip_paged* const* caches,
                               float* const* weights, size_t n, size_t ldw) {
    Gathered w{};
    uint32_t heads = 0;
    w.ld = ldw;
    w.pieces = static_cast<uint32_t>(std::min<size_t>((ldw + 255) / 256, 256));
    for (size_t i = 0; i < n; ++i) {
        if (weights[i]) {
            w.w[w.n] = weights[i];
            w.heads[w.n++] = static_cast<uint32_t>(caches[i]->n_kv_heads);
            heads = std::max(heads, static_cast<uint32_t>(caches[i]->n_kv_heads));
        }
        if (w.n == 0 || (w.n < kStores && i + 1 < n)) continue;
        const dim3 grid(heads * w.pieces, a.groups, w.n);
        if (a.beams <= 4)
            FOCR_LAUNCH(beam_weights_kernel<4>, grid, dim3(256), 0, s, a, w);
        else if (a.beams <= 8)
            FOCR_LAUNCH(beam_weights_kernel<8>, grid, dim3(256), 0, s, a, w);
        else if (a.beams <= 16)
            FOCR_LAUNCH(beam_weights_kernel<16>, grid, dim3(256), 0, s, a, w);
        else
            FOCR_LAUNCH(beam_weights_kernel<32>, grid, dim3(256), 0, s, a, w);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
        w.n = 0;
        heads = 0;
    }
    return hipSuccess;
}

hipError_t launch_beam_check(hipStream_t s, const BeamReorder& a, unsigned long long* err) {
    FOCR_LAUNCH(beam_check_kernel, dim3(a.groups), dim3(64), 0, s, a, err);
    return hipGetLastError();
}

}  // namespace focr
