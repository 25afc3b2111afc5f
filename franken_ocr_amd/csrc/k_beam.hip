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
constexpr int kPer = 16;                    // logits of a thread
constexpr int kChunk = kThreads * kPer;     // logits of a block

// The chunks' and rows' results: max and f64 sum of exp(x - max) per chunk,
// its W best keys (argmax_key order), then per row the sorted W best with
// their c.
struct Parts {
    float* max;     // [rows][nparts]
    double* sum;    // [rows][nparts]
    uint64_t* key;  // [rows][nparts][W], descending, 0 where there are fewer
    double* row_c;  // [rows][W]
    uint64_t* row_key;
};

__host__ __device__ inline Parts parts_of(void* p, int rows, int beams, int nparts) {
    Parts q;
    const size_t n = static_cast<size_t>(rows) * nparts, w = static_cast<size_t>(rows) * beams;
    q.sum = static_cast<double*>(p);
    q.row_c = q.sum + n;
    q.key = reinterpret_cast<uint64_t*>(q.row_c + w);
    q.row_key = q.key + n * beams;
    q.max = reinterpret_cast<float*>(q.row_key + w);
    return q;
}

// Grid (chunk, row): one pass over the chunk's logits, held in registers.
__global__ __launch_bounds__(kThreads) void beam_scan_kernel(BeamSelect a, Parts q) {
    __shared__ float s_max[kThreads / 64];
    __shared__ double s_sum[kThreads / 64];
    __shared__ uint64_t s_key[2][kThreads / 64];
    const int part = blockIdx.x;
    const int row = blockIdx.y;
    if (a.done && a.done[row]) return;  // its one candidate needs no logits
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const float* x = a.logits + static_cast<size_t>(row) * a.ld;
    const uint32_t* ban = a.ban_bits ? a.ban_bits + static_cast<size_t>(row) * a.ban_words : nullptr;
    float v[kPer];
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        const int t = part * kChunk + i * kThreads + static_cast<int>(threadIdx.x);
        v[i] = t < a.vocab ? x[t] : __uint_as_float(0x7FC00000u);  // NaN: no logit
    }
    float m = -INFINITY;
#pragma unroll
    for (int i = 0; i < kPer; ++i) m = fmaxf(m, v[i]);  // a NaN is skipped
    m = wave_max_f_full(m);
    if (lane == 0) s_max[wave] = m;
    __syncthreads();
    m = fmaxf(fmaxf(s_max[0], s_max[1]), fmaxf(s_max[2], s_max[3]));
    double sum = 0.0;
    if (m > -INFINITY) {
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            const double ex = v[i] == m ? 1.0 : exp(static_cast<double>(v[i]) - static_cast<double>(m));
            sum += v[i] == v[i] ? ex : 0.0;
        }
    }
    sum = wave_sum_d_full(sum);
    if (lane == 0) s_sum[wave] = sum;
    uint64_t key[kPer], best = 0ull;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        const int t = part * kChunk + i * kThreads + static_cast<int>(threadIdx.x);
        key[i] = argmax_key(v[i], static_cast<uint32_t>(t));
        if (ban && t < a.vocab && (ban[t >> 5] >> (t & 31) & 1u)) key[i] = 0ull;
        best = umax64(best, key[i]);
    }
    const size_t at = static_cast<size_t>(row) * a.nparts + part;
    for (int w = 0; w < a.beams; ++w) {
        const uint64_t mine = wave_max_u64_full(best);
        if (lane == 0) s_key[w & 1][wave] = mine;
        __syncthreads();
        const uint64_t* s = s_key[w & 1];
        const uint64_t top = umax64(umax64(s[0], s[1]), umax64(s[2], s[3]));
        if (threadIdx.x == 0) q.key[at * a.beams + w] = top;
        if (top == best && top != 0ull) {  // this thread's: its next best
            best = 0ull;
#pragma unroll
            for (int i = 0; i < kPer; ++i) {
                if (key[i] == top) key[i] = 0ull;
                best = umax64(best, key[i]);
            }
        }
    }
    if (threadIdx.x == 0) {
        q.max[at] = m;
        q.sum[at] = s_sum[0] + s_sum[1] + s_sum[2] + s_sum[3];
    }
}

// Keys of the descending list s[0..n) that are greater than k.
__device__ __forceinline__ int count_greater(const uint64_t* s, int n, uint64_t k) {
    int lo = 0, hi = n;
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (s[mid] > k)
            lo = mid + 1;
        else
            hi = mid;
    }
    return lo;
}

// Grid (row): L from the chunks, and the W best of the chunks' lists: a key's
// place is the number of greater ones, found in every list by bisection.
__global__ __launch_bounds__(kThreads) void beam_row_kernel(BeamSelect a, Parts q) {
    __shared__ double s_l;
    const int row = blockIdx.x;
    const int W = a.beams;
    double* rc = q.row_c + static_cast<size_t>(row) * W;
    uint64_t* rk = q.row_key + static_cast<size_t>(row) * W;
    const double score = static_cast<double>(a.scores[row]);
    const bool done = a.done && a.done[row];
    for (int i = threadIdx.x; i < W; i += kThreads) {
        rk[i] = done && i == 0 ? (1ull << 32) | (0xFFFFFFFFull - a.eos) : 0ull;
        rc[i] = done && i == 0 && score == score ? score : -INFINITY;
    }
    if (done) return;
    const size_t at = static_cast<size_t>(row) * a.nparts;
    if (threadIdx.x < 64) {
        float m = -INFINITY;
        for (int p = threadIdx.x; p < a.nparts; p += 64) m = fmaxf(m, q.max[at + p]);
        m = wave_max_f_full(m);
        double sum = 0.0;
        for (int p = threadIdx.x; p < a.nparts; p += 64)
            if (q.max[at + p] > -INFINITY)
                sum += q.sum[at + p] * (q.max[at + p] == m ? 1.0 : exp(static_cast<double>(q.max[at + p]) - static_cast<double>(m)));
        sum = wave_sum_d_full(sum);
        if (threadIdx.x == 0) s_l = static_cast<double>(m) + log(sum);
    }
    __syncthreads();
    const uint64_t* key = q.key + at * W;
    for (int i = threadIdx.x; i < a.nparts * W; i += kThreads) {
        const uint64_t k = key[i];
        if (k == 0ull) continue;
        int place = 0;
        for (int p = 0; p < a.nparts && place < W; ++p) place += count_greater(key + static_cast<size_t>(p) * W, W, k);
        if (place >= W) continue;
        const double c = score + (static_cast<double>(key_value(k)) - s_l);
        rk[place] = k;
        rc[place] = c == c ? c : -INFINITY;
    }
}

// Grid (group), a thread to a candidate: its place among the group's is the
// number before it in its own beam's list and, by bisection, in the others'.
__global__ __launch_bounds__(1024) void beam_pick_kernel(BeamSelect a, Parts q) {
    __shared__ double s_c[kBeamMax * kBeamMax];
    __shared__ uint64_t s_k[kBeamMax * kBeamMax];
    __shared__ int s_n[kBeamMax];  // candidates of a beam
    __shared__ uint8_t s_done[kBeamMax];
    const int W = a.beams;
    const int t = threadIdx.x;
    const size_t row0 = static_cast<size_t>(blockIdx.x) * W;
    const size_t at = row0 * W;
    if (t < W * W) {
        s_c[t] = q.row_c[at + t];
        s_k[t] = q.row_key[at + t];
    }
    if (t < W) s_done[t] = a.done ? a.done[row0 + t] : 0;
    __syncthreads();
    if (t < W) {
        int n = 0;
        while (n < W && s_k[t * W + n] != 0ull) ++n;
        s_n[t] = n;
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
__device__ __forceinline__ void permute_columns(const uint32_t* parent, int W, size_t n, int first, int step, At at) {
    for (size_t i = first; i < n; i += step) {
        V v[WB];
#pragma unroll
        for (int b = 0; b < WB; ++b)
            if (b < W && parent[b] != static_cast<uint32_t>(b)) v[b] = *at(parent[b], i);
#pragma unroll
        for (int b = 0; b < WB; ++b)
            if (b < W && parent[b] != static_cast<uint32_t>(b)) *at(b, i) = v[b];
    }
}

// Grid (head, group, store x {K, V} then one for histories and tables). A
// table's entries before the page in progress follow the parents; the page in
// progress and those after it stay with the slot, and the page's rows follow.
template <int WB>
__global__ __launch_bounds__(256) void beam_reorder_kernel(BeamReorder a, Stores st) {
    __shared__ uint32_t s_parent[WB], s_page[WB], s_len[WB];
    const int grp = blockIdx.y;
    const int W = a.beams;
    const size_t row0 = static_cast<size_t>(grp) * W;
    if (threadIdx.x < W) s_parent[threadIdx.x] = parent_of(a, grp, threadIdx.x);
    if (static_cast<int>(blockIdx.z) == 2 * st.n) {
        if (blockIdx.x == 0 && a.history) {
            if (threadIdx.x < W)
                s_len[threadIdx.x] = static_cast<uint32_t>(min(static_cast<size_t>(a.history_len[row0 + threadIdx.x]), a.cap));
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
    const uint32_t head = blockIdx.x;
    if (head >= s.heads) return;
    uint32_t rows = st.ring_rows;
    if (s.n_pages) {
        const Group g = group_of(a, grp);
        rows = g.len & ((1u << a.page_shift) - 1u);
        if (!g.ok || rows == 0) return;
        if (threadIdx.x < W) s_page[threadIdx.x] = a.tables[(row0 + threadIdx.x) * a.max_pages + (g.len >> a.page_shift)];
    } else if (threadIdx.x < W) {
        s_page[threadIdx.x] = static_cast<uint32_t>(row0 + threadIdx.x);
    }
    __syncthreads();
    if (s.n_pages)
        for (int b = 0; b < W; ++b)
            if (s_page[b] >= s.n_pages) return;
    char* base = (blockIdx.z & 1 ? s.v : s.k) + head * s.head_stride;
    const size_t n = static_cast<size_t>(rows) * s.slot_bytes / 16;
    permute_columns<WB, u4>(s_parent, W, n, threadIdx.x, 256, [&](uint32_t b, size_t i) {
        return reinterpret_cast<u4*>(base + s_page[b] * s.stride) + i;
    });
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
    const size_t n = static_cast<size_t>(rows) * nparts, w = static_cast<size_t>(rows) * beams;
    return n * 8 + w * 8 + n * beams * 8 + w * 8 + n * 4;
}

hipError_t launch_beam_select(hipStream_t s, const BeamSelect& a, focr_hip_ctx* ctx) {
    const int rows = a.groups * a.beams;
    const Parts q = parts_of(a.part, rows, a.beams, a.nparts);
    ProfScope ps(ctx, "beam_select");
    FOCR_LAUNCH(beam_scan_kernel, dim3(a.nparts, rows), dim3(kThreads), 0, s, a, q);
    FOCR_LAUNCH(beam_row_kernel, dim3(rows), dim3(kThreads), 0, s, a, q);
    const int t = (a.beams * a.beams + 63) / 64 * 64;
    FOCR_LAUNCH(beam_pick_kernel, dim3(a.groups), dim3(t), 0, s, a, q);
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
        uint32_t heads = 2;
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
                o.v = static_cast<char*>(c->v);
            } else {
                const focr_hip_rswa* c = rings[i + j - n_caches];
                o.slot_bytes = kHeadDim * sizeof(float);
                o.head_stride = static_cast<size_t>(kRingWindow) * o.slot_bytes;
                o.stride = c->stream_floats() * sizeof(float);
                o.heads = kNumHeads;
                o.n_pages = 0;
                o.k = reinterpret_cast<char*>(c->ring_k(0));
                o.v = reinterpret_cast<char*>(c->ring_v(0));
            }
            heads = std::max(heads, o.heads);
        }
        const dim3 grid(heads, a.groups, 2 * st.n + 1);
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

hipError_t launch_beam_check(hipStream_t s, const BeamReorder& a, unsigned long long* err) {
    FOCR_LAUNCH(beam_check_kernel, dim3(a.groups), dim3(64), 0, s, a, err);
    return hipGetLastError();
}

}  // namespace focr
