// k_paged.hip — one new token over a paged key-value cache: the write of its
// rows, the attention split over the cache's length, the join of the splits,
// the attention weight each key gathers, and eviction by that weight.
//
// Layout in HBM: K and V pools [n_pages][n_kv_heads][page_size][head_dim], so
// the slots of one (page, head) are contiguous. Key j of sequence s is slot
// j % page_size of page tables[s][j / page_size]. A call sees of n keys all,
// or (window w > 0) the first p = min(prefix, n) and the last w:
//   s_j = scale q.k_j, P_j = exp(s_j - max s) / sum exp, out = sum_j P_j v_j.
// Scores are kept times log2 e, so that the exponential is the hardware's
// exp2. Dots, the running maximum and sum and the outputs are f32; the only
// rounding to fewer bits is a written row's to the cache's type.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "focr_internal.hpp"
#include "k_common.hpp"
#include "k_paged_index.hpp"

namespace focr {
namespace {

constexpr float kLog2e = 1.4426950408889634f;

PoolGeom geom_of(const focr_hip_paged* c) {
    return PoolGeom{c->k, c->v, static_cast<uint32_t>(c->n_pages), c->page_shift,
                    static_cast<uint32_t>(c->n_kv_heads)};
}

typedef uint32_t u4 __attribute__((ext_vector_type(4)));

// 16 bytes of a row as floats, and back (round to nearest, ties to even).
template <typename T>
struct Row16;
template <>
struct Row16<float> {
    static constexpr int N = 4;
    static __device__ __forceinline__ void load(const u4& w, float* f) {
#pragma unroll
        for (int i = 0; i < 4; ++i) f[i] = __uint_as_float(w[i]);
    }
    static __device__ __forceinline__ u4 pack(const float* f) {
        u4 w;
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = __float_as_uint(f[i]);
        return w;
    }
};
template <>
struct Row16<__bf16> {
    static constexpr int N = 8;
    static __device__ __forceinline__ void load(const u4& w, float* f) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            f[2 * i] = __uint_as_float(w[i] << 16);
            f[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
        }
    }
    static __device__ __forceinline__ u4 pack(const float* f) {
        u4 w;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t lo = __builtin_bit_cast(uint16_t, static_cast<__bf16>(f[2 * i]));
            const uint32_t hi = __builtin_bit_cast(uint16_t, static_cast<__bf16>(f[2 * i + 1]));
            w[i] = lo | (hi << 16);
        }
        return w;
    }
};
template <>
struct Row16<_Float16> {
    static constexpr int N = 8;
    static __device__ __forceinline__ void load(const u4& w, float* f) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            f[2 * i] = static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(w[i] & 0xFFFFu)));
            f[2 * i + 1] = static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(w[i] >> 16)));
        }
    }
    static __device__ __forceinline__ u4 pack(const float* f) {
        u4 w;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t lo = __builtin_bit_cast(uint16_t, static_cast<_Float16>(f[2 * i]));
            const uint32_t hi = __builtin_bit_cast(uint16_t, static_cast<_Float16>(f[2 * i + 1]));
            w[i] = lo | (hi << 16);
        }
        return w;
    }
};

// Lane l's value with lane (l ^ M)'s: within a 16-lane row by DPP, across rows
// by v_permlane16_swap / v_permlane32_swap (VALU; a shuffle goes through LDS).
template <int M, typename Op>
__device__ __forceinline__ float xor_fold(float v, Op op) {
    if constexpr (M == 1) return op(v, __int_as_float(dpp_mov<0xB1>(__float_as_int(v))));
    if constexpr (M == 2) return op(v, __int_as_float(dpp_mov<0x4E>(__float_as_int(v))));
    if constexpr (M == 4) {  // after 1 and 2 every quad is uniform: the half row's mirror is the other quad
        return op(v, __int_as_float(dpp_mov<0x141>(__float_as_int(v))));
    }
    if constexpr (M == 8) return op(v, __int_as_float(dpp_mov<0x128>(__float_as_int(v))));  // row_ror:8
    if constexpr (M == 16) {
        const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        return op(__uint_as_float(r[0]), __uint_as_float(r[1]));
    }
    if constexpr (M == 32) {
        const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        return op(__uint_as_float(r[0]), __uint_as_float(r[1]));
    }
    return v;
}

struct Sum {
    __device__ __forceinline__ float operator()(float a, float b) const { return a + b; }
};
struct Max {
    __device__ __forceinline__ float operator()(float a, float b) const { return fmaxf(a, b); }
};

// Over the lanes that differ in the bits [A, B) of their number (powers of
// two); every lane gets the result. A = 1 or A >= 8.
template <int A, int B, typename Op>
__device__ __forceinline__ float fold_lanes(float v, Op op) {
    if constexpr (A < B) {
        v = xor_fold<A>(v, op);
        return fold_lanes<2 * A, B>(v, op);
    }
    return v;
}

// The rows of a split's keys b0 .. b0 + cnt, to LDS, with none behind them up
// to `padded`. Every table entry of a thread is requested before the first is
// used (one after the other they were eight waits of a loaded memory).
__device__ __forceinline__ void fill_rows(const PagedTables& t, const PoolGeom& g, const Seen& e, int s, uint32_t hk,
                                          uint32_t b0, int cnt, int padded, uint32_t* s_row) {
    constexpr int N = kPagedChunkMax / 256;
    uint32_t row[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
        if (i * 256 < cnt) {  // uniform; past the end a thread takes the last key's again
            const uint32_t at = b0 + min(static_cast<int>(threadIdx.x) + i * 256, cnt - 1);
            row[i] = row_of(t, g, s, hk, at < e.p ? at : at + e.shift);
        }
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int j = static_cast<int>(threadIdx.x) + i * 256;
        if (j < padded) s_row[j] = j < cnt ? row[i] : kBadRow;
    }
}

// The four waves' maxima, sums and outputs of GT heads joined and written as
// split z's part; row0: the first head's row of all [sequence][head].
template <int GT, int D>
__device__ __forceinline__ void join_waves(const PagedAttend& a, const float (*s_acc)[GT][D], const float2 (*s_ml)[GT],
                                           int g0, size_t row0, int z) {
    for (int at = threadIdx.x; at < GT * D; at += 256) {
        const int i = at / D, d = at - i * D;
        if (g0 + i >= a.group) break;
        const float m0 = s_ml[0][i].x, m1 = s_ml[1][i].x, m2 = s_ml[2][i].x, m3 = s_ml[3][i].x;
        const float mx = fmaxf(fmaxf(m0, m1), fmaxf(m2, m3));
        const float sf = mx == -INFINITY ? 0.0f : mx;
        const float w0 = __builtin_amdgcn_exp2f(m0 - sf), w1 = __builtin_amdgcn_exp2f(m1 - sf);
        const float w2 = __builtin_amdgcn_exp2f(m2 - sf), w3 = __builtin_amdgcn_exp2f(m3 - sf);
        const float o = s_acc[0][i][d] * w0 + s_acc[1][i][d] * w1 + s_acc[2][i][d] * w2 + s_acc[3][i][d] * w3;
        const size_t part = (row0 + i) * a.nsplit + z;
        a.part_acc[part * D + d] = o;
        if (d == 0)
            a.part_ml[part] = make_float2(mx, s_ml[0][i].y * w0 + s_ml[1][i].y * w1 + s_ml[2][i].y * w2 + s_ml[3][i].y * w3);
    }
}

// One split of one key head's keys, for its GT query heads (the group). Grid
// (split, key head, sequence), 4 waves. Every wave takes tiles of its own:
// C lanes hold a key's row (16 bytes each), 64 / C keys to a load
// instruction, U of those for K and U for V in flight at once; a lane keeps
// the same key's K and V, so the probabilities never leave their lanes, and
// there is no barrier until the four waves' maxima, sums and outputs are
// joined at the end. Bound by HBM: 128 sequences of up to 16384 keys, 2 key
// heads of 128 bf16, one query head each 204 us, 5.6 TB/s read (a large copy
// moves 4.7); 64 sequences in f32, 64 wide, 107 us. Eight f32 rows in flight
// for K and for V and four waves a SIMD are what the load latency takes.
template <typename T, int D, int GT, int U>
__global__ __launch_bounds__(256, GT == 1 ? 4 : 3) void paged_attend_kernel(PoolGeom g, PagedAttend a) {
    constexpr int E = Row16<T>::N;
    constexpr int C = D / E;
    constexpr int R = 64 / C;
    constexpr int TILE = U * R;
    static_assert(kPagedChunkUnit % TILE == 0 || TILE % kPagedChunkUnit == 0, "a padded split stays in s_row");
    __shared__ uint32_t s_row[kPagedChunkMax];
    __shared__ float s_acc[4][GT][D];
    __shared__ float2 s_ml[4][GT];
    const int z = blockIdx.x;
    const int hk = blockIdx.y;
    const int s = blockIdx.z;
    const Seen e = seen_of(a.t, a.prefix, a.window, a.k_steps != nullptr, s);
    if (z == 0 && blockIdx.y == 0 && threadIdx.x == 0)
        a.seen[s] = make_uint4(e.none ? kPagedNone : e.nvis, e.p, e.shift, e.own ? 1u : 0u);
    if (e.none) return;
    const uint32_t chunk = split_keys(e.nvis, a.nsplit, a.split_least);
    const uint32_t b0 = static_cast<uint32_t>(z) * chunk;
    if (b0 >= e.nvis) return;
    const int cnt = static_cast<int>(min(chunk, e.nvis - b0));
    const int padded = (cnt + TILE - 1) / TILE * TILE;
    fill_rows(a.t, g, e, s, hk, b0, cnt, padded, s_row);
    const int wave = threadIdx.x >> 6;
    const int lane = threadIdx.x & 63;
    const int cl = lane % C;  // which 16 bytes of a row
    const int r = lane / C;   // which key of a load instruction
    float q[GT][E];
    const float qscale = a.scale * kLog2e;
#pragma unroll
    for (int i = 0; i < GT; ++i) {
        const float* qr = a.q + static_cast<size_t>(s) * a.ldq + (static_cast<size_t>(hk) * GT + i) * D + cl * E;
#pragma unroll
        for (int j = 0; j < E; ++j) q[i][j] = qr[j] * qscale;
    }
    // the step's own row is the last key seen
    const int own = e.own && e.nvis - 1 - b0 < static_cast<uint32_t>(cnt) ? static_cast<int>(e.nvis - 1 - b0) : -1;
    float m[GT], l[GT], acc[GT][E];
#pragma unroll
    for (int i = 0; i < GT; ++i) {
        m[i] = -INFINITY;
        l[i] = 0.0f;
#pragma unroll
        for (int j = 0; j < E; ++j) acc[i][j] = 0.0f;
    }
    __syncthreads();
    const u4* kp = static_cast<const u4*>(g.k) + cl;
    const u4* vp = static_cast<const u4*>(g.v) + cl;
    const size_t head0 = static_cast<size_t>(hk) * GT;
    const size_t n_heads = static_cast<size_t>(g.kv_heads) * GT;
    for (int t0 = wave * TILE; t0 < cnt; t0 += 4 * TILE) {
        uint32_t row[U];
        bool all = true;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            row[u] = s_row[t0 + u * R + r];
            all = all && row[u] != kBadRow;
        }
        u4 kw[U], vw[U];
        if (__all(all)) {
#pragma unroll
            for (int u = 0; u < U; ++u) kw[u] = kp[static_cast<size_t>(row[u]) * C];
#pragma unroll
            for (int u = 0; u < U; ++u) vw[u] = vp[static_cast<size_t>(row[u]) * C];
        } else {  // slots that hold no key are not read: what lies there may be NaN
#pragma unroll
            for (int u = 0; u < U; ++u) kw[u] = row[u] != kBadRow ? kp[static_cast<size_t>(row[u]) * C] : u4{0, 0, 0, 0};
#pragma unroll
            for (int u = 0; u < U; ++u) vw[u] = row[u] != kBadRow ? vp[static_cast<size_t>(row[u]) * C] : u4{0, 0, 0, 0};
        }
        if (own >= t0 && own < t0 + TILE) {  // the step's row comes from the call and goes to its page
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (t0 + u * R + r == own && row[u] != kBadRow) {
                    const size_t at = static_cast<size_t>(s) * a.ldkv + static_cast<size_t>(hk) * D + cl * E;
                    float f[E];
#pragma unroll
                    for (int j = 0; j < E; ++j) f[j] = a.k_steps[at + j];
                    kw[u] = Row16<T>::pack(f);
#pragma unroll
                    for (int j = 0; j < E; ++j) f[j] = a.v_steps[at + j];
                    vw[u] = Row16<T>::pack(f);
                    static_cast<u4*>(g.k)[static_cast<size_t>(row[u]) * C + cl] = kw[u];
                    static_cast<u4*>(g.v)[static_cast<size_t>(row[u]) * C + cl] = vw[u];
                }
            }
        }
        float sc[U][GT];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            float f[E];
            Row16<T>::load(kw[u], f);
#pragma unroll
            for (int i = 0; i < GT; ++i) {
                float d = f[0] * q[i][0];
#pragma unroll
                for (int j = 1; j < E; ++j) d = fmaf(f[j], q[i][j], d);
                d = fold_lanes<1, C>(d, Sum());
                sc[u][i] = row[u] != kBadRow ? d : -INFINITY;
            }
        }
        if (a.scores) {
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int j = t0 + u * R + r;
                if (cl == 0 && j < cnt)
#pragma unroll
                    for (int i = 0; i < GT; ++i)
                        a.scores[(static_cast<size_t>(s) * n_heads + head0 + i) * a.score_ld + b0 + j] = sc[u][i];
            }
        }
        float safe[GT];
#pragma unroll
        for (int i = 0; i < GT; ++i) {
            float mx = sc[0][i];
#pragma unroll
            for (int u = 1; u < U; ++u) mx = fmaxf(mx, sc[u][i]);
            mx = fmaxf(fold_lanes<C, 64>(mx, Max()), m[i]);
            safe[i] = mx == -INFINITY ? 0.0f : mx;  // no key yet: every exponential is 0, not NaN
            const float corr = __builtin_amdgcn_exp2f(m[i] - safe[i]);
            m[i] = mx;
            l[i] *= corr;
#pragma unroll
            for (int j = 0; j < E; ++j) acc[i][j] *= corr;
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            float f[E];
            Row16<T>::load(vw[u], f);
#pragma unroll
            for (int i = 0; i < GT; ++i) {
                const float p = __builtin_amdgcn_exp2f(sc[u][i] - safe[i]);
                l[i] += p;
#pragma unroll
                for (int j = 0; j < E; ++j) acc[i][j] = fmaf(p, f[j], acc[i][j]);
            }
        }
    }
    // the R keys of a wave's lanes, then the waves
#pragma unroll
    for (int i = 0; i < GT; ++i) {
        l[i] = fold_lanes<C, 64>(l[i], Sum());
#pragma unroll
        for (int j = 0; j < E; ++j) acc[i][j] = fold_lanes<C, 64>(acc[i][j], Sum());
        if (lane == 0) s_ml[wave][i] = make_float2(m[i], l[i]);
        if (r == 0)
#pragma unroll
            for (int j = 0; j < E; ++j) s_acc[wave][i][cl * E + j] = acc[i][j];
    }
    __syncthreads();
    join_waves<GT, D>(a, s_acc, s_ml, 0, head0 + static_cast<size_t>(s) * n_heads, z);
}

// The same split on the matrix cores, for up to 16 query heads of a key head at
// once (grid (split, key head x tile of 16 heads, sequence)). A wave takes 16
// keys at a time; lane l = 16 a + b:
//   scores  S[key][head] = K q: A = K (lane: key b, the row's 16-byte pieces
//           a + 4 c), B = q (lane: head b, the same values of d). The result
//           leaves lane l with head b and the keys 4 a + i, i < 4 ...
//   output  O[head][d] = P V: ... which is what A takes here, so the
//           probabilities stay where they are; B = V (lane: keys 4 a + i, one
//           of the columns (b + 16 c) VE + j at a time).
// An f32 cache runs v_mfma_f32_16x16x4_f32. A 16-bit cache's K and V are exact
// operands of the 16-bit instructions (16x16x32 for the scores, 16x16x16 for
// the output, at eight and four times the f32 rate); q and P are f32 and are
// written as sums of 16-bit terms: three of bf16, cut off (exact), or two of
// f16, rounded. q's row is scaled by a power of two to below 2^15 and P by 2^14;
// the second f16 term is what the first leaves, times 2^12, with sums of its
// own: for values from 2^-14 on, the first is a normal number and the second
// holds the rest to 2^-23 of the value (unscaled, it would be subnormal below
// 2^-2). Values below 2^-14 have no such terms: 16 keys with a smaller
// probability (2^-28 of the reference's) take f32 products into the same sums,
// a row of q with a smaller coordinate takes them throughout. Infinities have no
// terms in either type (an infinite K times a term that is zero is NaN): a wave
// whose sums come out not finite does its keys again in f32 products. Where the
// scores of most keys are that far apart, f16 takes 126 us for the 120 below
// (128 wide 245 for 232, 256 wide 88 for 76, 32 sequences), f32 products for
// all 134; doing all of a wave's keys again at the first such probability 154.
// The running maximum is moved only where a score is well past it (any
// reference gives the same quotient, and f32 holds the sums), so the usual
// tile needs nothing from other lanes.
// 128 sequences of up to 16384 keys, 16 heads on 2 key heads, bf16: 64 wide 119
// us (4.8 TB/s), 128 wide 230 us (4.9); the f32 products alone took 134 and
// 275. Loading a second tile ahead cost more waves than it hid latency (163
// for 155 us then), as did two tiles at once (171 for 137).
typedef float v4f __attribute__((ext_vector_type(4)));
typedef uint32_t u2 __attribute__((ext_vector_type(2)));
typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef _Float16 v4h __attribute__((ext_vector_type(4)));
typedef short v4s __attribute__((ext_vector_type(4)));

template <typename T>
struct Terms {  // f32: its own products alone
    static constexpr bool kSplit = false;
    static constexpr int N = 1;
    static constexpr float kTop = 0.0f, kPast = 8.0f, kLeast = 0.0f, kApart = 1.0f;
    static __device__ void split2(float, float, uint32_t*) {}
    static __device__ v4f scores(const u4&, const u4&, v4f c) { return c; }
    static __device__ v4f output(const u2&, const u2&, v4f c) { return c; }
};
template <>
struct Terms<__bf16> {
    static constexpr bool kSplit = true;
    static constexpr int N = 3;
    static constexpr float kTop = 0.0f;   // the maximum's exponential is 2^kTop
    static constexpr float kPast = 8.0f;  // how far a score may pass the reference
    static constexpr float kLeast = 0.0f;  // the least value that the terms hold
    static constexpr float kApart = 1.0f;  // what the later terms are scaled by
    // two values' terms in one word each
    static __device__ __forceinline__ void split2(float x, float y, uint32_t* w) {
#pragma unroll
        for (int t = 0; t < N; ++t) {
            const uint32_t a = __float_as_uint(x), b = __float_as_uint(y);
            w[t] = __builtin_amdgcn_perm(b, a, 0x07060302u);
            x -= __uint_as_float(a & 0xFFFF0000u);
            y -= __uint_as_float(b & 0xFFFF0000u);
        }
    }
    static __device__ __forceinline__ v4f scores(const u4& k, const u4& q, v4f c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf, k), __builtin_bit_cast(v8bf, q), c, 0, 0, 0);
    }
    static __device__ __forceinline__ v4f output(const u2& p, const u2& v, v4f c) {
        return __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(__builtin_bit_cast(v4s, p), __builtin_bit_cast(v4s, v), c, 0, 0, 0);
    }
};
template <>
struct Terms<_Float16> {
    static constexpr bool kSplit = true;
    static constexpr int N = 2;
    static constexpr float kTop = 14.0f;
    static constexpr float kPast = 15.0f;
    static constexpr float kLeast = 0x1p-14f;
    static constexpr float kApart = 0x1p12f;
    static __device__ __forceinline__ void split2(float x, float y, uint32_t* w) {
#pragma unroll
        for (int t = 0; t < N; ++t) {
            const _Float16 a = static_cast<_Float16>(x), b = static_cast<_Float16>(y);
            w[t] = __builtin_bit_cast(uint16_t, a) | static_cast<uint32_t>(__builtin_bit_cast(uint16_t, b)) << 16;
            x = (x - static_cast<float>(a)) * kApart;
            y = (y - static_cast<float>(b)) * kApart;
        }
    }
    static __device__ __forceinline__ v4f scores(const u4& k, const u4& q, v4f c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8h, k), __builtin_bit_cast(v8h, q), c, 0, 0, 0);
    }
    static __device__ __forceinline__ v4f output(const u2& p, const u2& v, v4f c) {
        return __builtin_amdgcn_mfma_f32_16x16x16f16(__builtin_bit_cast(v4h, p), __builtin_bit_cast(v4h, v), c, 0, 0, 0);
    }
};

// A number's magnitude as a whole number of the same order, zero the greatest.
__device__ __forceinline__ uint32_t size_order(float v) { return (__float_as_uint(v) & 0x7FFFFFFFu) - 1u; }

template <typename T, int D>
__global__ __launch_bounds__(256, D == 256 ? 1 : 2) void paged_attend_mfma_kernel(PoolGeom g, PagedAttend a) {
    using TT = Terms<T>;
    constexpr int E = Row16<T>::N;
    constexpr int C = D / E;                 // 16-byte pieces of a row
    constexpr int KC = C / 4;                // K pieces of a lane
    constexpr int VE = C >= 16 ? E : E / 2;  // values of a V piece (8 bytes where a row has 8 pieces of 16)
    constexpr int VC = D / (16 * VE);        // V pieces of a lane and key
    __shared__ __align__(16) uint32_t s_row[kPagedChunkMax];
    __shared__ float s_acc[4][16][D];
    __shared__ float2 s_ml[4][16];
    const int z = blockIdx.x;
    const int tiles = (a.group + 15) / 16;
    const int hk = blockIdx.y / tiles;
    const int g0 = (blockIdx.y - hk * tiles) * 16;
    const int s = blockIdx.z;
    const Seen e = seen_of(a.t, a.prefix, a.window, a.k_steps != nullptr, s);
    if (z == 0 && blockIdx.y == 0 && threadIdx.x == 0)
        a.seen[s] = make_uint4(e.none ? kPagedNone : e.nvis, e.p, e.shift, e.own ? 1u : 0u);
    if (e.none) return;
    const uint32_t chunk = split_keys(e.nvis, a.nsplit, a.split_least);
    const uint32_t b0 = static_cast<uint32_t>(z) * chunk;
    if (b0 >= e.nvis) return;
    const int cnt = static_cast<int>(min(chunk, e.nvis - b0));
    const int padded = (cnt + 15) & ~15;
    fill_rows(a.t, g, e, s, hk, b0, cnt, padded, s_row);
    const int wave = threadIdx.x >> 6;
    const int lane = threadIdx.x & 63;
    const int la = lane >> 4;
    const int lb = lane & 15;
    const bool head = g0 + lb < a.group;
    const size_t head0 = static_cast<size_t>(hk) * a.group + g0;
    const size_t n_heads = static_cast<size_t>(g.kv_heads) * a.group;
    // a lane without a head reads the last one's row and takes zeros
    const float* qr = a.q + static_cast<size_t>(s) * a.ldq + (static_cast<size_t>(hk) * a.group + min(g0 + lb, a.group - 1)) * D + la * E;
    const float qscale = a.scale * kLog2e;
    const int own = e.own && e.nvis - 1 - b0 < static_cast<uint32_t>(cnt) ? static_cast<int>(e.nvis - 1 - b0) : -1;
    float m, l;         // of head lb, this lane's keys
    v4f acc[VC][VE];    // of heads 4 la + r, columns (lb + 16 c) VE + j
    const u4* kp = static_cast<const u4*>(g.k) + la;
    const auto vload = [&](uint32_t row, int c) -> u4 {
        const char* p = static_cast<const char*>(g.v) + (static_cast<size_t>(row) * D + (lb + 16 * c) * VE) * sizeof(T);
        if constexpr (VE * sizeof(T) == 8) {
            const u2 w = *reinterpret_cast<const u2*>(p);
            return u4{w[0], w[1], 0, 0};
        } else {
            return *reinterpret_cast<const u4*>(p);
        }
    };
    // false, and nothing done, where q has no terms
    const auto run = [&](auto f32_products) -> bool {
        constexpr bool EXACT = decltype(f32_products)::value;
        constexpr bool APART = !EXACT && TT::kApart != 1.0f;
        m = -INFINITY;
        l = 0.0f;
#pragma unroll
        for (int c = 0; c < VC; ++c)
#pragma unroll
            for (int j = 0; j < VE; ++j) acc[c][j] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
        float q[KC][E];
#pragma unroll
        for (int c = 0; c < KC; ++c)
#pragma unroll
            for (int j = 0; j < E; ++j) q[c][j] = qr[4 * E * c + j] * qscale;
#pragma unroll
        for (int c = 0; c < KC; ++c)
#pragma unroll
            for (int j = 0; j < E; ++j) q[c][j] = head ? q[c][j] : 0.0f;
        u4 qt[TT::N][KC];
        float unscale = 1.0f;
        if constexpr (!EXACT) {
            if constexpr (TT::kTop != 0.0f) {  // a power of two that brings the row below 2^15
                float big = 0.0f;
#pragma unroll
                for (int c = 0; c < KC; ++c)
#pragma unroll
                    for (int j = 0; j < E; ++j) big = fmaxf(big, fabsf(q[c][j]));
                big = fold_lanes<16, 64>(big, Max());
                const int up = big > 0.0f && big < INFINITY ? min(max(14 - ilogbf(big), -100), 100) : 0;
                unscale = ldexpf(1.0f, -up);
                const float by = ldexpf(1.0f, up);
#pragma unroll
                for (int c = 0; c < KC; ++c)
#pragma unroll
                    for (int j = 0; j < E; ++j) q[c][j] *= by;
                uint32_t least = ~0u;
#pragma unroll
                for (int c = 0; c < KC; ++c)
#pragma unroll
                    for (int j = 0; j < E; ++j) least = min(least, size_order(q[c][j]));
                if (__any(least < size_order(TT::kLeast))) return false;
            }
#pragma unroll
            for (int c = 0; c < KC; ++c)
#pragma unroll
                for (int j = 0; j < E; j += 2) {
                    uint32_t w[TT::N];
                    TT::split2(q[c][j], q[c][j + 1], w);
#pragma unroll
                    for (int t = 0; t < TT::N; ++t) qt[t][c][j / 2] = w[t];
                }
        }
        for (int t0 = wave * 16; t0 < cnt; t0 += 64) {
            const uint32_t krow = s_row[t0 + lb];
            const uint4 vrow4 = *reinterpret_cast<const uint4*>(s_row + t0 + 4 * la);
            const uint32_t vrow[4] = {vrow4.x, vrow4.y, vrow4.z, vrow4.w};
            u4 kw[KC], vw[4][VC];
            if (__all(krow != kBadRow)) {
#pragma unroll
                for (int c = 0; c < KC; ++c) kw[c] = kp[static_cast<size_t>(krow) * C + 4 * c];
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int c = 0; c < VC; ++c) vw[i][c] = vload(vrow[i], c);
            } else {  // slots that hold no key are not read: what lies there may be NaN
#pragma unroll
                for (int c = 0; c < KC; ++c) kw[c] = krow != kBadRow ? kp[static_cast<size_t>(krow) * C + 4 * c] : u4{0, 0, 0, 0};
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int c = 0; c < VC; ++c) vw[i][c] = vrow[i] != kBadRow ? vload(vrow[i], c) : u4{0, 0, 0, 0};
            }
            if (own >= t0 && own < t0 + 16) {  // the step's row comes from the call and goes to its page
                const size_t at = static_cast<size_t>(s) * a.ldkv + static_cast<size_t>(hk) * D;
                float f[8];
                if (t0 + lb == own && krow != kBadRow) {
#pragma unroll
                    for (int c = 0; c < KC; ++c) {
#pragma unroll
                        for (int j = 0; j < E; ++j) f[j] = a.k_steps[at + (la + 4 * c) * E + j];
                        kw[c] = Row16<T>::pack(f);
                        if (g0 == 0) static_cast<u4*>(g.k)[static_cast<size_t>(krow) * C + la + 4 * c] = kw[c];
                    }
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if (t0 + 4 * la + i == own && vrow[i] != kBadRow) {
#pragma unroll
                        for (int c = 0; c < VC; ++c) {
#pragma unroll
                            for (int j = 0; j < E; ++j) f[j] = j < VE ? a.v_steps[at + (lb + 16 * c) * VE + j] : 0.0f;
                            vw[i][c] = Row16<T>::pack(f);
                            if (g0 == 0) {
                                char* p = static_cast<char*>(g.v) + (static_cast<size_t>(vrow[i]) * D + (lb + 16 * c) * VE) * sizeof(T);
                                if constexpr (VE * sizeof(T) == 8)
                                    *reinterpret_cast<u2*>(p) = u2{vw[i][c][0], vw[i][c][1]};
                                else
                                    *reinterpret_cast<u4*>(p) = vw[i][c];
                            }
                        }
                    }
                }
            }
            v4f sc = {0.0f, 0.0f, 0.0f, 0.0f}, sc_low = sc;
#pragma unroll
            for (int c = 0; c < KC; ++c) {
                if constexpr (EXACT) {
                    float f[E];
                    Row16<T>::load(kw[c], f);
#pragma unroll
                    for (int j = 0; j < E; ++j) sc = __builtin_amdgcn_mfma_f32_16x16x4f32(f[j], q[c][j], sc, 0, 0, 0);
                } else {  // the small terms first
#pragma unroll
                    for (int t = TT::N - 1; t >= 0; --t) {
                        v4f& to = APART && t ? sc_low : sc;
                        to = TT::scores(kw[c], qt[t][c], to);
                    }
                }
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if constexpr (APART) sc[i] = fmaf(sc_low[i], 1.0f / TT::kApart, sc[i]);
                if constexpr (!EXACT && TT::kTop != 0.0f) sc[i] *= unscale;
                sc[i] = vrow[i] != kBadRow ? sc[i] : -INFINITY;
            }
            if (a.scores && head) {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (t0 + 4 * la + i < cnt)
                        a.scores[(static_cast<size_t>(s) * n_heads + head0 + lb) * a.score_ld + b0 + t0 + 4 * la + i] = sc[i];
            }
            float mx = fmaxf(fmaxf(sc[0], sc[1]), fmaxf(sc[2], sc[3]));
            if (__any(mx > m + TT::kPast)) {
                mx = fmaxf(fold_lanes<16, 64>(mx, Max()) - TT::kTop, m);
                const float corr = __builtin_amdgcn_exp2f(m - (mx == -INFINITY ? 0.0f : mx));
                m = mx;
                l *= corr;
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const float cr = __shfl(corr, 4 * la + r, 64);
#pragma unroll
                    for (int c = 0; c < VC; ++c)
#pragma unroll
                        for (int j = 0; j < VE; ++j) acc[c][j][r] *= cr;
                }
            }
            const float safe = m == -INFINITY ? 0.0f : m;
            float p[4];
            uint32_t least = ~0u;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                p[i] = __builtin_amdgcn_exp2f(sc[i] - safe);
                l += p[i];
                least = min(least, size_order(p[i]));
            }
            const bool few = APART && __any(least < size_order(TT::kLeast));
            if (EXACT || few) {
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int c = 0; c < VC; ++c) {
                        float f[E];
                        Row16<T>::load(vw[i][c], f);
#pragma unroll
                        for (int j = 0; j < VE; ++j) acc[c][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(p[i], f[j], acc[c][j], 0, 0, 0);
                    }
                // and zeros for the terms: as the other branch these products took 46 registers more at D = 256
                if constexpr (APART) p[0] = p[1] = p[2] = p[3] = 0.0f;
            }
            if constexpr (!EXACT) {
                uint32_t w0[TT::N], w1[TT::N];
                TT::split2(p[0], p[1], w0);
                TT::split2(p[2], p[3], w1);
#pragma unroll
                for (int c = 0; c < VC; ++c) {
                    u2 v[VE];
#pragma unroll
                    for (int j = 0; j < VE; ++j) {  // a column of the four keys: halves of their words
                        const uint32_t sel = j & 1 ? 0x07060302u : 0x05040100u;
                        v[j] = u2{__builtin_amdgcn_perm(vw[1][c][j / 2], vw[0][c][j / 2], sel),
                                  __builtin_amdgcn_perm(vw[3][c][j / 2], vw[2][c][j / 2], sel)};
                    }
                    if constexpr (APART) {
                        // the later term's sums of a tile alone: held over all tiles they took as many registers as acc
#pragma unroll
                        for (int j0 = 0; j0 < VE; j0 += 2) {
                            v4f low[2];
#pragma unroll
                            for (int j = 0; j < 2; ++j) low[j] = TT::output(u2{w0[1], w1[1]}, v[j0 + j], v4f{0.0f, 0.0f, 0.0f, 0.0f});
#pragma unroll
                            for (int j = 0; j < 2; ++j) acc[c][j0 + j] = TT::output(u2{w0[0], w1[0]}, v[j0 + j], acc[c][j0 + j]);
#pragma unroll
                            for (int j = 0; j < 2; ++j)
#pragma unroll
                                for (int r = 0; r < 4; ++r) acc[c][j0 + j][r] = fmaf(low[j][r], 1.0f / TT::kApart, acc[c][j0 + j][r]);
                        }
                    } else {
#pragma unroll
                        for (int t = TT::N - 1; t >= 0; --t)  // independent products between those of one sum
#pragma unroll
                            for (int j = 0; j < VE; ++j) acc[c][j] = TT::output(u2{w0[t], w1[t]}, v[j], acc[c][j]);
                    }
                }
            }
        }
        return true;
    };
    __syncthreads();
    if constexpr (!TT::kSplit) {
        run(std::true_type{});
    } else {
        bool again = !run(std::false_type{});
        if (!again) {
            float bad = l * 0.0f;  // NaN where a sum is not finite
#pragma unroll
            for (int c = 0; c < VC; ++c)
#pragma unroll
                for (int j = 0; j < VE; ++j)
#pragma unroll
                    for (int r = 0; r < 4; ++r) bad += acc[c][j][r] * 0.0f;
            again = __any(bad != bad);
        }
        if (again) run(std::true_type{});
    }
    l = fold_lanes<16, 64>(l, Sum());
    if (lane < 16) s_ml[wave][lane] = make_float2(m, l);
#pragma unroll
    for (int c = 0; c < VC; ++c)
#pragma unroll
        for (int j = 0; j < VE; ++j)
#pragma unroll
            for (int r = 0; r < 4; ++r) s_acc[wave][4 * la + r][(lb + 16 * c) * VE + j] = acc[c][j][r];
    __syncthreads();
    join_waves<16, D>(a, s_acc, s_ml, g0, head0 + static_cast<size_t>(s) * n_heads, z);
}

// The splits of a row joined, out = sum_z acc_z f_z / sum_z l_z f_z with f_z =
// exp2(m_z - max m), in the order of the splits within each of the NT / (D /
// 4) groups of lanes, then over the groups.
template <int D, int NT>
__device__ __forceinline__ void join_row(const PagedAttend& a, int h, int n_heads, int s, const uint4& e) {
    constexpr int L4 = D / 4;
    constexpr int G = NT / L4;
    __shared__ float4 s_acc[G][L4];
    __shared__ float s_l[G];
    __shared__ float s_m[NT / 64];
    const uint32_t nvis = e.x;
    const uint32_t keys = split_keys(nvis, a.nsplit, a.split_least);
    const int n = static_cast<int>((nvis + keys - 1) / keys);
    const size_t part = (static_cast<size_t>(s) * n_heads + h) * a.nsplit;
    float m = -INFINITY;
    for (int z = threadIdx.x; z < n; z += NT) m = fmaxf(m, a.part_ml[part + z].x);
    m = wave_max_f_full(m);
    if ((threadIdx.x & 63) == 0) s_m[threadIdx.x >> 6] = m;
    __syncthreads();
    m = s_m[0];
#pragma unroll
    for (int i = 1; i < NT / 64; ++i) m = fmaxf(m, s_m[i]);
    const float sf = m == -INFINITY ? 0.0f : m;
    const int gi = threadIdx.x / L4;
    const int d4 = threadIdx.x % L4;
    float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    float l = 0.0f;
#pragma unroll 4
    for (int z = gi; z < n; z += G) {
        const float2 ml = a.part_ml[part + z];
        const float4 v = reinterpret_cast<const float4*>(a.part_acc + (part + z) * D)[d4];
        const float f = __builtin_amdgcn_exp2f(ml.x - sf);
        l = fmaf(ml.y, f, l);
        acc.x = fmaf(v.x, f, acc.x);
        acc.y = fmaf(v.y, f, acc.y);
        acc.z = fmaf(v.z, f, acc.z);
        acc.w = fmaf(v.w, f, acc.w);
    }
    s_acc[gi][d4] = acc;
    if (d4 == 0) s_l[gi] = l;
    __syncthreads();
    if (threadIdx.x < D) {
        const float* f = reinterpret_cast<const float*>(s_acc);
        float o = 0.0f, lt = 0.0f;
#pragma unroll
        for (int i = 0; i < G; ++i) {
            o += f[i * D + threadIdx.x];
            lt += s_l[i];
        }
        // no keys: zeros; keys whose scores are all -inf: 0 / 0, as the formula has it
        a.out[static_cast<size_t>(s) * a.ldo + static_cast<size_t>(h) * D + threadIdx.x] = nvis == 0 ? 0.0f : o / lt;
    }
    if (a.lens_advance && h == 0 && threadIdx.x == 0 && e.w != 0) a.lens_advance[s] += 1;
}

// weights[key] += sum over the key head's query heads of exp2(score - M) / L
// for kWeightKeys keys from j0 on, M and L joined from the splits again.
constexpr int kWeightKeys = 512;
template <int NT>
__device__ __forceinline__ void add_weights(const PagedAttend& a, int hk, int kv_heads, int s, const uint4& e, uint32_t j0) {
    __shared__ float2 s_ml[64];
    const uint32_t nvis = e.x;
    if (j0 >= nvis) return;
    const uint32_t keys = split_keys(nvis, a.nsplit, a.split_least);
    const int n = static_cast<int>((nvis + keys - 1) / keys);
    const size_t head0 = (static_cast<size_t>(s) * kv_heads + hk) * a.group;
    for (int i = threadIdx.x >> 6; i < a.group; i += NT / 64) {  // a wave a head
        const float2* ml = a.part_ml + (head0 + i) * a.nsplit;
        float m = -INFINITY, l = 0.0f;
        for (int z = threadIdx.x & 63; z < n; z += 64) m = fmaxf(m, ml[z].x);
        m = wave_max_f_full(m);
        const float sf = m == -INFINITY ? 0.0f : m;
        for (int z = threadIdx.x & 63; z < n; z += 64) l = fmaf(ml[z].y, __builtin_amdgcn_exp2f(ml[z].x - sf), l);
        l = wave_sum_f_full(l);
        if ((threadIdx.x & 63) == 0) s_ml[i] = make_float2(sf, l);
    }
    __syncthreads();
    const uint32_t end = min(j0 + kWeightKeys, nvis);
    for (uint32_t j = j0 + threadIdx.x; j < end; j += NT) {
        float w = 0.0f;
        for (int i = 0; i < a.group; ++i)
            w += __builtin_amdgcn_exp2f(a.scores[(head0 + i) * a.score_ld + j] - s_ml[i].x) / s_ml[i].y;
        const uint32_t key = j < e.y ? j : j + e.z;
        a.weights[(static_cast<size_t>(s) * kv_heads + hk) * a.ldw + key] += w;
    }
}

// Grid (head, then chunk of keys x key head where weights are gathered;
// sequence). The lengths are read from what the splits' launch noted: a step
// counts them up here.
template <int D, int NT>
__global__ __launch_bounds__(NT) void paged_join_kernel(PagedAttend a, int kv_heads) {
    const int s = blockIdx.y;
    const uint4 e = a.seen[s];
    if (e.x == kPagedNone) return;
    const int n_heads = kv_heads * a.group;
    const int b = static_cast<int>(blockIdx.x) - n_heads;
    if (b < 0)
        join_row<D, NT>(a, blockIdx.x, n_heads, s, e);
    else
        add_weights<NT>(a, b % kv_heads, kv_heads, s, e, static_cast<uint32_t>(b / kv_heads) * kWeightKeys);
}

// Rows of k / v [rows][kv_heads * D] into the slots (seq, pos) of the cache;
// a thread takes 16 bytes of a row.
template <typename T>
__global__ __launch_bounds__(256) void paged_write_kernel(PoolGeom g, int D, const float* __restrict__ k,
                                                          const float* __restrict__ v, size_t ld, size_t rows,
                                                          const uint32_t* seq, const uint32_t* pos,
                                                          const uint32_t* tables, int n_seqs, size_t max_pages) {
    constexpr int E = Row16<T>::N;
    const int C = D / E;
    const size_t per = static_cast<size_t>(g.kv_heads) * C;
    const size_t at = static_cast<size_t>(blockIdx.x) * 256 + threadIdx.x;
    const size_t row = at / per;
    if (row >= rows) return;
    const uint32_t hk = static_cast<uint32_t>((at - row * per) / C);
    const int cl = static_cast<int>((at - row * per) % C);
    const uint32_t p = pos[row];
    const uint32_t s = seq ? seq[row] : static_cast<uint32_t>(row);
    if (p == kPagedNone || s >= static_cast<uint32_t>(n_seqs) || (p >> g.page_shift) >= max_pages) return;
    const PagedTables t{tables, nullptr, n_seqs, max_pages, 0};
    const uint32_t dst = row_of(t, g, static_cast<int>(s), hk, p);
    if (dst == kBadRow) return;
    const size_t src = row * ld + static_cast<size_t>(hk) * D + static_cast<size_t>(cl) * E;
    float f[E];
#pragma unroll
    for (int j = 0; j < E; ++j) f[j] = k[src + j];
    static_cast<u4*>(g.k)[static_cast<size_t>(dst) * C + cl] = Row16<T>::pack(f);
#pragma unroll
    for (int j = 0; j < E; ++j) f[j] = v[src + j];
    static_cast<u4*>(g.v)[static_cast<size_t>(dst) * C + cl] = Row16<T>::pack(f);
}

// ---- eviction --------------------------------------------------------------------

// A weight as a whole number of the same order: NaN lowest, -0 as +0.
__device__ __forceinline__ uint32_t weight_key(float v) {
    if (v != v) return 0u;
    if (v == 0.0f) v = 0.0f;
    const uint32_t u = __float_as_uint(v);
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

// The threshold is found by digits of 11, 11 and 10 bits of the keys, from the
// top: a histogram of the keys that share the digits found so far, then the
// digit in whose bin the last of the wanted ones falls.
constexpr int kBins = 2048;
constexpr int kSelThreads = 1024;
constexpr int kSelWaves = kSelThreads / 64;
constexpr int kDigitShift[3] = {21, 10, 0};

struct Pick {
    uint32_t found, want;  // the digits so far; how many of the keys that share them stay
};

// The sum of this lane's and the lower lanes' values: shifts within the 16-lane
// rows, then row 0's and 2's last lanes to the rows behind them, then lane 31's.
__device__ __forceinline__ uint32_t wave_prefix(uint32_t v) {
    int x = static_cast<int>(v);
    x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xF, 0xF, false);  // row_shr:1
    x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xF, 0xF, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xF, 0xF, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xF, 0xF, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xA, 0xF, false);  // row_bcast:15 into rows 1 and 3
    x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xC, 0xF, false);  // row_bcast:31 into rows 2 and 3
    return static_cast<uint32_t>(x);
}

// Bins from the top until `want` keys are counted; hist in LDS or registers:
// thread t holds the counts of bins 2047 - 2 t and 2046 - 2 t.
__device__ __forceinline__ Pick find_digit(uint32_t hi, uint32_t lo, Pick p, int shift, uint32_t* s_wave, Pick* s_pick) {
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const uint32_t sum = hi + lo;
    const uint32_t incl = wave_prefix(sum);
    if (lane == 63) s_wave[wave] = incl;
    __syncthreads();
    uint32_t before = incl - sum;
#pragma unroll
    for (int i = 0; i < kSelWaves; ++i) before += i < wave ? s_wave[i] : 0u;
    if (before < p.want && p.want - before <= sum) {
        const uint32_t bin = kBins - 1 - 2 * threadIdx.x;
        const bool up = p.want - before <= hi;
        s_pick->found = p.found | ((up ? bin : bin - 1) << shift);
        s_pick->want = p.want - before - (up ? 0u : hi);
    }
    __syncthreads();
    return *s_pick;
}

// A thread's keys of a tile of kSelThreads * KPT slots: slot (wave KPT + i) 64
// + lane of the tile, so that the slots of a wave follow each other.
template <int KPT>
struct SelTile {
    float v[KPT];
    uint32_t j0;
    __device__ __forceinline__ uint32_t slot(int i) const { return j0 + i * 64; }
    __device__ __forceinline__ void load(const float* w, const Cut& c, uint32_t tile) {
        j0 = tile * (kSelThreads * KPT) + (threadIdx.x >> 6) * (KPT * 64) + (threadIdx.x & 63);
#pragma unroll
        for (int i = 0; i < KPT; ++i) v[i] = slot(i) < c.n ? w[slot(i)] : 0.0f;
    }
    __device__ __forceinline__ bool middle(const Cut& c, int i) const { return slot(i) >= c.lo && slot(i) < c.hi; }
    __device__ __forceinline__ void count(const Cut& c, uint32_t found, int pass, uint32_t* s_hist) const {
        const int shift = kDigitShift[pass];
        const uint32_t mask = pass == 2 ? 1023u : kBins - 1u;
        const int known = pass == 0 ? 32 : kDigitShift[pass - 1];
#pragma unroll
        for (int i = 0; i < KPT; ++i) {
            const uint32_t k = weight_key(v[i]);
            if (middle(c, i) && (pass == 0 || (k >> known) == (found >> known))) atomicAdd(&s_hist[(k >> shift) & mask], 1u);
        }
    }
    // The slots that stay, in order, behind `above` slots above the threshold
    // and `equal` at it; advances both by the tile's.
    __device__ __forceinline__ void place(const Cut& c, Pick t, uint32_t& above, uint32_t& equal, uint32_t (*s_n)[kSelWaves],
                                          uint32_t* kept, float* dw) const {
        const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
        const uint64_t below = (1ull << lane) - 1;
        uint32_t na = 0, ne = 0;
#pragma unroll
        for (int i = 0; i < KPT; ++i) {
            na += __popcll(__ballot(is_above(c, t, i)));
            ne += __popcll(__ballot(is_equal(c, t, i)));
        }
        if (lane == 0) {
            s_n[0][wave] = na;
            s_n[1][wave] = ne;
        }
        __syncthreads();
        uint32_t wa = above, we = equal;
#pragma unroll
        for (int i = 0; i < kSelWaves; ++i) {
            wa += i < wave ? s_n[0][i] : 0u;
            we += i < wave ? s_n[1][i] : 0u;
            above += s_n[0][i];
            equal += s_n[1][i];
        }
#pragma unroll
        for (int i = 0; i < KPT; ++i) {
            const bool up = is_above(c, t, i), eq = is_equal(c, t, i);
            const uint64_t ma = __ballot(up), me = __ballot(eq);
            const uint32_t e0 = we + __popcll(me & below);  // equal ones before this slot
            if (up || (eq && e0 < t.want)) {
                const uint32_t to = wa + __popcll(ma & below) + min(e0, t.want);
                kept[to] = slot(i);
                dw[to] = v[i];
            }
            wa += __popcll(ma);
            we += __popcll(me);
        }
        __syncthreads();
    }
    __device__ __forceinline__ bool is_above(const Cut& c, Pick t, int i) const {
        return slot(i) < c.n && (c.whole || !middle(c, i) || (t.want != 0u && weight_key(v[i]) > t.found));
    }
    __device__ __forceinline__ bool is_equal(const Cut& c, Pick t, int i) const {
        return !c.whole && t.want != 0u && middle(c, i) && weight_key(v[i]) == t.found;
    }
};

// Grid (key head, sequence): a row of weights by one block, in registers where
// it fits a tile (read once), else a tile at a time in every pass.
template <int KPT>
__global__ __launch_bounds__(kSelThreads) void paged_select_kernel(PagedEvict a, uint32_t kv_heads) {
    __shared__ uint32_t s_hist[kBins];
    __shared__ uint32_t s_n[2][kSelWaves];
    __shared__ Pick s_pick;
    const int hk = blockIdx.x;
    const int s = blockIdx.y;
    const Cut c = cut_of(a, s);
    if (c.none) return;
    const size_t row = static_cast<size_t>(s) * kv_heads + hk;
    const float* w = a.weights + row * a.ldw;
    const uint32_t tiles = (c.n + kSelThreads * KPT - 1) / (kSelThreads * KPT);
    SelTile<KPT> t;
    t.load(w, c, 0);
    Pick p{0u, c.want};
    if (!c.whole && c.want != 0) {
        for (int pass = 0; pass < 3; ++pass) {
            s_hist[threadIdx.x] = s_hist[threadIdx.x + kSelThreads] = 0u;
            __syncthreads();
            for (uint32_t i = 0; i < tiles; ++i) {
                if (tiles > 1) t.load(w, c, i);
                t.count(c, p.found, pass, s_hist);
            }
            __syncthreads();
            p = find_digit(s_hist[kBins - 1 - 2 * threadIdx.x], s_hist[kBins - 2 - 2 * threadIdx.x], p, kDigitShift[pass], s_n[0], &s_pick);
        }
    }
    uint32_t above = 0, equal = 0;
    for (uint32_t i = 0; i < tiles; ++i) {
        if (tiles > 1) t.load(w, c, i);
        t.place(c, p, above, equal, s_n, a.kept + row * a.budget, a.dst_weights + row * a.dst_ldw);
    }
}

// The same for few long rows: a block to a tile of a row, a launch to a pass.
// Every block writes its histogram to [row][tile][pass]; the next launch's
// blocks each add up their row's and find its digit again.
constexpr int kLongKpt = 8;
constexpr uint32_t kLongTile = kSelThreads * kLongKpt;

// The digit of a pass from the row's histograms, and in `above` how many keys of
// this block's tile (own) or of the tiles before it lie past the digit, in
// `at` how many at it.
__device__ __forceinline__ Pick long_digit(const uint32_t* hist, uint32_t tiles, uint32_t tile, bool own, int pass, Pick p,
                                           uint32_t* s_wave, Pick* s_pick, uint32_t& above, uint32_t& at) {
    uint32_t hi = 0, lo = 0, mine_hi = 0, mine_lo = 0;
    const uint32_t* h = hist + static_cast<size_t>(pass) * kBins + (kBins - 2 - 2 * threadIdx.x);
#pragma unroll 8
    for (uint32_t i = 0; i < tiles; ++i) {
        const uint2 n = *reinterpret_cast<const uint2*>(h + static_cast<size_t>(i) * 3 * kBins);
        const bool m = own ? i == tile : i < tile;
        lo += n.x;
        hi += n.y;
        mine_lo += m ? n.x : 0u;
        mine_hi += m ? n.y : 0u;
    }
    p = find_digit(hi, lo, p, kDigitShift[pass], s_wave, s_pick);
    const uint32_t digit = (p.found >> kDigitShift[pass]) & (pass == 2 ? 1023u : kBins - 1u);
    const uint32_t bin = kBins - 1 - 2 * threadIdx.x;
    above = (bin > digit ? mine_hi : 0u) + (bin - 1 > digit ? mine_lo : 0u);
    at = bin == digit ? mine_hi : bin - 1 == digit ? mine_lo : 0u;
    return p;
}

// The block's sums of two counts, in every thread.
__device__ __forceinline__ void block_sum2(uint32_t& x, uint32_t& y, uint32_t (*s_n)[kSelWaves]) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        x += __shfl_xor(x, o, 64);
        y += __shfl_xor(y, o, 64);
    }
    __syncthreads();
    if ((threadIdx.x & 63) == 0) {
        s_n[0][threadIdx.x >> 6] = x;
        s_n[1][threadIdx.x >> 6] = y;
    }
    __syncthreads();
    x = y = 0;
#pragma unroll
    for (int i = 0; i < kSelWaves; ++i) {
        x += s_n[0][i];
        y += s_n[1][i];
    }
    __syncthreads();
}

// counts [row][tile][2]: the keys of a tile past the first and second digit.
struct LongRows {
    Pick* picks;       // [rows][2]
    uint32_t* counts;  // [rows][tiles][2]
    uint32_t* hist;    // [rows][tiles][3][kBins]
};

__global__ __launch_bounds__(kSelThreads) void paged_hist_kernel(PagedEvict a, uint32_t kv_heads, LongRows r, int pass) {
    __shared__ uint32_t s_hist[kBins];
    __shared__ uint32_t s_n[2][kSelWaves];
    __shared__ Pick s_pick;
    const uint32_t tile = blockIdx.x;
    const int s = blockIdx.z;
    const Cut c = cut_of(a, s);
    if (c.none || c.whole || c.want == 0 || tile * kLongTile >= c.n) return;
    const size_t row = static_cast<size_t>(s) * kv_heads + blockIdx.y;
    const uint32_t tiles = (c.n + kLongTile - 1) / kLongTile;
    uint32_t* rh = r.hist + row * gridDim.x * 3 * kBins;
    SelTile<kLongKpt> t;
    t.load(a.weights + row * a.ldw, c, tile);
    s_hist[threadIdx.x] = s_hist[threadIdx.x + kSelThreads] = 0u;
    Pick p{0u, c.want};
    if (pass > 0) {
        if (pass > 1) p = r.picks[row * 2];
        uint32_t above, at;
        p = long_digit(rh, tiles, tile, true, pass - 1, p, s_n[0], &s_pick, above, at);
        block_sum2(above, at, s_n);
        if (threadIdx.x == 0) {
            r.counts[(row * gridDim.x + tile) * 2 + pass - 1] = above;
            if (tile == 0) r.picks[row * 2 + pass - 1] = p;
        }
    }
    __syncthreads();
    t.count(c, p.found, pass, s_hist);
    __syncthreads();
    uint32_t* to = rh + (static_cast<size_t>(tile) * 3 + pass) * kBins;
    to[threadIdx.x] = s_hist[threadIdx.x];
    to[threadIdx.x + kSelThreads] = s_hist[threadIdx.x + kSelThreads];
}

__global__ __launch_bounds__(kSelThreads) void paged_place_kernel(PagedEvict a, uint32_t kv_heads, LongRows r) {
    __shared__ uint32_t s_n[2][kSelWaves];
    __shared__ Pick s_pick;
    const uint32_t tile = blockIdx.x;
    const int s = blockIdx.z;
    const Cut c = cut_of(a, s);
    if (c.none || tile * kLongTile >= c.n) return;
    const size_t row = static_cast<size_t>(s) * kv_heads + blockIdx.y;
    SelTile<kLongKpt> t;
    t.load(a.weights + row * a.ldw, c, tile);
    const uint32_t tiles = (c.n + kLongTile - 1) / kLongTile;
    Pick p{0u, c.want};
    uint32_t above = 0, equal = 0;
    if (!c.whole && c.want != 0) {
        p = long_digit(r.hist + row * gridDim.x * 3 * kBins, tiles, tile, false, 2, r.picks[row * 2 + 1], s_n[0], &s_pick, above, equal);
        for (uint32_t i = threadIdx.x; i < 2 * tile; i += kSelThreads) above += r.counts[row * gridDim.x * 2 + i];
        block_sum2(above, equal, s_n);
    }
    const uint32_t first = tile * kLongTile;  // and the slots before it that stay anyway
    above += c.whole ? first : min(first, c.lo) + (first > c.hi ? first - c.hi : 0u);
    t.place(c, p, above, equal, s_n, a.kept + row * a.budget, a.dst_weights + row * a.dst_ldw);
}

// Rows of a thread: 8 x 8192 -> 2048 slots took 52 us at 1, 53 at 2, 58 at 4 and
// 87 at 8; stores past the caches made that 46 at 2 (52 at 4).
constexpr int kGatherRows = 2;

// Grid (tile of kept slots, key head, sequence): their rows into the pages of
// dst_tables, 16 bytes a lane. The new lengths are written here: dst_lens may
// be lens, and min(length, budget) is the same of the old and the new.
template <int C>
__global__ __launch_bounds__(256) void paged_gather_kernel(PoolGeom g, PagedEvict a) {
    constexpr int R = 256 / C;  // rows a step
    constexpr int U = kGatherRows;
    const int hk = blockIdx.y;
    const int s = blockIdx.z;
    const uint32_t len = a.t.lens[s];
    const uint32_t n = min(min(len, a.t.max_len), a.budget);
    if (blockIdx.x == 0 && hk == 0 && threadIdx.x == 0) a.dst_lens[s] = len == kPagedNone ? kPagedNone : n;
    const uint32_t i0 = blockIdx.x * (R * U);
    if (len == kPagedNone || i0 >= n) return;
    const int cl = threadIdx.x % C;
    const uint32_t* kept = a.kept + (static_cast<size_t>(s) * g.kv_heads + hk) * a.budget;
    const PagedTables dst{a.dst_tables, nullptr, a.t.n_seqs, a.dst_max_pages, 0};
    uint32_t from[U], to[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const uint32_t i = i0 + u * R + threadIdx.x / C;
        from[u] = to[u] = kBadRow;
        if (i < n) {
            from[u] = row_of(a.t, g, s, hk, kept[i]);
            to[u] = row_of(dst, g, s, hk, i);
        }
        if (from[u] == kBadRow) to[u] = kBadRow;
    }
    u4 kw[U], vw[U];
    const u4* kp = static_cast<const u4*>(g.k) + cl;
    const u4* vp = static_cast<const u4*>(g.v) + cl;
#pragma unroll
    for (int u = 0; u < U; ++u) {
        if (to[u] != kBadRow) {
            kw[u] = kp[static_cast<size_t>(from[u]) * C];
            vw[u] = vp[static_cast<size_t>(from[u]) * C];
        }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
        if (to[u] != kBadRow) {
            __builtin_nontemporal_store(kw[u], static_cast<u4*>(g.k) + static_cast<size_t>(to[u]) * C + cl);
            __builtin_nontemporal_store(vw[u], static_cast<u4*>(g.v) + static_cast<size_t>(to[u]) * C + cl);
        }
    }
}

// ---- checks, for calls that ask for them ---------------------------------------------

__device__ __forceinline__ void fault(unsigned long long* err, uint32_t row, int code) {
    atomicMin(err, (static_cast<unsigned long long>(row) << 8) | static_cast<unsigned long long>(code));
}

__global__ void paged_check_kernel(PoolGeom g, PagedTables t, uint32_t add, const uint32_t* prefix, uint32_t window,
                                   unsigned long long* err) {
    const int s = blockIdx.x;
    const uint32_t len = t.lens[s];
    if (len == kPagedNone) return;
    if (len > t.max_len || t.max_len - len < add) {
        if (threadIdx.x == 0) fault(err, s, kFaultLen);
        return;
    }
    const Seen e = seen_of(t, prefix, window, add != 0, s);
    const uint32_t unit = 1u << g.page_shift;
    // every page that holds a key that is seen
    for (uint32_t pg = threadIdx.x; static_cast<uint64_t>(pg) * unit < e.n; pg += blockDim.x) {
        const uint32_t first = pg * unit, last = min(first + unit, e.n);
        const bool used = first < e.p || last > e.p + e.shift;
        if (used && t.tables[static_cast<size_t>(s) * t.max_pages + pg] >= g.n_pages) fault(err, s, kFaultPage);
    }
}

__global__ void paged_check_rows_kernel(PoolGeom g, size_t rows, const uint32_t* seq, const uint32_t* pos,
                                        const uint32_t* tables, int n_seqs, size_t max_pages,
                                        unsigned long long* err) {
    const size_t row = static_cast<size_t>(blockIdx.x) * blockDim.x + threadIdx.x;
    if (row >= rows) return;
    const uint32_t p = pos[row];
    if (p == kPagedNone) return;
    const uint32_t s = seq ? seq[row] : static_cast<uint32_t>(row);
    const uint32_t at = static_cast<uint32_t>(row);
    if (s >= static_cast<uint32_t>(n_seqs)) return fault(err, at, kFaultSeq);
    if ((p >> g.page_shift) >= max_pages) return fault(err, at, kFaultLen);
    if (tables[static_cast<size_t>(s) * max_pages + (p >> g.page_shift)] >= g.n_pages) fault(err, at, kFaultPage);
}

__global__ void clear_words_kernel(uint32_t* p, size_t n) {
    const size_t i = static_cast<size_t>(blockIdx.x) * blockDim.x + threadIdx.x;
    if (i < n) p[i] = 0u;
}

// marks: a bit for every page that a sequence reads
__global__ void paged_mark_kernel(PoolGeom g, PagedTables t, uint32_t* marks) {
    const int s = blockIdx.x;
    const uint32_t len = t.lens[s];
    if (len == kPagedNone) return;
    const uint32_t n = min(len, t.max_len);
    for (uint32_t pg = threadIdx.x; (static_cast<uint64_t>(pg) << g.page_shift) < n; pg += blockDim.x) {
        const uint32_t page = t.tables[static_cast<size_t>(s) * t.max_pages + pg];
        if (page < g.n_pages) atomicOr(marks + (page >> 5), 1u << (page & 31));
    }
}

// the pages written: of the pool, read by none, each written once
__global__ void paged_check_dst_kernel(PoolGeom g, PagedEvict a, uint32_t* marks, unsigned long long* err) {
    const int s = blockIdx.x;
    const uint32_t len = a.t.lens[s];
    if (len == kPagedNone) return;
    const uint32_t n = min(min(len, a.t.max_len), a.budget);
    for (uint32_t pg = threadIdx.x; (static_cast<uint64_t>(pg) << g.page_shift) < n; pg += blockDim.x) {
        const uint32_t page = a.dst_tables[static_cast<size_t>(s) * a.dst_max_pages + pg];
        if (page >= g.n_pages) {
            fault(err, s, kFaultDstPage);
            continue;
        }
        if (atomicOr(marks + (page >> 5), 1u << (page & 31)) & (1u << (page & 31))) fault(err, s, kFaultDstShared);
    }
}

template <typename T, int D>
void attend(hipStream_t s, const focr_hip_paged* c, const PagedAttend& a) {
    const PoolGeom g = geom_of(c);
    const int kv = static_cast<int>(c->n_kv_heads);
    const auto grid = [&](int gt) { return dim3(a.nsplit, kv * ((a.group + gt - 1) / gt), a.t.n_seqs); };
    // By query heads to a key head (one, two, three, four), VALU kernel / matrix
    // cores, us; ragged sequences of up to 16384 keys on 2 key heads, 560 MB in all:
    //   bf16  64 wide  106/108  109/111  115/113  136/115
    //   bf16 128 wide  109/113  114/115  119/117  131/119
    //   bf16 256 wide  113/133  119/136  125/139  135/142
    //   f16   64 wide  106/108  109/111  114/114  131/115
    //   f16  128 wide  109/114  114/117  119/119  124/120
    //   f16  256 wide  113/119  118/122  125/124  134/126
    //   f32   64 wide  106/112  109/113  112/115  116/117
    //   f32  128 wide  110/117  113/119  116/121  121/122
    //   f32  256 wide  107/140  112/142  116/143  121/146
    // One rule for all of them: three heads in f32, and three and four in bf16
    // and f32 at 256 wide, are the faster on the VALU by what stands here.
    if (a.group > 2)
        FOCR_LAUNCH((paged_attend_mfma_kernel<T, D>), grid(16), dim3(256), 0, s, g, a);
    else if (a.group == 2)
        FOCR_LAUNCH((paged_attend_kernel<T, D, 2, 8>), grid(2), dim3(256), 0, s, g, a);
    else
        FOCR_LAUNCH((paged_attend_kernel<T, D, 1, 8>), grid(1), dim3(256), 0, s, g, a);
}

template <int D, int NT>
void launch_join(hipStream_t s, dim3 grid, const PagedAttend& a, int kv) {
    FOCR_LAUNCH((paged_join_kernel<D, NT>), grid, dim3(NT), 0, s, a, kv);
}

template <typename T>
void attend_dim(hipStream_t s, const focr_hip_paged* c, const PagedAttend& a) {
    if (c->head_dim == 64)
        attend<T, 64>(s, c, a);
    else if (c->head_dim == 128)
        attend<T, 128>(s, c, a);
    else
        attend<T, 256>(s, c, a);
}

}  // namespace

PagedSplits paged_pick_splits(size_t n_seqs, size_t kv_heads, int group, uint32_t max_seen, bool window, int cu_count) {
    return pick_splits(n_seqs, kv_heads, group, max_seen, window, cu_count);
}

hipError_t launch_paged_attend(hipStream_t s, const focr_hip_paged* c, const PagedAttend& a, focr_hip_ctx* ctx) {
    const int kv = static_cast<int>(c->n_kv_heads);
    {
        ProfScope ps(ctx, "paged_attend");
        if (c->dtype == FOCR_HIP_DT_F32)
            attend_dim<float>(s, c, a);
        else if (c->dtype == FOCR_HIP_DT_F16)
            attend_dim<_Float16>(s, c, a);
        else
            attend_dim<__bf16>(s, c, a);
    }
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    ProfScope ps(ctx, "paged_join");
    const uint32_t chunks = a.weights ? static_cast<uint32_t>((a.score_ld + kWeightKeys - 1) / kWeightKeys) : 0;
    const dim3 grid(kv * (a.group + chunks), a.t.n_seqs);
    // 1024 threads where a row has many splits to join (64 rows of 256 splits: 10
    // -> 7.5 us). Whole calls at 256 / 1024 threads, us: 2 x 16384 keys, 32 heads
    // on 8, 32.7 / 32.2, 2 x 131071 171 / 169, 64 x 65536, 16 on 2, 233 / 234;
    // with weights, whose blocks then have 512 keys for 1024 threads, 36.1 / 35.5,
    // 204 / 216, 352 / 394.
    const bool many = a.nsplit > 64;
    if (c->head_dim == 64)
        many ? launch_join<64, 1024>(s, grid, a, kv) : launch_join<64, 256>(s, grid, a, kv);
    else if (c->head_dim == 128)
        many ? launch_join<128, 1024>(s, grid, a, kv) : launch_join<128, 256>(s, grid, a, kv);
    else
        many ? launch_join<256, 1024>(s, grid, a, kv) : launch_join<256, 256>(s, grid, a, kv);
    return hipGetLastError();
}

hipError_t launch_paged_write(hipStream_t s, const focr_hip_paged* c, const float* k, const float* v, size_t ld,
                              size_t rows, const uint32_t* seq, const uint32_t* pos, const uint32_t* tables,
                              int n_seqs, size_t max_pages) {
    const PoolGeom g = geom_of(c);
    const int D = static_cast<int>(c->head_dim);
    const size_t units = rows * c->n_kv_heads * c->head_dim * c->esize() / 16;
    const dim3 grid(static_cast<uint32_t>((units + 255) / 256));
    if (c->dtype == FOCR_HIP_DT_F32)
        FOCR_LAUNCH(paged_write_kernel<float>, grid, dim3(256), 0, s, g, D, k, v, ld, rows, seq, pos, tables, n_seqs,
                    max_pages);
    else if (c->dtype == FOCR_HIP_DT_F16)
        FOCR_LAUNCH(paged_write_kernel<_Float16>, grid, dim3(256), 0, s, g, D, k, v, ld, rows, seq, pos, tables,
                    n_seqs, max_pages);
    else
        FOCR_LAUNCH(paged_write_kernel<__bf16>, grid, dim3(256), 0, s, g, D, k, v, ld, rows, seq, pos, tables, n_seqs,
                    max_pages);
    return hipGetLastError();
}

// A block to a row keeps up to 16384 keys in registers and reads longer rows in
// every pass; a block to a tile takes four dependent launches. Whole evictions,
// block to a row / to a tile, us: 10 rows of 12000 slots 25 / 30, of 20000 44 /
// 32, of 33000 62 / 34; 80 rows 27 / 34, 46 / 35, 64 / 48; 240 rows 35 / 57,
// 54 / 70, 74 / 91.
size_t paged_evict_hist_words(size_t rows, uint32_t max_len, int cu_count) {
    const size_t tiles = (static_cast<size_t>(max_len) + kLongTile - 1) / kLongTile;
    return max_len > 16 * kSelThreads && 2 * rows <= static_cast<size_t>(cu_count) ? rows * (4 + tiles * (2 + 3 * kBins)) : 0;
}

hipError_t launch_paged_evict(hipStream_t s, const focr_hip_paged* c, const PagedEvict& a, focr_hip_ctx* ctx) {
    const PoolGeom g = geom_of(c);
    {
        ProfScope ps(ctx, "paged_select");
        const dim3 rows(g.kv_heads, a.t.n_seqs), block(kSelThreads);
        if (a.hist) {
            const dim3 grid((a.t.max_len + kLongTile - 1) / kLongTile, g.kv_heads, a.t.n_seqs);
            const size_t n = static_cast<size_t>(a.t.n_seqs) * g.kv_heads;
            const LongRows r{reinterpret_cast<Pick*>(a.hist), a.hist + 4 * n, a.hist + 4 * n + 2 * n * grid.x};
            for (int pass = 0; pass < 3; ++pass) FOCR_LAUNCH(paged_hist_kernel, grid, block, 0, s, a, g.kv_heads, r, pass);
            FOCR_LAUNCH(paged_place_kernel, grid, block, 0, s, a, g.kv_heads, r);
        } else if (a.t.max_len <= 2 * kSelThreads) {
            FOCR_LAUNCH(paged_select_kernel<2>, rows, block, 0, s, a, g.kv_heads);
        } else if (a.t.max_len <= 8 * kSelThreads) {
            FOCR_LAUNCH(paged_select_kernel<8>, rows, block, 0, s, a, g.kv_heads);
        } else {
            FOCR_LAUNCH(paged_select_kernel<16>, rows, block, 0, s, a, g.kv_heads);
        }
    }
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    ProfScope ps(ctx, "paged_gather");
    const uint32_t most = std::min(a.budget, a.t.max_len);
    const int lanes = static_cast<int>(c->head_dim * c->esize() / 16);
    const uint32_t rows = kGatherRows * (256 / lanes);
    const dim3 grid(std::max<uint32_t>((most + rows - 1) / rows, 1), g.kv_heads, a.t.n_seqs);
    if (lanes == 8)
        FOCR_LAUNCH(paged_gather_kernel<8>, grid, dim3(256), 0, s, g, a);
    else if (lanes == 16)
        FOCR_LAUNCH(paged_gather_kernel<16>, grid, dim3(256), 0, s, g, a);
    else if (lanes == 32)
        FOCR_LAUNCH(paged_gather_kernel<32>, grid, dim3(256), 0, s, g, a);
    else
        FOCR_LAUNCH(paged_gather_kernel<64>, grid, dim3(256), 0, s, g, a);
    return hipGetLastError();
}

hipError_t launch_paged_check(hipStream_t s, const focr_hip_paged* c, const PagedTables& t, uint32_t add,
                              const uint32_t* prefix, uint32_t window, unsigned long long* err) {
    FOCR_LAUNCH(paged_check_kernel, dim3(t.n_seqs), dim3(256), 0, s, geom_of(c), t, add, prefix, window, err);
    return hipGetLastError();
}

hipError_t launch_paged_check_rows(hipStream_t s, const focr_hip_paged* c, size_t rows, const uint32_t* seq,
                                   const uint32_t* pos, const uint32_t* tables, int n_seqs, size_t max_pages,
                                   unsigned long long* err) {
    FOCR_LAUNCH(paged_check_rows_kernel, dim3(static_cast<uint32_t>((rows + 255) / 256)), dim3(256), 0, s, geom_of(c),
                rows, seq, pos, tables, n_seqs, max_pages, err);
    return hipGetLastError();
}

hipError_t launch_clear_words(hipStream_t s, uint32_t* p, size_t n) {
    FOCR_LAUNCH(clear_words_kernel, dim3(static_cast<uint32_t>((n + 255) / 256)), dim3(256), 0, s, p, n);
    return hipGetLastError();
}

hipError_t launch_paged_check_dst(hipStream_t s, const focr_hip_paged* c, const PagedEvict& a, uint32_t* marks,
                                  unsigned long long* err) {
    const PoolGeom g = geom_of(c);
    hipError_t e = launch_clear_words(s, marks, (c->n_pages + 31) / 32);
    if (e != hipSuccess) return e;
    FOCR_LAUNCH(paged_mark_kernel, dim3(a.t.n_seqs), dim3(256), 0, s, g, a.t, marks);
    FOCR_LAUNCH(paged_check_dst_kernel, dim3(a.t.n_seqs), dim3(256), 0, s, g, a, marks, err);
    return hipGetLastError();
}

}  // namespace focr
