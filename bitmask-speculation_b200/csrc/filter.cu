// Filtered sampling: temperature, top-k, top-p and min-p over masked rows, one given uniform per row.
//
// For a row x under mask A at temperature T > 0, order the valid finite tokens by (x descending, token ascending);
// w_i = exp((x_i - max) / T) in float64.  Kept is the shortest of three prefixes of that order: the first
// top_k tokens; of their total mass the tokens whose preceding mass is below top_p * total; the tokens
// with w >= min_p.  The result is the lowest kept token whose running mass in token order exceeds u * kept mass.
//
// A cluster of C CTAs owns a row, each CTA a contiguous slice, each warp a contiguous span of it.  The
// row is streamed from HBM once (maximum, counts, NaN); later passes hit L2, because only the rows in
// flight are live there.  Order keys are 64-bit: ordered float bits, then the complement of the token, so that ties
// are part of the key and every prefix is "key >= cut".
//
// Passes.  The first one also gives a lower bound of the k-th largest score for free: G disjoint
// groups of lanes each hold a token at or above the smallest of their maxima, so at least G tokens reach it.
//  * Few tokens in play (k small, min-p alone, or a sparse mask): they are collected into shared
//    memory, sorted, weighed and cut there; only they are ever exponentiated.
//  * Otherwise one counting pass over value bins estimates where the nucleus ends, one weighing pass
//    sums the exact masses above and below a bracket of bins around that place and collects the
//    bracket's tokens, whose sorted prefix gives the exact cut; if the estimate missed or a
//    bracket overflows (runs of equal scores), the cut is bisected over the order keys instead.
//    A last pass weighs the kept tokens by spans, and one CTA walks the span that holds u.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cfloat>
#include <cmath>
#include <cstring>

#include "../../include/bms_b200.h"
#include "abi_common.cuh"

namespace bms {
namespace {

namespace cg = cooperative_groups;

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxCluster = 16;
constexpr int kCap = 4096;   // tokens that the list path holds
constexpr int kBins = 8192;  // value bins of the counting pass
constexpr int kPerThread = kBins / kThreads;

struct FilterParams {
    const void* logits;
    const int32_t* masks;
    const int32_t* mask_rows;
    int64_t mask_table_rows, rows, vocab, words;
    double temperature, top_p, min_p;
    int64_t top_k;
    const float *temperatures, *top_ps, *min_ps;
    const int32_t* top_ks;
    const double* uniforms;
    int64_t* tokens;
    int64_t* kept;
    int32_t* status;
};

struct RowStats {
    float max;               // maximum of the valid tokens
    float low[3];            // smallest maximum of the groups of 32, 8 and 1 lanes
    uint32_t finite, flags;  // valid finite tokens; 1 NaN, 2 some valid token
};

__device__ __forceinline__ void merge(RowStats& a, const RowStats& o) {
    a.max = fmaxf(a.max, o.max);
#pragma unroll
    for (int i = 0; i < 3; ++i) a.low[i] = fminf(a.low[i], o.low[i]);
    a.finite += o.finite;
    a.flags |= o.flags;
}

struct MassCount {
    double mass;
    int64_t count;
};

struct Shared {
    union {
        uint64_t list[kCap];
        uint32_t bins[kBins];  // this CTA's counts, until every CTA has read them
    };
    double weight[kCap];
    uint32_t merged[kBins];
    double spans[kMaxCluster * kWarps];
    MassCount part[2][kMaxCluster];
    RowStats stats[kMaxCluster];
    double warp_mass[kWarps];
    int64_t warp_count[kWarps];
    double exp_table[64];  // 2^(j / 64)
    uint64_t cut;
    double above[kMaxCluster], below[kMaxCluster];
    uint32_t list_counts[kMaxCluster];
    uint32_t list_count, list_base;
    int32_t bin[3];
    uint32_t bin_count;
    float goal;
    int32_t found, owner;
    double before;
    uint32_t pick;
    int64_t token;
};

__device__ __forceinline__ uint32_t order_bits(float x) {
    const uint32_t b = __float_as_uint(x + 0.0f);  // -0 ranks with +0
    return b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u);
}

__device__ __forceinline__ float order_value(uint32_t k) { return __uint_as_float((k >> 31) ? k ^ 0x80000000u : ~k); }

__device__ __forceinline__ uint64_t order_key(float x, uint32_t token) {
    return (static_cast<uint64_t>(order_bits(x)) << 32) | (0xffffffffu - token);
}

__device__ __forceinline__ float widen(float x) { return x; }
__device__ __forceinline__ float widen(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float widen(__half x) { return __half2float(x); }

template <typename T>
__device__ __forceinline__ T narrow(float x) {
    if constexpr (sizeof(T) == 4) return x;
    else return T(x);
}

// Eight consecutive tokens of a row, aligned to 16 bytes of the row's own address, and their mask bits.
template <typename T>
struct RowView {
    const T* row;
    const int32_t* mask;
    int64_t vocab;
    int32_t skew;  // elements from the 16-byte boundary below the row's start
    __device__ int64_t groups() const { return (vocab + skew + 7) / 8; }
    __device__ __forceinline__ int64_t first(int64_t g) const { return g * 8 - skew; }
    struct Raw {
        uint4 v[sizeof(T) / 2];
    };
    __device__ __forceinline__ Raw fetch(int64_t g) const {
        const int64_t t = first(g);
        Raw r;
        if (t >= 0 && t + 8 <= vocab) {
#pragma unroll
            for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i) r.v[i] = __ldg(reinterpret_cast<const uint4*>(row + t) + i);
        } else {  // the row's ends
            T e[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) e[i] = t + i >= 0 && t + i < vocab ? row[t + i] : narrow<T>(-INFINITY);
            memcpy(&r, e, sizeof r);
        }
        return r;
    }
    static __device__ __forceinline__ void expand(const Raw& r, float (&x)[8]) {
        T e[8];
        memcpy(e, &r, sizeof r);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = widen(e[i]);
    }
    __device__ __forceinline__ void load(int64_t g, float (&x)[8]) const { expand(fetch(g), x); }
    __device__ __forceinline__ uint32_t bits(int64_t g) const {
        const int64_t t = first(g);
        uint32_t b = 0xffu;
        if (mask != nullptr) {
            if (t >= 0) {
                const int64_t w = t >> 5;
                const int sh = t & 31;
                b = static_cast<uint32_t>(mask[w]) >> sh;
                if (sh > 24 && (w + 1) * 32 < vocab) b |= static_cast<uint32_t>(mask[w + 1]) << (32 - sh);
            } else {
                b = static_cast<uint32_t>(mask[0]) << -t;
            }
            b &= 0xffu;
        }
        if (t < 0) b &= 0xffu << -t;
        if (t + 8 > vocab) b &= 0xffu >> (t + 8 - vocab);
        return b;
    }
};

// exp((x - top) * inv_t), float64: z = n ln2 / 64 + r, |r| <= ln2 / 128; 2^(n / 64) from a 64-entry table and the exponent
// field, e^r by its series to r^5 (the next term is below 4e-17).  Relative error about 1e-16 + |z| 2^-53, far
// below what decides a token; a third of the instructions of the library's exp.  Weights that come near the
// subnormals (z < -690) take that.
__device__ __forceinline__ double weight_of(float x, double top, double inv_t, const double* table) {
    const double z = (static_cast<double>(x) - top) * inv_t;
    if (z < -690.0) return exp(z);
    constexpr double kMagic = 6755399441055744.0;  // 1.5 * 2^52: adding it rounds to an integer in the low bits
    const double shifted = fma(z, 92.332482616893656877, kMagic);  // 64 / ln 2
    const int n = __double2loint(shifted);
    const double r = fma(shifted - kMagic, -0.010830424696249145, z);  // ln 2 / 64
    double e = fma(r, 1.0 / 120.0, 1.0 / 24.0);
    e = fma(e, r, 1.0 / 6.0);
    e = fma(e, r, 0.5);
    e = fma(e, r, 1.0);
    e = fma(e, r, 1.0);
    e *= table[n & 63];
    return __hiloint2double(__double2hiint(e) + (n >> 6) * 1048576, __double2loint(e));
}

// Calls f(token of element 0, x[8], valid bits) for the groups [g0, g1) with any valid token; several groups' loads are
// in flight at once.
template <typename T, typename F>
__device__ __forceinline__ void each_group(const RowView<T>& v, int64_t g0, int64_t g1, F f) {
    constexpr int kBatch = sizeof(T) == 4 ? 2 : 4;
    for (int64_t g = g0 + (threadIdx.x & 31); g < g1; g += 32 * kBatch) {
        uint32_t b[kBatch];
        typename RowView<T>::Raw raw[kBatch];
#pragma unroll
        for (int i = 0; i < kBatch; ++i) b[i] = g + 32 * i < g1 ? v.bits(g + 32 * i) : 0u;
#pragma unroll
        for (int i = 0; i < kBatch; ++i)
            if (b[i]) raw[i] = v.fetch(g + 32 * i);
#pragma unroll
        for (int i = 0; i < kBatch; ++i)
            if (b[i]) {
                float x[8];
                v.expand(raw[i], x);
                f(v.first(g + 32 * i), x, b[i]);
            }
    }
}

__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
    for (int d = 16; d; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
    return v;
}
__device__ __forceinline__ int64_t warp_sum(int64_t v) {
#pragma unroll
    for (int d = 16; d; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
    return v;
}

// Mass and count over the cluster of the tokens with key > cut_above and key >= floor_key, in a fixed order of sums.
template <typename T>
__device__ MassCount sum_above(cg::cluster_group& cluster, Shared& sh, const RowView<T>& v, int64_t g0, int64_t g1, double top, double inv_t,
                               uint64_t above, uint64_t floor_key, bool weigh, int& turn) {
    double mass = 0.0;
    int64_t count = 0;
    each_group(v, g0, g1, [&](int64_t t, const float(&x)[8], uint32_t b) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if (!((b >> i) & 1) || !(x[i] > -INFINITY)) continue;
            const uint64_t k = order_key(x[i], static_cast<uint32_t>(t + i));
            if (k > above && k >= floor_key) {
                if (weigh) mass += weight_of(x[i], top, inv_t, sh.exp_table);
                ++count;
            }
        }
    });
    mass = warp_sum(mass);
    count = warp_sum(count);
    const int warp = threadIdx.x >> 5;
    if ((threadIdx.x & 31) == 0) sh.warp_mass[warp] = mass, sh.warp_count[warp] = count;
    __syncthreads();
    const int c = cluster.num_blocks(), rank = cluster.block_rank();
    if (threadIdx.x < c) {
        MassCount mc{0.0, 0};
        for (int w = 0; w < kWarps; ++w) mc.mass += sh.warp_mass[w], mc.count += sh.warp_count[w];
        *cluster.map_shared_rank(&sh.part[turn][rank], threadIdx.x) = mc;
    }
    cluster.sync();
    MassCount all{0.0, 0};
    for (int r = 0; r < c; ++r) all.mass += sh.part[turn][r].mass, all.count += sh.part[turn][r].count;
    turn ^= 1;
    return all;
}

// Sorts the first n (<= kCap) entries descending; entries behind n must be 0.  m: n rounded up to a power of two.
__device__ void sort_desc(uint64_t* a, int m) {
    for (int size = 2; size <= m; size <<= 1)
        for (int step = size >> 1; step > 0; step >>= 1) {
            __syncthreads();
            for (int i = threadIdx.x; i < m / 2; i += kThreads) {
                const int lo = 2 * i - (i & (step - 1)), hi = lo + step;
                const bool down = (lo & size) == 0;
                const uint64_t x = a[lo], y = a[hi];
                if ((x < y) == down) a[lo] = y, a[hi] = x;
            }
        }
    __syncthreads();
}

// Inclusive scan of a[0, n) in place.
__device__ void scan_in_place(double* a, int n, Shared& sh) {
    const int per = (n + kThreads - 1) / kThreads;
    const int lo = min(n, static_cast<int>(threadIdx.x) * per), hi = min(n, lo + per);
    double s = 0.0;
    for (int i = lo; i < hi; ++i) s += a[i], a[i] = s;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    double run = s;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const double up = __shfl_up_sync(0xffffffffu, run, d);
        if (lane >= d) run += up;
    }
    __syncthreads();
    if (lane == 31) sh.warp_mass[warp] = run;
    __syncthreads();
    double before = 0.0;
    for (int w = 0; w < warp; ++w) before += sh.warp_mass[w];
    const double up = __shfl_up_sync(0xffffffffu, run, 1);
    if (lane > 0) before += up;
    for (int i = lo; i < hi; ++i) a[i] += before;
    __syncthreads();
}

// Sum of the values of the threads before this one, and of all (through `all`).
template <typename V>
__device__ V block_before(V v, V* warp_totals, V& all) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    V run = v;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const V up = __shfl_up_sync(0xffffffffu, run, d);
        if (lane >= d) run += up;
    }
    __syncthreads();
    if (lane == 31) warp_totals[warp] = run;
    __syncthreads();
    V before = 0;
    all = 0;
    for (int w = 0; w < kWarps; ++w) {
        if (w == warp) before = all;
        all += warp_totals[w];
    }
    return before + run - v;
}

__device__ __forceinline__ int round_pow2(int n) {
    int m = 2;
    while (m < n) m <<= 1;
    return m;
}

// The list path: all tokens in play are in sh.list (unsorted).  Returns through token / kept.
__device__ void finish_list(Shared& sh, int n, double top, double inv_t, int64_t k, double p, double min_p, double u, int64_t* token,
                            int64_t* kept_out) {
    const int m = round_pow2(n);
    for (int i = n + threadIdx.x; i < m; i += kThreads) sh.list[i] = 0;
    sort_desc(sh.list, m);
    int keep = static_cast<int>(min(static_cast<int64_t>(n), k));
    for (int i = threadIdx.x; i < keep; i += kThreads) sh.weight[i] = weight_of(order_value(static_cast<uint32_t>(sh.list[i] >> 32)), top, inv_t, sh.exp_table);
    __syncthreads();
    if (threadIdx.x == 0) sh.pick = 0;
    __syncthreads();
    if (min_p > 0.0) {
        uint32_t mine = 0;
        for (int i = threadIdx.x; i < keep; i += kThreads) mine += sh.weight[i] >= min_p;
        if (mine) atomicAdd(&sh.pick, mine);
        __syncthreads();
    }
    const int by_min = min_p > 0.0 ? static_cast<int>(sh.pick) : keep;
    int by_p = keep;
    if (p < 1.0) {
        scan_in_place(sh.weight, keep, sh);
        const double limit = p * sh.weight[keep - 1];
        if (threadIdx.x == 0) sh.pick = 0;
        __syncthreads();
        uint32_t mine = 0;
        for (int i = threadIdx.x; i < keep; i += kThreads) mine += i == 0 || sh.weight[i - 1] < limit;
        if (mine) atomicAdd(&sh.pick, mine);
        __syncthreads();
        by_p = static_cast<int>(sh.pick);
    }
    keep = min(by_p, by_min);
    // Token order: descending keys of the complement of the token.
    const int mk = round_pow2(keep);
    __syncthreads();
    for (int i = threadIdx.x; i < mk; i += kThreads)
        sh.list[i] = i < keep ? (sh.list[i] << 32) | (sh.list[i] >> 32) : 0;
    sort_desc(sh.list, mk);
    for (int i = threadIdx.x; i < keep; i += kThreads) sh.weight[i] = weight_of(order_value(static_cast<uint32_t>(sh.list[i])), top, inv_t, sh.exp_table);
    __syncthreads();
    scan_in_place(sh.weight, keep, sh);
    const double total = sh.weight[keep - 1], target = u * total;
    if (threadIdx.x == 0) sh.pick = 0xffffffffu;
    __syncthreads();
    // First entry whose running mass exceeds the target; after rounding, the first that reaches the total.
    for (int i = threadIdx.x; i < keep; i += kThreads)
        if (sh.weight[i] > target || sh.weight[i] >= total) {
            atomicMin(&sh.pick, static_cast<uint32_t>(i));
            break;
        }
    __syncthreads();
    if (threadIdx.x == 0) {
        *token = 0xffffffffu - static_cast<uint32_t>(sh.list[sh.pick] >> 32);
        *kept_out = keep;
    }
}

template <typename T>
__global__ void __launch_bounds__(kThreads, 2) filter_sample_kernel(const FilterParams p) {
    extern __shared__ __align__(16) unsigned char smem_raw[];
    Shared& sh = *reinterpret_cast<Shared*>(smem_raw);
    cg::cluster_group cluster = cg::this_cluster();
    const int c = cluster.num_blocks(), rank = cluster.block_rank();
    const int64_t r = blockIdx.x / c;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;

    const double temp = p.temperatures ? static_cast<double>(p.temperatures[r]) : p.temperature;
    const double top_p = p.top_ps ? static_cast<double>(p.top_ps[r]) : p.top_p;
    const double min_p = p.min_ps ? static_cast<double>(p.min_ps[r]) : p.min_p;
    const int64_t top_k = p.top_ks ? p.top_ks[r] : p.top_k;
    const double u = p.uniforms[r];
    const int64_t mrow = p.mask_rows ? p.mask_rows[r] : r;
    int32_t code = BMS_STATUS_OK;
    if (!(temp >= 0.0) || temp > DBL_MAX || !(top_p > 0.0) || top_p > 1.0 || !(min_p >= 0.0) || min_p > 1.0 || top_k < 0)
        code = BMS_STATUS_BAD_PARAMETER;
    else if (p.masks != nullptr && p.mask_rows != nullptr && (mrow < 0 || mrow >= p.mask_table_rows))
        code = BMS_STATUS_BAD_MASK_ROW;
    auto finish = [&](int64_t token, int64_t kept, int32_t status) {
        p.tokens[r] = token;
        p.kept[r] = kept;
        p.status[r] = status;
    };
    if (code != BMS_STATUS_OK) {
        if (rank == 0 && threadIdx.x == 0) finish(-1, 0, code);
        return;
    }
    const T* row = static_cast<const T*>(p.logits) + r * p.vocab;
    const RowView<T> view{row, p.masks ? p.masks + mrow * p.words : nullptr, p.vocab,
                          static_cast<int32_t>((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(T))};
    const int64_t groups = view.groups();
    const int64_t c0 = groups * rank / c, c1 = groups * (rank + 1) / c;
    const int64_t g0 = c0 + (c1 - c0) * warp / kWarps, g1 = c0 + (c1 - c0) * (warp + 1) / kWarps;

    if (threadIdx.x < 64) sh.exp_table[threadIdx.x] = exp2(threadIdx.x / 64.0);

    // Pass 1: maximum and count of valid finite tokens, NaN anywhere.
    RowStats st{-INFINITY, {}, 0, 0};
    {
        constexpr int kBatch = sizeof(T) == 4 ? 2 : 4;
        for (int64_t g = g0 + lane; g < g1; g += 32 * kBatch) {
            uint32_t b[kBatch];
            typename RowView<T>::Raw raw[kBatch];
#pragma unroll
            for (int i = 0; i < kBatch; ++i)
                if (g + 32 * i < g1) raw[i] = view.fetch(g + 32 * i);
#pragma unroll
            for (int i = 0; i < kBatch; ++i) b[i] = g + 32 * i < g1 ? view.bits(g + 32 * i) : 0u;
#pragma unroll
            for (int i = 0; i < kBatch; ++i) {
                if (g + 32 * i >= g1) break;
                float x[8];
                view.expand(raw[i], x);
                if (b[i]) st.flags |= 2;
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    if (x[j] != x[j]) st.flags |= 1;
                    const float xv = (b[i] >> j) & 1 ? x[j] : -INFINITY;
                    st.max = fmaxf(st.max, xv);
                    st.finite += xv > -INFINITY;
                }
            }
        }
        float m = st.max;
        st.low[2] = m;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
            if (d == 4) st.low[1] = m;
        }
        st.low[0] = st.max = m;
#pragma unroll
        for (int d = 16; d; d >>= 1) {
            st.low[1] = fminf(st.low[1], __shfl_xor_sync(0xffffffffu, st.low[1], d));
            st.low[2] = fminf(st.low[2], __shfl_xor_sync(0xffffffffu, st.low[2], d));
            st.finite += __shfl_xor_sync(0xffffffffu, st.finite, d);
            st.flags |= __shfl_xor_sync(0xffffffffu, st.flags, d);
        }
    }
    RowStats* warp_stats = reinterpret_cast<RowStats*>(sh.weight);
    if (lane == 0) warp_stats[warp] = st;
    if (threadIdx.x == 0) sh.list_count = 0;
    __syncthreads();
    if (threadIdx.x < c) {
        RowStats a = warp_stats[0];
        for (int w = 1; w < kWarps; ++w) merge(a, warp_stats[w]);
        *cluster.map_shared_rank(&sh.stats[rank], threadIdx.x) = a;
    }
    cluster.sync();
    st = sh.stats[0];
    for (int i = 1; i < c; ++i) merge(st, sh.stats[i]);
    const bool greedy = temp == 0.0;
    if (st.flags & 1) code = BMS_STATUS_NAN;
    else if (!greedy && st.max == INFINITY) code = BMS_STATUS_POS_INF;
    else if (!(st.flags & 2)) code = BMS_STATUS_EMPTY;
    else if (!greedy && st.finite == 0) code = BMS_STATUS_NO_MASS;
    else if (!greedy && !(u >= 0.0 && u < 1.0)) code = BMS_STATUS_BAD_UNIFORM;
    if (code != BMS_STATUS_OK) {
        if (rank == 0 && threadIdx.x == 0) finish(-1, 0, code);
        return;  // nothing remote is outstanding: the statistics arrived before the barrier
    }
    const float topf = st.max;
    const double top = topf;
    int turn = 0;

    if (greedy) {  // lowest valid token that holds the maximum
        if (threadIdx.x == 0) sh.pick = 0xffffffffu;
        cluster.sync();
        uint32_t best = 0xffffffffu;
        for (int64_t g = g0 + lane; g < g1 && best == 0xffffffffu; g += 32) {
            const uint32_t b = view.bits(g);
            if (b == 0) continue;
            float x[8];
            view.load(g, x);
#pragma unroll
            for (int i = 7; i >= 0; --i)
                if (((b >> i) & 1) && x[i] == topf) best = static_cast<uint32_t>(view.first(g) + i);
        }
        best = __reduce_min_sync(0xffffffffu, best);
        if (lane == 0 && best != 0xffffffffu) atomicMin(cluster.map_shared_rank(&sh.pick, 0), best);
        cluster.sync();
        if (rank == 0 && threadIdx.x == 0) finish(sh.pick, 1, BMS_STATUS_OK);
        return;
    }

    const double inv_t = fmin(1.0 / temp, DBL_MAX);
    const int64_t k = top_k > 0 ? min(top_k, static_cast<int64_t>(st.finite)) : st.finite;
    const bool k_cuts = k < st.finite;

    // Collects the keys of the finite tokens that `in(x)` accepts into rank 0's list; returns their number in the whole row
    // (above kCap: the list is not complete).
    auto collect = [&](auto in) -> uint32_t {
        __syncthreads();
        if (threadIdx.x == 0) sh.list_count = 0;
        __syncthreads();
        each_group(view, g0, g1, [&](int64_t t, const float(&x)[8], uint32_t b) {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (((b >> i) & 1) && x[i] > -INFINITY && in(x[i])) {
                    const uint32_t at = atomicAdd(&sh.list_count, 1u);
                    if (at < kCap) sh.list[at] = order_key(x[i], static_cast<uint32_t>(t + i));
                }
        });
        __syncthreads();
        if (c == 1) return sh.list_count;
        if (threadIdx.x < c) *cluster.map_shared_rank(&sh.list_counts[rank], threadIdx.x) = sh.list_count;
        cluster.sync();
        uint32_t before = 0, all = 0;
        for (int i = 0; i < c; ++i) {
            if (i < rank) before += sh.list_counts[i];
            all += sh.list_counts[i];
        }
        if (all <= kCap && rank != 0) {
            uint64_t* dst = cluster.map_shared_rank(sh.list, 0) + before;
            for (uint32_t i = threadIdx.x; i < sh.list_count; i += kThreads) dst[i] = sh.list[i];
        }
        cluster.sync();
        return all;
    };
    auto from_list = [&](uint32_t n) {
        if (rank == 0) {
            finish_list(sh, static_cast<int>(n), top, inv_t, k, top_p, min_p, u, &p.tokens[r], &p.kept[r]);
            if (threadIdx.x == 0) p.status[r] = BMS_STATUS_OK;
        }
    };

    // The tokens that can be kept, where a bound is known without another pass.
    if (st.finite <= kCap) return from_list(collect([](float) { return true; }));
    if (k_cuts) {
        const float low = k <= kWarps * c ? st.low[0] : k <= 4 * kWarps * c ? st.low[1] : st.low[2];
        if (k <= kThreads * c && low > -INFINITY) {
            const uint32_t n = collect([&](float x) { return x >= low; });
            if (n <= kCap) return from_list(n);
        }
    } else if (min_p > 0.0 && top_p >= 1.0) {
        // A little below the smallest weight kept, so that rounding here decides nothing.
        const double floor_x = top + temp * (log(min_p) - 1e-9) - 1e-12 * (fabs(top) + 1.0);
        const float low = __double2float_rd(floor_x);
        const uint32_t n = collect([&](float x) { return x >= low; });
        if (n <= kCap) return from_list(n);
    }

    // Counts of the tokens with key >= from by value bins of width span / kBins below the maximum, in sh.merged (a
    // token further down is in the last bin), the same in every CTA.
    const float span = static_cast<float>(fmin(40.0 * temp, 1e30));
    const float bin_scale = 2.0f * kBins / span;
    auto bin_of = [&](float x) { return static_cast<int>(fminf((0.5f * topf - 0.5f * x) * bin_scale, kBins - 1.0f)); };
    auto count_bins = [&](uint64_t from) {
        for (int i = threadIdx.x; i < kBins; i += kThreads) sh.bins[i] = 0;
        __syncthreads();
        each_group(view, g0, g1, [&](int64_t t, const float(&x)[8], uint32_t b) {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (((b >> i) & 1) && x[i] > -INFINITY && (from == 0 || order_key(x[i], static_cast<uint32_t>(t + i)) >= from))
                    atomicAdd(&sh.bins[bin_of(x[i])], 1u);
        });
        cluster.sync();
        for (int i = threadIdx.x; i < kBins; i += kThreads) {
            uint32_t n = 0;
            for (int q = 0; q < c; ++q) n += cluster.map_shared_rank(sh.bins, q)[i];
            sh.merged[i] = n;
        }
        cluster.sync();
    };

    // Cut of the first k tokens: exact counts find the bin that holds rank k; its tokens, sorted, give the key.
    uint64_t cut = 0;
    if (k_cuts) {
        count_bins(0);
        uint32_t mine = 0, all;
        for (int i = 0; i < kPerThread; ++i) mine += sh.merged[threadIdx.x * kPerThread + i];
        uint32_t run = block_before(mine, reinterpret_cast<uint32_t*>(sh.warp_mass), all);
        if (run < k && k <= run + mine) {
            int i = threadIdx.x * kPerThread;
            while (run + sh.merged[i] < k) run += sh.merged[i++];
            sh.bin[0] = i;
            sh.bin_count = run;
        }
        __syncthreads();
        const int bin = sh.bin[0];
        const uint32_t before = sh.bin_count, inside = sh.merged[bin];
        if (before + inside <= kCap && bin < kBins - 1) return from_list(collect([&](float x) { return bin_of(x) <= bin; }));
        if (inside <= kCap) {
            const uint32_t n = collect([&](float x) { return bin_of(x) == bin; });
            if (rank == 0) {
                const int m = round_pow2(n);
                for (int i = n + threadIdx.x; i < m; i += kThreads) sh.list[i] = 0;
                sort_desc(sh.list, m);
                if (threadIdx.x < c) *cluster.map_shared_rank(&sh.cut, threadIdx.x) = sh.list[k - before - 1];
            }
            cluster.sync();
            cut = sh.cut;
        } else {
            uint64_t lo = 0, hi = ~0ull;
            while (lo < hi) {
                const uint64_t mid = lo + (hi - lo) / 2;
                if (sum_above(cluster, sh, view, g0, g1, top, inv_t, mid, 0, false, turn).count < k) hi = mid;
                else lo = mid + 1;
            }
            cut = lo;
        }
    }
    if (top_p < 1.0) {
        // Where the nucleus ends, by the bins' counts and middle weights.  The estimate is good to about a part
        // in a thousand of the mass; a miss tells the exact masses around the bracket, which place the next one.
        count_bins(cut);
        const float step = span / kBins * static_cast<float>(inv_t) * 1.44269504f;
        float mine = 0.f, all;
        for (int i = 0; i < kPerThread; ++i) {
            const int at = threadIdx.x * kPerThread + i;
            mine += sh.merged[at] * exp2f(-(at + 0.5f) * step);
        }
        const float run = block_before(mine, reinterpret_cast<float*>(sh.warp_mass), all);
        float goal = static_cast<float>(top_p) * all, slack = 1e-3f;
        bool found = false;
        uint64_t nucleus = 0;
        for (int attempt = 0; attempt < 3 && !found; ++attempt, slack = 2e-4f) {
            __syncthreads();
            if (threadIdx.x == 0) sh.bin[0] = 0, sh.bin[1] = sh.bin[2] = kBins - 1, sh.bin_count = 0;
            __syncthreads();
#pragma unroll
            for (int side = 0; side < 3; ++side) {
                const float want = side == 0 ? goal - slack * all : side == 1 ? goal + slack * all : goal;
                if (run < want && want <= run + mine) {
                    float before = run;
                    int i = threadIdx.x * kPerThread;
                    for (const int last = i + kPerThread - 1; i < last; ++i) {
                        const float m = sh.merged[i] * exp2f(-(i + 0.5f) * step);
                        if (before + m >= want) break;
                        before += m;
                    }
                    sh.bin[side] = i;
                }
            }
            __syncthreads();
            int b0 = max(sh.bin[0] - 1, 0), b1 = min(sh.bin[1] + 1, kBins - 1);
            uint32_t inside = 0;
            for (int i = b0 + threadIdx.x; i <= b1; i += kThreads) inside += sh.merged[i];
            inside = __reduce_add_sync(0xffffffffu, inside);
            if (lane == 0) atomicAdd(&sh.bin_count, inside);
            __syncthreads();
            inside = sh.bin_count;
            if (inside > kCap) b0 = b1 = sh.bin[2], inside = sh.merged[b0];
            if (inside > kCap || inside == 0) break;
            double above = 0.0, below = 0.0;
            __syncthreads();
            if (threadIdx.x == 0) sh.list_count = 0;
            __syncthreads();
            each_group(view, g0, g1, [&](int64_t t, const float(&x)[8], uint32_t b) {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    if (!((b >> i) & 1) || !(x[i] > -INFINITY)) continue;
                    const uint64_t key = order_key(x[i], static_cast<uint32_t>(t + i));
                    if (key < cut) continue;
                    const int bin = bin_of(x[i]);
                    if (bin >= b0 && bin <= b1) {
                        sh.list[atomicAdd(&sh.list_count, 1u)] = key;
                    } else {
                        const double w = weight_of(x[i], top, inv_t, sh.exp_table);
                        if (bin < b0) above += w;
                        else below += w;
                    }
                }
            });
            above = warp_sum(above), below = warp_sum(below);
            __syncthreads();
            if (lane == 0) sh.warp_mass[warp] = above, sh.spans[warp] = below;
            __syncthreads();
            if (threadIdx.x == 0) {
                above = below = 0.0;
                for (int w = 0; w < kWarps; ++w) above += sh.warp_mass[w], below += sh.spans[w];
                *cluster.map_shared_rank(&sh.above[rank], 0) = above;
                *cluster.map_shared_rank(&sh.below[rank], 0) = below;
            }
            if (threadIdx.x < c) *cluster.map_shared_rank(&sh.list_counts[rank], threadIdx.x) = sh.list_count;
            cluster.sync();
            uint32_t mine = 0, n = 0;
            for (int i = 0; i < c; ++i) {
                if (i < rank) mine += sh.list_counts[i];
                n += sh.list_counts[i];
            }
            if (rank != 0) {
                uint64_t* dst = cluster.map_shared_rank(sh.list, 0) + mine;
                for (uint32_t i = threadIdx.x; i < sh.list_count; i += kThreads) dst[i] = sh.list[i];
            }
            cluster.sync();
            if (rank == 0) {
                above = below = 0.0;
                for (int i = 0; i < c; ++i) above += sh.above[i], below += sh.below[i];
                const int m = round_pow2(n);
                for (int i = n + threadIdx.x; i < m; i += kThreads) sh.list[i] = 0;
                sort_desc(sh.list, m);
                for (int i = threadIdx.x; i < n; i += kThreads)
                    sh.weight[i] = weight_of(order_value(static_cast<uint32_t>(sh.list[i] >> 32)), top, inv_t, sh.exp_table);
                if (threadIdx.x == 0) sh.pick = 0;
                __syncthreads();
                scan_in_place(sh.weight, n, sh);
                const double limit = top_p * (above + sh.weight[n - 1] + below);
                uint32_t kept = 0;
                for (int i = threadIdx.x; i < n; i += kThreads) kept += above + (i ? sh.weight[i - 1] : 0.0) < limit;
                if (kept) atomicAdd(&sh.pick, kept);
                __syncthreads();
                // Outside the bracket: not one of its tokens kept, or all of them with more below.
                const bool ends_inside = sh.pick > 0 && (above + sh.weight[n - 1] >= limit || b1 == kBins - 1);
                if (threadIdx.x < c) {
                    *cluster.map_shared_rank(&sh.cut, threadIdx.x) = ends_inside ? sh.list[sh.pick - 1] : 0;
                    *cluster.map_shared_rank(&sh.found, threadIdx.x) = ends_inside;
                    // How far the end lies before the bracket (negative) or behind it.
                    *cluster.map_shared_rank(&sh.goal, threadIdx.x) = static_cast<float>(sh.pick == 0 ? limit - above : limit - above - sh.weight[n - 1]);
                }
            }
            cluster.sync();
            found = sh.found;
            nucleus = sh.cut;
            if (!found) {  // the same correction from the estimated mass at the bracket's edge
                const float off = sh.goal;
                __syncthreads();
                const int edge = off <= 0.f ? b0 : b1 + 1;
                if (edge / kPerThread == threadIdx.x) {
                    float e = run;
                    for (int i = threadIdx.x * kPerThread; i < edge; ++i) e += sh.merged[i] * exp2f(-(i + 0.5f) * step);
                    sh.goal = e + off;
                }
                __syncthreads();
                goal = sh.goal;
            }
        }
        if (!found) {
            const double limit = top_p * sum_above(cluster, sh, view, g0, g1, top, inv_t, 0, cut, true, turn).mass;
            uint64_t lo = cut, hi = ~0ull;
            while (lo < hi) {
                const uint64_t mid = lo + (hi - lo) / 2;
                if (sum_above(cluster, sh, view, g0, g1, top, inv_t, mid, 0, true, turn).mass < limit) hi = mid;
                else lo = mid + 1;
            }
            nucleus = lo;
        }
        cut = max(cut, nucleus);
    }
    // Kept mass of every warp's span, in token order.
    double mass = 0.0;
    int64_t count = 0;
    each_group(view, g0, g1, [&](int64_t t, const float(&x)[8], uint32_t b) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if (!((b >> i) & 1) || !(x[i] > -INFINITY) || order_key(x[i], static_cast<uint32_t>(t + i)) < cut) continue;
            const double w = weight_of(x[i], top, inv_t, sh.exp_table);
            if (w >= min_p) mass += w, ++count;
        }
    });
    mass = warp_sum(mass);
    count = warp_sum(count);
    if (lane == 0) sh.warp_count[warp] = count;
    if (lane < c) *cluster.map_shared_rank(&sh.spans[rank * kWarps + warp], lane) = mass;
    __syncthreads();
    if (threadIdx.x == 0) {
        int64_t all = 0;
        for (int w = 0; w < kWarps; ++w) all += sh.warp_count[w];
        cluster.map_shared_rank(&sh.part[turn][rank], 0)->count = all;
    }
    cluster.sync();
    if (threadIdx.x == 0) {
        double total = 0.0;
        for (int i = 0; i < c * kWarps; ++i) total += sh.spans[i];
        const double target = u * total;
        double run = 0.0;
        int owner = -1;
        for (int i = 0; i < c * kWarps; ++i) {
            if (sh.spans[i] > 0.0) {
                owner = i;
                sh.before = run;
                if (run + sh.spans[i] > target) break;
            }
            run += sh.spans[i];
        }
        sh.owner = owner;
        sh.weight[0] = target;
    }
    __syncthreads();
    if (rank == 0 && threadIdx.x == 0) {
        int64_t all = 0;
        for (int i = 0; i < c; ++i) all += sh.part[turn][i].count;
        p.kept[r] = all;
        p.status[r] = BMS_STATUS_OK;
    }
    if (sh.owner / kWarps != rank) return;
    // The owner CTA walks the span that holds the target, one group per thread and round.
    const double target = sh.weight[0];
    double before = sh.before;
    const int w0 = sh.owner % kWarps;
    const int64_t s0 = c0 + (c1 - c0) * w0 / kWarps, s1 = c0 + (c1 - c0) * (w0 + 1) / kWarps;
    if (threadIdx.x == 0) sh.token = -1, sh.found = 0;
    __syncthreads();
    for (int64_t base = s0; base < s1; base += kThreads) {
        const int64_t g = base + threadIdx.x;
        double w[8], sum = 0.0;
        int last = -1;
#pragma unroll
        for (int i = 0; i < 8; ++i) w[i] = 0.0;
        if (g < s1) {
            const uint32_t b = view.bits(g);
            float x[8];
            if (b) view.load(g, x);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                if (!((b >> i) & 1) || !(x[i] > -INFINITY) || order_key(x[i], static_cast<uint32_t>(view.first(g) + i)) < cut) continue;
                const double wi = weight_of(x[i], top, inv_t, sh.exp_table);
                if (wi >= min_p && wi > 0.0) w[i] = wi, sum += wi, last = i;
            }
        }
        double run = sum;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const double up = __shfl_up_sync(0xffffffffu, run, d);
            if (lane >= d) run += up;
        }
        __syncthreads();
        if (lane == 31) sh.warp_mass[warp] = run;
        __syncthreads();
        double start = before, all = before;
        for (int i = 0; i < kWarps; ++i) {
            if (i < warp) start += sh.warp_mass[i];
            all += sh.warp_mass[i];
        }
        const double upv = __shfl_up_sync(0xffffffffu, run, 1);
        if (lane > 0) start += upv;
        // Tokens are in thread order: the first crossing thread wins; without one (rounding at the very
        // end) the last token with mass.
        double at = start;
        int hit = -1;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            at += w[i];
            if (hit < 0 && w[i] > 0.0 && at > target) hit = i;
        }
        if (threadIdx.x == 0) sh.pick = 0xffffffffu;
        __syncthreads();
        if (hit >= 0) atomicMin(&sh.pick, threadIdx.x);
        __syncthreads();
        const bool crossed = sh.pick != 0xffffffffu;
        if (crossed) {
            if (sh.pick == threadIdx.x) sh.token = view.first(g) + hit;
            break;
        }
        // Remember the last token with mass so far.
        const int any = __syncthreads_or(last >= 0);
        if (any) {
            if (threadIdx.x == 0) sh.list_base = 0;
            __syncthreads();
            if (last >= 0) atomicMax(&sh.list_base, threadIdx.x);
            __syncthreads();
            if (sh.list_base == threadIdx.x) sh.token = view.first(g) + last;
        }
        before = all;
        __syncthreads();
    }
    __syncthreads();
    if (threadIdx.x == 0) p.tokens[r] = sh.token;
}

template <typename T>
int launch_filter(const FilterParams& p, int device, cudaStream_t stream) {
    static bool ready[kMaxDevices];
    static int sms[kMaxDevices];
    auto kernel = filter_sample_kernel<T>;
    if (!ready[device]) {
        BMS_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(sizeof(Shared))), "cudaFuncSetAttribute(smem)");
        BMS_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1), "cudaFuncSetAttribute(cluster)");
        BMS_CUDA(cudaDeviceGetAttribute(&sms[device], cudaDevAttrMultiProcessorCount, device), "sm count");
        ready[device] = true;
    }
    int c = 1;
    while (c < 8 && p.rows * c * 2 <= sms[device] && p.vocab / (2 * c) >= 4096) c *= 2;
    if (p.rows * c > 2147483647LL) return fail(BMS_ERROR_UNSUPPORTED, "too many rows");
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(static_cast<unsigned>(p.rows * c));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = sizeof(Shared);
    cfg.stream = stream;
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = c, attr.val.clusterDim.y = 1, attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    BMS_CUDA(cudaLaunchKernelEx(&cfg, kernel, p), "filtered sampler launch");
    return BMS_SUCCESS;
}

}  // namespace
}  // namespace bms

using namespace bms;

extern "C" int bms_filtered_sample_batch(const void* logits, int32_t dtype, const int32_t* masks, const int32_t* mask_rows,
                                         int64_t mask_table_rows, int64_t rows, int64_t vocab, const bms_filter* filter,
                                         const double* uniforms, int64_t* tokens, int64_t* kept, int32_t* status, int32_t device,
                                         void* stream) {
    if (dtype != BMS_FLOAT32 && dtype != BMS_BFLOAT16 && dtype != BMS_FLOAT16)
        return fail(BMS_ERROR_INVALID_ARGUMENT, "logits must be float32, bfloat16 or float16 (dtype code %d)", dtype);
    if (vocab <= 0 || vocab > 2147483647LL) return fail(BMS_ERROR_INVALID_ARGUMENT, "invalid vocabulary size");
    if (rows < 0) return fail(BMS_ERROR_INVALID_ARGUMENT, "rows must not be negative");
    if (filter == nullptr) return fail(BMS_ERROR_INVALID_ARGUMENT, "filter must not be NULL");
    const bms_filter& f = *filter;
    if (!f.temperatures && !(f.temperature >= 0.0 && f.temperature <= DBL_MAX)) return fail(BMS_ERROR_INVALID_ARGUMENT, "invalid temperature");
    if (!f.top_ps && !(f.top_p > 0.0 && f.top_p <= 1.0)) return fail(BMS_ERROR_INVALID_ARGUMENT, "top_p must be in (0, 1]");
    if (!f.min_ps && !(f.min_p >= 0.0 && f.min_p <= 1.0)) return fail(BMS_ERROR_INVALID_ARGUMENT, "min_p must be in [0, 1]");
    if (!f.top_ks && f.top_k < 0) return fail(BMS_ERROR_INVALID_ARGUMENT, "top_k must not be negative");
    if (mask_rows != nullptr && (masks == nullptr || mask_table_rows <= 0))
        return fail(BMS_ERROR_INVALID_ARGUMENT, "mask_rows needs a mask table");
    if (rows == 0) return BMS_SUCCESS;
    cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;  // pointer queries are allowed during a capture in this mode only
    cudaThreadExchangeStreamCaptureMode(&mode);
    struct Restore {
        cudaStreamCaptureMode* m;
        ~Restore() { cudaThreadExchangeStreamCaptureMode(m); }
    } restore{&mode};
    BMS_CHECK(check_device(device));
    BMS_CHECK(check_ptr(logits, device, "logits", dtype == BMS_FLOAT32 ? 4 : 2));
    if (masks) BMS_CHECK(check_ptr(masks, device, "masks", 4));
    if (mask_rows) BMS_CHECK(check_ptr(mask_rows, device, "mask_rows", 4));
    if (f.temperatures) BMS_CHECK(check_ptr(f.temperatures, device, "temperatures", 4));
    if (f.top_ks) BMS_CHECK(check_ptr(f.top_ks, device, "top_ks", 4));
    if (f.top_ps) BMS_CHECK(check_ptr(f.top_ps, device, "top_ps", 4));
    if (f.min_ps) BMS_CHECK(check_ptr(f.min_ps, device, "min_ps", 4));
    BMS_CHECK(check_ptr(uniforms, device, "uniforms", 8));
    BMS_CHECK(check_ptr(tokens, device, "tokens", 8));
    BMS_CHECK(check_ptr(kept, device, "kept", 8));
    BMS_CHECK(check_ptr(status, device, "status", 4));
    DeviceGuard guard;
    BMS_CUDA(guard.enter(device), "cudaSetDevice");
    const FilterParams p{logits, masks, mask_rows, mask_table_rows, rows, vocab, (vocab + 31) / 32, f.temperature, f.top_p, f.min_p, f.top_k,
                         f.temperatures, f.top_ps, f.min_ps, f.top_ks, uniforms, tokens, kept, status};
    const auto st = static_cast<cudaStream_t>(stream);
    if (dtype == BMS_FLOAT32) return launch_filter<float>(p, device, st);
    if (dtype == BMS_BFLOAT16) return launch_filter<__nv_bfloat16>(p, device, st);
    return launch_filter<__half>(p, device, st);
}
