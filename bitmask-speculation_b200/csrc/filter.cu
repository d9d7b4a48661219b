// Filtered sampling: temperature, top-k, top-p and min-p over masked rows, one given uniform per row.
//
// For a row x under mask A at temperature T > 0, order the valid finite tokens by (x descending, token ascending);
// w_i = exp((x_i - max) / T) in float64.  Kept is the shortest of three prefixes of that order: the first
// top_k tokens; of their total mass the tokens whose preceding mass is below top_p * total; the tokens
// with w >= min_p.  The result is the lowest kept token whose running mass in token order exceeds u * kept mass.
//
// A cluster of C CTAs owns a row, each a contiguous slice, each warp a contiguous span of it.  The
// row is streamed from HBM once (maximum, counts, NaN); later passes over it hit L2, because only the
// rows in flight are live there.  Order keys are 64-bit: ordered float bits, then the complement of the token, so that ties
// are part of the key and every prefix is "key >= cut".
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cfloat>
#include <cmath>

#include "../../include/bms_b200.h"
#include "abi_common.cuh"

namespace bms {
namespace {

namespace cg = cooperative_groups;

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxCluster = 16;
constexpr int kCap = 4096;   // tokens that the list path holds
constexpr int kBins = 2048;  // value bins of the counting pass

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
    float max, low;  // row maximum of valid tokens; smallest of the threads' maxima
    uint32_t finite, flags;  // valid finite tokens; 1 NaN, 2 some valid token
};

struct MassCount {
    double mass;
    int64_t count;
};

struct Shared {
    uint64_t list[kCap];
    double weight[kCap];
    uint32_t bins[kBins];
    uint32_t merged[kBins];
    double spans[kMaxCluster * kWarps];
    MassCount part[2][kMaxCluster];
    RowStats stats[kMaxCluster];
    double warp_mass[kWarps];
    int64_t warp_count[kWarps];
    uint32_t list_count, remote_count, list_base;
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

// Eight consecutive tokens of a row, aligned to 16 bytes of the row's own address, and their mask bits.
template <typename T>
struct RowView {
    const T* row;
    const int32_t* mask;
    int64_t vocab;
    int32_t skew;  // elements from the 16-byte boundary below the row's start
    __device__ int64_t groups() const { return (vocab + skew + 7) / 8; }
    __device__ __forceinline__ int64_t first(int64_t g) const { return g * 8 - skew; }
    __device__ __forceinline__ void load(int64_t g, float (&x)[8]) const {
        const int64_t t = first(g);
        if (t >= 0 && t + 8 <= vocab) {
            if constexpr (sizeof(T) == 4) {
                const float4 a = *reinterpret_cast<const float4*>(row + t), b = *reinterpret_cast<const float4*>(row + t + 4);
                x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
            } else {
                const uint4 a = *reinterpret_cast<const uint4*>(row + t);
                const T* v = reinterpret_cast<const T*>(&a);
#pragma unroll
                for (int i = 0; i < 8; ++i) x[i] = widen(v[i]);
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = t + i >= 0 && t + i < vocab ? widen(row[t + i]) : -INFINITY;
        }
    }
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

__device__ __forceinline__ double weight_of(float x, float top, double inv_t) {
    return exp((static_cast<double>(x) - static_cast<double>(top)) * inv_t);
}

// Calls f(token of element 0, x[8], valid bits) for the groups [g0, g1) of this warp's span with any valid token.
template <typename T, typename F>
__device__ __forceinline__ void each_group(const RowView<T>& v, int64_t g0, int64_t g1, F f) {
    for (int64_t g = g0 + (threadIdx.x & 31); g < g1; g += 32) {
        const uint32_t b = v.bits(g);
        if (b == 0) continue;
        float x[8];
        v.load(g, x);
        f(v.first(g), x, b);
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
__device__ MassCount sum_above(cg::cluster_group& cluster, Shared& sh, const RowView<T>& v, int64_t g0, int64_t g1, float top, double inv_t,
                               uint64_t above, uint64_t floor_key, int& turn) {
    double mass = 0.0;
    int64_t count = 0;
    each_group(v, g0, g1, [&](int64_t t, const float(&x)[8], uint32_t b) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if (!((b >> i) & 1) || !(x[i] > -INFINITY)) continue;
            const uint64_t k = order_key(x[i], static_cast<uint32_t>(t + i));
            if (k > above && k >= floor_key) mass += weight_of(x[i], top, inv_t), ++count;
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

__device__ __forceinline__ int round_pow2(int n) {
    int m = 2;
    while (m < n) m <<= 1;
    return m;
}

// The list path: all tokens in play are in sh.list (unsorted).  Returns through token / kept.
__device__ void finish_list(Shared& sh, int n, float top, double inv_t, int64_t k, double p, double min_p, double u, int64_t* token,
                            int64_t* kept_out) {
    const int m = round_pow2(n);
    for (int i = n + threadIdx.x; i < m; i += kThreads) sh.list[i] = 0;
    sort_desc(sh.list, m);
    int keep = static_cast<int>(min(static_cast<int64_t>(n), k));
    for (int i = threadIdx.x; i < keep; i += kThreads) sh.weight[i] = weight_of(order_value(static_cast<uint32_t>(sh.list[i] >> 32)), top, inv_t);
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
    for (int i = threadIdx.x; i < keep; i += kThreads) sh.weight[i] = weight_of(order_value(static_cast<uint32_t>(sh.list[i])), top, inv_t);
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

    // Pass 1: maximum and count of valid finite tokens, NaN anywhere.
    RowStats st{-INFINITY, 0.f, 0, 0};
    for (int64_t g = g0 + lane; g < g1; g += 32) {
        const uint32_t b = view.bits(g);
        float x[8];
        view.load(g, x);
        if (b) st.flags |= 2;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if (x[i] != x[i]) st.flags |= 1;
            const float xv = (b >> i) & 1 ? x[i] : -INFINITY;
            st.max = fmaxf(st.max, xv);
            st.finite += xv > -INFINITY;
        }
    }
    st.low = st.max;
#pragma unroll
    for (int d = 16; d; d >>= 1) {
        st.max = fmaxf(st.max, __shfl_xor_sync(0xffffffffu, st.max, d));
        st.low = fminf(st.low, __shfl_xor_sync(0xffffffffu, st.low, d));
        st.finite += __shfl_xor_sync(0xffffffffu, st.finite, d);
        st.flags |= __shfl_xor_sync(0xffffffffu, st.flags, d);
    }
    RowStats* warp_stats = reinterpret_cast<RowStats*>(sh.weight);
    if (lane == 0) warp_stats[warp] = st;
    __syncthreads();
    if (threadIdx.x < c) {
        RowStats a = warp_stats[0];
        for (int w = 1; w < kWarps; ++w) {
            const RowStats o = warp_stats[w];
            a.max = fmaxf(a.max, o.max), a.low = fminf(a.low, o.low), a.finite += o.finite, a.flags |= o.flags;
        }
        *cluster.map_shared_rank(&sh.stats[rank], threadIdx.x) = a;
    }
    if (threadIdx.x == 0) sh.list_count = sh.remote_count = 0;
    cluster.sync();
    st = sh.stats[0];
    for (int i = 1; i < c; ++i) {
        const RowStats o = sh.stats[i];
        st.max = fmaxf(st.max, o.max), st.low = fminf(st.low, o.low), st.finite += o.finite, st.flags |= o.flags;
    }
    const bool greedy = temp == 0.0;
    if (st.flags & 1) code = BMS_STATUS_NAN;
    else if (!greedy && st.max == INFINITY) code = BMS_STATUS_POS_INF;
    else if (!(st.flags & 2)) code = BMS_STATUS_EMPTY;
    else if (!greedy && st.finite == 0) code = BMS_STATUS_NO_MASS;
    else if (!greedy && !(u >= 0.0 && u < 1.0)) code = BMS_STATUS_BAD_UNIFORM;
    if (code != BMS_STATUS_OK) {
        if (rank == 0 && threadIdx.x == 0) finish(-1, 0, code);
        cluster.sync();
        return;
    }
    const float top = st.max;
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
                if (((b >> i) & 1) && x[i] == top) best = static_cast<uint32_t>(view.first(g) + i);
        }
        best = __reduce_min_sync(0xffffffffu, best);
        if (lane == 0 && best != 0xffffffffu) atomicMin(cluster.map_shared_rank(&sh.pick, 0), best);
        cluster.sync();
        if (rank == 0 && threadIdx.x == 0) finish(sh.pick, 1, BMS_STATUS_OK);
        return;
    }

    const double inv_t = fmin(1.0 / temp, DBL_MAX);
    const int64_t k = top_k > 0 ? min(top_k, static_cast<int64_t>(st.finite)) : st.finite;

    if (st.finite <= kCap) {
        each_group(view, g0, g1, [&](int64_t t, const float(&x)[8], uint32_t b) {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (((b >> i) & 1) && x[i] > -INFINITY) sh.list[atomicAdd(&sh.list_count, 1u)] = order_key(x[i], static_cast<uint32_t>(t + i));
        });
        __syncthreads();
        if (c > 1) {
            if (rank != 0) {
                if (threadIdx.x == 0) sh.list_base = atomicAdd(cluster.map_shared_rank(&sh.remote_count, 0), sh.list_count);
            }
            cluster.sync();
            // Rank 0's own entries come first; the others follow in the order of their reservations.
            if (rank != 0) {
                const uint32_t base = *cluster.map_shared_rank(&sh.list_count, 0) + sh.list_base;
                uint64_t* dst = cluster.map_shared_rank(sh.list, 0);
                for (uint32_t i = threadIdx.x; i < sh.list_count; i += kThreads) dst[base + i] = sh.list[i];
            }
            cluster.sync();
        }
        if (rank == 0) finish_list(sh, static_cast<int>(st.finite), top, inv_t, k, top_p, min_p, u, &p.tokens[r], &p.kept[r]);
        if (rank == 0 && threadIdx.x == 0) p.status[r] = BMS_STATUS_OK;
        return;
    }

    // Cuts by bisection over the order keys: the smallest key whose preceding count (mass) is below the limit.
    uint64_t cut = 0;
    if (k < st.finite) {
        uint64_t lo = 0, hi = ~0ull;
        while (lo < hi) {
            const uint64_t mid = lo + (hi - lo) / 2;
            const MassCount mc = sum_above(cluster, sh, view, g0, g1, top, 0.0, mid, 0, turn);
            if (mc.count < k) hi = mid;
            else lo = mid + 1;
        }
        cut = lo;
    }
    if (top_p < 1.0) {
        const double limit = top_p * sum_above(cluster, sh, view, g0, g1, top, inv_t, 0, cut, turn).mass;
        uint64_t lo = cut, hi = ~0ull;
        while (lo < hi) {
            const uint64_t mid = lo + (hi - lo) / 2;
            const MassCount mc = sum_above(cluster, sh, view, g0, g1, top, inv_t, mid, 0, turn);
            if (mc.mass < limit) hi = mid;
            else lo = mid + 1;
        }
        cut = lo;
    }
    // Kept mass of every warp's span, in token order.
    double mass = 0.0;
    int64_t count = 0;
    each_group(view, g0, g1, [&](int64_t t, const float(&x)[8], uint32_t b) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if (!((b >> i) & 1) || !(x[i] > -INFINITY) || order_key(x[i], static_cast<uint32_t>(t + i)) < cut) continue;
            const double w = weight_of(x[i], top, inv_t);
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
                const double wi = weight_of(x[i], top, inv_t);
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
