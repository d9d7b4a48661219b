// Filtered sampling: temperature, top-k, top-p and min-p over masked rows, one given uniform per row.
//
// For a row x under mask A at temperature T > 0, order the valid finite tokens by (x descending, token ascending);
// w_i = exp((x_i - max) / T) in float64.  Kept is the shortest of three prefixes of that order: the first
// top_k tokens; of their total mass the tokens whose preceding mass is below top_p * total; the tokens
// with w >= min_p.  The result is the lowest kept token whose running mass in token order exceeds u * kept mass.
//
// Bound.  A row has to be read once (497 KB for 248,320 bfloat16 scores), which is the first pass's work: 0.21 ms of the
// 0.64 for 1,152 rows whose bytes alone take 0.09.  All passes issue instructions at 70 % of what the schedulers can: a round
// of 256 tokens costs a warp about 120 in the first pass, twice that where a sparse mask's tokens are kept.  Few rows are
// bound by latency: 8 rows with top-k 21 us, 7 of them the first pass.
//
// A cluster of C CTAs owns a row, each CTA a contiguous slice, each warp a contiguous span of it.  The
// row is streamed from HBM once (maximum, counts, NaN); later passes hit L2, because only the rows in
// flight are live there.  A place in the order is a score and a token (`Place`); every filter ends at one.
//
// Passes.  The first one also gives a lower bound of the k-th largest score for free: G disjoint
// groups of lanes each hold a token at or above the smallest of their maxima, so at least G tokens reach it.
//  * Few tokens in play (k small, min-p alone, or a sparse mask): the first pass or one more collects them in token order into
//    shared memory (vectors whose maximum stays below the bound cost a handful of instructions), and
//    one CTA orders, weighs, cuts and draws there; only these tokens are ever exponentiated.
//  * Otherwise, for bfloat16, one pass counts the tokens by score, which gives every filter's end exactly, and one weighs
//    the kept ones by spans; one CTA walks the span that holds u.
//  * For the other types one counting pass over value bins estimates where the nucleus ends, one weighing pass
//    sums the exact masses above and below a bracket of bins around that place and collects the
//    bracket's tokens, whose prefix gives the exact end (they are put into token order first: sums do not depend on
//    timing); if the estimate missed, the exact masses place the next bracket, and if a bracket overflows (runs of equal scores) the end is bisected over the
//    64-bit order keys instead.  (bfloat16 rows whose filters end near zero go this way, too.)  By scores 1,152 rows of
//    248,320 with top-p took 0.84 ms, by brackets 1.15 (masked rows); with the present streams 0.64.  Unmasked rows take 0.85 by
//    scores, 1.24 (float16) and 1.50 (float32) by brackets; 8 rows of 151,936 equal scores 0.69 by bisection.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <cfloat>
#include <cmath>
#include <cstring>
#include <type_traits>

#include "../../include/bms_b200.h"
#include "abi_common.cuh"
#include "ptx.cuh"

namespace bms {
namespace {

namespace cg = cooperative_groups;

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxCluster = 16;
constexpr int kCap = 4096;   // tokens that the list path holds
constexpr int kSegment = 480;  // of them in one warp's span (two CTAs fill an SM's shared memory)
constexpr int kTable = 512;    // powers 2^(j / 512)
constexpr int kBins = 4096;   // value bins of the counting pass
// A warp's queue: 63 tokens left over and a round of one 16-byte vector per lane.
template <typename T>
constexpr int kQueue = 64 + 32 * 16 / static_cast<int>(sizeof(T));
constexpr int kPerThread = kBins / kThreads;
constexpr int32_t kNear = 120 << 7;  // bfloat16 magnitudes below 2^-7 have no bin of their own (see score_bin)
constexpr int32_t kAllTies = 0x7fffffff;
constexpr int kWide = kCap / kThreads;  // list entries per thread

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
    float low;               // smallest maximum of the half-lanes
    uint32_t finite, flags;  // valid finite tokens; 1 NaN, 2 some valid token, 4 a full segment
};

__device__ __forceinline__ void merge(RowStats& a, const RowStats& o) {
    a.max = fmaxf(a.max, o.max);
    a.low = fminf(a.low, o.low);
    a.finite += o.finite;
    a.flags |= o.flags;
}

// A place in the order of a row's tokens, as an order key or in parts: tokens up to it are kept.
struct Place {
    float x;
    uint32_t t;
    __device__ __forceinline__ bool keeps(float y, uint32_t s) const { return y > x || (y == x && s <= t); }
};

struct MassCount {
    double mass;
    int64_t count;
};

// A warp's rounds in flight: a vector per lane and the round's mask words, copied without registers (cp.async).  (Loads
// ahead into rotating registers stall at the first move.)
constexpr int kAhead = 4;
struct Ring {
    uint4 vec[kAhead][32];
    uint32_t mask[kAhead][12];
};

struct Shared {
    double top, rate, top_p, u;     // the row: maximum, 512 / (T ln 2), nucleus, uniform
    float topf, floor_x;            // maximum; lowest score that min-p keeps
    float width, bin_scale, bin_at; // value bins: their width, and a score's bin is bin_at - x * bin_scale
    int32_t shift;                  // order bits that the scores' type leaves constant
    int32_t top_rank;               // bfloat16: the maximum's rank (see score_bin)
    int64_t k;                      // tokens that top-k keeps
    uint64_t first_k;               // order key of the last of them
    int32_t bounds[kWarps + 1];     // the warps' spans, in groups
    int32_t b0, b1;                 // bracket of bins
    alignas(16) unsigned char view[64];  // RowView
    union {
        uint64_t list[kCap];  // order keys
        struct {
            uint32_t bins[kBins];    // this CTA's counts, until every CTA has read them
            uint32_t merged[kBins];  // the row's counts
        };
        double score_weight[kBins];  // bfloat16: of the kept scores
        Ring first_ring[kWarps];  // of the passes that collect, which write the list at their end
    };
    union {
        struct {
            uint32_t queue[kWarps][2 * kQueue<float>];
            Ring ring[kWarps];       // of the passes over single tokens
        };
        uint64_t segment[kWarps][kSegment];  // keys that a warp collected, until they are in the list
    };
    RowStats warp_stats[kWarps];
    uint32_t fills[kWarps];  // tokens in the warps' segments
    double exp_table[kTable];
    double spans[kMaxCluster * kWarps];
    uint32_t warp_counts[kMaxCluster * kWarps];
    float group_max[kMaxCluster * kWarps * 4];  // of the 8-lane groups of every warp
    MassCount part[2][kMaxCluster];
    RowStats stats[kMaxCluster];
    double warp_mass[kWarps], warp_below[kWarps], step_mass[2][kWarps];
    int64_t warp_count[kWarps], counts[kMaxCluster];
    double above[kMaxCluster], below[kMaxCluster];
    double target, before;
    uint64_t cut;
    uint32_t list_counts[kMaxCluster];
    uint32_t list_count, bin_count, pick, last, passed, low_bits;
    int32_t bin[3];
    float goal;
    int32_t found, owner, token;
    // The cut by exact scores: tokens above `threshold` are kept, and the first `ties` at it.
    float threshold;
    int32_t ties, tie_limit;  // of the row; of the drawn token's span
    int32_t k_bin, k_need;    // the last kept bin, and how many of its tokens
    struct Outside {
        double mass;
        int64_t count;
    } outside[2][kMaxCluster];  // tokens near zero and below the bins
};

__device__ __forceinline__ uint32_t order_bits(float x) {
    const uint32_t b = __float_as_uint(x + 0.0f);  // -0 ranks with +0
    return b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u);
}

__device__ __forceinline__ float order_value(uint32_t k) { return __uint_as_float((k >> 31) ? k ^ 0x80000000u : ~k); }

__device__ __forceinline__ uint64_t order_key(float x, uint32_t token) {
    return (static_cast<uint64_t>(order_bits(x)) << 32) | (0xffffffffu - token);
}

__device__ __forceinline__ Place place_of(uint64_t key) { return {order_value(static_cast<uint32_t>(key >> 32)), 0xffffffffu - static_cast<uint32_t>(key)}; }

__device__ __forceinline__ float widen(float x) { return x; }
__device__ __forceinline__ float widen(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float widen(__half x) { return __half2float(x); }

// Two 16-bit scores in a word.
template <typename T>
struct Pair;
template <>
struct Pair<__nv_bfloat16> {
    static constexpr uint32_t kInf = 0x7f807f80u;
    static __device__ __forceinline__ uint32_t max(uint32_t a, uint32_t b) { return ptx::max_bf16x2(a, b); }
    static __device__ __forceinline__ uint32_t max_nan(uint32_t a, uint32_t b) { return ptx::max_nan_bf16x2(a, b); }
    static __device__ __forceinline__ uint32_t min(uint32_t a, uint32_t b) {
        uint32_t r;
        asm("min.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
        return r;
    }
    static __device__ __forceinline__ float lo(uint32_t u) { return __uint_as_float(u << 16); }
    static __device__ __forceinline__ float hi(uint32_t u) { return __uint_as_float(u & 0xffff0000u); }
};
template <>
struct Pair<__half> {
    static constexpr uint32_t kInf = 0x7c007c00u;
    static __device__ __forceinline__ uint32_t max(uint32_t a, uint32_t b) { return ptx::max_f16x2(a, b); }
    static __device__ __forceinline__ uint32_t max_nan(uint32_t a, uint32_t b) { return ptx::max_nan_f16x2(a, b); }
    static __device__ __forceinline__ uint32_t min(uint32_t a, uint32_t b) {
        uint32_t r;
        asm("min.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
        return r;
    }
    static __device__ __forceinline__ float lo(uint32_t u) { return __half2float(__ushort_as_half(static_cast<unsigned short>(u))); }
    static __device__ __forceinline__ float hi(uint32_t u) { return __half2float(__ushort_as_half(static_cast<unsigned short>(u >> 16))); }
};
template <>
struct Pair<float> {
    static constexpr uint32_t kInf = 0;
    static __device__ __forceinline__ float lo(uint32_t u) { return __uint_as_float(u); }
};

template <typename T>
__device__ __forceinline__ T narrow(float x) {
    if constexpr (sizeof(T) == 4) return x;
    else return T(x);
}

// A row as 16-byte vectors ("groups") on 16-byte boundaries, whatever the row's own address, and their mask bits.
// Groups [full0, full1) lie wholly in the row; the few tokens before and behind them (`edge`) are taken one per lane.
template <typename T>
struct RowView {
    static constexpr int kVec = 16 / sizeof(T);
    static constexpr uint32_t kAll = (1u << kVec) - 1u;
    const T* row;
    const int32_t* mask;
    uint32_t vocab;
    int32_t skew;  // elements from the 16-byte boundary below the row's start
    int32_t groups, full0, full1;
    RowView() = default;
    __device__ RowView(const T* r, const int32_t* m, int64_t n) : row(r), mask(m), vocab(static_cast<uint32_t>(n)) {
        skew = static_cast<int32_t>((reinterpret_cast<uintptr_t>(r) & 15) / sizeof(T));
        groups = static_cast<int32_t>((n + skew + kVec - 1) / kVec);
        full0 = skew ? 1 : 0;
        full1 = max(full0, static_cast<int32_t>((n + skew) / kVec));
    }
    __device__ __forceinline__ int32_t first(int32_t g) const { return g * kVec - skew; }
    // A group of [full0, full1).
    __device__ __forceinline__ uint4 fetch(int32_t g) const { return __ldg(reinterpret_cast<const uint4*>(row - skew) + g); }
    static __device__ __forceinline__ void expand(const uint4& r, float (&x)[kVec]) {
        if constexpr (sizeof(T) == 4) {
            x[0] = __uint_as_float(r.x), x[1] = __uint_as_float(r.y), x[2] = __uint_as_float(r.z), x[3] = __uint_as_float(r.w);
        } else {
            x[0] = Pair<T>::lo(r.x), x[1] = Pair<T>::hi(r.x), x[2] = Pair<T>::lo(r.y), x[3] = Pair<T>::hi(r.y);
            x[4] = Pair<T>::lo(r.z), x[5] = Pair<T>::hi(r.z), x[6] = Pair<T>::lo(r.w), x[7] = Pair<T>::hi(r.w);
        }
    }
    __device__ __forceinline__ uint32_t bits(int32_t g) const {
        if (mask == nullptr) return kAll;
        const uint32_t t = static_cast<uint32_t>(first(g)), w = t >> 5, sh = t & 31;
        uint32_t b = static_cast<uint32_t>(__ldg(mask + w)) >> sh;
        if (sh > 32 - kVec) b |= static_cast<uint32_t>(__ldg(mask + w + 1)) << (32 - sh);
        return b & kAll;
    }
    // This lane's token outside the full groups of [g0, g1), or -1.
    __device__ __forceinline__ int32_t edge(int32_t g0, int32_t g1) const {
        const int lane = threadIdx.x & 31;
        if (lane < kVec) return g0 == 0 && g1 > 0 && full0 && lane < min(first(1), static_cast<int32_t>(vocab)) ? lane : -1;
        const int32_t t = first(full1) + lane - kVec;
        return full1 >= g0 && full1 < g1 && full1 < groups && lane < 2 * kVec && t < static_cast<int32_t>(vocab) ? t : -1;
    }
    __device__ __forceinline__ bool valid(int32_t t) const { return mask == nullptr || (static_cast<uint32_t>(mask[t >> 5]) >> (t & 31) & 1); }
};

// The full groups of a warp's span, a round of one vector per lane at a time, kAhead - 1 rounds ahead.  Callers pass through a
// warp-wide vote between two rounds, so that no lane's copy overwrites mask words that another one has yet to read.
template <typename T>
struct Stream {
    static constexpr int kVec = RowView<T>::kVec;
    static constexpr int kWords = kVec + 1;  // mask words that a round's 32 kVec bits can touch; rounds are whole words apart
    const RowView<T>& v;
    Ring& ring;
    const uint4* from;     // this lane's next vector to copy
    const int32_t* words;  // its next mask word to copy, among the round's
    const int32_t* words_end;
    int32_t z, lane;
    int32_t g, ahead;      // this lane's groups: of the current round, of the next one to copy
    uint32_t slot = 0;
    uint32_t shift, word;  // where this lane's bits start in every round's words
    __device__ __forceinline__ void copy(uint32_t to) {
        if (ahead < z) ptx::cp_async_16(ptx::smem_addr(&ring.vec[to][lane]), from);
        // Like the vectors, only what some round takes: the space has later uses.
        if (words < words_end && ahead - lane < z) ptx::cp_async_4(ptx::smem_addr(&ring.mask[to][lane]), words);
        asm volatile("cp.async.commit_group;" ::: "memory");
        ahead += 32, from += 32, words += kVec;
    }
    __device__ __forceinline__ Stream(const RowView<T>& view, Ring& r, int32_t g0, int32_t g1) : v(view), ring(r), z(min(g1, view.full1)), lane(threadIdx.x & 31) {
        g = ahead = max(g0, view.full0) + lane;
        from = reinterpret_cast<const uint4*>(v.row - v.skew) + ahead;
        const uint32_t t0 = static_cast<uint32_t>(v.first(g - lane)), t = static_cast<uint32_t>(v.first(g));
        word = (t >> 5) - (t0 >> 5), shift = t & 31;
        words = v.mask + (t0 >> 5) + lane;
        words_end = v.mask != nullptr && lane < kWords ? v.mask + ((v.vocab - 1) >> 5) + 1 : words;
        for (int i = 0; i < kAhead - 1; ++i) copy(i);
    }
    __device__ __forceinline__ bool more() const { return g - lane < z; }
    // The current round's vector, and its bits (0 behind the span's end); starts the copy of a later one.
    __device__ __forceinline__ uint32_t take(uint4& now) {
        copy((slot + kAhead - 1) % kAhead);
        asm volatile("cp.async.wait_group %0;" ::"n"(kAhead - 1) : "memory");
        __syncwarp();
        now = ring.vec[slot][lane];
        if (g >= z) return 0;
        if (v.mask == nullptr) return RowView<T>::kAll;
        return __funnelshift_r(ring.mask[slot][word], ring.mask[slot][word + 1], shift) & RowView<T>::kAll;
    }
    __device__ __forceinline__ void next() { slot = (slot + 1) % kAhead, g += 32; }
    // Element j of the current round's vector.
    __device__ __forceinline__ float element(int j) const { return widen(reinterpret_cast<const T*>(&ring.vec[slot][lane])[j]); }
    __device__ __forceinline__ uint32_t raw_element(int j) const {
        if constexpr (sizeof(T) == 2) return reinterpret_cast<const uint16_t*>(&ring.vec[slot][lane])[j];
        else return reinterpret_cast<const uint32_t*>(&ring.vec[slot][lane])[j];
    }
};

// exp((x - top) / T), float64: t = (x - top) * rate in units of 2^(1/512) splits into an integer n and |r| <= 1/2; 2^(n / 512)
// comes from a table and the exponent field, 2^(r / 512) from its series to r^3 (the next term is below 1e-14
// relative), far below what decides a token.  Branch-free, a quarter of the instructions of the library's exp.
// Weights between 2^-1022 and 2^-1075 stay near 2^-1022, smaller ones are 0.
__device__ __forceinline__ double weight_of(float x, double top, double rate, const double* table) {
    constexpr double kMagic = 6755399441055744.0;  // 1.5 * 2^52: adding it rounds to an integer in the low bits
    constexpr double kLn = 0.0013538030870311432;  // ln 2 / 512
    const double t = (static_cast<double>(x) - top) * rate;
    const double shifted = t + kMagic;
    const int n = __double2loint(shifted);
    const double r = t - (shifted - kMagic);
    double e = fma(r, kLn * kLn * kLn / 6.0, kLn * kLn / 2.0);
    e = fma(e, r, kLn);
    e = fma(e, r, 1.0);
    e *= table[n & (kTable - 1)];
    e = __hiloint2double(__double2hiint(e) + (max(n, -1022 * kTable) >> 9) * 1048576, __double2loint(e));
    return t < -1075.0 * kTable ? 0.0 : e;
}

// The valid tokens with x >= low of a vector, one bit each.
template <typename T>
__device__ __forceinline__ uint32_t reaching(const uint4& now, uint32_t bits, float low) {
    constexpr int kVec = RowView<T>::kVec;
    float x[kVec];
    RowView<T>::expand(now, x);
    uint32_t in = 0;
#pragma unroll
    for (int j = 0; j < kVec; ++j) in |= static_cast<uint32_t>(x[j] >= low) << j;
    return in & bits;
}

// Calls f(x, token, live) for the valid tokens of the warp's span.  Rounds (one vector per lane) in which every token is
// valid go straight from the registers, unrolled; in others the valid tokens go through the warp's queue in shared
// memory, two per lane at a time, so that f's cost follows their number and not the vocabulary (grammar
// masks keep 0.1 - 60 % of it).  A queue entry is 16 bits of score and 16 of offset for 16-bit types, 8 bytes
// for float32.
template <typename T, typename F>
__device__ __forceinline__ void each_token(Shared& sh, const RowView<T>& v, F f) {
    constexpr bool kHalf = sizeof(T) == 2;
    constexpr int kVec = RowView<T>::kVec;
    constexpr int kGroups = 65536 / kVec;  // offsets stay within 16 bits
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int32_t g0 = sh.bounds[warp], g1 = sh.bounds[warp + 1];
    uint32_t* queue = sh.queue[warp];
    const uint32_t below = (1u << lane) - 1u;
    auto push = [&](int to, uint32_t value, uint32_t offset) {
        if constexpr (kHalf) queue[to] = value | (offset << 16);
        else reinterpret_cast<uint2*>(queue)[to] = make_uint2(value, offset);
    };
    for (int32_t base = max(g0, v.full0); base < min(g1, v.full1); base += kGroups) {
        const int32_t last = min(min(g1, v.full1), base + kGroups);
        const int32_t t0 = v.first(base);
        int fill = 0;
        for (Stream<T> stream(v, sh.ring[warp], base, last); stream.more(); stream.next()) {
            uint4 now;
            const uint32_t bits = stream.take(now);
            const uint32_t at = (stream.g - base) * kVec;
            if (__all_sync(0xffffffffu, bits == RowView<T>::kAll)) {
                float x[kVec];
                v.expand(now, x);
#pragma unroll
                for (int j = 0; j < kVec; ++j) f(x[j], static_cast<uint32_t>(t0 + at + j), x[j] > -INFINITY);
                continue;
            }
            const int most = __reduce_max_sync(0xffffffffu, __popc(bits));
            if (most > 3) {
#pragma unroll
                for (int j = 0; j < kVec; ++j) {
                    const bool in = (bits >> j) & 1;
                    const uint32_t who = __ballot_sync(0xffffffffu, in);
                    if (in) push(fill + __popc(who & below), (&now.x)[kHalf ? j >> 1 : j] >> (kHalf && (j & 1) ? 16 : 0) & (kHalf ? 0xffffu : 0xffffffffu), at + j);
                    fill += __popc(who);
                }
            } else {  // a few tokens per lane: one per lane and step
                uint32_t rest = bits;
#pragma unroll 1
                for (int i = 0; i < most; ++i, rest &= rest - 1) {
                    const uint32_t who = __ballot_sync(0xffffffffu, rest != 0);
                    if (rest) {
                        const int j = __ffs(rest) - 1;
                        push(fill + __popc(who & below), stream.raw_element(j), at + j);
                    }
                    fill += __popc(who);
                }
            }
            __syncwarp();
            const bool ends = stream.g - lane + 32 >= stream.z;  // the last round empties the queue
#pragma unroll 1
            while (fill >= 64 || (ends && fill > 0)) {
                const int from = max(fill - 64, 0);
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const int k = from + 32 * i + lane;
                    float x = -INFINITY;
                    uint32_t t = 0;
                    if (k < fill) {
                        if constexpr (kHalf) {
                            const uint32_t e = queue[k];
                            x = Pair<T>::lo(e);
                            t = t0 + (e >> 16);
                        } else {
                            const uint2 e = reinterpret_cast<const uint2*>(queue)[k];
                            x = __uint_as_float(e.x);
                            t = t0 + e.y;
                        }
                    }
                    f(x, t, x > -INFINITY);
                }
                fill = from;
                __syncwarp();
            }
        }
        // A queue left by sparse rounds before a last dense one.
        while (fill > 0) {
            const int from = max(fill - 32, 0);
            float x = -INFINITY;
            uint32_t t = 0;
            if (from + lane < fill) {
                if constexpr (kHalf) x = Pair<T>::lo(queue[from + lane]), t = t0 + (queue[from + lane] >> 16);
                else x = __uint_as_float(queue[2 * (from + lane)]), t = t0 + queue[2 * (from + lane) + 1];
            }
            f(x, t, x > -INFINITY);
            fill = from;
        }
        __syncwarp();
    }
    const int32_t t = v.edge(g0, g1);
    if (__any_sync(0xffffffffu, t >= 0)) {
        const float x = t >= 0 && v.valid(t) ? widen(v.row[t]) : -INFINITY;
        f(x, static_cast<uint32_t>(t), x > -INFINITY);
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

// Where the shortest of the first k tokens and the nucleus ends among the list's n (<= kCap) tokens, in any order:
// the order key of the last one kept.  `above` is the mass before the list, `rest` the mass behind it (both 0 where
// the list is the whole row); through `kept` how many of the list's tokens the nucleus keeps, through `mass`
// the mass of the first k.  By bisection: over the scores' order bits, 10 - 30 steps of a block-wide sum over keys in
// registers, then, where the end falls inside a run of equal scores, over tokens.  (A bitonic sort of the list
// took 2.5 times as long at 250 tokens, and far longer at 4,096.)
__device__ __noinline__ uint64_t list_cut(Shared& sh, int n, int64_t k, double p, double above, double rest, int& kept, double& mass) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int rounds = (n + kThreads - 1) / kThreads;
    uint32_t v[kWide], t[kWide];
    double w[kWide];
    uint32_t lo = 0xffffffffu, hi = 0;
#pragma unroll
    for (int r = 0; r < kWide; ++r) {
        const int i = r * kThreads + threadIdx.x;
        v[r] = 0, t[r] = 0xffffffffu, w[r] = 0.0;
        if (i < n) {
            const uint64_t key = sh.list[i];
            v[r] = static_cast<uint32_t>(key >> 32) >> sh.shift, t[r] = 0xffffffffu - static_cast<uint32_t>(key);
            if (p < 1.0) w[r] = weight_of(order_value(static_cast<uint32_t>(key >> 32)), sh.top, sh.rate, sh.exp_table);
            lo = min(lo, v[r]), hi = max(hi, v[r]);
        }
    }
    __syncthreads();
    if (threadIdx.x == 0) sh.pick = 0xffffffffu, sh.last = 0;
    __syncthreads();
    lo = __reduce_min_sync(0xffffffffu, lo), hi = __reduce_max_sync(0xffffffffu, hi);
    if (lane == 0) atomicMin(&sh.pick, lo), atomicMax(&sh.last, hi);
    __syncthreads();
    const uint32_t lowest = sh.pick, highest = sh.last;
    int turn = 0;
    // Sums over the list, alternating between two sets of warp totals so that one barrier per step does.
    auto count = [&](auto in) {
        uint32_t c = 0;
#pragma unroll
        for (int r = 0; r < kWide; ++r)
            if (r < rounds) c += in(v[r], t[r]);
        c = __reduce_add_sync(0xffffffffu, c);
        uint32_t* totals = reinterpret_cast<uint32_t*>(sh.step_mass[turn ^= 1]);
        if (lane == 0) totals[warp] = c;
        __syncthreads();
        return __reduce_add_sync(0xffffffffu, lane < kWarps ? totals[lane] : 0u);
    };
    auto weigh = [&](auto in) {
        double m = 0.0;
#pragma unroll
        for (int r = 0; r < kWide; ++r)
            if (r < rounds && in(v[r], t[r])) m += w[r];
        m = warp_sum(m);
        double* totals = sh.step_mass[turn ^= 1];
        if (lane == 0) totals[warp] = m;
        __syncthreads();
        return warp_sum(lane < kWarps ? totals[lane] : 0.0);
    };
    // The token of the j-th (from 1) of the equal scores x, in token order.
    auto token_of = [&](uint32_t x, uint32_t j) {
        uint32_t a = 0, b = 0xfffffffeu;
        while (a < b) {
            const uint32_t mid = a + (b - a) / 2;
            if (count([&](uint32_t y, uint32_t s) { return y == x && s <= mid; }) >= j) b = mid;
            else a = mid + 1;
        }
        return a;
    };
    uint32_t cut_v = lowest, cut_t = 0xfffffffeu;  // all of the list; entries behind it carry token 0xffffffff
    kept = n;
    if (k < n) {
        uint32_t a = lowest, b = highest;
        while (a < b) {
            const uint32_t mid = a + (b - a) / 2;
            if (count([&](uint32_t y, uint32_t) { return y > mid; }) < k) b = mid;
            else a = mid + 1;
        }
        cut_v = a;
        const uint32_t need = static_cast<uint32_t>(k) - count([&](uint32_t y, uint32_t) { return y > cut_v; });
        if (need < count([&](uint32_t y, uint32_t s) { return y == cut_v && s != 0xffffffffu; })) cut_t = token_of(cut_v, need);
        kept = static_cast<int>(k);
    }
    mass = 0.0;
    if (p < 1.0) {
        auto first_k = [&](uint32_t y, uint32_t s) { return y > cut_v || (y == cut_v && s <= cut_t); };
        mass = weigh(first_k);
        const double limit = p * (above + mass + rest);
        uint32_t a = lowest, b = highest;
        while (a < b) {
            const uint32_t mid = a + (b - a) / 2;
            if (above + weigh([&](uint32_t y, uint32_t s) { return y > mid && first_k(y, s); }) < limit) b = mid;
            else a = mid + 1;
        }
        const double before = above + weigh([&](uint32_t y, uint32_t s) { return y > a && first_k(y, s); });
        const uint32_t ahead = count([&](uint32_t y, uint32_t s) { return y > a && first_k(y, s); });
        const uint32_t ties = count([&](uint32_t y, uint32_t s) { return y == a && s != 0xffffffffu && first_k(y, s); });
        // The j-th of the equal scores is kept iff before + (j - 1) of their weights is below the limit.
        const double one = weight_of(order_value(sh.shift == 0 ? a : (a << sh.shift) | ((a >> (31 - sh.shift)) ? 0u : (1u << sh.shift) - 1u)), sh.top, sh.rate, sh.exp_table);
        uint32_t j = 0;
        for (uint32_t bit = 1u << 12; bit; bit >>= 1)
            if (j + bit <= ties && before + (j + bit - 1) * one < limit) j += bit;
        kept = static_cast<int>(ahead + j);
        if (j < ties) {
            if (j > 0) {
                cut_t = token_of(a, j);
                cut_v = a;
            } else {  // not even the first: only where the limit lies in the mass above the list
                cut_v = a + 1, cut_t = 0;
            }
        } else if (a > cut_v) {
            cut_v = a, cut_t = 0xfffffffeu;
        }
    }
    __syncthreads();
    // Back to a full order key: the constant low bits are zeros for positive scores and ones for negative ones.
    const uint32_t bits = sh.shift == 0 ? cut_v : (cut_v << sh.shift) | ((cut_v >> (31 - sh.shift)) ? 0u : (1u << sh.shift) - 1u);
    return (static_cast<uint64_t>(bits) << 32) | (0xffffffffu - cut_t);
}

// bfloat16 scores.  A row's scores are few: 128 per octave.  So a bin per score holds the whole row, but for magnitudes below
// 2^-7 (octaves without end; 0.3 % of normal logits) and for what lies 4,096 scores below the maximum.  The masses by bin
// are then exact, count times weight, with a weight per score and not per token, and the filters' end follows from them: a
// score, and how many of the tokens at it are kept.  One pass counts, one weighs the kept tokens by spans.
template <typename T>
constexpr bool kScoreBins = std::is_same_v<T, __nv_bfloat16>;

// A score's rank is 0 at 2^-7, grows with the score from there on, and is -1 at -2^-7 (and for a maximum near zero); its bin
// is how far it lies below the maximum.
__device__ __forceinline__ int32_t score_rank(uint32_t u) {
    const int32_t d = static_cast<int32_t>(u & 0x7fffu) - kNear;
    return d < 0 ? -1 : d ^ -static_cast<int32_t>(u >> 15);
}

// -1: near zero; kBins and more: below the bins.
__device__ __forceinline__ int32_t score_bin(uint32_t u, int32_t top_rank) {
    const int32_t d = static_cast<int32_t>(u & 0x7fffu) - kNear;
    const int32_t bin = top_rank - (d ^ -static_cast<int32_t>(u >> 15));
    return d < 0 ? -1 : bin;
}

__device__ __forceinline__ float bin_score(int32_t bin, int32_t top_rank) {
    const int32_t rank = top_rank - bin;
    const uint32_t u = rank >= 0 ? rank + kNear : 0x8000u | static_cast<uint32_t>(~rank + kNear);
    return __uint_as_float(u << 16);
}

// The end of the first k tokens and of the nucleus among them, from counts by score and c CTAs' sh.outside: sh.threshold and sh.ties; false where
// it lies among the tokens without a bin.  Every CTA computes the same.
__device__ __noinline__ bool cut_scores(Shared& sh, const uint32_t* counts, int c, bool k_cuts) {
    const int32_t top_rank = sh.top_rank, near_at = max(top_rank + 1, 0);  // the tokens near zero come before this bin
    Shared::Outside near{0.0, 0}, low{0.0, 0};
    for (int i = 0; i < c; ++i) {
        near.mass += sh.outside[0][i].mass, near.count += sh.outside[0][i].count;
        low.mass += sh.outside[1][i].mass, low.count += sh.outside[1][i].count;
    }
    if (near_at >= kBins) low.mass += near.mass, low.count += near.count;
    const int first = threadIdx.x * kPerThread;
    double mass = 0.0;
    int64_t count = 0;
    // Calls f(bin, tokens, weight) for this thread's bins in order; the tokens near zero are bin -1 and weigh their whole mass.
    auto each_bin = [&](auto f) {
#pragma unroll 1
        for (int b = first; b < first + kPerThread; ++b) {
            if (b == near_at && near.count) f(-1, near.count, near.mass);
            const uint32_t n = counts[b];
            if (n) f(b, static_cast<int64_t>(n), weight_of(bin_score(b, top_rank), sh.top, sh.rate, sh.exp_table));
        }
    };
    each_bin([&](int b, int64_t n, double w) { mass += b < 0 ? w : n * w, count += n; });
    double all_mass;
    int64_t all_count;
    const double mass_before = block_before(mass, sh.warp_mass, all_mass);
    const int64_t count_before = block_before(count, sh.warp_count, all_count);
    const int64_t k = sh.k;
    if (threadIdx.x == 0) sh.found = 1, sh.k_bin = kBins, sh.last = 0, sh.target = all_mass + low.mass;
    __syncthreads();
    if (k_cuts) {
        if (k > all_count) return false;
        if (count_before < k && k <= count_before + count) {
            int64_t n0 = count_before;
            double m = mass_before;
            bool done = false;
            each_bin([&](int b, int64_t n, double w) {
                if (done) return;
                if (k > n0 + n) {
                    n0 += n, m += b < 0 ? w : n * w;
                    return;
                }
                done = true;
                if (b < 0) sh.found = 0;
                sh.k_bin = b, sh.k_need = static_cast<int32_t>(k - n0);
                sh.target = m + (k - n0) * w;
            });
        }
        __syncthreads();
        if (!sh.found) return false;
    }
    if (sh.top_p < 1.0) {
        const double limit = sh.top_p * sh.target;
        if (!k_cuts && low.count && all_mass < limit) return false;
        // The last thread with tokens before which the mass is below the limit holds the end.
        if (count && (mass_before < limit)) atomicMax(&sh.last, threadIdx.x + 1);
        __syncthreads();
        if (threadIdx.x + 1 == sh.last) {
            double m = mass_before, before = 0.0, weight = 0.0;
            int bin = -1;
            int64_t tokens = 0;
            each_bin([&](int b, int64_t n, double w) {
                if (m < limit || bin < 0 && tokens == 0) bin = b, tokens = n, before = m, weight = w;
                m += b < 0 ? w : n * w;
            });
            int64_t j = 1;  // tokens at the score that the nucleus keeps: (j - 1) of their weights lie below the limit
            for (int64_t bit = 1ll << 30; bit; bit >>= 1)
                if (j + bit <= tokens && before + (j + bit - 1) * weight < limit) j += bit;
            if (bin < 0) sh.found = 0;
            if (bin < sh.k_bin || (bin == sh.k_bin && j < sh.k_need)) sh.k_bin = bin, sh.k_need = j == tokens ? kAllTies : static_cast<int32_t>(j);
        }
        __syncthreads();
        if (!sh.found) return false;
    }
    if (threadIdx.x == 0) {
        const float x = bin_score(sh.k_bin, top_rank);
        sh.threshold = fmaxf(x, sh.floor_x);
        if (x < sh.floor_x) {  // min-p keeps every token at its score: the last bin that reaches it, -1 where only scores near zero do
            int lo = bin_score(0, top_rank) >= sh.floor_x ? 0 : -1, hi = max(lo, sh.k_bin);
            while (lo >= 0 && lo < hi) {
                const int mid = (lo + hi + 1) / 2;
                if (bin_score(mid, top_rank) >= sh.floor_x) lo = mid;
                else hi = mid - 1;
            }
            sh.k_bin = lo, sh.k_need = kAllTies;
        }
        sh.ties = sh.k_need;
    }
    __syncthreads();
    return true;
}

// list_cut for bfloat16 by counts of the list's scores: the order key of the last kept token, or 0 where they do not give it.
// (256 rows of mixed filters 131 us by bisection and 126 by counts, 1,152 rows with top-p 659 and 635.)
__device__ __noinline__ uint64_t list_cut_scores(Shared& sh, int n, bool k_cuts) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int32_t top_rank = sh.top_rank;
    static_assert(sizeof sh.segment >= kBins * sizeof(uint32_t), "space of the counts");
    uint32_t* counts = reinterpret_cast<uint32_t*>(sh.segment);  // their tokens are in the list
    __syncthreads();
    for (int i = threadIdx.x; i < kBins; i += kThreads) counts[i] = 0;
    __syncthreads();
    double near_mass = 0.0, low_mass = 0.0;
    int near_count = 0, low_count = 0;
    for (int i = threadIdx.x; i < n; i += kThreads) {
        const float x = order_value(static_cast<uint32_t>(sh.list[i] >> 32));
        const int32_t bin = score_bin(__float_as_uint(x) >> 16, top_rank);
        if (static_cast<uint32_t>(bin) < kBins) {
            atomicAdd(&counts[bin], 1u);
            continue;
        }
        const double w = weight_of(x, sh.top, sh.rate, sh.exp_table);
        if (bin < 0) near_mass += w, ++near_count;
        else low_mass += w, ++low_count;
    }
    near_mass = warp_sum(near_mass), low_mass = warp_sum(low_mass);
    near_count = __reduce_add_sync(0xffffffffu, near_count), low_count = __reduce_add_sync(0xffffffffu, low_count);
    if (lane == 0) {
        sh.warp_mass[warp] = near_mass, sh.warp_below[warp] = low_mass;
        sh.warp_count[warp] = static_cast<int64_t>(low_count) << 32 | static_cast<uint32_t>(near_count);
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        Shared::Outside near{0.0, 0}, low{0.0, 0};
        for (int w = 0; w < kWarps; ++w) {
            near.mass += sh.warp_mass[w], near.count += sh.warp_count[w] & 0xffffffff;
            low.mass += sh.warp_below[w], low.count += sh.warp_count[w] >> 32;
        }
        sh.outside[0][0] = near, sh.outside[1][0] = low;
    }
    __syncthreads();
    if (!cut_scores(sh, counts, 1, k_cuts)) return 0;
    const uint32_t bits = order_bits(sh.threshold);
    if (sh.ties == kAllTies) return static_cast<uint64_t>(bits) << 32;
    // The list is in token order: its entry that is the last kept one of the threshold's.
    const int per = (n + kThreads - 1) / kThreads, first = threadIdx.x * per;
    int mine = 0, all;
    for (int i = first; i < min(first + per, n); ++i) mine += static_cast<uint32_t>(sh.list[i] >> 32) == bits;
    const int ahead = block_before(mine, reinterpret_cast<int*>(sh.warp_count), all);
    if (ahead < sh.ties && sh.ties <= ahead + mine) {
        int left = sh.ties - ahead;
        for (int i = first; left; ++i)
            if (static_cast<uint32_t>(sh.list[i] >> 32) == bits && --left == 0) sh.cut = sh.list[i];
    }
    __syncthreads();
    return sh.cut;
}

// The list path: the tokens in play are in sh.list, in token order.  Cuts, weighs and draws.
__device__ __noinline__ void finish_list(Shared& sh, int n, int64_t* token, int64_t* kept_out) {
    const double top = sh.top, rate = sh.rate, p = sh.top_p, u = sh.u;
    const int64_t k = sh.k;
    const float floor_x = sh.floor_x;
    uint64_t cut = 0;
    if (n <= kThreads && (k < n || p < 1.0)) {
        // A thread per token counts and weighs the tokens ahead of its own in the order: no barriers on the way.
        double* weights = reinterpret_cast<double*>(sh.segment);
        const int i = threadIdx.x;
        const uint64_t key = i < n ? sh.list[i] : 0;
        const double w = i < n ? weight_of(order_value(static_cast<uint32_t>(key >> 32)), top, rate, sh.exp_table) : 0.0;
        weights[i] = w;
        __syncthreads();
        int ahead = 0;
        double before = 0.0;
        if ((i & ~31) < n) {
#pragma unroll 4
            for (int j = 0; j < n; ++j)
                if (sh.list[j] > key) ++ahead, before += weights[j];
        }
        const bool in = i < n && ahead < k;
        double total;
        block_before(in ? w : 0.0, sh.warp_mass, total);
        const bool keep = in && (p >= 1.0 || before < p * total);
        if (threadIdx.x == 0) sh.cut = ~0ull;
        __syncthreads();
        if (keep) atomicMin(reinterpret_cast<unsigned long long*>(&sh.cut), static_cast<unsigned long long>(key));
        __syncthreads();
        cut = sh.cut;
    } else if (k < n || p < 1.0) {
        int kept;
        double mass;
        if (sh.shift == 16) cut = list_cut_scores(sh, n, k < n);
        if (cut == 0) cut = list_cut(sh, n, k, p, 0.0, 0.0, kept, mass);
    }
    cut = max(cut, static_cast<uint64_t>(order_bits(floor_x)) << 32);
    // Running masses in token order, consecutive tokens per thread.
    constexpr int kPer = kWide;
    const int per = (n + kThreads - 1) / kThreads, first = threadIdx.x * per;
    double w[kPer], sum = 0.0;
    int count = 0;
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
        w[j] = 0.0;
        if (j < per && first + j < n) {
            const uint64_t key = sh.list[first + j];
            if (key >= cut) w[j] = weight_of(order_value(static_cast<uint32_t>(key >> 32)), top, rate, sh.exp_table), ++count;
            sum += w[j];
        }
    }
    double total;
    double run = block_before(sum, sh.warp_mass, total);
    const double target = u * total;
    int kept;
    block_before(count, reinterpret_cast<int*>(sh.warp_count), kept);
    if (threadIdx.x == 0) sh.pick = 0xffffffffu, sh.last = 0;
    __syncthreads();
    // The first token whose running mass exceeds the target; without one (rounding at the very end) the last with mass.
    int hit = -1, last = -1;
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
        run += w[j];
        if (w[j] > 0.0) {
            last = first + j;
            if (hit < 0 && run > target) hit = first + j;
        }
    }
    if (hit >= 0) atomicMin(&sh.pick, static_cast<uint32_t>(hit));
    if (last >= 0) atomicMax(&sh.last, static_cast<uint32_t>(last));
    __syncthreads();
    if (threadIdx.x == 0) {
        *token = 0xffffffffu - static_cast<uint32_t>(sh.list[sh.pick != 0xffffffffu ? sh.pick : sh.last]);
        *kept_out = kept;
    }
}

// A score's bin: one rounding, so higher scores never lie in later bins.
__device__ __forceinline__ int bin_of(float x, float at, float scale) {
    return __float_as_int(fminf(fmaxf(fmaf(x, -scale, at), 0.f), kBins - 1.f) + 8388608.f) & (kBins - 1);  // adding 2^23 rounds to an integer
}

// The passes below are functions of their own, with the row's state in shared memory: inlined together they would
// share one register budget (64, for two CTAs of 512 per SM) and spill in their loops.

// Mass (0 unless `weigh`) and count over the cluster of the tokens with key > above and key >= floor_key, summed in a fixed order.
template <typename T>
__device__ __noinline__ MassCount sum_above(Shared& sh, const RowView<T>& shared_view, uint64_t above, uint64_t floor_key, bool weigh, int& turn) {
    cg::cluster_group cluster = cg::this_cluster();
    const RowView<T> view = shared_view;
    const int c = cluster.num_blocks(), rank = cluster.block_rank(), warp = threadIdx.x >> 5;
    double mass = 0.0;
    int64_t count = 0;
    each_token(sh, view, [&](float x, uint32_t t, bool live) {
        const uint64_t k = order_key(x, t);
        if (live && k > above && k >= floor_key) {
            if (weigh) mass += weight_of(x, sh.top, sh.rate, sh.exp_table);
            ++count;
        }
    });
    mass = warp_sum(mass);
    count = warp_sum(count);
    if ((threadIdx.x & 31) == 0) sh.warp_mass[warp] = mass, sh.warp_count[warp] = count;
    __syncthreads();
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

// The smallest order key whose preceding count (weigh: mass) is below the limit, by bisection from `lo`.
template <typename T>
__device__ __noinline__ uint64_t bisect(Shared& sh, const RowView<T>& view, uint64_t lo, double limit, bool weigh, int& turn) {
    uint64_t hi = ~0ull;
    while (lo < hi) {
        const uint64_t mid = lo + (hi - lo) / 2;
        const MassCount mc = sum_above(sh, view, mid, 0, weigh, turn);
        if ((weigh ? mc.mass : static_cast<double>(mc.count)) < limit) hi = mid;
        else lo = mid + 1;
    }
    return lo;
}

// Appends this lane's tokens `in` of the current round (tokens from t on) to the warp's segment in token order.
template <typename T>
__device__ __forceinline__ void append(uint64_t* segment, uint32_t& fill, uint32_t in, const Stream<T>& stream, int32_t t) {
    const int lane = threadIdx.x & 31;
    if (!__any_sync(0xffffffffu, in & (in - 1))) {  // at most one per lane
        const uint32_t who = __ballot_sync(0xffffffffu, in != 0), to = fill + __popc(who & ((1u << lane) - 1u));
        if (in && to < kSegment) {
            const int j = __ffs(in) - 1;
            segment[to] = order_key(stream.element(j), static_cast<uint32_t>(t + j));
        }
        fill += __popc(who);
        return;
    }
    uint32_t run = __popc(in);
    uint32_t at = fill - run;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const uint32_t up = __shfl_up_sync(0xffffffffu, run, d);
        if (lane >= d) run += up;
    }
    at += run;
    fill += __shfl_sync(0xffffffffu, run, 31);
#pragma unroll 1
    for (; in; in &= in - 1, ++at) {
        const int j = __ffs(in) - 1;
        if (at < kSegment) segment[at] = order_key(stream.element(j), static_cast<uint32_t>(t + j));
    }
}

// Drops a segment's tokens with x < low, in place; returns how many stay.
__device__ __forceinline__ uint32_t filter(uint64_t* segment, uint32_t have, float low) {
    const int lane = threadIdx.x & 31;
    const uint64_t key = static_cast<uint64_t>(order_bits(low)) << 32;
    uint32_t fill = 0;
    for (uint32_t i = 0; i < have; i += 32) {  // entries only move forward
        const uint64_t k = i + lane < have ? segment[i + lane] : 0;
        const uint32_t who = __ballot_sync(0xffffffffu, k >= key);
        __syncwarp();
        if (k >= key) segment[fill + __popc(who & ((1u << lane) - 1u))] = k;
        __syncwarp();
        fill += __popc(who);
    }
    return fill;
}

// A row's edge tokens (front or back of the full groups), one per lane, likewise.
template <typename T>
__device__ __forceinline__ void append_edge(const RowView<T>& view, uint64_t* segment, uint32_t& fill, float low, int32_t g0, int32_t g1, bool front) {
    const int lane = threadIdx.x & 31;
    const int32_t t = view.edge(g0, g1);
    const float x = t >= 0 && (lane < RowView<T>::kVec) == front && view.valid(t) ? widen(view.row[t]) : -INFINITY;
    const uint32_t who = __ballot_sync(0xffffffffu, x >= low);
    const uint32_t at = fill + __popc(who & ((1u << lane) - 1u));
    if (x >= low && at < kSegment) segment[at] = order_key(x, static_cast<uint32_t>(t));
    fill += __popc(who);
}

// The first pass: statistics of the row over the cluster, and, while it streams, the tokens that can matter: a warp keeps
// those that reach a bound which only rises.  mode 1 (top-k of at most 32): the smallest of its lanes' maxima so far,
// which at least 32 tokens reach (about 32 ln 32 of them stay: they fit the segment); mode 2 (min-p): its maximum
// so far less `drop`; mode 0: none, for sparse masks.  A warp whose segment is full stops keeping, and the row needs
// another pass.
template <typename T>
__device__ __noinline__ RowStats first_pass(Shared& sh, const RowView<T>& shared_view, int mode, float drop) {
    cg::cluster_group cluster = cg::this_cluster();
    const RowView<T> view = shared_view;
    const int c = cluster.num_blocks(), rank = cluster.block_rank(), lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int32_t g0 = sh.bounds[warp], g1 = sh.bounds[warp + 1];
    constexpr int kVec = RowView<T>::kVec;
    uint64_t* segment = sh.segment[warp];
    uint32_t fill = 0, finite = 0, some = 0, nan2 = Pair<T>::kInf ^ 0x80008000u, max2 = nan2;
    float nan1 = -INFINITY, max_a = -INFINITY, max_b = -INFINITY, low = -FLT_MAX;
    append_edge(view, segment, fill, low, g0, g1, true);
#pragma unroll 1
    for (Stream<T> stream(view, sh.first_ring[warp], g0, g1); stream.more(); stream.next()) {
        uint4 now;
        const uint32_t bits = stream.take(now);
        if (stream.g >= stream.z) now = make_uint4(0, 0, 0, 0);
        const uint32_t w[4] = {now.x, now.y, now.z, now.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if constexpr (sizeof(T) == 2) nan2 = Pair<T>::max_nan(nan2, w[j]);
            else nan1 = ptx::max_nan(nan1, __uint_as_float(w[j]));
        }
        if (!__any_sync(0xffffffffu, bits != 0)) continue;
        finite += __popc(bits);
        some |= bits;
        float best, least = INFINITY;  // of this vector's valid tokens
        if constexpr (sizeof(T) == 2) {  // two tokens per instruction; hidden ones become -inf (for the minimum +inf)
            const uint32_t lo = (bits & 0xfu) * 0x10204080u, hi = (bits >> 4) * 0x10204080u;
            uint32_t top2 = Pair<T>::kInf ^ 0x80008000u, min2 = Pair<T>::kInf;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint32_t keep = ptx::prmt(j < 2 ? lo : hi, 0u, j & 1 ? 0xBBAAu : 0x9988u);
                top2 = Pair<T>::max(top2, ptx::select_bits(w[j], keep, Pair<T>::kInf ^ 0x80008000u));
                min2 = Pair<T>::min(min2, ptx::select_bits(w[j], keep, Pair<T>::kInf));
            }
            max2 = Pair<T>::max(max2, top2);
            best = fmaxf(Pair<T>::lo(top2), Pair<T>::hi(top2));
            least = fminf(Pair<T>::lo(min2), Pair<T>::hi(min2));
        } else {
            float m[kVec];
#pragma unroll
            for (int j = 0; j < kVec; ++j) {
                const bool in = (bits >> j) & 1;
                m[j] = in ? __uint_as_float(w[j]) : -INFINITY;
                least = fminf(least, in ? __uint_as_float(w[j]) : INFINITY);
            }
            const float a = fmaxf(m[0], m[1]), o = fmaxf(m[2], m[3]);
            max_a = fmaxf(max_a, a), max_b = fmaxf(max_b, o);
            best = fmaxf(a, o);
        }
        const bool never = __any_sync(0xffffffffu, least == -INFINITY);
        if (never) finite -= __popc(bits & ~reaching<T>(now, bits, -FLT_MAX));  // valid, never drawn
        if (fill <= kSegment && __any_sync(0xffffffffu, best >= low)) {
            if (mode == 0 && fill + __reduce_add_sync(0xffffffffu, __popc(bits)) * ((stream.z - stream.g + lane) / 32) > 2 * kSegment) {
                fill = kSegment + 1;  // as dense as this, the span would not fit
                continue;
            }
            // No room for a whole round: drop what the bound has passed.  What stays full is given up.
            if (fill + 32 * kVec > kSegment && mode) fill = filter(segment, fill, low);
            append<T>(segment, fill, mode == 0 && !never ? bits : reaching<T>(now, bits, low), stream, view.first(stream.g));
            if (mode) {
                if constexpr (sizeof(T) == 2) max_a = Pair<T>::lo(max2), max_b = Pair<T>::hi(max2);
                const float lane_bound = fmaxf(max_a, max_b);
                const uint32_t o = order_bits(lane_bound);
                low = mode == 1 ? order_value(__reduce_min_sync(0xffffffffu, o)) : __fsub_rd(order_value(__reduce_max_sync(0xffffffffu, o)), drop);
                low = fmaxf(low, -FLT_MAX);
            }
        }
    }
    if (fill <= kSegment) append_edge(view, segment, fill, low, g0, g1, false);
    if constexpr (sizeof(T) == 2) {
        max_a = Pair<T>::lo(max2), max_b = Pair<T>::hi(max2);
        nan1 = ptx::max_nan(Pair<T>::lo(nan2), Pair<T>::hi(nan2));
    }
    RowStats st{-INFINITY, fminf(max_a, max_b), 0, 0};
    st.max = fmaxf(max_a, max_b);
    const int32_t t = view.edge(g0, g1);
    if (t >= 0) {
        const float x = widen(view.row[t]);
        nan1 = ptx::max_nan(nan1, x);
        if (view.valid(t)) st.max = fmaxf(st.max, x), some = 1, finite += x > -INFINITY;
    }
    st.finite = finite;
    st.flags = (nan1 != nan1 ? 1u : 0u) | (some ? 2u : 0u);
    // The other CTAs' shared memory exists once they have started: the kernel arrived at its start, the wait ends here.
    if (c > 1) {
        __syncwarp();
        ptx::cluster_wait();
    }
    float m = st.max;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
        if (d == 4 && (lane & 7) == 0)
            for (int i = 0; i < c; ++i) cluster.map_shared_rank(sh.group_max, i)[(rank * kWarps + warp) * 4 + lane / 8] = m;
    }
    st.max = m;
#pragma unroll
    for (int d = 16; d; d >>= 1) {
        st.low = fminf(st.low, __shfl_xor_sync(0xffffffffu, st.low, d));
        st.finite += __shfl_xor_sync(0xffffffffu, st.finite, d);
        st.flags |= __shfl_xor_sync(0xffffffffu, st.flags, d);
    }
    if (fill > kSegment) st.flags |= 4;
    if (lane == 0) sh.warp_stats[warp] = st, sh.fills[warp] = fill;
    __syncthreads();
    if (threadIdx.x < c) {
        RowStats a = sh.warp_stats[0];
        for (int w = 1; w < kWarps; ++w) merge(a, sh.warp_stats[w]);
        *cluster.map_shared_rank(&sh.stats[rank], threadIdx.x) = a;
    }
    cluster.sync();
    st = sh.stats[0];
    for (int i = 1; i < c; ++i) merge(st, sh.stats[i]);
    return st;
}

// The segments' tokens with x >= low into rank 0's list, in token order; returns their number in the whole row, or more
// than kCap where the list overflowed.  Every warp's segment is whole.
__device__ __noinline__ uint32_t gather(Shared& sh, float low) {
    cg::cluster_group cluster = cg::this_cluster();
    const int c = cluster.num_blocks(), rank = cluster.block_rank(), lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    uint64_t* segment = sh.segment[warp];
    const uint32_t fill = filter(segment, sh.fills[warp], low);
    if (lane < c) *cluster.map_shared_rank(&sh.warp_counts[rank * kWarps + warp], lane) = fill;
    cluster.sync();
    uint32_t before = 0, all = 0;
    for (int i = lane; i < c * kWarps; i += 32) {
        const uint32_t n = sh.warp_counts[i];
        all += n;
        if (i < rank * kWarps + warp) before += n;
    }
    before = __reduce_add_sync(0xffffffffu, before);
    all = __reduce_add_sync(0xffffffffu, all);
    if (all <= kCap) {
        uint64_t* dst = cluster.map_shared_rank(sh.list, 0) + before;
        for (uint32_t i = lane; i < fill; i += 32) dst[i] = segment[i];
    }
    cluster.sync();
    return all;
}

// A score that at least k tokens reach, close to the k-th: the k-th largest of the maxima of disjoint groups of lanes,
// whole warps' where these are enough (about -G ln(1 - k / G) tokens reach the k-th of G), else of 8 lanes (at most
// kThreads of them in the cluster).
__device__ __noinline__ float kth_maximum(Shared& sh, int k, int c) {
    const int n = 4 * kWarps * c, step = k * 5 <= 4 * kWarps * c ? 4 : 1, i = threadIdx.x;
    float mine = -INFINITY;
    if (i < n && i % step == 0)
        for (int j = 0; j < step; ++j) mine = fmaxf(mine, sh.group_max[i + j]);
    __syncthreads();
    if (i < n && i % step == 0) sh.group_max[i] = mine;
    if (i == 0) sh.low_bits = 0;
    __syncthreads();
    int ahead = 0;
    if (i < n && i % step == 0)
#pragma unroll 4
        for (int j = 0; j < n; j += step) ahead += sh.group_max[j] > mine || (sh.group_max[j] == mine && j < i);
    if (i < n && i % step == 0 && ahead == k - 1) sh.low_bits = order_bits(mine);
    __syncthreads();
    return sh.low_bits ? order_value(sh.low_bits) : -INFINITY;
}

// A pass that collects the tokens with x >= low into rank 0's list, in token order; returns as gather does, or more
// than kCap where a segment overflowed.
template <typename T>
__device__ __noinline__ uint32_t collect(Shared& sh, const RowView<T>& shared_view, float low) {
    cg::cluster_group cluster = cg::this_cluster();
    const RowView<T> view = shared_view;
    const int c = cluster.num_blocks(), lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int32_t g0 = sh.bounds[warp], g1 = sh.bounds[warp + 1];
    constexpr int kVec = RowView<T>::kVec;
    uint32_t fill = 0;
    uint64_t* segment = sh.segment[warp];
    __syncthreads();  // the segments' space had other uses
    append_edge(view, segment, fill, low, g0, g1, true);
#pragma unroll 1
    for (Stream<T> stream(view, sh.first_ring[warp], g0, g1); stream.more(); stream.next()) {
        uint4 now;
        const uint32_t bits = stream.take(now);
        float best = -INFINITY;
        if (bits) {
            float x[kVec];
            view.expand(now, x);
#pragma unroll
            for (int j = 0; j < kVec; ++j) best = fmaxf(best, x[j]);
        }
        if (__any_sync(0xffffffffu, best >= low)) append<T>(segment, fill, bits ? reaching<T>(now, bits, low) : 0u, stream, view.first(stream.g));
    }
    append_edge(view, segment, fill, low, g0, g1, false);
    if (lane == 0) sh.fills[warp] = min(fill, static_cast<uint32_t>(kSegment));
    const int over = __syncthreads_or(fill > kSegment);
    if (threadIdx.x < c) *cluster.map_shared_rank(&sh.list_counts[cluster.block_rank()], threadIdx.x) = over;
    cluster.sync();
    uint32_t any = 0;
    for (int i = 0; i < c; ++i) any |= sh.list_counts[i];
    const uint32_t n = gather(sh, low);
    return any ? kCap + 1 : n;
}

// Counts of the tokens up to sh.first_k by value bins of width sh.width below the maximum, in sh.merged (a token further
// down is in the last bin), the same in every CTA.
template <typename T, bool kEnd>
__device__ __noinline__ void count_bins_to(Shared& sh, const RowView<T>& shared_view) {
    cg::cluster_group cluster = cg::this_cluster();
    const RowView<T> view = shared_view;
    const int c = cluster.num_blocks();
    const Place end = place_of(sh.first_k);
    __syncthreads();
    for (int i = threadIdx.x; i < kBins; i += kThreads) sh.bins[i] = 0;
    __syncthreads();
    const float at = sh.bin_at, scale = sh.bin_scale;
    each_token(sh, view, [&](float x, uint32_t t, bool live) {
        if (live && (!kEnd || end.keeps(x, t))) atomicAdd(&sh.bins[bin_of(x, at, scale)], 1u);
    });
    cluster.sync();
    for (int i = threadIdx.x; i < kBins; i += kThreads) {
        uint32_t n = 0;
        for (int q = 0; q < c; ++q) n += cluster.map_shared_rank(sh.bins, q)[i];
        sh.merged[i] = n;
    }
    cluster.sync();
}

template <typename T>
__device__ __forceinline__ void count_bins(Shared& sh, const RowView<T>& view) {
    if (place_of(sh.first_k).x > -INFINITY) count_bins_to<T, true>(sh, view);
    else count_bins_to<T, false>(sh, view);
}

// Moves every CTA's sh.list (sh.list_count keys, in no order) behind rank 0's; returns their number.
__device__ __noinline__ uint32_t pool(Shared& sh) {
    cg::cluster_group cluster = cg::this_cluster();
    const int c = cluster.num_blocks(), rank = cluster.block_rank();
    __syncthreads();
    if (threadIdx.x < c) *cluster.map_shared_rank(&sh.list_counts[rank], threadIdx.x) = sh.list_count;
    cluster.sync();
    uint32_t before = 0, all = 0;
    for (int i = 0; i < c; ++i) {
        if (i < rank) before += sh.list_counts[i];
        all += sh.list_counts[i];
    }
    if (rank != 0) {
        uint64_t* dst = cluster.map_shared_rank(sh.list, 0) + before;
        for (uint32_t i = threadIdx.x; i < sh.list_count; i += kThreads) dst[i] = sh.list[i];
    }
    cluster.sync();
    return all;
}

// Brings sh.list's n keys into token order, so that sums over it come out the same in every call, in whatever order the tokens
// were collected.  Counts by up to 512 ranges of 2^s tokens, then every key's rank in its range.
__device__ __noinline__ void order_list(Shared& sh, int n, uint32_t vocab) {
    static_assert(kThreads == 1 << 9 && sizeof sh.segment >= kCap * sizeof(uint64_t) + (2 * kThreads + 1) * sizeof(uint32_t), "space of the order");
    uint64_t* parted = &sh.segment[0][0];  // its tokens are in the list
    uint32_t* first = reinterpret_cast<uint32_t*>(parted + kCap);  // [kThreads + 1] where each range starts
    uint32_t* next = first + kThreads + 1;
    const int s = max(32 - __clz(vocab - 1) - 9, 0);
    auto range_of = [&](uint64_t key) { return (0xffffffffu - static_cast<uint32_t>(key)) >> s; };
    __syncthreads();
    next[threadIdx.x] = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += kThreads) atomicAdd(&next[range_of(sh.list[i])], 1u);
    __syncthreads();
    uint32_t all;
    const uint32_t before = block_before(next[threadIdx.x], reinterpret_cast<uint32_t*>(sh.warp_count), all);
    first[threadIdx.x] = next[threadIdx.x] = before;
    if (threadIdx.x == 0) first[kThreads] = n;
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += kThreads) parted[atomicAdd(&next[range_of(sh.list[i])], 1u)] = sh.list[i];
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += kThreads) {
        const uint64_t key = parted[i];
        const uint32_t r = range_of(key);
        uint32_t at = first[r];
        for (uint32_t j = first[r]; j < first[r + 1]; ++j) at += static_cast<uint32_t>(parted[j]) > static_cast<uint32_t>(key);  // lower tokens
        sh.list[at] = key;
    }
    __syncthreads();
}

// The keys of bin b's tokens into sh.list (no order).
template <typename T>
__device__ __noinline__ void collect_bin(Shared& sh, const RowView<T>& shared_view, int b) {
    const RowView<T> view = shared_view;
    __syncthreads();
    if (threadIdx.x == 0) sh.list_count = 0;
    __syncthreads();
    const float at = sh.bin_at, scale = sh.bin_scale;
    each_token(sh, view, [&](float x, uint32_t t, bool live) {
        if (live && bin_of(x, at, scale) == b) sh.list[atomicAdd(&sh.list_count, 1u)] = order_key(x, t);
    });
}

// The weighing pass around the bracket [sh.b0, sh.b1] of bins, among the tokens up to sh.first_k: masses above and below
// it and the number of kept tokens above it to rank 0 (sh.above, sh.below, sh.counts, sh.spans), the bracket's keys
// into sh.list.
template <typename T, bool kEnd, bool kFloor>
__device__ __noinline__ void weigh_bracket_to(Shared& sh, const RowView<T>& shared_view) {
    cg::cluster_group cluster = cg::this_cluster();
    const RowView<T> view = shared_view;
    const int rank = cluster.block_rank(), lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const Place end = place_of(sh.first_k);
    const double top = sh.top, rate = sh.rate;
    const int b0 = sh.b0, b1 = sh.b1;
    const float at = sh.bin_at, scale = sh.bin_scale, floor_x = sh.floor_x;
    double above = 0.0, below = 0.0, kept_above = 0.0;
    int count = 0;
    each_token(sh, view, [&](float x, uint32_t t, bool live) {
        if (!live || (kEnd && !end.keeps(x, t))) return;
        const int bin = bin_of(x, at, scale);
        if (bin >= b0 && bin <= b1) {
            sh.list[atomicAdd(&sh.list_count, 1u)] = order_key(x, t);
            return;
        }
        const double w = weight_of(x, top, rate, sh.exp_table);
        if (bin > b1) below += w;
        else above += w;
        if (kFloor && bin < b0 && x >= floor_x) kept_above += w;
        count += bin < b0 && (!kFloor || x >= floor_x);
    });
    if (!kFloor) kept_above = above;
    above = warp_sum(above), below = warp_sum(below), kept_above = warp_sum(kept_above);
    count = __reduce_add_sync(0xffffffffu, count);
    if (lane == 0) {
        sh.warp_mass[warp] = above, sh.warp_below[warp] = below, sh.warp_count[warp] = count;
        *cluster.map_shared_rank(&sh.spans[rank * kWarps + warp], 0) = kept_above;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        double a = 0.0, b = 0.0;
        int64_t n = 0;
        for (int w = 0; w < kWarps; ++w) a += sh.warp_mass[w], b += sh.warp_below[w], n += sh.warp_count[w];
        *cluster.map_shared_rank(&sh.above[rank], 0) = a;
        *cluster.map_shared_rank(&sh.below[rank], 0) = b;
        *cluster.map_shared_rank(&sh.counts[rank], 0) = n;
    }
}

template <typename T>
__device__ __forceinline__ void weigh_bracket(Shared& sh, const RowView<T>& view) {
    const bool end = place_of(sh.first_k).x > -INFINITY, floor = sh.floor_x > -INFINITY;
    if (end) floor ? weigh_bracket_to<T, true, true>(sh, view) : weigh_bracket_to<T, true, false>(sh, view);
    else floor ? weigh_bracket_to<T, false, true>(sh, view) : weigh_bracket_to<T, false, false>(sh, view);
}

// Mass of the tokens up to `end` by spans, and their number, to rank 0.
template <typename T, bool kEnd>
__device__ __noinline__ void weigh_spans(Shared& sh, const RowView<T>& shared_view, Place end) {
    cg::cluster_group cluster = cg::this_cluster();
    const RowView<T> view = shared_view;
    const int rank = cluster.block_rank(), lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const double top = sh.top, rate = sh.rate;
    double mass = 0.0;
    int count = 0;
    each_token(sh, view, [&](float x, uint32_t t, bool live) {
        if (live && (!kEnd || end.keeps(x, t))) mass += weight_of(x, top, rate, sh.exp_table), ++count;
    });
    mass = warp_sum(mass);
    count = __reduce_add_sync(0xffffffffu, count);
    __syncthreads();
    if (lane == 0) {
        sh.warp_count[warp] = count;
        *cluster.map_shared_rank(&sh.spans[rank * kWarps + warp], 0) = mass;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        int64_t all = 0;
        for (int w = 0; w < kWarps; ++w) all += sh.warp_count[w];
        *cluster.map_shared_rank(&sh.counts[rank], 0) = all;
    }
    cluster.sync();
}

// The nucleus: the place where it ends in sh.cut and the kept masses by spans on rank 0, or false where the estimate
// or the list does not serve.
template <typename T>
__device__ __noinline__ bool find_nucleus(Shared& sh, const RowView<T>& shared_view, int64_t* kept_out, int32_t* status_out) {
    cg::cluster_group cluster = cg::this_cluster();
    const int c = cluster.num_blocks(), rank = cluster.block_rank(), lane = threadIdx.x & 31;
    const int64_t groups = shared_view.groups;
    // Where the nucleus ends, by the bins' counts and middle weights.  The estimate is good to about a part
    // in a thousand of the mass; a miss tells the exact masses around the bracket, which place the next one.
    count_bins<T>(sh, shared_view);
    const float step = sh.width * static_cast<float>(sh.rate / kTable);  // log2 of the weights' ratio from bin to bin
    float mine = 0.f, all;
    for (int i = 0; i < kPerThread; ++i) {
        const int at = threadIdx.x * kPerThread + i;
        mine += sh.merged[at] * exp2f(-at * step);
    }
    const float run = block_before(mine, reinterpret_cast<float*>(sh.warp_mass), all);
    float goal = static_cast<float>(sh.top_p) * all, slack = 1e-3f;
    bool found = false;
    for (int attempt = 0; attempt < 3 && !found; ++attempt, slack = 2e-4f) {
        __syncthreads();
        if (threadIdx.x == 0) sh.bin[0] = 0, sh.bin[1] = sh.bin[2] = kBins - 1, sh.bin_count = 0, sh.list_count = 0;
        __syncthreads();
#pragma unroll 1
        for (int side = 0; side < 3; ++side) {
            const float want = side == 0 ? goal - slack * all : side == 1 ? goal + slack * all : goal;
            if (run < want && want <= run + mine) {
                float before = run;
                int i = threadIdx.x * kPerThread;
                for (const int last = i + kPerThread - 1; i < last; ++i) {
                    const float m = sh.merged[i] * exp2f(-i * step);
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
        if (threadIdx.x == 0) sh.b0 = b0, sh.b1 = b1;
        __syncthreads();
        weigh_bracket<T>(sh, shared_view);
        const uint32_t n = pool(sh);
        if (rank == 0) {
            double above = 0.0, below = 0.0;
            for (int i = 0; i < c; ++i) above += sh.above[i], below += sh.below[i];
            int kept;
            double mass;
            order_list(sh, static_cast<int>(n), shared_view.vocab);
            const uint64_t key = list_cut(sh, static_cast<int>(n), n, sh.top_p, above, below, kept, mass);
            const double limit = sh.top_p * (above + mass + below);
            // Outside the bracket: not one of its tokens kept, or all of them with more below.
            const bool ends_inside = kept > 0 && (above + mass >= limit || b1 == kBins - 1);
            if (ends_inside) {
                // The bracket's kept tokens join their spans, a warp per span: they lie side by side in the list.
                if (threadIdx.x == 0) sh.passed = 0;
                __syncthreads();
                uint32_t passed = 0;
                int32_t* begins = reinterpret_cast<int32_t*>(sh.segment);  // of the spans in the list
                static_assert(kMaxCluster * kWarps < kThreads, "a start per thread");
                if (threadIdx.x <= c * kWarps) {
                    const int q = threadIdx.x / kWarps, w = threadIdx.x % kWarps;
                    const int64_t from = groups * q / c, len = groups * (q + 1) / c - from;
                    const int64_t t = (from + len * w / kWarps) * RowView<T>::kVec - shared_view.skew;  // of span c * kWarps: the row's end
                    int lo = 0, hi = static_cast<int>(n);
                    while (lo < hi) {
                        const int mid = (lo + hi) >> 1;
                        if (static_cast<int64_t>(0xffffffffu - static_cast<uint32_t>(sh.list[mid])) < t) lo = mid + 1;
                        else hi = mid;
                    }
                    begins[threadIdx.x] = lo;
                }
                __syncthreads();
                for (int span = threadIdx.x / 32; span < c * kWarps; span += kWarps) {
                    const int end = begins[span + 1];
                    double sum = 0.0;
                    for (int i = begins[span] + lane; i < end; i += 32) {
                        const Place at = place_of(sh.list[i]);
                        if (sh.list[i] < key || at.x < sh.floor_x) continue;
                        ++passed;
                        sum += weight_of(at.x, sh.top, sh.rate, sh.exp_table);
                    }
                    sum = warp_sum(sum);
                    if (lane == 0) sh.spans[span] += sum;
                }
                if (passed) atomicAdd(&sh.passed, passed);
                __syncthreads();
                if (threadIdx.x == 0) {
                    int64_t all_count = sh.passed;
                    for (int i = 0; i < c; ++i) all_count += sh.counts[i];
                    *kept_out = all_count;
                    *status_out = BMS_STATUS_OK;
                }
            }
            if (threadIdx.x < c) {
                *cluster.map_shared_rank(&sh.cut, threadIdx.x) = key;
                *cluster.map_shared_rank(&sh.found, threadIdx.x) = ends_inside;
                // How far the end lies before the bracket (negative) or behind it.
                *cluster.map_shared_rank(&sh.goal, threadIdx.x) = static_cast<float>(kept == 0 ? limit - above : limit - above - mass);
            }
        }
        cluster.sync();
        found = sh.found;
        if (!found) {  // the same correction from the estimated mass at the bracket's edge
            const float off = sh.goal;
            count_bins<T>(sh, shared_view);  // the list has taken the counts' place
            const int edge = off <= 0.f ? b0 : b1 + 1;
            if (edge / kPerThread == threadIdx.x) {
                float e = run;
                for (int i = threadIdx.x * kPerThread; i < edge; ++i) e += sh.merged[i] * exp2f(-i * step);
                sh.goal = e + off;
            }
            __syncthreads();
            goal = sh.goal;
        }
    }
    return found;
}

// Counts by score in sh.merged, tokens without a bin in sh.outside; the same in every CTA.
template <typename T>
__device__ __noinline__ void count_scores(Shared& sh, const RowView<T>& shared_view) {
    cg::cluster_group cluster = cg::this_cluster();
    const RowView<T> view = shared_view;
    constexpr int kVec = RowView<T>::kVec;
    const int c = cluster.num_blocks(), rank = cluster.block_rank(), lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    __syncthreads();
    for (int i = threadIdx.x; i < kBins; i += kThreads) sh.bins[i] = 0;
    __syncthreads();
    const int32_t top_rank = sh.top_rank, g0 = sh.bounds[warp], g1 = sh.bounds[warp + 1];
    double near_mass = 0.0, low_mass = 0.0;
    int near_count = 0, low_count = 0;
    auto count = [&](uint32_t u) {  // true where the token has a bin
        const uint32_t bin = static_cast<uint32_t>(score_bin(u, top_rank));
        if (bin < kBins) atomicAdd(&sh.bins[bin], 1u);
        return bin < kBins;
    };
    auto weigh = [&](uint32_t u) {
        const float x = Pair<T>::lo(u);
        if (!(x > -INFINITY)) return;
        const double w = weight_of(x, sh.top, sh.rate, sh.exp_table);
        if (score_bin(u, top_rank) < 0) near_mass += w, ++near_count;
        else low_mass += w, ++low_count;
    };
#pragma unroll 1
    for (Stream<T> stream(view, sh.ring[warp], g0, g1); stream.more(); stream.next()) {
        uint4 now;
        const uint32_t bits = stream.take(now);
        const int most = __reduce_max_sync(0xffffffffu, __popc(bits));
        uint32_t out = 0;  // this lane's tokens without a bin
        if (most > 3) {
            const uint32_t w[4] = {now.x, now.y, now.z, now.w};
#pragma unroll
            for (int j = 0; j < kVec; ++j)
                if ((bits >> j & 1) && !count(w[j >> 1] >> (j & 1 ? 16 : 0) & 0xffffu)) out |= 1u << j;
        } else {
#pragma unroll 1
            for (uint32_t rest = bits; rest; rest &= rest - 1) {
                const int j = __ffs(rest) - 1;
                if (!count(stream.raw_element(j))) out |= 1u << j;
            }
        }
        if (__any_sync(0xffffffffu, out != 0)) {
#pragma unroll 1
            for (; out; out &= out - 1) weigh(stream.raw_element(__ffs(out) - 1));
        }
    }
    const int32_t t = view.edge(g0, g1);
    if (t >= 0 && view.valid(t)) {
        const uint32_t u = __float_as_uint(widen(view.row[t])) >> 16;
        if (!count(u)) weigh(u);
    }
    near_mass = warp_sum(near_mass), low_mass = warp_sum(low_mass);
    near_count = __reduce_add_sync(0xffffffffu, near_count), low_count = __reduce_add_sync(0xffffffffu, low_count);
    if (lane == 0) {
        sh.warp_mass[warp] = near_mass, sh.warp_below[warp] = low_mass;
        sh.warp_count[warp] = static_cast<int64_t>(low_count) << 32 | static_cast<uint32_t>(near_count);
    }
    __syncthreads();
    if (threadIdx.x < c) {
        Shared::Outside near{0.0, 0}, low{0.0, 0};
        for (int w = 0; w < kWarps; ++w) {
            near.mass += sh.warp_mass[w], near.count += sh.warp_count[w] & 0xffffffff;
            low.mass += sh.warp_below[w], low.count += sh.warp_count[w] >> 32;
        }
        *cluster.map_shared_rank(&sh.outside[0][rank], threadIdx.x) = near;
        *cluster.map_shared_rank(&sh.outside[1][rank], threadIdx.x) = low;
    }
    cluster.sync();
    for (int i = threadIdx.x; i < kBins; i += kThreads) {
        uint32_t n = 0;
        for (int q = 0; q < c; ++q) n += cluster.map_shared_rank(sh.bins, q)[i];
        sh.merged[i] = n;
    }
    cluster.sync();
}

// Masses of the kept tokens by spans, less the ones at the last score where some of those are dropped, the number of
// these by spans, and the number of the others, to rank 0.
template <typename T>
__device__ __noinline__ void weigh_kept(Shared& sh, const RowView<T>& shared_view) {
    cg::cluster_group cluster = cg::this_cluster();
    const RowView<T> view = shared_view;
    constexpr int kVec = RowView<T>::kVec;
    const int rank = cluster.block_rank(), lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int32_t top_rank = sh.top_rank, g0 = sh.bounds[warp], g1 = sh.bounds[warp + 1];
    const uint32_t whole = sh.ties == kAllTies ? sh.k_bin + 1 : sh.k_bin;  // bins below it are kept whole
    for (int b = threadIdx.x; b <= sh.k_bin; b += kThreads) sh.score_weight[b] = weight_of(bin_score(b, top_rank), sh.top, sh.rate, sh.exp_table);
    __syncthreads();
    const float threshold = sh.threshold;
    double mass = 0.0;
    int count = 0, ties = 0;
    auto take = [&](uint32_t u) {  // true for a token near zero
        const uint32_t bin = static_cast<uint32_t>(score_bin(u, top_rank));
        if (bin < whole) mass += sh.score_weight[bin], ++count;
        else ties += bin == whole;
        return bin == 0xffffffffu;
    };
    auto near_zero = [&](uint32_t u) {
        const float x = Pair<T>::lo(u);
        if (x >= threshold) mass += weight_of(x, sh.top, sh.rate, sh.exp_table), ++count;
    };
#pragma unroll 1
    for (Stream<T> stream(view, sh.ring[warp], g0, g1); stream.more(); stream.next()) {
        uint4 now;
        uint32_t bits = stream.take(now);
        if (bits) bits = reaching<T>(now, bits, threshold);  // few tokens are kept of many: cheaper than their bins
        const int most = __reduce_max_sync(0xffffffffu, __popc(bits));
        uint32_t near = 0;
        if (most > 3) {
            const uint32_t w[4] = {now.x, now.y, now.z, now.w};
#pragma unroll
            for (int j = 0; j < kVec; ++j)
                if ((bits >> j & 1) && take(w[j >> 1] >> (j & 1 ? 16 : 0) & 0xffffu)) near |= 1u << j;
        } else {
#pragma unroll 1
            for (uint32_t rest = bits; rest; rest &= rest - 1) {
                const int j = __ffs(rest) - 1;
                if (take(stream.raw_element(j))) near |= 1u << j;
            }
        }
        if (__any_sync(0xffffffffu, near != 0)) {
#pragma unroll 1
            for (; near; near &= near - 1) near_zero(stream.raw_element(__ffs(near) - 1));
        }
    }
    const int32_t t = view.edge(g0, g1);
    if (t >= 0 && view.valid(t)) {
        const uint32_t u = __float_as_uint(widen(view.row[t])) >> 16;
        if (take(u)) near_zero(u);
    }
    if (sh.ties == kAllTies) ties = 0;  // the first bin that is not kept
    mass = warp_sum(mass);
    count = __reduce_add_sync(0xffffffffu, count), ties = __reduce_add_sync(0xffffffffu, ties);
    if (lane == 0) {
        sh.warp_count[warp] = count;
        *cluster.map_shared_rank(&sh.spans[rank * kWarps + warp], 0) = mass;
        *cluster.map_shared_rank(&sh.warp_counts[rank * kWarps + warp], 0) = ties;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        int64_t all = 0;
        for (int w = 0; w < kWarps; ++w) all += sh.warp_count[w];
        *cluster.map_shared_rank(&sh.counts[rank], 0) = all;
    }
    cluster.sync();
}

// The lowest valid token with the score, through rank 0's sh.pick.
template <typename T>
__device__ __noinline__ uint32_t lowest_at(Shared& sh, const RowView<T>& shared_view, float score) {
    cg::cluster_group cluster = cg::this_cluster();
    const RowView<T> view = shared_view;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int32_t g0 = sh.bounds[warp], g1 = sh.bounds[warp + 1];
    constexpr int kVec = RowView<T>::kVec;
    if (threadIdx.x == 0) sh.pick = 0xffffffffu;
    cluster.sync();
    uint32_t best = 0xffffffffu;
    for (int32_t g = max(g0, view.full0) + lane; g < min(g1, view.full1) && best == 0xffffffffu; g += 32) {
        const uint32_t b = view.bits(g);
        if (b == 0) continue;
        float x[kVec];
        view.expand(view.fetch(g), x);
#pragma unroll
        for (int i = kVec - 1; i >= 0; --i)
            if (((b >> i) & 1) && x[i] == score) best = static_cast<uint32_t>(view.first(g) + i);
    }
    const int32_t t = view.edge(g0, g1);
    if (t >= 0 && view.valid(t) && widen(view.row[t]) == score) best = min(best, static_cast<uint32_t>(t));
    best = __reduce_min_sync(0xffffffffu, best);
    if (lane == 0 && best != 0xffffffffu) atomicMin(cluster.map_shared_rank(&sh.pick, 0), best);
    cluster.sync();
    return sh.pick;
}

// Finds the drawn token (sh.token) in the span that holds the target: every warp weighs a part of it, and the part that holds
// the target is walked, one token per thread and round.  Of the tokens up to `end` that score as it does, the span keeps the
// first `ties`.  (Walking the whole span took 40 us more of 750 for 1,152 rows.)
template <typename T>
__device__ __noinline__ void walk_span(Shared& sh, const RowView<T>& shared_view, int span, Place end, int32_t ties) {
    const RowView<T> view = shared_view;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const double target = sh.target;
    double before = sh.before;
    int32_t s0 = max(view.first(sh.bounds[span]), 0);
    int32_t s1 = static_cast<int32_t>(min(static_cast<int64_t>(view.vocab), static_cast<int64_t>(sh.bounds[span + 1]) * RowView<T>::kVec - view.skew));
    auto score = [&](int32_t t) {  // of a token up to `end`, else -inf
        const float x = t < s1 && view.valid(t) ? widen(view.row[t]) : -INFINITY;
        return end.keeps(x, static_cast<uint32_t>(t)) ? x : -INFINITY;
    };
    auto weigh = [&](float x) { return weight_of(x, sh.top, sh.rate, sh.exp_table); };
    if (threadIdx.x == 0) sh.token = -1;
    const int32_t part = ((s1 - s0 + kWarps - 1) / kWarps + 31) & ~31;
    const int32_t stop = min(s1, s0 + (warp + 1) * part);
    double mass = 0.0;
    int equal = 0;
#pragma unroll 4
    for (int32_t t = s0 + warp * part + lane; t < stop; t += 32) {
        const float x = score(t);
        if (ties != kAllTies && x == end.x) ++equal;
        else if (x > -INFINITY) mass += weigh(x);
    }
    mass = warp_sum(mass);
    equal = __reduce_add_sync(0xffffffffu, equal);
    __syncthreads();
    if (lane == 0) sh.warp_mass[warp] = mass, sh.warp_count[warp] = equal;
    __syncthreads();
    // The first part whose running mass exceeds the target; without one (rounding at the very end) the last with mass.
    double run = before, from = before;
    int32_t left = ties, left_from = ties, owner = 0;
    const double one = ties != kAllTies ? weigh(end.x) : 0.0;
    for (int w = 0; w < kWarps; ++w) {
        const int32_t keep = min(static_cast<int32_t>(sh.warp_count[w]), left);
        const double m = sh.warp_mass[w] + keep * one;
        if (m > 0.0) owner = w, from = run, left_from = left;
        run += m;
        if (ties != kAllTies) left -= keep;
        if (m > 0.0 && run > target) break;
    }
    before = from, ties = left_from;
    s0 += owner * part;
    s1 = min(s1, s0 + part);
    for (int32_t base = s0; base < s1; base += kThreads) {
        const int32_t t = base + threadIdx.x;
        const float x = score(t);
        bool in = x > -INFINITY;
        if (ties != kAllTies) {
            int64_t all;
            const int64_t ahead = block_before(static_cast<int64_t>(in && x == end.x), sh.warp_count, all);
            in = in && (x != end.x || ahead < ties);
            ties -= static_cast<int32_t>(min(all, static_cast<int64_t>(ties)));
        }
        const double w = in ? weigh(x) : 0.0;
        double all;
        const double run_here = before + block_before(w, sh.warp_mass, all) + w;
        // The first token that crosses the target; without one the last one with mass.
        if (threadIdx.x == 0) sh.pick = 0xffffffffu, sh.last = 0;
        __syncthreads();
        if (w > 0.0) {
            if (run_here > target) atomicMin(&sh.pick, threadIdx.x);
            atomicMax(&sh.last, threadIdx.x + 1);
        }
        __syncthreads();
        if (threadIdx.x == 0) {
            if (sh.pick != 0xffffffffu) sh.token = base + static_cast<int32_t>(sh.pick);
            else if (sh.last) sh.token = base + static_cast<int32_t>(sh.last) - 1;
        }
        if (sh.pick != 0xffffffffu) break;
        before += all;
    }
    __syncthreads();
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
    if (c > 1) ptx::cluster_arrive_relaxed();  // first_pass waits for it before it stores into other CTAs
    RowView<T>& view = *reinterpret_cast<RowView<T>*>(sh.view);
    static_assert(sizeof(RowView<T>) <= sizeof sh.view, "space of the view");
    if (threadIdx.x == 0) {
        view = RowView<T>(static_cast<const T*>(p.logits) + r * p.vocab, p.masks ? p.masks + mrow * p.words : nullptr, p.vocab);
        const int64_t g = view.groups, c0 = g * rank / c, slice = g * (rank + 1) / c - c0;
        for (int w = 0; w <= kWarps; ++w) sh.bounds[w] = static_cast<int32_t>(c0 + slice * w / kWarps);
    }
    static_assert(2 * kQueue<float> >= kQueue<__half>, "queue space");
    __syncthreads();

    // What the first pass can keep: see there.  (A greedy row keeps nothing that is used.)
    const int mode = top_k > 0 && top_k <= 32 ? 1 : min_p > 0.0 && top_p >= 1.0 ? 2 : 0;
    const float drop = mode == 2 ? __double2float_ru(-temp * (log(min_p) - 1e-6)) : 0.f;
    RowStats st = first_pass<T>(sh, view, mode, drop);
    const bool greedy = temp == 0.0;
    int turn = 0;
    if (st.flags & 1) code = BMS_STATUS_NAN;
    else if (!greedy && st.max == INFINITY) code = BMS_STATUS_POS_INF;
    else if (!(st.flags & 2)) code = BMS_STATUS_EMPTY;
    else if (!greedy && st.finite == 0) code = BMS_STATUS_NO_MASS;
    else if (!greedy && !(u >= 0.0 && u < 1.0)) code = BMS_STATUS_BAD_UNIFORM;
    if (code != BMS_STATUS_OK) {
        if (rank == 0 && threadIdx.x == 0) finish(-1, 0, code);
        return;  // nothing remote is outstanding: the statistics arrived before the barrier
    }
    if (greedy) {
        const uint32_t token = lowest_at<T>(sh, view, st.max);
        if (rank == 0 && threadIdx.x == 0) finish(token, 1, BMS_STATUS_OK);
        return;
    }
    const int64_t k = top_k > 0 ? min(top_k, static_cast<int64_t>(st.finite)) : st.finite;
    const bool k_cuts = k < st.finite;
    static_assert(kTable == kThreads, "an entry per thread");
    sh.exp_table[threadIdx.x] = exp2(threadIdx.x / static_cast<double>(kTable));
    if (threadIdx.x == 64) {
        sh.topf = st.max, sh.top = st.max;
        sh.top_p = top_p, sh.u = u, sh.k = k;
        sh.rate = fmin(kTable / 0.69314718055994530942 / temp, DBL_MAX);
        sh.width = static_cast<float>(fmin(40.0 * temp, 1e30)) / kBins;  // 40 T below the maximum weighs 4e-18
        sh.bin_scale = 1.0f / sh.width;
        sh.bin_at = sh.topf * sh.bin_scale;
        sh.shift = sizeof(T) == 4 ? 0 : std::is_same_v<T, __half> ? 13 : 16;
        sh.top_rank = score_rank(__float_as_uint(st.max) >> 16);
        sh.first_k = static_cast<uint64_t>(order_bits(-INFINITY)) << 32;
    }
    __syncthreads();
    if (warp == 0) {
        // min-p as a score: the lowest float whose weight reaches it (weights grow with the score), by a 33-way search.
        uint32_t lo = order_bits(-FLT_MAX), hi = order_bits(st.max);
        while (min_p > 0.0 && lo < hi) {
            const uint32_t at = lo + static_cast<uint32_t>((static_cast<uint64_t>(hi - lo) * (lane + 1)) / 33);
            const uint32_t reach = __ballot_sync(0xffffffffu, weight_of(order_value(at), sh.top, sh.rate, sh.exp_table) >= min_p);
            const int first = reach ? __ffs(reach) - 1 : 32;
            const uint32_t base = lo, width = hi - lo;
            if (first < 32) hi = base + static_cast<uint32_t>((static_cast<uint64_t>(width) * (first + 1)) / 33);
            if (first > 0) lo = base + static_cast<uint32_t>((static_cast<uint64_t>(width) * first) / 33) + 1;
        }
        if (lane == 0) sh.floor_x = min_p > 0.0 ? order_value(hi) : -INFINITY;
    }
    __syncthreads();
    auto from_list = [&](uint32_t n) {
        if (rank == 0) {
            finish_list(sh, static_cast<int>(n), &p.tokens[r], &p.kept[r]);
            if (threadIdx.x == 0) p.status[r] = BMS_STATUS_OK;
        }
    };

    // The tokens that can be kept, where a bound is known: the first pass has them, or another pass collects them.
    float low = -INFINITY;
    if (k_cuts) low = k * 5 <= 4 * 4 * kWarps * c && 4 * kWarps * c <= kThreads ? kth_maximum(sh, static_cast<int>(k), c) : k <= 2 * kThreads * c ? st.low : -INFINITY;
    else if (top_p >= 1.0) low = sh.floor_x;
    const bool have = !(st.flags & 4) && (mode != 0 || st.finite <= kCap || low > -INFINITY);
    if (have || st.finite <= kCap || low > -INFINITY) {
        low = fmaxf(low, -FLT_MAX);
        const uint32_t n = have ? gather(sh, low) : collect<T>(sh, view, low);
        if (n <= kCap) return from_list(n);
    }

    bool by_score = false;
    if constexpr (kScoreBins<T>) {
        if (k_cuts || top_p < 1.0) {
            count_scores<T>(sh, view);
            by_score = cut_scores(sh, sh.merged, c, k_cuts);
            if (by_score) weigh_kept<T>(sh, view);
        }
    }

    // End of the first k tokens: exact counts find the bin that holds rank k; its tokens, sorted, give the place.
    if (k_cuts && !by_score) {
        count_bins<T>(sh, view);
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
        if (before + inside <= kCap && bin < kBins - 1) {
            // A score a little below the bin: all of the first k tokens lie above it.
            low = sh.topf - (bin + 1) * sh.width - 1e-5f * (fabsf(sh.topf) + sh.width * kBins);
            if (bin_of(low, sh.bin_at, sh.bin_scale) > bin) {
                const uint32_t n = collect<T>(sh, view, fmaxf(low, -FLT_MAX));
                if (n <= kCap) return from_list(n);
            }
        }
        if (inside <= kCap) {
            collect_bin<T>(sh, view, bin);
            const uint32_t n = pool(sh);
            if (rank == 0) {
                int kept;
                double mass;
                const uint64_t key = list_cut(sh, static_cast<int>(n), k - before, 1.0, 0.0, 0.0, kept, mass);
                if (threadIdx.x < c) *cluster.map_shared_rank(&sh.cut, threadIdx.x) = key;
            }
            cluster.sync();
        } else {
            const uint64_t key = bisect<T>(sh, view, 0, static_cast<double>(k), false, turn);
            if (threadIdx.x == 0) sh.cut = key;
        }
        __syncthreads();
        if (threadIdx.x == 0) sh.first_k = sh.cut;
        __syncthreads();
    }
    uint64_t cut = sh.first_k;
    bool have_spans = by_score;
    if (top_p < 1.0 && !by_score) {
        have_spans = find_nucleus<T>(sh, view, &p.kept[r], &p.status[r]);
        if (!have_spans) {
            const double limit = top_p * sum_above<T>(sh, view, 0, cut, true, turn).mass;
            cut = bisect<T>(sh, view, cut, limit, true, turn);
        } else {
            cut = max(cut, sh.cut);
        }
    }
    // min-p: no token below its score, any token at it.
    const Place end = by_score ? Place{sh.threshold, 0xffffffffu} : place_of(max(cut, static_cast<uint64_t>(order_bits(sh.floor_x)) << 32));
    // Kept masses by spans, unless the nucleus left them; rank 0 finds the span that holds the target.
    if (!have_spans) {
        if (end.x > -INFINITY) weigh_spans<T, true>(sh, view, end);
        else weigh_spans<T, false>(sh, view, end);
        if (rank == 0 && threadIdx.x == 0) {
            int64_t all = 0;
            for (int i = 0; i < c; ++i) all += sh.counts[i];
            p.kept[r] = all;
            p.status[r] = BMS_STATUS_OK;
        }
    }
    if (rank == 0) {
        __syncthreads();
        // Running masses of the spans, in token order.
        static_assert(kMaxCluster * kWarps <= kThreads, "a span per thread");
        double mine = threadIdx.x < c * kWarps ? sh.spans[threadIdx.x] : 0.0;
        int32_t limit = kAllTies;
        if (by_score) {  // the kept tokens at the threshold, the first of the row
            int64_t all;
            const int64_t have = threadIdx.x < c * kWarps ? sh.warp_counts[threadIdx.x] : 0;
            const int64_t ahead = block_before(have, sh.warp_count, all);
            const int64_t keep = min(max(sh.ties - ahead, static_cast<int64_t>(0)), have);
            mine += keep * weight_of(sh.threshold, sh.top, sh.rate, sh.exp_table);
            if (keep < have) limit = static_cast<int32_t>(keep);
            if (threadIdx.x == 0) {
                int64_t n = min(static_cast<int64_t>(sh.ties), all);
                for (int i = 0; i < c; ++i) n += sh.counts[i];
                p.kept[r] = n;
                p.status[r] = BMS_STATUS_OK;
            }
        }
        double total;
        const double before = block_before(mine, sh.warp_mass, total);
        const double target = u * total;
        if (threadIdx.x == 0) sh.pick = 0xffffffffu, sh.last = 0;
        __syncthreads();
        // The first span whose running mass exceeds the target; without one (rounding at the very end) the last with mass.
        if (mine > 0.0) {
            if (before + mine > target) atomicMin(&sh.pick, threadIdx.x);
            atomicMax(&sh.last, threadIdx.x);
        }
        __syncthreads();
        const uint32_t owner = sh.pick != 0xffffffffu ? sh.pick : sh.last;
        if (threadIdx.x == owner) {
            for (int i = 0; i < c; ++i) {
                *cluster.map_shared_rank(&sh.owner, i) = static_cast<int32_t>(owner);
                *cluster.map_shared_rank(&sh.target, i) = target;
                *cluster.map_shared_rank(&sh.before, i) = before;
                *cluster.map_shared_rank(&sh.tie_limit, i) = limit;
            }
        }
    }
    cluster.sync();
    if (sh.owner / kWarps == rank) {
        walk_span<T>(sh, view, sh.owner % kWarps, end, sh.tie_limit);
        if (threadIdx.x == 0) p.tokens[r] = sh.token;
    }
}

template <typename T>
int launch_filter(const FilterParams& p, int device, cudaStream_t stream) {
    static std::atomic<int> sm_counts[kMaxDevices];  // 0: not set up; calls of several threads may set up twice, to the same end
    auto kernel = filter_sample_kernel<T>;
    constexpr size_t smem = sizeof(Shared);
    static_assert(2 * (smem + 1024) <= 228 * 1024, "two CTAs per SM");
    int sms = sm_counts[device].load(std::memory_order_acquire);
    if (sms == 0) {
        BMS_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem)), "cudaFuncSetAttribute(smem)");
        BMS_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1), "cudaFuncSetAttribute(cluster)");
        BMS_CUDA(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device), "sm count");
        sm_counts[device].store(sms, std::memory_order_release);
    }
    // CTAs per row.  Few rows are split for latency, as long as the parts run side by side (two CTAs per SM): with 1 / 2 / 4 / 8 CTAs,
    // rows of 151,936 with top-p 0.9 take 107 / 66 / 46 / 37 us for 8 of them, 108 / 66 / 46 / 52 for 32, 108 / 67 / 65 / 99 for 64
    // and 108 / 96 / 125 / 184 for 128; 64 float32 rows of 50,257 with min-p 54 / 36 / 25 with 1 / 2 / 4.  Two keep a row that takes long (a wide nucleus) from ending the launch alone: 256 rows of
    // mixed filters and masks take 166 / 133 / 149 / 224 us.  Many rows keep the SMs busy by themselves (600: 398 / 405 / 505 / 799).
    int c = p.rows * 16 <= sms ? 8 : p.rows * 2 <= sms ? 4 : p.rows <= 2 * sms ? 2 : 1;
    while (c > 1 && p.vocab / c < 4096) c /= 2;
    if (p.rows * c > 2147483647LL) return fail(BMS_ERROR_UNSUPPORTED, "too many rows");
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(static_cast<unsigned>(p.rows * c));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = smem;
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
    if (vocab > 2147479552LL) return fail(BMS_ERROR_UNSUPPORTED, "vocabulary beyond 2^31 - 4096 tokens");  // 32-bit token arithmetic
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
    if (device >= kMaxDevices) return fail(BMS_ERROR_UNSUPPORTED, "device %d", device);
    DeviceGuard guard;
    BMS_CUDA(guard.enter(device), "cudaSetDevice");
    const FilterParams p{logits, masks, mask_rows, mask_table_rows, rows, vocab, (vocab + 31) / 32, f.temperature, f.top_p, f.min_p, f.top_k,
                         f.temperatures, f.top_ps, f.min_ps, f.top_ks, uniforms, tokens, kept, status};
    const auto st = static_cast<cudaStream_t>(stream);
    if (dtype == BMS_FLOAT32) return launch_filter<float>(p, device, st);
    if (dtype == BMS_BFLOAT16) return launch_filter<__nv_bfloat16>(p, device, st);
    return launch_filter<__half>(p, device, st);
}
