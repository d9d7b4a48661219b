// Paged key/value cache: page planning, rotary append, and attention of a chunk of new tokens.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <cfloat>
#include <cmath>

#include "../../include/bms_b200.h"
#include "abi_common.cuh"

namespace bms {
namespace {

constexpr int kMaxPlanSeqs = 8192;

// Entry points may be called while the caller's stream is being captured: pointer queries are
// allowed there in the relaxed mode only.
struct RelaxedCapture {
    cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
    RelaxedCapture() { cudaThreadExchangeStreamCaptureMode(&mode); }
    ~RelaxedCapture() { cudaThreadExchangeStreamCaptureMode(&mode); }
};

template <typename T>
struct Convert;
template <>
struct Convert<float> {
    static __device__ __forceinline__ float up(float x) { return x; }
    static __device__ __forceinline__ float down(float x) { return x; }
};
template <>
struct Convert<__nv_bfloat16> {
    static __device__ __forceinline__ float up(__nv_bfloat16 x) { return __bfloat162float(x); }
    static __device__ __forceinline__ __nv_bfloat16 down(float x) { return __float2bfloat16_rn(x); }
};
template <>
struct Convert<__half> {
    static __device__ __forceinline__ float up(__half x) { return __half2float(x); }
    static __device__ __forceinline__ __half down(float x) { return __float2half_rn(x); }
};

// ---------------------------------------------------------------- page plan
struct PlanParams {
    const int32_t *past, *fresh, *held, *free_count;
    int32_t *table, *free_pages;
    int32_t *query_start, *seq_lens, *positions, *held_out, *free_count_out, *status;
    int64_t* slots;
    int32_t seqs, width, pages, page_size, tokens;
};

constexpr int kPlanThreads = 512;

__device__ __forceinline__ int64_t warp_scan(int64_t v, int lane) {
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const int64_t up = __shfl_up_sync(0xffffffffu, v, d);
        if (lane >= d) v += up;
    }
    return v;
}

// Inclusive block scan of three values per thread; `carry` holds the running totals before the block.
__device__ __forceinline__ void block_scan3(int64_t (&v)[3], int64_t (&carry)[3], int64_t (*warp_tot)[3]) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    constexpr int kWarps = kPlanThreads / 32;
#pragma unroll
    for (int i = 0; i < 3; ++i) v[i] = warp_scan(v[i], lane);
    __syncthreads();
    if (lane == 31) {
#pragma unroll
        for (int i = 0; i < 3; ++i) warp_tot[warp][i] = v[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 3; ++i) {
        int64_t before = carry[i], all = carry[i];
        for (int w = 0; w < kWarps; ++w) {
            const int64_t t = warp_tot[w][i];
            if (w < warp) before += t;
            all += t;
        }
        v[i] += before;
        carry[i] = all;
    }
}

// Every CTA scans all sequences (new tokens, pages given back, pages taken; 12 bytes each, from L2)
// into shared memory, then does its share: sequences s = blockIdx.x, blockIdx.x + gridDim.x, ... (table
// entries, per-sequence outputs) and a contiguous range of tokens, each found by a binary search
// over the starts.  One launch and no exchange between CTAs; the scan is repeated instead, which
// costs about a microsecond at 1,024 sequences against a second launch.  Nothing a CTA writes is read by
// another one: given-back pages are read from entries [need, held) of shrinking rows, taken ones
// written to entries [held, need) of growing rows; the stack is read below free_count and written
// from it on.  Bound by latency: 6.3 us for 32 sequences, 10.5 for 1,024 (two scans of a chain of loads, a binary search per
// token, one dependent table load); the host's part of a call is longer than that.
__global__ void __launch_bounds__(kPlanThreads) page_plan_kernel(const PlanParams p) {
    extern __shared__ int32_t plan_smem[];
    __shared__ int64_t warp_tot[kPlanThreads / 32][3];
    int32_t* start = plan_smem;              // [seqs + 1] first token
    int32_t* drop_at = start + p.seqs + 1;   // [seqs + 1] pages given back by earlier sequences
    int32_t* grab_at = drop_at + p.seqs + 1; // [seqs] pages taken by earlier sequences, -1: failed
    const int64_t page = p.page_size;
    const int32_t count = min(max(*p.free_count, 0), p.pages);

    int64_t carry[3] = {0, 0, 0};
    if (threadIdx.x == 0) start[0] = drop_at[0] = 0;
    for (int base = 0; base < p.seqs; base += kPlanThreads) {
        const int s = base + threadIdx.x;
        int64_t v[3] = {0, 0, 0};
        int64_t past = 0, fresh = 0, held = 0;
        if (s < p.seqs) {
            past = p.past[s], fresh = p.fresh[s], held = p.held[s];
            v[0] = fresh > 0 ? fresh : 0;
        }
        // Whether the step's token capacity holds the sequence depends on the starts: scan them first.
        int64_t first[3] = {v[0], 0, 0}, c0[3] = {carry[0], 0, 0};
        block_scan3(first, c0, warp_tot);
        const bool good = s < p.seqs && past >= 0 && fresh >= 0 && held >= 0 && held <= p.width && past <= held * page &&
                          past + fresh <= p.width * page && first[0] <= p.tokens;
        const int64_t need = good ? (past + fresh + page - 1) / page : held;
        v[0] = 0;
        v[1] = held > need ? held - need : 0;
        v[2] = need > held ? need - held : 0;
        const int64_t grab = v[2];
        int64_t c12[3] = {0, carry[1], carry[2]};
        block_scan3(v, c12, warp_tot);
        carry[0] = c0[0], carry[1] = c12[1], carry[2] = c12[2];
        if (s < p.seqs) {
            start[s + 1] = static_cast<int32_t>(min(first[0], static_cast<int64_t>(p.tokens)));
            drop_at[s + 1] = static_cast<int32_t>(v[1]);
            grab_at[s] = good ? static_cast<int32_t>(v[2] - grab) : -1;
        }
    }
    __syncthreads();
    const int32_t level = count + drop_at[p.seqs];  // pages that can be handed out

    // A sequence's demand is met iff all demands up to its own fit: later ones cannot overtake it.
    auto shape = [&](int s, int32_t& held, int32_t& need, bool& good, bool& enough) {
        held = p.held[s];
        good = grab_at[s] >= 0;
        need = good ? static_cast<int32_t>((static_cast<int64_t>(p.past[s]) + p.fresh[s] + page - 1) / page) : held;
        enough = need <= held || static_cast<int64_t>(grab_at[s]) + need - held <= level;
        good = good && enough;
    };
    // Entry `pos` of the stack of free and given-back pages.
    auto stack_page = [&](int32_t pos) {
        if (pos < count) return p.free_pages[pos];
        const int32_t j = pos - count;
        int lo = 0, hi = p.seqs - 1;  // the sequence s with drop_at[s] <= j < drop_at[s + 1]
        while (lo < hi) {
            const int mid = (lo + hi) >> 1;
            if (drop_at[mid + 1] > j) hi = mid;
            else lo = mid + 1;
        }
        const int32_t need = static_cast<int32_t>((static_cast<int64_t>(p.past[lo]) + p.fresh[lo] + page - 1) / page);
        return p.table[static_cast<int64_t>(lo) * p.width + need + (j - drop_at[lo])];
    };

    const int lane = threadIdx.x & 31;
    const int warps = gridDim.x * (kPlanThreads / 32);
    for (int s = blockIdx.x * (kPlanThreads / 32) + (threadIdx.x >> 5); s < p.seqs; s += warps) {
        int32_t held, need;
        bool good, enough;
        shape(s, held, need, good, enough);
        if (good) {
            int32_t* row = p.table + static_cast<int64_t>(s) * p.width;
            for (int32_t i = held + lane; i < need; i += 32) row[i] = stack_page(level - 1 - grab_at[s] - (i - held));
        }
        if (lane == 0) {
            p.query_start[s + 1] = start[s + 1];
            p.seq_lens[s] = good ? p.past[s] + p.fresh[s] : 0;
            p.held_out[s] = good ? need : held;
            p.status[s] = good ? BMS_STATUS_OK : (enough ? BMS_STATUS_BAD_LENGTH : BMS_STATUS_NO_PAGES);
        }
    }
    // Pages left on the stack above the old free ones: given back and not taken.
    int32_t taken = 0;
    {
        // The last sequence whose demand is met ends the taken range: demands are met in order.
        int32_t most = 0;
        for (int s = threadIdx.x; s < p.seqs; s += kPlanThreads) {
            int32_t held, need;
            bool good, enough;
            shape(s, held, need, good, enough);
            if (good && need > held) most = max(most, grab_at[s] + need - held);
        }
#pragma unroll
        for (int d = 16; d; d >>= 1) most = max(most, __shfl_xor_sync(0xffffffffu, most, d));
        __syncthreads();
        if (lane == 0) warp_tot[threadIdx.x >> 5][0] = most;
        __syncthreads();
        for (int w = 0; w < kPlanThreads / 32; ++w) taken = max(taken, static_cast<int32_t>(warp_tot[w][0]));
    }
    const int32_t left = min(level - taken, p.pages);
    for (int32_t i = count + blockIdx.x * kPlanThreads + threadIdx.x; i < left; i += gridDim.x * kPlanThreads)
        p.free_pages[i] = stack_page(i);
    if (blockIdx.x == 0 && threadIdx.x == 0) {
        p.query_start[0] = 0;
        *p.free_count_out = left;
    }

    const int32_t total = start[p.seqs];
    for (int32_t t = blockIdx.x * kPlanThreads + threadIdx.x; t < p.tokens; t += gridDim.x * kPlanThreads) {
        int32_t position = -1;
        int64_t slot = -1;
        if (t < total) {
            int lo = 0, hi = p.seqs - 1;  // the sequence s with start[s] <= t < start[s + 1]
            while (lo < hi) {
                const int mid = (lo + hi) >> 1;
                if (start[mid + 1] > t) hi = mid;
                else lo = mid + 1;
            }
            int32_t held, need;
            bool good, enough;
            shape(lo, held, need, good, enough);
            if (good) {
                position = p.past[lo] + (t - start[lo]);
                const int32_t i = position / p.page_size;
                const int32_t pg = i < held ? p.table[static_cast<int64_t>(lo) * p.width + i]
                                            : stack_page(level - 1 - grab_at[lo] - (i - held));
                if (pg >= 0 && pg < p.pages) slot = static_cast<int64_t>(pg) * p.page_size + position % p.page_size;
            }
        }
        p.positions[t] = position;
        p.slots[t] = slot;
    }
}

// ---------------------------------------------------------------- rotary append
struct AppendParams {
    const void *q, *k, *v;
    void *q_out, *k_cache, *v_cache;
    const float *cos, *sin;
    const int32_t* positions;
    const int64_t* slots;
    int32_t* status;
    int64_t tokens, max_positions, total_slots;
    int64_t q_tok, q_head, k_tok, k_head, v_tok, v_head;
    int64_t kc_page, kc_slot, kc_head, vc_page, vc_slot, vc_head;
    int32_t heads, kv_heads, half, page_size;
};

template <typename T, int kVec>
struct alignas(sizeof(T) * kVec) Pack {
    T v[kVec];
};

// Inputs are read once and results not read here: both stream through the caches, which leaves the L2 to the
// rotation's tables and whatever else is live (24 prompts, 445 MB: 84 us without the hints, 78 with the loads', 70 with both,
// at two rows per thread).
template <typename P>
__device__ __forceinline__ P load_once(const void* x) {
    if constexpr (sizeof(P) == 16) {
        const uint4 r = __ldcs(reinterpret_cast<const uint4*>(x));
        return *reinterpret_cast<const P*>(&r);
    } else {
        return *reinterpret_cast<const P*>(x);
    }
}
template <typename P>
__device__ __forceinline__ void store_once(void* x, const P& v) {
    if constexpr (sizeof(P) == 16) __stcs(reinterpret_cast<uint4*>(x), *reinterpret_cast<const uint4*>(&v));
    else *reinterpret_cast<P*>(x) = v;
}

// A token's rows are its query heads, key heads (rotate) and value heads (copy).  A block has one token (blockIdx.y: a share
// of its rows): threadIdx.x is a vector of kVec elements of each half, threadIdx.y a row, and a thread takes up to
// kBatch rows, blockDim.y apart.  Their loads go out before anything that depends on the position, and before any
// store.  Bound by HBM for long steps: 445 MB in 68 us, the measured copy rate.  (8 blocks per SM leave 64 registers:
// three rows in flight fit but for 32 bytes of 16-bit types that spill; with fewer registers the step takes 90 us and more.)
template <typename T, int kVec, int kBatch>
__global__ void __launch_bounds__(128, 8) rotary_append_kernel(const AppendParams p) {
    const int64_t t = blockIdx.x;
    const int32_t position = p.positions[t];
    const int64_t slot = p.slots[t];
    using P = Pack<T, kVec>;
    const int64_t dim = 2 * static_cast<int64_t>(p.half);
    const int row0 = blockIdx.y * kBatch * blockDim.y + threadIdx.y, rows = p.heads + 2 * p.kv_heads;
    for (int c = threadIdx.x * kVec; c < p.half; c += blockDim.x * kVec) {
        P a[kBatch], b[kBatch];
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
            const int row = row0 + u * blockDim.y;
            if (row >= rows) break;
            const T* from = row < p.heads ? static_cast<const T*>(p.q) + t * p.q_tok + row * p.q_head
                            : row < p.heads + p.kv_heads ? static_cast<const T*>(p.k) + t * p.k_tok + (row - p.heads) * p.k_head
                                                         : static_cast<const T*>(p.v) + t * p.v_tok + (row - p.heads - p.kv_heads) * p.v_head;
            a[u] = load_once<P>(from + c), b[u] = load_once<P>(from + p.half + c);
        }
        const bool bad_position = position >= p.max_positions, bad_slot = slot >= p.total_slots;
        if (p.status != nullptr && row0 == 0 && c == 0) p.status[t] = bad_position ? BMS_STATUS_BAD_POSITION : bad_slot ? BMS_STATUS_BAD_PAGE : BMS_STATUS_OK;
        if (position < 0 || bad_position || bad_slot) return;
        float cs[kVec], sn[kVec];
        const float* cr = p.cos + static_cast<int64_t>(position) * p.half + c;
        const float* sr = p.sin + static_cast<int64_t>(position) * p.half + c;
#pragma unroll
        for (int i = 0; i < kVec; ++i) cs[i] = cr[i], sn[i] = sr[i];
        const int64_t pg = max(slot, static_cast<int64_t>(0)) / p.page_size, off = max(slot, static_cast<int64_t>(0)) - pg * p.page_size;
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
            const int row = row0 + u * blockDim.y;
            if (row >= rows || (row >= p.heads && slot < 0)) break;
            if (row < p.heads + p.kv_heads) {
#pragma unroll
                for (int i = 0; i < kVec; ++i) {
                    const float lo = Convert<T>::up(a[u].v[i]), hi = Convert<T>::up(b[u].v[i]);
                    a[u].v[i] = Convert<T>::down(fmaf(lo, cs[i], -hi * sn[i]));
                    b[u].v[i] = Convert<T>::down(fmaf(lo, sn[i], hi * cs[i]));
                }
            }
            T* to = row < p.heads ? static_cast<T*>(p.q_out) + (t * p.heads + row) * dim
                    : row < p.heads + p.kv_heads ? static_cast<T*>(p.k_cache) + pg * p.kc_page + off * p.kc_slot + (row - p.heads) * p.kc_head
                                                 : static_cast<T*>(p.v_cache) + pg * p.vc_page + off * p.vc_slot + (row - p.heads - p.kv_heads) * p.vc_head;
            store_once(to + c, a[u]);
            store_once(to + p.half + c, b[u]);
        }
    }
}

template <typename T>
int launch_append(const AppendParams& p, int sms, cudaStream_t stream) {
    constexpr int kVec = 16 / sizeof(T);
    auto aligned = [](const void* x) { return reinterpret_cast<uintptr_t>(x) % 16 == 0; };
    const int64_t strides[] = {p.q_tok, p.q_head, p.k_tok, p.k_head, p.v_tok, p.v_head, p.kc_page, p.kc_slot, p.kc_head, p.vc_page, p.vc_slot, p.vc_head};
    bool wide = p.half % kVec == 0 && aligned(p.q) && aligned(p.k) && aligned(p.v) && aligned(p.q_out) && aligned(p.k_cache) && aligned(p.v_cache);
    for (const int64_t s : strides) wide = wide && s % kVec == 0;
    const int rows = p.heads + 2 * p.kv_heads;
    const int x = std::min(p.half / (wide ? kVec : 1), 128);
    // Rows per thread: one for short steps (latency: 72 tokens of 48 rows of 128 take 2.2 us with 1 and 2.8 with 3), three for long ones
    // (bandwidth: 5,000 take 22.7 and 18.9, the largest step 85 and 68); the two meet near 1,024 vectors per SM.
    const int batch = p.tokens * rows * x < 1024LL * sms ? 1 : 3;
    const int shares = (rows + batch - 1) / batch;
    const int y = std::min(shares, std::max(128 / x, 1)), z = (shares + y - 1) / y;
    if (z > 65535) return fail(BMS_ERROR_UNSUPPORTED, "too many heads");
    const dim3 grid(static_cast<unsigned>(p.tokens), z), block(x, (shares + z - 1) / z);
    auto kernel = wide ? (batch == 1 ? rotary_append_kernel<T, kVec, 1> : rotary_append_kernel<T, kVec, 3>)
                       : (batch == 1 ? rotary_append_kernel<T, 1, 1> : rotary_append_kernel<T, 1, 3>);
    kernel<<<grid, block, 0, stream>>>(p);
    BMS_CUDA(cudaGetLastError(), "rotary append launch");
    return BMS_SUCCESS;
}

// ---------------------------------------------------------------- chunk attention
struct AttendParams {
    const void* q;
    const void *k, *v;
    void* out;
    float* lse;
    const int32_t *table, *seq_lens, *query_start;
    int32_t* status;
    int64_t tokens, q_tok, q_head;
    int64_t k_page, k_slot, k_head, v_page, v_slot, v_head;
    int64_t pages, window, sinks;
    int32_t seqs, width, page_size, heads, kv_heads, dim;
    float scale;
};

// Whether a sequence's rows lie in the step and its tokens in its table row.
__device__ __forceinline__ bool lengths_fit(const AttendParams& a, int s) {
    const int64_t x = a.query_start[s], y = a.query_start[s + 1], len = a.seq_lens[s];
    return x >= 0 && y >= x && y <= a.tokens && len >= y - x && len <= static_cast<int64_t>(a.width) * a.page_size;
}

// Starts in order give every sequence rows of its own.  Broken ones (malformed input) need not: then a row belongs to the one
// sequence that fits and claims it; where several do, all of them fail, and the row is nobody's.
__device__ __forceinline__ bool start_broken(const AttendParams& a, int s) {
    const int32_t x = a.query_start[s], y = a.query_start[s + 1];
    return x < 0 || y < x || y > a.tokens;
}

// Whether another sequence that fits claims rows of sequence s, which fits.  All threads of the block take part, here and below.
__device__ bool shares_rows(const AttendParams& a, int s) {
    const int32_t x = a.query_start[s], y = a.query_start[s + 1];
    int hit = 0;
    for (int t = threadIdx.x; t < a.seqs; t += blockDim.x)
        hit |= t != s && max(a.query_start[t], x) < min(a.query_start[t + 1], y) && lengths_fit(a, t);
    return __syncthreads_or(hit) != 0;
}

constexpr int kClaimWords = 2048;  // a bitmap of 65,536 rows

// Zeroes the rows of a failed sequence, as far as they lie in the step.  If the starts are broken and its own lengths do not fit, it
// may reach over rows of others: the ones that any fitting sequence claims are left to that one.
template <typename T>
__device__ void clear_rows(const AttendParams& p, int s, bool broken, uint32_t* claimed) {
    const int64_t a = max(p.query_start[s], 0), b = min(static_cast<int64_t>(p.query_start[s + 1]), p.tokens);
    const int64_t row = static_cast<int64_t>(p.heads) * p.dim;
    const bool others = broken && !lengths_fit(p, s);
    T* out = static_cast<T*>(p.out);
    for (int64_t r0 = a; r0 < b; r0 += kClaimWords * 32) {
        const int64_t r1 = min(b, r0 + kClaimWords * 32);
        if (others) {
            __syncthreads();
            for (int i = threadIdx.x; i < kClaimWords; i += blockDim.x) claimed[i] = 0;
            __syncthreads();
            for (int t = threadIdx.x; t < p.seqs; t += blockDim.x) {
                if (!lengths_fit(p, t)) continue;
                const int from = static_cast<int>(max(p.query_start[t] - r0, static_cast<int64_t>(0)));
                const int to = static_cast<int>(min(static_cast<int64_t>(p.query_start[t + 1]), r1) - r0);
                for (int w = from >> 5; 32 * w < to; ++w) {  // word by word
                    const int lo = max(from - 32 * w, 0), hi = min(to - 32 * w, 32);
                    atomicOr(&claimed[w], (0xffffffffu >> (32 - hi)) & (0xffffffffu << lo));
                }
            }
            __syncthreads();
        }
        auto free_row = [&](int64_t r) { return !others || !(claimed[(r - r0) >> 5] >> ((r - r0) & 31) & 1); };
        for (int64_t i = r0 * row + threadIdx.x; i < r1 * row; i += blockDim.x)
            if (free_row(i / row)) out[i] = Convert<T>::down(0.f);
        if (p.lse != nullptr)
            for (int64_t i = r0 * p.heads + threadIdx.x; i < r1 * p.heads; i += blockDim.x)
                if (free_row(i / p.heads)) p.lse[i] = -INFINITY;
    }
}

// Status of each sequence's lengths, and through *broken whether the starts are (written by the first block).
__global__ void __launch_bounds__(256) attend_check_kernel(const AttendParams p, int32_t* broken) {
    for (int s = blockIdx.x * 256 + threadIdx.x; s < p.seqs; s += gridDim.x * 256) p.status[s] = lengths_fit(p, s) ? BMS_STATUS_OK : BMS_STATUS_BAD_LENGTH;
    if (blockIdx.x != 0) return;
    int bad = 0;
    for (int s = threadIdx.x; s < p.seqs; s += 256) bad |= start_broken(p, s);
    bad = __syncthreads_or(bad);
    if (threadIdx.x == 0) *broken = bad;
}

template <typename T>
__global__ void __launch_bounds__(256) attend_clear_kernel(const AttendParams p, const int32_t* broken) {
    __shared__ uint32_t claimed[kClaimWords];
    const int s = blockIdx.x;
    int32_t code = p.status[s];
    if (*broken && lengths_fit(p, s) && shares_rows(p, s)) code = BMS_STATUS_BAD_LENGTH;
    __syncthreads();
    if (code == BMS_STATUS_OK) return;
    if (threadIdx.x == 0) p.status[s] = code;
    clear_rows<T>(p, s, *broken, claimed);
}

// One warp computes one row (token, head) with plain arithmetic: 32 keys at a time, one per lane, for
// the scores, a running maximum and sum, then the lanes share the value row's elements.  Keys that
// the row does not see are never loaded.  This is the form for float32, odd dims, pages and strides, and for rows that see
// non-finite values; no tensor cores, no sharing of keys between rows, and loads that touch a line per lane: 8 single tokens
// over 600 keys take about 330 us where the tiles take 24, 64 windows of 9 over long caches 74 ms (0.4), and prompts of 2,000
// tokens 1.4 s (1.5 ms), 3 to 25 times as long as elementary torch operations.
template <typename T>
__device__ void attend_row(const AttendParams& p, int s, int64_t token, int head, float* qs) {
    const int lane = threadIdx.x & 31;
    const int64_t n = p.query_start[s + 1] - p.query_start[s];
    const int64_t pos = p.seq_lens[s] - n + (token - p.query_start[s]);
    const int kvh = head / (p.heads / p.kv_heads);
    const T* q = static_cast<const T*>(p.q) + token * p.q_tok + head * p.q_head;
    __syncwarp();
    for (int d = lane; d < p.dim; d += 32) qs[d] = Convert<T>::up(q[d]);
    __syncwarp();
    const int32_t* row = p.table + static_cast<int64_t>(s) * p.width;
    const int64_t low = p.window > 0 ? max(pos + 1 - p.window, static_cast<int64_t>(0)) : 0;
    const int64_t sinks = min(p.sinks, low);
    const int64_t visible = sinks + (pos + 1 - low);
    const float sc = p.scale * 1.4426950408889634f;
    float m = -INFINITY, l = 0.f, acc[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) acc[i] = 0.f;
    bool bad = false;
    for (int64_t j0 = 0; j0 < visible; j0 += 32) {
        const int64_t i = j0 + lane;
        const int64_t key = i < sinks ? i : low + (i - sinks);
        float x = -INFINITY;
        int64_t v_at = 0;
        const bool live = i < visible;
        if (live) {
            const int32_t pg = row[key / p.page_size];
            const int64_t off = key % p.page_size;
            if (pg < 0 || pg >= p.pages) {
                bad = true;
            } else {
                const T* kr = static_cast<const T*>(p.k) + pg * p.k_page + off * p.k_slot + kvh * p.k_head;
                v_at = pg * p.v_page + off * p.v_slot + kvh * p.v_head;
                float dot = 0.f;
                for (int d = 0; d < p.dim; ++d) dot = fmaf(qs[d], Convert<T>::up(kr[d]), dot);
                x = dot * sc;
            }
        }
        if (__any_sync(0xffffffffu, bad)) break;
        float mx = x;
#pragma unroll
        for (int d = 16; d; d >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, d));
        const float mn = fmaxf(m, mx);
        const float keep = m == -INFINITY ? 0.f : exp2f(m - mn);
        const float w = live && x != -INFINITY ? exp2f(x - mn) : 0.f;  // while all scores are -inf the maximum is, too
        float sum = w;
#pragma unroll
        for (int d = 16; d; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
        l = l * keep + sum;
        m = mn;
#pragma unroll
        for (int i8 = 0; i8 < 8; ++i8) acc[i8] *= keep;
        const int live_keys = static_cast<int>(min(visible - j0, static_cast<int64_t>(32)));
        for (int u = 0; u < live_keys; ++u) {
            const float wu = __shfl_sync(0xffffffffu, w, u);
            const T* vr = static_cast<const T*>(p.v) + __shfl_sync(0xffffffffu, v_at, u);
#pragma unroll
            for (int i8 = 0; i8 < 8; ++i8) {
                const int d = lane + 32 * i8;
                if (d < p.dim) acc[i8] = fmaf(wu, Convert<T>::up(vr[d]), acc[i8]);
            }
        }
    }
    if (__any_sync(0xffffffffu, bad)) {
        if (lane == 0) atomicMax(&p.status[s], static_cast<int32_t>(BMS_STATUS_BAD_PAGE));
        return;
    }
    T* out = static_cast<T*>(p.out) + (token * p.heads + head) * p.dim;
#pragma unroll
    for (int i8 = 0; i8 < 8; ++i8) {
        const int d = lane + 32 * i8;
        if (d < p.dim) out[d] = Convert<T>::down(acc[i8] / l);
    }
    if (lane == 0 && p.lse != nullptr) p.lse[token * p.heads + head] = m * 0.6931471805599453f + logf(l);
}

template <typename T>
__global__ void __launch_bounds__(256) attend_rows_kernel(const AttendParams p, const int32_t* broken) {
    __shared__ float qs[8][256];
    const int64_t rows = p.tokens * p.heads;
    for (int64_t r = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5); r < rows; r += static_cast<int64_t>(gridDim.x) * 8) {
        const int64_t token = r / p.heads;
        int lo = 0;
        if (!*broken) {
            int hi = p.seqs;  // the last s with query_start[s] <= token
            while (lo < hi) {
                const int mid = (lo + hi) >> 1;
                if (p.query_start[mid + 1] > token) hi = mid;
                else lo = mid + 1;
            }
            if (lo >= p.seqs || p.query_start[lo] > token || p.status[lo] == BMS_STATUS_BAD_LENGTH) continue;
        } else {  // any that fits: of several all fail
            int mine = p.seqs;
            for (int s = threadIdx.x & 31; s < p.seqs && mine == p.seqs; s += 32)
                if (p.query_start[s] <= token && token < p.query_start[s + 1] && lengths_fit(p, s)) mine = s;
            lo = __reduce_min_sync(0xffffffffu, mine);
            if (lo >= p.seqs) continue;
        }
        attend_row<T>(p, lo, token, static_cast<int>(r % p.heads), qs[threadIdx.x >> 5]);
    }
}

}  // namespace
}  // namespace bms

#include "attend.cuh"

namespace bms {
namespace {

using EncodeTiled = decltype(&cuTensorMapEncodeTiled);

// The driver's tensor-map encoder, looked up once (the library links no driver stub).
EncodeTiled encode_tiled() {
    static const EncodeTiled fn = [] {
        void* f = nullptr;
        cudaDriverEntryPointQueryResult found;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &found) != cudaSuccess || found != cudaDriverEntryPointSuccess) {
            cudaGetLastError();
            f = nullptr;
        }
        return reinterpret_cast<EncodeTiled>(f);
    }();
    return fn;
}

// Where the tile kernel takes a call: 16-bit types, dim 64 or 128, pages that divide or are divided by a tile's 128 keys
// and hold whole 8-row swizzle groups, everything on 16-byte boundaries (TMA, 16-byte query loads and
// result stores), at most 128 query heads per key head.  Other calls go row by row.
bool tiles_fit(const AttendParams& p, int dtype) {
    if (dtype == BMS_FLOAT32 || (p.dim != 64 && p.dim != 128) || p.page_size % 8 != 0) return false;
    if (tc::kTile % p.page_size != 0 && p.page_size % tc::kTile != 0) return false;
    if (tc::kTile / std::min(p.page_size, tc::kTile) > 16 || p.heads / p.kv_heads > tc::kTile || encode_tiled() == nullptr) return false;
    for (const void* x : {p.q, p.k, p.v, static_cast<const void*>(p.out)})
        if (reinterpret_cast<uintptr_t>(x) % 16 != 0) return false;
    const int64_t strides[][2] = {{p.q_tok, p.tokens}, {p.q_head, p.heads}, {p.k_page, p.pages}, {p.k_slot, p.page_size}, {p.k_head, p.kv_heads},
                                  {p.v_page, p.pages}, {p.v_slot, p.page_size}, {p.v_head, p.kv_heads}};
    for (const auto& [s, n] : strides)  // a tensor map has no stride of 0: broadcast inputs go row by row
        if (s % 8 != 0 || s >= (1LL << 38) || (s == 0 && n > 1)) return false;
    return true;
}

int page_map(CUtensorMap* map, const AttendParams& p, int dtype, const void* base, int64_t page, int64_t slot, int64_t head) {
    const cuuint64_t dims[4] = {static_cast<cuuint64_t>(p.dim), static_cast<cuuint64_t>(p.kv_heads), static_cast<cuuint64_t>(p.page_size),
                                static_cast<cuuint64_t>(p.pages)};
    // A dimension of one entry may have any stride: 16 bytes stand in for one of 0.
    const cuuint64_t strides[3] = {static_cast<cuuint64_t>(std::max<int64_t>(head * 2, 16)), static_cast<cuuint64_t>(std::max<int64_t>(slot * 2, 16)),
                                   static_cast<cuuint64_t>(std::max<int64_t>(page * 2, 16))};
    const cuuint32_t box[4] = {64, 1, static_cast<cuuint32_t>(std::min(p.page_size, tc::kTile)), 1};
    const cuuint32_t steps[4] = {1, 1, 1, 1};
    const CUresult rc = encode_tiled()(map, dtype == BMS_BFLOAT16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4,
                                       const_cast<void*>(base), dims, strides, box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                                       CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (rc != CUDA_SUCCESS) return fail(BMS_ERROR_CUDA, "tensor map of the cache (driver error %d)", static_cast<int>(rc));
    return BMS_SUCCESS;
}

int query_map(CUtensorMap* map, const AttendParams& p, int dtype, int group, int tile_tokens) {
    const cuuint64_t dims[3] = {static_cast<cuuint64_t>(p.dim), static_cast<cuuint64_t>(p.heads), static_cast<cuuint64_t>(p.tokens)};
    const cuuint64_t strides[2] = {static_cast<cuuint64_t>(std::max<int64_t>(p.q_head * 2, 16)), static_cast<cuuint64_t>(std::max<int64_t>(p.q_tok * 2, 16))};
    const cuuint32_t box[3] = {64, static_cast<cuuint32_t>(group), static_cast<cuuint32_t>(tile_tokens)};
    const cuuint32_t steps[3] = {1, 1, 1};
    const CUresult rc = encode_tiled()(map, dtype == BMS_BFLOAT16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3,
                                       const_cast<void*>(p.q), dims, strides, box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                                       CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (rc != CUDA_SUCCESS) return fail(BMS_ERROR_CUDA, "tensor map of the queries (driver error %d)", static_cast<int>(rc));
    return BMS_SUCCESS;
}

int64_t tiles_workspace(int64_t ctas, int64_t dim) { return 256 + ctas * 2 * 256 * (dim + 1) * 4 + ((ctas * 4 + 255) / 256) * 256; }

std::atomic<int32_t> g_hold_pages{0};  // bms_hold_pages

template <typename T, int D>
int launch_tiles(const AttendParams& a, int dtype, int device, int sms, void* workspace, cudaStream_t stream) {
    static std::atomic<bool> ready[kMaxDevices];  // calls of several threads may set up twice, to the same end
    auto kernel = tc::attend_tiles_kernel<T, D>;
    if (!ready[device].load(std::memory_order_acquire)) {
        BMS_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, tc::Layout<D>::kSmem), "cudaFuncSetAttribute(smem)");
        ready[device].store(true, std::memory_order_release);
    }
    const int group = a.heads / a.kv_heads;
    CUtensorMap q_map, k_map, v_map;
    BMS_CHECK(query_map(&q_map, a, dtype, group, tc::kTile / group));
    BMS_CHECK(page_map(&k_map, a, dtype, a.k, a.k_page, a.k_slot, a.k_head));
    BMS_CHECK(page_map(&v_map, a, dtype, a.v, a.v_page, a.v_slot, a.v_head));
    tc::Params p{};
    p.a = a;
    p.flags = static_cast<int32_t*>(workspace);
    unsigned char* rest = static_cast<unsigned char*>(workspace) + ((sms * 4 + 255) / 256) * 256;
    p.parts = reinterpret_cast<float*>(rest);
    p.part_lse = p.parts + static_cast<int64_t>(sms) * 2 * 256 * D;
    p.scale2 = std::max(std::fabs(a.scale) * 1.4426950408889634f, FLT_MIN);  // a factor of 0 would turn masked scores into NaN
    p.negate = a.scale < 0.f ? 0x80000000u : 0u;
    p.group = group;
    p.tile_tokens = tc::kTile / p.group;
    p.group_inv = (65536 + p.group - 1) / p.group;
    p.hold = g_hold_pages.load(std::memory_order_relaxed);
    // Both launches are programmatic dependents: their prologues run while the launch before them ends.
    cudaLaunchAttribute overlap{};
    overlap.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    overlap.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(sms), cfg.blockDim = dim3(tc::kThreads), cfg.dynamicSmemBytes = tc::Layout<D>::kSmem, cfg.stream = stream;
    cfg.attrs = &overlap, cfg.numAttrs = 1;
    BMS_CUDA(cudaLaunchKernelEx(&cfg, kernel, q_map, k_map, v_map, p), "chunk attention launch");
    cfg.gridDim = dim3(sms, 4), cfg.blockDim = dim3(tc::kFinishThreads), cfg.dynamicSmemBytes = 0;
    BMS_CUDA(cudaLaunchKernelEx(&cfg, tc::attend_finish_kernel<T, D>, p), "chunk attention launch");
    return BMS_SUCCESS;
}

template <typename T>
int launch_attend(const AttendParams& p, int sms, void* workspace, cudaStream_t stream) {
    int32_t* broken = static_cast<int32_t*>(workspace);
    attend_check_kernel<<<(p.seqs + 255) / 256, 256, 0, stream>>>(p, broken);
    const int64_t blocks = std::min<int64_t>((p.tokens * p.heads + 7) / 8, 16LL * sms);
    if (blocks > 0) attend_rows_kernel<T><<<static_cast<unsigned>(blocks), 256, 0, stream>>>(p, broken);
    attend_clear_kernel<T><<<p.seqs, 256, 0, stream>>>(p, broken);
    BMS_CUDA(cudaGetLastError(), "chunk attention launch");
    return BMS_SUCCESS;
}

int sm_count(int device, int& sms) {
    static std::atomic<int> table[kMaxDevices];
    if (device >= kMaxDevices) return fail(BMS_ERROR_UNSUPPORTED, "device %d", device);
    sms = table[device].load(std::memory_order_relaxed);
    if (sms == 0) {
        BMS_CUDA(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device), "sm count");
        table[device].store(sms, std::memory_order_relaxed);
    }
    return BMS_SUCCESS;
}

int check_row_strides(const int64_t* s) {
    if (s == nullptr) return fail(BMS_ERROR_INVALID_ARGUMENT, "strides must not be NULL");
    if (s[0] < 0 || s[1] < 0) return fail(BMS_ERROR_INVALID_ARGUMENT, "strides must not be negative");
    return BMS_SUCCESS;
}

int check_cache_shape(const bms_paged_cache* c) {
    if (c == nullptr) return fail(BMS_ERROR_INVALID_ARGUMENT, "cache must not be NULL");
    if (c->pages <= 0 || c->page_size <= 0 || c->kv_heads <= 0 || c->dim <= 0 || c->pages > 2147483647LL || c->page_size > 65536 || c->kv_heads > 65535)
        return fail(BMS_ERROR_INVALID_ARGUMENT, "invalid cache shape");
    for (int i = 0; i < 3; ++i)
        if (c->k_stride[i] < 0 || c->v_stride[i] < 0) return fail(BMS_ERROR_INVALID_ARGUMENT, "cache strides must not be negative");
    return BMS_SUCCESS;
}

int check_cache(const bms_paged_cache* c, int device, int size) {
    BMS_CHECK(check_ptr(c->k, device, "cache k", size));
    return check_ptr(c->v, device, "cache v", size);
}

int check_kind(int dtype) {
    if (dtype != BMS_FLOAT32 && dtype != BMS_BFLOAT16 && dtype != BMS_FLOAT16)
        return fail(BMS_ERROR_INVALID_ARGUMENT, "q, k and v must be float32, bfloat16 or float16 (dtype code %d)", dtype);
    return BMS_SUCCESS;
}

}  // namespace
}  // namespace bms

using namespace bms;

extern "C" {

int bms_page_plan(const int32_t* past_lens, const int32_t* new_lens, const int32_t* held, int64_t seqs, int32_t* table, int64_t width,
                  int32_t* free_pages, int64_t pages, const int32_t* free_count, int64_t page_size, int64_t tokens, int32_t* query_start,
                  int32_t* seq_lens, int32_t* positions, int64_t* slots, int32_t* held_out, int32_t* free_count_out, int32_t* status,
                  int32_t device, void* stream) {
    if (seqs <= 0 || width <= 0 || pages <= 0 || page_size <= 0 || tokens < 0)
        return fail(BMS_ERROR_INVALID_ARGUMENT, "seqs, width, pages and page_size must be positive and tokens not negative");
    if (seqs > kMaxPlanSeqs) return fail(BMS_ERROR_UNSUPPORTED, "at most %d sequences per plan", kMaxPlanSeqs);
    if (pages > 1073741823LL || page_size > 65536 || tokens > 1073741823LL || seqs * width > 1073741823LL || width * page_size > 2147483647LL)
        return fail(BMS_ERROR_UNSUPPORTED, "pages, tokens or table beyond the 32-bit range");
    RelaxedCapture relaxed;
    BMS_CHECK(check_device(device));
    const void* in[] = {past_lens, new_lens, held, free_count, table, free_pages};
    const char* in_names[] = {"past_lens", "new_lens", "held", "free_count", "table", "free_pages"};
    void* outs[] = {query_start, seq_lens, held_out, free_count_out, status, tokens ? positions : nullptr, tokens ? slots : nullptr};
    const char* out_names[] = {"query_start", "seq_lens", "held_out", "free_count_out", "status", "positions", "slots"};
    for (int i = 0; i < 6; ++i) BMS_CHECK(check_ptr(in[i], device, in_names[i], 4));
    for (int i = 0; i < (tokens ? 7 : 5); ++i) {
        BMS_CHECK(check_ptr(outs[i], device, out_names[i], i == 6 ? 8 : 4));
        for (const void* x : in)
            if (x == outs[i]) return fail(BMS_ERROR_INVALID_ARGUMENT, "%s must not alias an input", out_names[i]);
    }
    DeviceGuard guard;
    BMS_CUDA(guard.enter(device), "cudaSetDevice");
    int sms = 0;
    BMS_CHECK(sm_count(device, sms));
    const size_t smem = (3 * static_cast<size_t>(seqs) + 2) * sizeof(int32_t);
    BMS_CUDA(cudaFuncSetAttribute(page_plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 3 * (kMaxPlanSeqs + 1) * 4), "cudaFuncSetAttribute");
    const int64_t blocks = std::clamp<int64_t>(std::max((tokens + kPlanThreads - 1) / kPlanThreads, (seqs * 32 + kPlanThreads - 1) / kPlanThreads), 1, sms);
    const PlanParams p{past_lens, new_lens, held, free_count, table, free_pages, query_start, seq_lens, positions, held_out, free_count_out, status, slots,
                       static_cast<int32_t>(seqs), static_cast<int32_t>(width), static_cast<int32_t>(pages), static_cast<int32_t>(page_size),
                       static_cast<int32_t>(tokens)};
    page_plan_kernel<<<static_cast<unsigned>(blocks), kPlanThreads, smem, static_cast<cudaStream_t>(stream)>>>(p);
    BMS_CUDA(cudaGetLastError(), "page plan launch");
    return BMS_SUCCESS;
}

int bms_rotary_append(const void* q, const void* k, const void* v, int32_t dtype, int64_t tokens, int64_t heads, const int64_t q_stride[2],
                      const int64_t k_stride[2], const int64_t v_stride[2], const float* cos, const float* sin, int64_t max_positions,
                      const int32_t* positions, const int64_t* slots, void* q_out, const bms_paged_cache* cache, int32_t* status, int32_t device,
                      void* stream) {
    BMS_CHECK(check_kind(dtype));
    if (tokens < 0 || heads <= 0 || heads > 65535 || max_positions <= 0)
        return fail(BMS_ERROR_INVALID_ARGUMENT, "tokens, heads and max_positions must be positive");
    for (const int64_t* s : {q_stride, k_stride, v_stride}) BMS_CHECK(check_row_strides(s));
    BMS_CHECK(check_cache_shape(cache));
    if (cache->dim % 2 != 0 || cache->dim > 65536) return fail(BMS_ERROR_INVALID_ARGUMENT, "dim must be even");
    if (tokens > 2147483647LL) return fail(BMS_ERROR_UNSUPPORTED, "at most 2^31 - 1 tokens per call");  // a block each
    const int size = dtype == BMS_FLOAT32 ? 4 : 2;
    RelaxedCapture relaxed;
    BMS_CHECK(check_device(device));
    BMS_CHECK(check_cache(cache, device, size));
    if (tokens == 0) return BMS_SUCCESS;
    const void* ptrs[] = {q, k, v, q_out};
    const char* names[] = {"q", "k", "v", "q_out"};
    for (int i = 0; i < 4; ++i) BMS_CHECK(check_ptr(ptrs[i], device, names[i], size));
    BMS_CHECK(check_ptr(cos, device, "cos", 4));
    BMS_CHECK(check_ptr(sin, device, "sin", 4));
    BMS_CHECK(check_ptr(positions, device, "positions", 4));
    BMS_CHECK(check_ptr(slots, device, "slots", 8));
    if (status != nullptr) BMS_CHECK(check_ptr(status, device, "status", 4));
    DeviceGuard guard;
    BMS_CUDA(guard.enter(device), "cudaSetDevice");
    int sms = 0;
    BMS_CHECK(sm_count(device, sms));
    const AppendParams p{q, k, v, q_out, cache->k, cache->v, cos, sin, positions, slots, status, tokens, max_positions, cache->pages * cache->page_size,
                         q_stride[0], q_stride[1], k_stride[0], k_stride[1], v_stride[0], v_stride[1], cache->k_stride[0], cache->k_stride[1],
                         cache->k_stride[2], cache->v_stride[0], cache->v_stride[1], cache->v_stride[2], static_cast<int32_t>(heads),
                         static_cast<int32_t>(cache->kv_heads), static_cast<int32_t>(cache->dim / 2), static_cast<int32_t>(cache->page_size)};
    const auto st = static_cast<cudaStream_t>(stream);
    if (dtype == BMS_FLOAT32) return launch_append<float>(p, sms, st);
    if (dtype == BMS_BFLOAT16) return launch_append<__nv_bfloat16>(p, sms, st);
    return launch_append<__half>(p, sms, st);
}

int64_t bms_attention_workspace_bytes(int32_t device, int64_t tokens, int64_t heads, int64_t seqs, int64_t dim) {
    int sms = 0;
    if (device < 0 || tokens < 0 || heads <= 0 || seqs <= 0 || dim <= 0 || sm_count(device, sms) != BMS_SUCCESS) return -1;
    return dim == 64 || dim == 128 ? tiles_workspace(sms, dim) : 256;
}

int bms_chunk_attention(const void* q, int32_t dtype, int64_t tokens, int64_t heads, const int64_t q_stride[2], const bms_paged_cache* cache,
                        const int32_t* table, int64_t seqs, int64_t width, const int32_t* seq_lens, const int32_t* query_start, double scale,
                        int64_t window, int64_t sinks, void* out, float* lse, int32_t* status, void* workspace, int64_t workspace_bytes,
                        int32_t device, void* stream) {
    BMS_CHECK(check_kind(dtype));
    if (tokens < 0 || heads <= 0 || heads > 65535 || seqs <= 0 || width <= 0 || seqs > 1048576)
        return fail(BMS_ERROR_INVALID_ARGUMENT, "tokens, heads, seqs and width must be positive");
    if (window < 0 || sinks < 0) return fail(BMS_ERROR_INVALID_ARGUMENT, "window and sinks must not be negative");
    if (!std::isfinite(scale) || std::fabs(scale) > 1e30) return fail(BMS_ERROR_INVALID_ARGUMENT, "scale must be finite");
    BMS_CHECK(check_row_strides(q_stride));
    BMS_CHECK(check_cache_shape(cache));
    if (cache->dim > 256) return fail(BMS_ERROR_UNSUPPORTED, "dim is at most 256");
    if (heads % cache->kv_heads != 0) return fail(BMS_ERROR_INVALID_ARGUMENT, "heads must be a multiple of the cache's kv_heads");
    if (tokens > 1073741823LL || width > 2147483391LL / cache->page_size)  // positions, rounded up to a tile, fit int32
        return fail(BMS_ERROR_UNSUPPORTED, "lengths beyond the 32-bit range");
    const int size = dtype == BMS_FLOAT32 ? 4 : 2;
    RelaxedCapture relaxed;
    BMS_CHECK(check_device(device));
    BMS_CHECK(check_cache(cache, device, size));
    BMS_CHECK(check_ptr(table, device, "table", 4));
    BMS_CHECK(check_ptr(seq_lens, device, "seq_lens", 4));
    BMS_CHECK(check_ptr(query_start, device, "query_start", 4));
    BMS_CHECK(check_ptr(status, device, "status", 4));
    if (tokens > 0) {
        BMS_CHECK(check_ptr(q, device, "q", size));
        BMS_CHECK(check_ptr(out, device, "out", size));
        if (out == q) return fail(BMS_ERROR_INVALID_ARGUMENT, "out must not be q");  // rows are read again after others are written
        if (lse != nullptr) BMS_CHECK(check_ptr(lse, device, "lse", 4));
    }
    const int64_t need = bms_attention_workspace_bytes(device, tokens, heads, seqs, cache->dim);
    BMS_CHECK(check_ptr(workspace, device, "workspace", 256));
    if (workspace_bytes < need) return fail(BMS_ERROR_INVALID_ARGUMENT, "workspace needs %lld bytes", static_cast<long long>(need));
    DeviceGuard guard;
    BMS_CUDA(guard.enter(device), "cudaSetDevice");
    int sms = 0;
    BMS_CHECK(sm_count(device, sms));
    const AttendParams p{q, cache->k, cache->v, out, lse, table, seq_lens, query_start, status, tokens, q_stride[0], q_stride[1],
                         cache->k_stride[0], cache->k_stride[1], cache->k_stride[2], cache->v_stride[0], cache->v_stride[1], cache->v_stride[2],
                         cache->pages, window, sinks, static_cast<int32_t>(seqs), static_cast<int32_t>(width), static_cast<int32_t>(cache->page_size),
                         static_cast<int32_t>(heads), static_cast<int32_t>(cache->kv_heads), static_cast<int32_t>(cache->dim), static_cast<float>(scale)};
    const auto st = static_cast<cudaStream_t>(stream);
    if (dtype == BMS_FLOAT32) return launch_attend<float>(p, sms, workspace, st);
    const bool bf16 = dtype == BMS_BFLOAT16;
    if (tokens > 0 && tiles_fit(p, dtype)) {
        if (p.dim == 64)
            return bf16 ? launch_tiles<__nv_bfloat16, 64>(p, dtype, device, sms, workspace, st) : launch_tiles<__half, 64>(p, dtype, device, sms, workspace, st);
        return bf16 ? launch_tiles<__nv_bfloat16, 128>(p, dtype, device, sms, workspace, st) : launch_tiles<__half, 128>(p, dtype, device, sms, workspace, st);
    }
    return bf16 ? launch_attend<__nv_bfloat16>(p, sms, workspace, st) : launch_attend<__half>(p, sms, workspace, st);
}

int bms_hold_pages(int32_t hold) {
    g_hold_pages.store(hold != 0, std::memory_order_relaxed);
    return BMS_SUCCESS;
}

}  // extern "C"
