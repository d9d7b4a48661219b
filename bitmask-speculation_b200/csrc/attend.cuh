// Chunk attention on the tensor cores (tcgen05), for 16-bit types, dim 64 or 128 and pages that tile 128 keys.
//
// Work.  An item is (sequence, key head, query tile).  The group's query heads share their key head, so the rows of
// an item are (token, head of the group) pairs.  If a sequence's rows fit 128 they form one tile, and the two
// softmax warpgroups take even and odd key tiles, each with its own running maximum, sum and output, merged at the
// end; else an item is two tiles of 128 rows that read every key tile together.  Key tiles that no row of the item
// sees (causal bound, window, sinks) are not part of it.
//
// Split.  All items' steps (a key tile, or a pair of them for one-tile items) form one line, cut into equal
// parts, one per CTA: few long sequences fill the GPU as well as many short ones.  An item that a cut divides leaves
// float32 partials (normalised output and log2 of the sum) in the workspace, and attend_finish_kernel joins them in
// the order of the CTAs, so that results do not depend on timing.
//
// Pipeline (384 threads, one CTA per SM).  A producer warp loads pages by TMA (one box of up to 128 slots x 64
// elements per page, 128-byte swizzle) into a ring of key and value tiles in the order the products consume them.  One
// thread issues the products: S = Q K^T into TMEM, and O += P V with P in TMEM (over S) and V as an MN-major
// operand, so neither P nor V is transposed or copied.  While a warpgroup turns S into P the tensor cores work for
// the other one.  A softmax thread owns a row: no shuffles.  O is rescaled only when a row's maximum grew by more
// than a threshold (2^8 for bfloat16); sums stay float32, weights are rounded once to the inputs' type for the
// second product, because the tensor cores take both operands in that type.
//
// Hidden keys.  Scores of keys that a row does not see are replaced, so any bits there vanish.  Values cannot be:
// 0 * NaN is NaN.  In tiles that are not seen by every row, non-finite values of keys that some row does not see are
// zeroed in shared memory before the product; if another row does see such a key the CTA flags its range, and
// attend_finish_kernel computes those items again row by row.
#pragma once
#include <cuda.h>

#include "ptx.cuh"

namespace bms {
namespace tc {

constexpr int kTile = 128;              // keys per tile, rows per query tile
constexpr int kThreads = 384;           // 2 softmax warpgroups, one with the producer and the product warp
constexpr int kProducerWarp = 8, kMmaWarp = 9;
constexpr uint64_t kWaitNs = 1000000000ull;

template <int D>
struct Layout {
    static constexpr int kTileBytes = kTile * D * 2;
    static constexpr int kStages = D == 128 ? 5 : 12;
    static constexpr int kQBytes = 2 * kTileBytes;  // also the exchange of one-tile items: 128 x D float32
    static constexpr int kSmem = 1024 + kQBytes + kStages * kTileBytes;
};

struct Control {
    uint64_t full[12], empty[12];
    uint64_t q_full, s_full[2], p_full[2], o_full[2];
    float ref[kTile], sum[kTile];
    int64_t scan[kThreads / 32];
    int64_t total, start_off;
    int32_t start_seq;
    uint32_t tmem, poison, abort;
};

struct Params {
    AttendParams a;
    float* parts;      // [ctas][2][256][D]
    float* part_lse;   // [ctas][2][256], log2
    int32_t* flags;    // [ctas]: 1 poisoned values, 2 a wait ran out
    float scale2;      // |scale| log2(e)
    uint32_t negate;   // sign bits for queries of a negative scale
    int32_t group, tile_tokens;
};

// ---- schedule ---------------------------------------------------------------------------------
struct Shape {
    int64_t total;  // steps of one key head over all query tiles
    int32_t n, past, tiles;
    bool wide;
};

struct Range {  // one query tile's key tiles
    int32_t first, end;        // tokens of the sequence's chunk
    int32_t pmin, pmax;        // positions
    int32_t sink_tiles, low_tile, tiles, steps;
    __device__ __forceinline__ int32_t tile(int i) const { return i < sink_tiles ? i : low_tile + (i - sink_tiles); }
};

__device__ __forceinline__ Range query_range(const Params& p, int32_t n, int32_t past, bool wide, int qt) {
    Range r;
    const int32_t per = wide ? 2 * p.tile_tokens : p.tile_tokens;
    r.first = qt * per;
    r.end = min(n, r.first + per);
    r.pmin = past + r.first;
    r.pmax = past + r.end - 1;
    int32_t low = 0, sinks = 0;
    if (p.a.window > 0) {
        low = static_cast<int32_t>(max(static_cast<int64_t>(0), r.pmin + 1 - p.a.window));
        sinks = static_cast<int32_t>(min(p.a.sinks, static_cast<int64_t>(low)));
    }
    r.low_tile = low / kTile;
    r.sink_tiles = min((sinks + kTile - 1) / kTile, r.low_tile);
    r.tiles = r.sink_tiles + r.pmax / kTile + 1 - r.low_tile;
    r.steps = wide ? r.tiles : (r.tiles + 1) / 2;
    return r;
}

__device__ __forceinline__ bool lengths_fit(const AttendParams& a, int s) {
    const int64_t x = a.query_start[s], y = a.query_start[s + 1], len = a.seq_lens[s];
    return x >= 0 && y >= x && y <= a.tokens && len >= y - x && len <= static_cast<int64_t>(a.width) * a.page_size;
}

__device__ __forceinline__ Shape sequence_shape(const Params& p, int s) {
    Shape h{0, 0, 0, 0, false};
    if (!lengths_fit(p.a, s)) return h;
    h.n = p.a.query_start[s + 1] - p.a.query_start[s];
    if (h.n == 0) return h;
    h.past = p.a.seq_lens[s] - h.n;
    h.wide = h.n > p.tile_tokens;
    const int32_t per = h.wide ? 2 * p.tile_tokens : p.tile_tokens;
    h.tiles = (h.n + per - 1) / per;
    for (int q = 0; q < h.tiles; ++q) h.total += query_range(p, h.n, h.past, h.wide, q).steps;
    return h;
}

// Walks the items of a CTA's part of the line of steps.
struct Walk {
    int32_t s, head, qt;
    int64_t left;       // steps of the part not yet walked
    int32_t st0, st1;   // steps of the current item that belong to the part
    Shape shape;
    Range range;
    __device__ __forceinline__ void start(const Params& p, int seq, int64_t off, int64_t count) {
        s = seq, left = count;
        head = qt = st0 = 0;
        if (count <= 0) return;
        shape = sequence_shape(p, s);
        head = static_cast<int32_t>(off / shape.total);
        int64_t rest = off % shape.total;
        for (;; ++qt) {
            range = query_range(p, shape.n, shape.past, shape.wide, qt);
            if (rest < range.steps) break;
            rest -= range.steps;
        }
        st0 = static_cast<int32_t>(rest);
    }
    __device__ __forceinline__ bool valid() {
        if (left <= 0) return false;
        st1 = static_cast<int32_t>(min(static_cast<int64_t>(range.steps), st0 + left));
        return true;
    }
    __device__ __forceinline__ void next(const Params& p) {
        left -= st1 - st0;
        st0 = 0;
        if (left <= 0) return;
        if (++qt == shape.tiles) {
            qt = 0;
            if (++head == p.a.kv_heads) {
                head = 0;
                do shape = sequence_shape(p, ++s);
                while (shape.total == 0);
            }
        }
        range = query_range(p, shape.n, shape.past, shape.wide, qt);
    }
    __device__ __forceinline__ int tile0() const { return shape.wide ? st0 : 2 * st0; }
    __device__ __forceinline__ int tile1() const { return shape.wide ? st1 : min(2 * st1, range.tiles); }
    __device__ __forceinline__ bool whole() const { return st0 == 0 && st1 == range.steps; }
};

// Total steps, and the sequence and offset at which part `c` of `parts` starts.  All threads of the block take part.
template <int kBlock>
__device__ void locate(const Params& p, int64_t* scan, int64_t& total, int64_t& off, int32_t& seq, int c, int ctas) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    constexpr int kW = kBlock / 32;
    int64_t target = -1, run = 0;
    for (int pass = 0; pass < 2; ++pass) {
        run = 0;
        for (int base = 0; base < p.a.seqs; base += kBlock) {
            const int s = base + threadIdx.x;
            const int64_t mine = s < p.a.seqs ? sequence_shape(p, s).total * p.a.kv_heads : 0;
            int64_t v = mine;
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) {
                const int64_t up = __shfl_up_sync(0xffffffffu, v, d);
                if (lane >= d) v += up;
            }
            __syncthreads();
            if (lane == 31) scan[warp] = v;
            __syncthreads();
            int64_t all = run;
            for (int w = 0; w < kW; ++w) {
                if (w == warp) v += all;
                all += scan[w];
            }
            if (pass == 1 && mine > 0 && target >= v - mine && target < v) seq = s, off = target - (v - mine);
            run = all;
        }
        if (pass == 0) {
            if (threadIdx.x == 0) total = run, seq = -1, off = 0;
            const int64_t parts = min(static_cast<int64_t>(ctas), run);
            target = c < parts ? run * c / parts : -1;
        }
        __syncthreads();
    }
}

__device__ __forceinline__ int64_t part_begin(int64_t total, int c, int ctas) {
    const int64_t parts = min(static_cast<int64_t>(ctas), total);
    return c >= parts ? total : total * c / parts;
}

// ---- tcgen05 ------------------------------------------------------------------------------------
__device__ __forceinline__ void tmem_alloc(uint32_t* dst, uint32_t cols) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(ptx::smem_addr(dst)), "r"(cols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
}
__device__ __forceinline__ void tmem_free(uint32_t addr, uint32_t cols) {
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(addr), "r"(cols));
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool add) {
    asm volatile(
        "{ .reg .pred p; setp.ne.u32 p, %4, 0; tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p; }" ::"r"(d), "l"(a), "l"(b), "r"(idesc),
        "r"(static_cast<uint32_t>(add))
        : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool add) {
    asm volatile(
        "{ .reg .pred p; setp.ne.u32 p, %4, 0; tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p; }" ::"r"(d), "r"(a), "l"(b), "r"(idesc),
        "r"(static_cast<uint32_t>(add))
        : "memory");
}
__device__ __forceinline__ void mma_commit(uint64_t* bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(ptx::smem_addr(bar)) : "memory");
}
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void fence_async_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

#define BMS_R8(r, o) "=r"(r[o]), "=r"(r[o + 1]), "=r"(r[o + 2]), "=r"(r[o + 3]), "=r"(r[o + 4]), "=r"(r[o + 5]), "=r"(r[o + 6]), "=r"(r[o + 7])
#define BMS_W8(r, o) "r"(r[o]), "r"(r[o + 1]), "r"(r[o + 2]), "r"(r[o + 3]), "r"(r[o + 4]), "r"(r[o + 5]), "r"(r[o + 6]), "r"(r[o + 7])
// 32 columns of this thread's lane.
__device__ __forceinline__ void tmem_ld32(uint32_t addr, uint32_t* r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, "
        "%20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : BMS_R8(r, 0), BMS_R8(r, 8), BMS_R8(r, 16), BMS_R8(r, 24)
        : "r"(addr));
}
__device__ __forceinline__ void tmem_st32(uint32_t addr, const uint32_t* r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, "
        "%19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31};" ::BMS_W8(r, 0),
        BMS_W8(r, 8), BMS_W8(r, 16), BMS_W8(r, 24), "r"(addr)
        : "memory");
}
#undef BMS_R8
#undef BMS_W8

// Shared-memory operand with 128-byte swizzle: start address, leading and stride offsets in 16-byte units, version 1.
__device__ __forceinline__ uint64_t smem_desc(uint32_t addr, uint32_t lead, uint32_t stride) {
    return static_cast<uint64_t>((addr >> 4) & 0x3fff) | (static_cast<uint64_t>((lead >> 4) & 0x3fff) << 16) |
           (static_cast<uint64_t>((stride >> 4) & 0x3fff) << 32) | (1ull << 46) | (2ull << 61);
}

// float32 accumulator, 16-bit inputs (kind: 0 float16, 1 bfloat16), A K-major, B K- or MN-major, M = 128.
__host__ __device__ constexpr uint32_t instr_desc(uint32_t kind, bool b_mn, uint32_t n) {
    return (1u << 4) | (kind << 7) | (kind << 10) | (static_cast<uint32_t>(b_mn) << 16) | ((n >> 3) << 17) | ((128u >> 4) << 24);
}

__device__ __forceinline__ void tma_page(uint32_t dst, const CUtensorMap* map, int x, int head, int slot, int page, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(dst), "l"(map),
        "r"(bar), "r"(x), "r"(head), "r"(slot), "r"(page)
        : "memory");
}

// Waits at most about a second; after that the CTA's abort flag ends every wait at once.
__device__ __forceinline__ void wait_bar(Control& c, uint64_t* bar, uint32_t parity) {
    const uint32_t addr = ptx::smem_addr(bar);
    if (ptx::mbar_try_wait(addr, parity)) return;
    const uint64_t t0 = ptx::globaltimer();
    volatile uint32_t* abort = &c.abort;
    while (!ptx::mbar_try_wait(addr, parity)) {
        if (*abort) return;
        if (ptx::globaltimer() - t0 > kWaitNs) {
            *abort = 1;
            return;
        }
    }
}

__device__ __forceinline__ uint32_t pack_pair(float lo, float hi, __nv_bfloat16) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ uint32_t pack_pair(float lo, float hi, __half) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}

template <typename T>
struct Kind;
template <>
struct Kind<__half> {
    static constexpr uint32_t code = 0, exponent = 0x7c00u;
    // Weights are kept 2^10 above the running maximum's so that small ones stay normal numbers; with the threshold
    // of 2^4 the largest is 2^14.
    static constexpr float bias = 10.f, grow = 4.f;
};
template <>
struct Kind<__nv_bfloat16> {
    static constexpr uint32_t code = 1, exponent = 0x7f80u;
    static constexpr float bias = 0.f, grow = 8.f;
};

// Zeroes non-finite values of keys that some row of the item does not see; true if another row sees one of them.
template <typename T, int D>
__device__ bool clean_values(uint32_t tile, int32_t key0, const Range& r, int64_t window, int64_t sinks, int tid) {
    constexpr uint32_t e = Kind<T>::exponent;
    bool poison = false;
    const int32_t key = key0 + tid;  // one key per thread
    const bool inside = key < sinks;
    const bool by_all = key <= r.pmin && (window == 0 || key > r.pmax - window || inside);
    if (by_all) return false;
    const bool by_some = key <= r.pmax && (window == 0 || key > r.pmin - window || inside);
#pragma unroll 4
    for (int c = 0; c < D / 8; ++c) {
        const uint32_t at = tile + (c >> 3) * (kTile * 128) + tid * 128 + (((c & 7) ^ (tid & 7)) << 4);
        uint32_t w[4];
        asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(at));
        bool bad = false;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if ((w[i] & e) == e) w[i] &= 0xffff0000u, bad = true;
            if ((w[i] & (e << 16)) == (e << 16)) w[i] &= 0x0000ffffu, bad = true;
        }
        if (bad) {
            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]) : "memory");
            poison |= by_some;
        }
    }
    return poison;
}

template <typename T, int D>
__global__ void __launch_bounds__(kThreads, 1)
attend_tiles_kernel(const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map, const Params p) {
    using L = Layout<D>;
    constexpr int kStages = L::kStages;
    extern __shared__ unsigned char tiles_smem[];
    __shared__ Control ctl;
    const uint32_t smem = (ptx::smem_addr(tiles_smem) + 1023u) & ~1023u;
    const uint32_t q_smem = smem, ring = smem + L::kQBytes;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const AttendParams& a = p.a;

    if (threadIdx.x == 0) {
        for (int i = 0; i < kStages; ++i) ptx::mbar_init(ptx::smem_addr(&ctl.full[i]), 1), ptx::mbar_init(ptx::smem_addr(&ctl.empty[i]), 1);
        ptx::mbar_init(ptx::smem_addr(&ctl.q_full), 8);
        for (int i = 0; i < 2; ++i) {
            ptx::mbar_init(ptx::smem_addr(&ctl.s_full[i]), 1);
            ptx::mbar_init(ptx::smem_addr(&ctl.p_full[i]), 4);
            ptx::mbar_init(ptx::smem_addr(&ctl.o_full[i]), 1);
        }
        ptx::fence_mbarrier_init();
        ctl.poison = ctl.abort = 0;
    }
    if (warp == kMmaWarp) tmem_alloc(&ctl.tmem, 512);
    fence_before();
    locate<kThreads>(p, ctl.scan, ctl.total, ctl.start_off, ctl.start_seq, blockIdx.x, gridDim.x);
    __syncthreads();
    fence_after();
    const uint32_t tmem = ctl.tmem;
    const int64_t begin = part_begin(ctl.total, blockIdx.x, gridDim.x), end = part_begin(ctl.total, blockIdx.x + 1, gridDim.x);
    // Registers: launched with 168 a thread; 2 x 128 x 224 + 128 x 40 is below 384 x 168.  Each role sets its own
    // share inside its branch: after a join the compiler would have to assume the smaller one.
    if (warp >= kProducerWarp) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 40;");
        Walk walk;
        walk.start(p, ctl.start_seq, ctl.start_off, end - begin);
        if (warp == kProducerWarp) {
            uint32_t seq = 0;  // tiles loaded so far
            auto load = [&](const CUtensorMap* map, int tile) {
                const uint32_t stage = seq % kStages, round = seq / kStages;
                ++seq;
                wait_bar(ctl, &ctl.empty[stage], (round & 1) ^ 1);
                const int32_t key0 = walk.range.tile(tile) * kTile;
                const int32_t box = min(a.page_size, kTile);
                const int32_t key = key0 + lane * box;  // lane i loads the tile's box i
                bool mine = lane < kTile / box && key <= walk.range.pmax;
                if (mine && a.window > 0) mine = key + box - 1 > walk.range.pmin - a.window || key < a.sinks;
                int32_t page = 0;
                if (mine) {
                    page = a.table[static_cast<int64_t>(walk.s) * a.width + key / a.page_size];
                    mine = page >= 0 && page < a.pages;  // attend_finish_kernel reports the others
                }
                const uint32_t boxes = __popc(__ballot_sync(0xffffffffu, mine));
                const uint32_t bar = ptx::smem_addr(&ctl.full[stage]);
                if (lane == 0) ptx::mbar_arrive_expect_tx(bar, boxes * box * D * 2);
                __syncwarp();
                if (mine && !*static_cast<volatile uint32_t*>(&ctl.abort)) {
                    const uint32_t dst = ring + stage * L::kTileBytes + lane * box * 128;
#pragma unroll
                    for (int half = 0; half < D / 64; ++half) tma_page(dst + half * (kTile * 128), map, half * 64, walk.head, key % a.page_size, page, bar);
                }
            };
            for (; walk.valid(); walk.next(p)) {
                const int t0 = walk.tile0(), t1 = walk.tile1(), ahead = walk.shape.wide ? 1 : 2;
                for (int t = t0; t < min(t0 + ahead, t1); ++t) load(&k_map, t);
                for (int t = t0; t < t1; ++t) {
                    load(&v_map, t);
                    if (t + ahead < t1) load(&k_map, t + ahead);
                }
            }
            // After an abort copies may still be in flight: they land before the shared memory goes away.
            if (*static_cast<volatile uint32_t*>(&ctl.abort)) {
                const uint64_t t0 = ptx::globaltimer();
                for (uint32_t i = seq > kStages ? seq - kStages : 0; i < seq; ++i)
                    while (!ptx::mbar_try_wait(ptx::smem_addr(&ctl.full[i % kStages]), (i / kStages) & 1) && ptx::globaltimer() - t0 < kWaitNs / 5) {
                    }
            }
        } else if (warp == kMmaWarp) {
            if (lane == 0) {
                constexpr uint32_t s_desc = instr_desc(Kind<T>::code, false, kTile), o_desc = instr_desc(Kind<T>::code, true, D);
                uint32_t seq = 0, item = 0, p_round[2] = {0, 0};
                auto ready = [&](uint32_t i) { wait_bar(ctl, &ctl.full[i % kStages], (i / kStages) & 1); };
                auto stage_at = [&](uint32_t i) { return ring + (i % kStages) * L::kTileBytes; };
                // Rolled loops: unrolled ones keep dozens of operand descriptors in registers and spill.
                auto score = [&](int wg, int q_tile, uint32_t i) {
#pragma unroll 1
                    for (int k = 0; k < D / 16; ++k) {
                        const uint32_t off = (k >> 2) * (kTile * 128) + (k & 3) * 32;
                        mma_ss(tmem + wg * kTile, smem_desc(q_smem + q_tile * L::kTileBytes + off, 16, 1024), smem_desc(stage_at(i) + off, 16, 1024), s_desc, k > 0);
                    }
                    mma_commit(&ctl.s_full[wg]);
                };
                auto output = [&](int wg, uint32_t i, bool add) {
                    wait_bar(ctl, &ctl.p_full[wg], p_round[wg] & 1);
                    ++p_round[wg];
                    fence_after();
#pragma unroll 1
                    for (int k = 0; k < kTile / 16; ++k)
                        mma_ts(tmem + 2 * kTile + wg * D, tmem + wg * kTile + k * 8, smem_desc(stage_at(i) + k * 2048, D == 128 ? kTile * 128 : 1024, 1024), o_desc, add || k > 0);
                };
                for (; walk.valid(); walk.next(p), ++item) {
                    const int n = walk.tile1() - walk.tile0();
                    wait_bar(ctl, &ctl.q_full, item & 1);
                    fence_after();
                    if (walk.shape.wide) {
                        ready(seq);
                        fence_after();
                        score(0, 0, seq);
                        score(1, 1, seq);
                        mma_commit(&ctl.empty[seq % kStages]);
                        for (int t = 0; t < n; ++t) {
                            const uint32_t v_at = seq + 2 * t + 1, k_at = v_at + 1;
                            ready(v_at);
                            if (t + 1 < n) ready(k_at);
                            fence_after();
                            for (int wg = 0; wg < 2; ++wg) {
                                output(wg, v_at, t > 0);
                                if (t + 1 == n) mma_commit(&ctl.o_full[wg]);
                                if (wg == 1) mma_commit(&ctl.empty[v_at % kStages]);
                                if (t + 1 < n) score(wg, wg, k_at);
                            }
                            if (t + 1 < n) mma_commit(&ctl.empty[k_at % kStages]);
                        }
                        seq += 2 * n;
                    } else {
                        for (int t = 0; t < min(n, 2); ++t) {
                            ready(seq);
                            fence_after();
                            score(t, 0, seq);
                            mma_commit(&ctl.empty[seq % kStages]);
                            ++seq;
                        }
                        for (int t = 0; t < n; ++t) {
                            const int wg = t & 1;
                            ready(seq);
                            fence_after();
                            output(wg, seq, t > 1);
                            if (t + 2 >= n) mma_commit(&ctl.o_full[wg]);
                            mma_commit(&ctl.empty[seq % kStages]);
                            ++seq;
                            if (t + 2 < n) {
                                ready(seq);
                                fence_after();
                                score(wg, 0, seq);
                                mma_commit(&ctl.empty[seq % kStages]);
                                ++seq;
                            }
                        }
                    }
                }
            }
            __syncwarp();
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 224;");
        Walk walk;
        walk.start(p, ctl.start_seq, ctl.start_off, end - begin);
        // ---- softmax warpgroups -------------------------------------------------------------------
        const int wg = warp >> 2, row = threadIdx.x & 127;
        const uint32_t lane_base = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16);
        const uint32_t s_addr = lane_base + wg * kTile, o_addr = lane_base + 2 * kTile + wg * D;
        uint32_t seq = 0, s_round = 0, o_round = 0;
        for (; walk.valid(); walk.next(p)) {
            const Range& r = walk.range;
            const bool wide = walk.shape.wide;
            const int t0 = walk.tile0(), n = walk.tile1() - t0;
            const int32_t q_first = a.query_start[walk.s];
            // Both warpgroups have read the last item's output: every product is done with Q.
            ptx::named_sync(1, 256);
            for (int i = threadIdx.x; i < (wide ? 2 : 1) * kTile * (D / 8); i += 256) {
                const int c = i % (D / 8), rr = i / (D / 8), half_tile = rr >> 7, lr = rr & 127;
                const int32_t token = r.first + half_tile * p.tile_tokens + lr / p.group;
                uint4 x = make_uint4(0, 0, 0, 0);
                if (lr < p.tile_tokens * p.group && token < r.end) {
                    const int head = walk.head * p.group + lr % p.group;
                    x = *reinterpret_cast<const uint4*>(static_cast<const T*>(a.q) + static_cast<int64_t>(q_first + token) * a.q_tok + head * a.q_head + c * 8);
                    x.x ^= p.negate, x.y ^= p.negate, x.z ^= p.negate, x.w ^= p.negate;
                }
                const uint32_t at = q_smem + half_tile * L::kTileBytes + (c >> 3) * (kTile * 128) + lr * 128 + (((c & 7) ^ (lr & 7)) << 4);
                asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(x.x), "r"(x.y), "r"(x.z), "r"(x.w) : "memory");
            }
            fence_async_smem();
            fence_before();
            __syncwarp();
            if (lane == 0) ptx::mbar_arrive(ptx::smem_addr(&ctl.q_full));

            const int32_t token = r.first + (wide ? wg * p.tile_tokens : 0) + row / p.group;
            const bool live = row < p.tile_tokens * p.group && token < r.end;
            const bool warp_live = __any_sync(0xffffffffu, live);
            const int32_t pos = live ? walk.shape.past + token : -1;
            // Positions of this warpgroup's rows: a tile they all see needs no mask.
            const int32_t wg_first = r.first + (wide ? wg * p.tile_tokens : 0), wg_end = min(r.end, wg_first + p.tile_tokens);
            const int32_t wg_min = walk.shape.past + wg_first, wg_max = walk.shape.past + wg_end - 1;
            float ref = -INFINITY, sum = 0.f;
            const int mine = wide ? n : (n + 1 - wg) / 2;
            for (int i = 0; i < mine; ++i) {
                const int t = wide ? i : 2 * i + wg;
                const int32_t key0 = r.tile(t0 + t) * kTile;
                const bool seen_by_item = key0 + kTile - 1 <= r.pmin && (a.window == 0 || key0 > r.pmax - a.window || key0 + kTile <= a.sinks);
                const bool seen = key0 + kTile - 1 <= wg_min && (a.window == 0 || key0 > wg_max - a.window || key0 + kTile <= a.sinks);
                wait_bar(ctl, &ctl.s_full[wg], s_round & 1);
                ++s_round;
                fence_after();
                if (warp_live) {
                    uint32_t x[kTile];
#pragma unroll
                    for (int c = 0; c < kTile; c += 32) tmem_ld32(s_addr + c, x + c);
                    wait_ld();
                    if (!seen) {
                        const int32_t hi = pos - key0;  // columns up to hi
                        const int32_t lo = a.window > 0 ? static_cast<int32_t>(max(static_cast<int64_t>(-1), pos - a.window - key0)) : -1;
                        const int32_t sk = a.window > 0 ? static_cast<int32_t>(min(max(a.sinks - key0, static_cast<int64_t>(0)), static_cast<int64_t>(kTile))) : 0;
#pragma unroll
                        for (int c = 0; c < kTile; ++c)
                            if (!(c <= hi && (c > lo || c < sk))) x[c] = 0xff800000u;
                    }
                    float m0 = -INFINITY, m1 = -INFINITY, m2 = -INFINITY, m3 = -INFINITY;
#pragma unroll
                    for (int c = 0; c < kTile; c += 4) {
                        m0 = fmaxf(m0, __uint_as_float(x[c]));
                        m1 = fmaxf(m1, __uint_as_float(x[c + 1]));
                        m2 = fmaxf(m2, __uint_as_float(x[c + 2]));
                        m3 = fmaxf(m3, __uint_as_float(x[c + 3]));
                    }
                    const float top = fmaxf(fmaxf(m0, m1), fmaxf(m2, m3)) * p.scale2 - Kind<T>::bias;
                    const bool raise = top > ref + Kind<T>::grow || (ref == -INFINITY && top > -INFINITY);
                    if (__any_sync(0xffffffffu, raise)) {
                        const float factor = raise ? (ref == -INFINITY ? 0.f : ptx::ex2(ref - top)) : 1.f;
                        if (raise) ref = top;
                        sum *= factor;
                        if (i > 0) {
#pragma unroll
                            for (int c = 0; c < D; c += 32) {
                                uint32_t o[32];
                                tmem_ld32(o_addr + c, o);
                                wait_ld();
#pragma unroll
                                for (int j = 0; j < 32; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * factor);
                                tmem_st32(o_addr + c, o);
                            }
                        }
                    }
                    const float shift = ref == -INFINITY ? 0.f : -ref;
                    float s0 = 0.f, s1 = 0.f;
#pragma unroll
                    for (int c = 0; c < kTile; c += 2) {
                        const float e0 = ptx::ex2(fmaf(__uint_as_float(x[c]), p.scale2, shift));
                        const float e1 = ptx::ex2(fmaf(__uint_as_float(x[c + 1]), p.scale2, shift));
                        s0 += e0, s1 += e1;
                        x[c / 2] = pack_pair(e0, e1, T{});
                    }
                    sum += s0 + s1;
                    tmem_st32(s_addr, x);
                    tmem_st32(s_addr + 32, x + 32);
                    wait_st();
                }
                if (!seen_by_item) {
                    const uint32_t v_at = seq + (wide ? 2 * t + 1 : min(n, 2) + t + min(t, max(n - 2, 0)));
                    wait_bar(ctl, &ctl.full[v_at % kStages], (v_at / kStages) & 1);
                    if (clean_values<T, D>(ring + (v_at % kStages) * L::kTileBytes, key0, r, a.window, a.sinks, row)) ctl.poison = 1;
                    fence_async_smem();
                }
                fence_before();
                __syncwarp();
                if (lane == 0) ptx::mbar_arrive(ptx::smem_addr(&ctl.p_full[wg]));
            }
            seq += 2 * n;
            if (mine > 0) {
                wait_bar(ctl, &ctl.o_full[wg], o_round & 1);
                ++o_round;
                fence_after();
            }
            // Merge of a one-tile item's halves through the space of Q (the second half is done with it: its output
            // was committed after every score product).
            float mine_w = 1.f, other_w = 0.f;
            const bool merge = !wide && n > 1;
            float* exchange = reinterpret_cast<float*>(tiles_smem + (q_smem - ptx::smem_addr(tiles_smem)));
            if (merge && wg == 1) {
                if (warp_live) {
#pragma unroll
                    for (int c = 0; c < D; c += 32) {
                        uint32_t o[32];
                        tmem_ld32(o_addr + c, o);
                        wait_ld();
#pragma unroll
                        for (int j = 0; j < 32; ++j) exchange[(c + j) * kTile + row] = __uint_as_float(o[j]);
                    }
                    ctl.ref[row] = ref, ctl.sum[row] = sum;
                }
            }
            if (merge) ptx::named_sync(1, 256);
            if (merge && wg == 0 && live) {
                const float ref1 = ctl.ref[row], sum1 = ctl.sum[row];
                const float best = fmaxf(ref, ref1);
                if (best > -INFINITY) {
                    mine_w = ptx::ex2(ref - best), other_w = ptx::ex2(ref1 - best);
                    sum = sum * mine_w + sum1 * other_w;
                    ref = best;
                }
            }
            if (warp_live && (wide || wg == 0)) {
                const bool whole = walk.whole();
                const float inv = sum != 0.f ? 1.f / sum : 0.f;
                const int head = walk.head * p.group + row % p.group;
                const int64_t out_row = static_cast<int64_t>(q_first + token) * a.heads + head;
                const int64_t slot = (static_cast<int64_t>(blockIdx.x) * 2 + (walk.st0 == 0 ? 1 : 0)) * 256 + wg * kTile + row;
                const float lse2 = sum != 0.f ? ref + log2f(sum) : -INFINITY;
#pragma unroll
                for (int c = 0; c < D; c += 32) {
                    uint32_t o[32];
                    tmem_ld32(o_addr + c, o);
                    wait_ld();
                    if (live) {
                        float f[32];
#pragma unroll
                        for (int j = 0; j < 32; ++j) {
                            float y = __uint_as_float(o[j]);
                            if (merge) y = y * mine_w + exchange[(c + j) * kTile + row] * other_w;
                            f[j] = y * inv;
                        }
                        if (whole) {
                            uint4* dst = reinterpret_cast<uint4*>(static_cast<T*>(a.out) + out_row * D + c);
#pragma unroll
                            for (int j = 0; j < 4; ++j)
                                dst[j] = make_uint4(pack_pair(f[8 * j], f[8 * j + 1], T{}), pack_pair(f[8 * j + 2], f[8 * j + 3], T{}),
                                                    pack_pair(f[8 * j + 4], f[8 * j + 5], T{}), pack_pair(f[8 * j + 6], f[8 * j + 7], T{}));
                        } else {
                            float4* dst = reinterpret_cast<float4*>(p.parts + slot * D + c);
#pragma unroll
                            for (int j = 0; j < 8; ++j) dst[j] = make_float4(f[4 * j], f[4 * j + 1], f[4 * j + 2], f[4 * j + 3]);
                        }
                    }
                }
                if (live) {
                    if (!whole) p.part_lse[slot] = lse2;
                    else if (a.lse != nullptr) a.lse[out_row] = lse2 * 0.6931471805599453f;
                }
            }
            fence_before();
        }
    }
    __syncthreads();
    fence_after();
    if (threadIdx.x == 0) p.flags[blockIdx.x] = ctl.poison | (ctl.abort << 1);
    if (warp == kMmaWarp) tmem_free(tmem, 512);
}

constexpr int kFinishThreads = 256;

// After the tiles: joins the parts of divided items (the CTA in whose part an item ends owns it), computes
// flagged items again row by row, writes every sequence's status and clears the rows of failed ones.
template <typename T, int D>
__global__ void __launch_bounds__(kFinishThreads) attend_finish_kernel(const Params p) {
    __shared__ int64_t scan[kFinishThreads / 32];
    __shared__ int64_t total, start_off;
    __shared__ int32_t start_seq;
    __shared__ float qs[kFinishThreads / 32][256];
    const AttendParams& a = p.a;
    const int c = blockIdx.x, ctas = gridDim.x, warp = threadIdx.x >> 5;
    locate<kFinishThreads>(p, scan, total, start_off, start_seq, c, ctas);

    // Whether all pages that the sequence's rows see lie in the cache.  All threads of the block take part.
    auto failed = [&](int s) -> int {
        if (!lengths_fit(a, s)) return BMS_STATUS_BAD_LENGTH;
        const int32_t n = a.query_start[s + 1] - a.query_start[s], len = a.seq_lens[s];
        if (n == 0) return 0;
        const int64_t low = a.window > 0 ? max(static_cast<int64_t>(0), len - n + 1 - a.window) : 0;
        int bad = 0;
        for (int32_t i = threadIdx.x; i < (len + a.page_size - 1) / a.page_size; i += kFinishThreads) {
            const int64_t key = static_cast<int64_t>(i) * a.page_size;
            if (key + a.page_size <= low && key >= a.sinks) continue;
            const int32_t pg = a.table[static_cast<int64_t>(s) * a.width + i];
            bad |= pg < 0 || pg >= a.pages;
        }
        return __syncthreads_or(bad) ? BMS_STATUS_BAD_PAGE : 0;
    };

    const int64_t begin = part_begin(total, c, ctas), end = part_begin(total, c + 1, ctas);
    int abort = 0;
    for (int i = threadIdx.x; i < ctas; i += kFinishThreads) abort |= p.flags[i] & 2;
    abort = __syncthreads_or(abort);
    Walk walk;
    walk.start(p, start_seq, start_off, end - begin);
    int64_t at = begin;
    for (bool first = true; walk.valid(); at += walk.st1 - walk.st0, walk.next(p), first = false) {
        if (!first && p.flags[c] == 0) break;                     // later items that end here are whole
        if (walk.st1 != walk.range.steps) break;                  // ends in a later part
        const int64_t item_begin = at - walk.st0;
        if (walk.st0 == 0 && p.flags[c] == 0) continue;           // whole and clean
        int from = c;
        while (from > 0 && part_begin(total, from, ctas) > item_begin) --from;
        int poison = 0;
        for (int i = from; i <= c; ++i) poison |= p.flags[i] & 1;
        if (walk.st0 == 0 && !poison) continue;
        if (failed(walk.s)) continue;
        const int32_t q_first = a.query_start[walk.s];
        const int tokens = walk.range.end - walk.range.first;
        if (poison) {
            for (int i = warp; i < tokens * p.group; i += kFinishThreads / 32)
                attend_row<T>(a, walk.s, q_first + walk.range.first + i / p.group, walk.head * p.group + i % p.group, qs[warp]);
            continue;
        }
        constexpr int kVecs = D / 4;
        for (int i = threadIdx.x; i < tokens * p.group * kVecs; i += kFinishThreads) {
            const int v = i % kVecs, rr = i / kVecs;
            const int tok = rr / p.group, j = rr % p.group;
            const int tile = tok / p.tile_tokens;
            const int local = tile * kTile + (tok - tile * p.tile_tokens) * p.group + j;
            auto slot = [&](int cta) { return (static_cast<int64_t>(cta) * 2 + (cta == from ? 1 : 0)) * 256 + local; };
            float best = -INFINITY;
            for (int k = from; k <= c; ++k) best = fmaxf(best, p.part_lse[slot(k)]);
            float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
            float sum = 0.f;
            for (int k = from; k <= c; ++k) {
                const float lse = p.part_lse[slot(k)];
                // A part whose rows saw nothing weighs 0; NaN passes on.
                const float w = lse == -INFINITY ? 0.f : exp2f(lse - best);
                const float4 x = *reinterpret_cast<const float4*>(p.parts + slot(k) * D + 4 * v);
                o.x += w * x.x, o.y += w * x.y, o.z += w * x.z, o.w += w * x.w;
                sum += w;
            }
            const float inv = 1.f / sum;
            const int64_t out_row = static_cast<int64_t>(q_first + walk.range.first + tok) * a.heads + walk.head * p.group + j;
            uint2 packed = make_uint2(pack_pair(o.x * inv, o.y * inv, T{}), pack_pair(o.z * inv, o.w * inv, T{}));
            *reinterpret_cast<uint2*>(static_cast<T*>(a.out) + out_row * D + 4 * v) = packed;
            if (v == 0 && a.lse != nullptr) a.lse[out_row] = (best + log2f(sum)) * 0.6931471805599453f;
        }
    }
    for (int s = c; s < a.seqs; s += ctas) {
        int code = failed(s);
        if (code == 0 && abort) code = BMS_STATUS_TIMEOUT;
        if (threadIdx.x == 0) a.status[s] = code;
        if (code != 0) clear_rows<T>(a, s);
    }
}

}  // namespace tc
}  // namespace bms
