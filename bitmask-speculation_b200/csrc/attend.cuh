// Chunk attention on the tensor cores (tcgen05), for 16-bit types, dim 64 or 128 and pages that tile 128 keys.
//
// Work.  An item is (sequence, key head, query tile).  The group's query heads share their key head, so the rows of
// an item are (token, head of the group) pairs.  If a sequence's rows fit 128 they form one tile, and the two
// softmax warpgroups take even and odd key tiles, each with its own running maximum, sum and output, merged at the
// end; else an item is two tiles of 128 rows that read every key tile together.  Key tiles that no row of the item
// sees (causal bound, window, sinks) are not part of it.
//
// Split.  All items, with their steps (a key tile, or a pair of them for one-tile items), form one line, cut into equal
// parts, one per CTA: few long sequences fill the GPU as well as many short ones.  An item that a cut divides leaves
// float32 partials (normalised output and log2 of the sum) in the workspace, and attend_finish_kernel joins them in
// the order of the CTAs, so that results do not depend on timing.
//
// Pipeline (384 threads, one CTA per SM).  A producer warp loads pages by TMA (one box of up to 128 slots x 64
// elements per page, 128-byte swizzle) into a ring of key and value tiles in the order the products consume them, another
// one the queries of the next item as soon as the last one's are done with.  One thread issues the products: S = Q K^T into TMEM, and O += P V with P in TMEM (over S) and V as an MN-major
// operand, so neither P nor V is transposed or copied.  While a warpgroup turns S into P the tensor cores work for
// the other one.  A softmax thread owns a row: no shuffles.  O is rescaled only when a row's maximum grew by more
// than a threshold (2^8 for bfloat16); sums stay float32, weights are rounded once to the inputs' type for the
// second product, because the tensor cores take both operands in that type.  Exponentials are ex2.approx (2 ulp): 2^-22 beside
// the weights' 2^-8 (2^-11 for float16).
//
// Hidden keys.  Scores of keys that a row does not see are replaced, so any bits there vanish.  Values cannot be:
// 0 * NaN is NaN.  In tiles that are not seen by every row, non-finite values of keys that some row does not see are
// zeroed in shared memory before the product; if another row does see such a key the CTA flags its range, and
// attend_finish_kernel computes those items again row by row.
//
// Bound.  Prompt chunks (dim 128) run at 0.86 - 0.9 PFLOP/s, 1.0 in the steady state: a warpgroup's step is a chain (scores 0.4 us,
// load 0.1, maximum 0.15, exponentials 1.2, second half of the output product 0.2), and the two warpgroups' chains overlap; TMEM
// has no room for a second score tile of each (2 x 128 columns of scores, 2 x 128 of output).  Verification windows over long
// caches read them at 4.2 - 4.5 TB/s (6.5 in the steady state).  What is lost lies between items, about 14 us of it per CTA and item
// (output, first scores), at the start (13 us to the first scores, the search for the part's start and cold code in it)
// and in the joining kernel (18 - 27 us for the longest cases); single tokens over short caches take 24 us of that alone.
// Tried without gain: a warp of its own for the cleaning of values, handing the first half of the weights over later, looking up
// the joined items before the tiles are done.
#pragma once
#include <cuda.h>

#include "ptx.cuh"

namespace bms {
namespace tc {

constexpr int kTile = 128;              // keys per tile, rows per query tile
constexpr int kThreads = 384;           // 2 softmax warpgroups, one with the key/value, product and query warps
constexpr int kProducerWarp = 8, kMmaWarp = 9, kQueryWarp = 10;
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
    uint64_t q_full, q_free, s_full[2], p_full[2][2], o_full[2], drained;
    float ref[kTile], sum[kTile];
    int32_t item_tiles[2], item_wide[2];  // of the item whose queries are in place, by the item's parity; 0 tiles: no more
    uint32_t tmem, poison, abort, broken;
};

struct Params {
    AttendParams a;
    float* parts;      // [ctas][2][D / 4][256][4]: lanes (rows) side by side
    float* part_lse;   // [ctas][2][256], log2
    int32_t* flags;    // [ctas]: 1 poisoned values, 2 a wait ran out, 4 row starts are broken
    float scale2;      // |scale| log2(e)
    uint32_t negate;   // sign bit for the scores of a negative scale
    int32_t group, tile_tokens;
    int32_t group_inv;  // 65536 / group, rounded up: r / group = r * group_inv >> 16 for rows r < 128
    int32_t hold;       // of tests: no page is loaded, so that the waits for them run out
};

// ---- schedule ---------------------------------------------------------------------------------
struct Shape {
    int64_t total;  // length of one key head's items over all query tiles
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

// A sequence without its total.
__device__ __forceinline__ Shape sequence_shape(const Params& p, int s) {
    Shape h{0, 0, 0, 0, false};
    if (!lengths_fit(p.a, s)) return h;
    h.n = p.a.query_start[s + 1] - p.a.query_start[s];
    h.past = p.a.seq_lens[s] - h.n;
    h.wide = h.n > p.tile_tokens;
    const int32_t per = h.wide ? 2 * p.tile_tokens : p.tile_tokens;
    h.tiles = (h.n + per - 1) / per;
    return h;
}

// Where a part of the line of steps starts.
struct Start {
    int64_t total, off;  // the line's length; the part's start within its sequence
    int32_t seq;
    Shape shape;
};

// Walks the items of a CTA's part of the line.  An item is kItemCost + steps long: what an item costs beside its steps
// (queries in, result out, the pipeline's filling) counts as that many steps, so that many short items and few long
// ones balance (64 verifying sequences of 2,048 to 24,576 keys took 432, 425 and 407 us at a cost of 0, 1 and 2 steps, 16
// windowed ones 166, 161 and 153, four long prompt chunks 1,535, 1,506 and 1,530).  A part that ends inside an item's fixed
// length leaves all of its steps to the next part.
constexpr int kItemCost = 2;
struct Walk {
    int32_t s, head, qt;
    int64_t left;       // length of the part not yet walked
    int64_t at;         // where in the item the part continues
    int32_t st0, st1;   // steps of the current item that belong to the part
    Shape shape;
    Range range;
    __device__ __forceinline__ void start(const Params& p, const Start& from, int64_t count) {
        s = from.seq, left = count;
        head = qt = st0 = st1 = 0;
        at = 0;
        if (count <= 0) return;
        shape = from.shape;
        head = static_cast<int32_t>(from.off / shape.total);
        at = from.off % shape.total;
        for (;; ++qt) {
            range = query_range(p, shape.n, shape.past, shape.wide, qt);
            if (at < kItemCost + range.steps) break;
            at -= kItemCost + range.steps;
        }
    }
    // Moves on to the next item with steps in the part; false at the part's end.
    __device__ __forceinline__ bool valid(const Params& p) {
        while (left > 0) {
            st0 = static_cast<int32_t>(max(at - kItemCost, static_cast<int64_t>(0)));
            st1 = static_cast<int32_t>(min(static_cast<int64_t>(range.steps), at + left - kItemCost));
            if (st1 > st0) return true;
            next(p);
        }
        return false;
    }
    __device__ __forceinline__ void next(const Params& p) {
        left -= kItemCost + range.steps - at;
        at = 0;
        if (left <= 0) return;
        if (++qt == shape.tiles) {
            qt = 0;
            if (++head == p.a.kv_heads) {
                head = 0;
                do shape = sequence_shape(p, ++s);
                while (shape.n == 0);
            }
        }
        range = query_range(p, shape.n, shape.past, shape.wide, qt);
    }
    __device__ __forceinline__ int tile0() const { return shape.wide ? st0 : 2 * st0; }
    __device__ __forceinline__ int tile1() const { return shape.wide ? st1 : min(2 * st1, range.tiles); }
    __device__ __forceinline__ bool whole() const { return st0 == 0 && st1 == range.steps; }
};

// Finds where part `c` of `ctas` starts.  All threads of the block take part; the sequences' totals come one per thread,
// or, for prompts of many query tiles, one per warp with the tiles over its lanes.  True where this thread met a broken start.
template <int kBlock>
struct LocateSpace {
    int64_t totals[kBlock], scan[kBlock / 32];
    Start start;
};

template <int kBlock>
__device__ bool locate(const Params& p, LocateSpace<kBlock>& sp, int c, int ctas) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    constexpr int kW = kBlock / 32;
    const bool by_warp = p.a.tokens > 2LL * p.tile_tokens * p.a.seqs;
    const bool once = p.a.seqs <= kBlock;  // one round: the second pass has the totals already
    int64_t target = -1, mine = 0, v = 0;
    bool broken = false;
    for (int pass = 0; pass < 2; ++pass) {
        int64_t run = 0;
        for (int base = 0; base < p.a.seqs; base += kBlock) {
            const int s = base + threadIdx.x;
            if (pass == 0 || !once) {
                __syncthreads();
                if (by_warp) {
                    for (int i = warp; i < kBlock && base + i < p.a.seqs; i += kW) {
                        const Shape h = sequence_shape(p, base + i);
                        broken |= h.n == 0 && start_broken(p.a, base + i);
                        int64_t t = 0;  // beyond 2^31 from 1.05 million new tokens with 128 heads per key head on
                        for (int q = lane; q < h.tiles; q += 32) t += kItemCost + query_range(p, h.n, h.past, h.wide, q).steps;
#pragma unroll
                        for (int d = 16; d; d >>= 1) t += __shfl_xor_sync(0xffffffffu, t, d);
                        if (lane == 0) sp.totals[i] = t;
                    }
                } else if (s < p.a.seqs) {
                    const Shape h = sequence_shape(p, s);
                    broken |= h.n == 0 && start_broken(p.a, s);
                    int64_t t = 0;
                    for (int q = 0; q < h.tiles; ++q) t += kItemCost + query_range(p, h.n, h.past, h.wide, q).steps;
                    sp.totals[threadIdx.x] = t;
                }
                __syncthreads();
                mine = s < p.a.seqs ? sp.totals[threadIdx.x] * p.a.kv_heads : 0;
                v = mine;
#pragma unroll
                for (int d = 1; d < 32; d <<= 1) {
                    const int64_t up = __shfl_up_sync(0xffffffffu, v, d);
                    if (lane >= d) v += up;
                }
                if (lane == 31) sp.scan[warp] = v;
                __syncthreads();
                int64_t all = run;
                for (int w = 0; w < kW; ++w) {
                    if (w == warp) v += all;
                    all += sp.scan[w];
                }
                run = all;
            }
            if (pass == 1 && mine > 0 && target >= v - mine && target < v) {
                sp.start.seq = s, sp.start.off = target - (v - mine);
                sp.start.shape = sequence_shape(p, s);
                sp.start.shape.total = mine / p.a.kv_heads;
            }
        }
        if (pass == 0) {
            if (threadIdx.x == 0) sp.start.total = run;
            const int64_t parts = min(static_cast<int64_t>(ctas), run);
            target = c < parts ? run * c / parts : -1;
        }
        __syncthreads();
    }
    return broken;
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
// Operand descriptors come as their low word and a high word that all operands of one layout share: an address step is one
// 32-bit addition, and the issuing thread keeps few registers.
__device__ __forceinline__ void mma_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t high, uint32_t idesc, bool add) {
    asm volatile(
        "{ .reg .pred p; .reg .b64 da, db; setp.ne.u32 p, %5, 0; mov.b64 da, {%1, %3}; mov.b64 db, {%2, %3};\n"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %4, p; }" ::"r"(d),
        "r"(a), "r"(b), "r"(high), "r"(idesc), "r"(static_cast<uint32_t>(add))
        : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t high, uint32_t idesc, bool add) {
    asm volatile(
        "{ .reg .pred p; .reg .b64 db; setp.ne.u32 p, %5, 0; mov.b64 db, {%2, %3};\n"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %4, p; }" ::"r"(d),
        "r"(a), "r"(b), "r"(high), "r"(idesc), "r"(static_cast<uint32_t>(add))
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

// Shared-memory operand with 128-byte swizzle: start address and leading offset in the low word, stride offset, version 1
// and the swizzle mode in the high one (addresses and offsets in units of 16 bytes).
__device__ __forceinline__ uint32_t desc_low(uint32_t addr, uint32_t lead) { return ((addr >> 4) & 0x3fff) | (lead >> 4) << 16; }
constexpr uint32_t kDescHigh = (1024 >> 4) | (1u << 14) | (2u << 29);  // 8 rows of 128 bytes from group to group

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

__device__ __forceinline__ void tma_rows(uint32_t dst, const CUtensorMap* map, int x, int head, int token, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(dst), "l"(map), "r"(bar),
        "r"(x), "r"(head), "r"(token)
        : "memory");
}

// Waits at most about a second; after that the CTA's abort flag ends every wait.  Nothing more is loaded or multiplied then; the
// softmax warpgroups walk on through their items without tiles, because they meet at barriers; and copies and products
// in flight land (`drain`) before the CTA gives its memory back.
__device__ __forceinline__ bool wait_bar(Control& c, uint64_t* bar, uint32_t parity) {
    const uint32_t addr = ptx::smem_addr(bar);
    volatile uint32_t* abort = &c.abort;
    uint64_t t0 = 0;
    for (uint32_t i = 0; !ptx::mbar_try_wait(addr, parity); ++i) {
        if (*abort) return false;
        if ((i & 63u) != 63u) continue;
        const uint64_t now = ptx::globaltimer();
        if (t0 == 0) t0 = now;
        else if (now - t0 > kWaitNs) *abort = 1;
    }
    return true;
}

// For what is in flight already: lands in microseconds, whether the CTA gave up or not; the limit is for hardware that failed.
__device__ __forceinline__ void drain(uint64_t* bar, uint32_t parity) {
    const uint32_t addr = ptx::smem_addr(bar);
    const uint64_t t0 = ptx::globaltimer();
    while (!ptx::mbar_try_wait(addr, parity) && ptx::globaltimer() - t0 < kWaitNs / 5) {
    }
}

__device__ __forceinline__ bool aborted(const Control& c) { return *static_cast<const volatile uint32_t*>(&c.abort) != 0; }

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
attend_tiles_kernel(const __grid_constant__ CUtensorMap q_map, const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map,
                    const Params p) {
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
        ptx::mbar_init(ptx::smem_addr(&ctl.q_full), 1), ptx::mbar_init(ptx::smem_addr(&ctl.q_free), 8);
        for (int i = 0; i < 2; ++i) {
            ptx::mbar_init(ptx::smem_addr(&ctl.s_full[i]), 1);
            ptx::mbar_init(ptx::smem_addr(&ctl.p_full[i][0]), 4), ptx::mbar_init(ptx::smem_addr(&ctl.p_full[i][1]), 4);
            ptx::mbar_init(ptx::smem_addr(&ctl.o_full[i]), 1);
        }
        ptx::mbar_init(ptx::smem_addr(&ctl.drained), 1);
        ptx::fence_mbarrier_init();
        ctl.poison = ctl.abort = ctl.broken = 0;
    }
    if (warp == kMmaWarp) tmem_alloc(&ctl.tmem, 512);
    fence_before();
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;");  // not before the wait: the dependent reads this call's inputs early
    // The space of Q serves the search before the first item.
    LocateSpace<kThreads>& located = *reinterpret_cast<LocateSpace<kThreads>*>(tiles_smem + (q_smem - ptx::smem_addr(tiles_smem)));
    if (locate<kThreads>(p, located, blockIdx.x, gridDim.x)) ctl.broken = 1;
    fence_after();
    const uint32_t tmem = ctl.tmem;
    const Start start = located.start;
    fence_async_smem();
    __syncthreads();  // everyone has it before Q comes in
    const int64_t begin = part_begin(start.total, blockIdx.x, gridDim.x), end = part_begin(start.total, blockIdx.x + 1, gridDim.x);
    // Registers: launched with 168 a thread; 2 x 128 x 224 + 128 x 56 is exactly 384 x 168.  Each role sets its own
    // share inside its branch: after a join the compiler would have to assume the smaller one.
    if (warp >= kProducerWarp) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
        if (warp == kProducerWarp) {
            Walk walk;
            walk.start(p, start, end - begin);
            uint32_t seq = 0;  // tiles loaded so far
            bool stop = p.hold != 0;
            // Lane i loads box i of a tile.  Its page index (-1: nothing to load) is fetched a tile ahead of its use.
            const int32_t box = min(a.page_size, kTile);
            auto page_of = [&](int tile) {
                const int32_t key = walk.range.tile(tile) * kTile + lane * box;
                bool mine = lane < kTile / box && key <= walk.range.pmax;
                if (mine && a.window > 0) mine = key + box - 1 > walk.range.pmin - a.window || key < a.sinks;
                int32_t page = mine ? a.table[static_cast<int64_t>(walk.s) * a.width + key / a.page_size] : -1;
                return page < a.pages ? page : -1;  // attend_finish_kernel reports pages outside the cache
            };
            auto load = [&](const CUtensorMap* map, int tile, int32_t page) {
                if (stop) return;
                const uint32_t stage = seq % kStages, round = seq / kStages;
                // All lanes go on or none does: a barrier expects just the boxes that are on their way.
                stop = __any_sync(0xffffffffu, !wait_bar(ctl, &ctl.empty[stage], (round & 1) ^ 1));
                if (stop) return;
                ++seq;
                const bool mine = page >= 0;
                const uint32_t boxes = __popc(__ballot_sync(0xffffffffu, mine));
                const uint32_t bar = ptx::smem_addr(&ctl.full[stage]);
                if (lane == 0) ptx::mbar_arrive_expect_tx(bar, boxes * box * D * 2);
                __syncwarp();
                if (mine) {
                    const int32_t slot = (walk.range.tile(tile) * kTile + lane * box) % a.page_size;
                    const uint32_t dst = ring + stage * L::kTileBytes + lane * box * 128;
#pragma unroll
                    for (int half = 0; half < D / 64; ++half) tma_page(dst + half * (kTile * 128), map, half * 64, walk.head, slot, page, bar);
                }
            };
            for (; !stop && walk.valid(p); walk.next(p)) {
                const int t0 = walk.tile0(), t1 = walk.tile1(), ahead = walk.shape.wide ? 1 : 2;
                auto fetch = [&](int t) { return t < t1 ? page_of(t) : -1; };
                // Pages of tiles t, t + 1, t + 2: values trail their keys by `ahead` tiles.
                int32_t pg0 = fetch(t0), pg1 = fetch(t0 + 1), pg2 = fetch(t0 + 2);
                load(&k_map, t0, pg0);
                if (ahead == 2 && t0 + 1 < t1) load(&k_map, t0 + 1, pg1);
                for (int t = t0; t < t1 && !stop; ++t) {
                    const int32_t pg3 = fetch(t + 3);
                    load(&v_map, t, pg0);
                    if (t + ahead < t1) load(&k_map, t + ahead, ahead == 1 ? pg1 : pg2);
                    pg0 = pg1, pg1 = pg2, pg2 = pg3;
                }
            }
            for (uint32_t i = seq > kStages ? seq - kStages : 0; i < seq; ++i) drain(&ctl.full[i % kStages], (i / kStages) & 1);
        } else if (warp == kQueryWarp) {
            // Queries of the next item as soon as the last one's space is free: rows are (token, head of the group) pairs, and a
            // box of the group's heads by the tile's tokens is just that.  Boxes may run into the next sequence's tokens
            // (rows that nobody reads) and behind the last token (zeros).
            Walk walk;
            walk.start(p, start, end - begin);
            uint32_t item = 0;
            bool stop = false;
            for (; walk.valid(p); walk.next(p), ++item) {
                stop = __any_sync(0xffffffffu, !wait_bar(ctl, &ctl.q_free, (item & 1) ^ 1));
                if (stop) break;
                if (lane == 0) {
                    const int tiles = walk.shape.wide ? 2 : 1;
                    const uint32_t bar = ptx::smem_addr(&ctl.q_full);
                    ctl.item_tiles[item & 1] = walk.tile1() - walk.tile0(), ctl.item_wide[item & 1] = walk.shape.wide;
                    ptx::mbar_arrive_expect_tx(bar, tiles * p.tile_tokens * p.group * D * 2);
                    for (int t = 0; t < tiles; ++t)
                        for (int half = 0; half < D / 64; ++half)
                            tma_rows(q_smem + t * L::kTileBytes + half * (kTile * 128), &q_map, half * 64, walk.head * p.group,
                                     a.query_start[walk.s] + walk.range.first + t * p.tile_tokens, bar);
                }
                __syncwarp();
            }
            if (!stop) stop = __any_sync(0xffffffffu, !wait_bar(ctl, &ctl.q_free, (item & 1) ^ 1));
            if (stop) {
                if (item > 0) drain(&ctl.q_full, (item - 1) & 1);
            } else if (lane == 0) {
                ctl.item_tiles[item & 1] = 0;
                ptx::mbar_arrive(ptx::smem_addr(&ctl.q_full));
            }
        } else if (warp == kMmaWarp) {
            if (lane == 0) {
                constexpr uint32_t s_desc = instr_desc(Kind<T>::code, false, kTile), o_desc = instr_desc(Kind<T>::code, true, D);
                uint32_t seq = 0, p_round = 0;  // p_round: a bit per half, the parity of its next round
                auto ready = [&](uint32_t i) { wait_bar(ctl, &ctl.full[i % kStages], (i / kStages) & 1); };
                auto stage_at = [&](uint32_t i) { return ring + (i % kStages) * L::kTileBytes; };
                auto score = [&](int wg, int q_tile, uint32_t i) {
                    const uint32_t q_low = desc_low(q_smem + q_tile * L::kTileBytes, 16), k_low = desc_low(stage_at(i), 16);
#pragma unroll
                    for (int k = 0; k < D / 16; ++k) {
                        const uint32_t off = ((k >> 2) * (kTile * 128) + (k & 3) * 32) >> 4;
                        mma_ss(tmem + wg * kTile, q_low + off, k_low + off, kDescHigh, s_desc, k > 0);
                    }
                    mma_commit(&ctl.s_full[wg]);
                };
                auto output = [&](int wg, uint32_t i, bool add) {
                    const uint32_t v_low = desc_low(stage_at(i), D == 128 ? kTile * 128 : 1024);
                    const uint32_t o_at = tmem + 2 * kTile + wg * D, p_at = tmem + wg * kTile;
#pragma unroll
                    for (int half = 0; half < 2; ++half) {  // the weights come in two halves
                        wait_bar(ctl, &ctl.p_full[wg][half], p_round >> wg & 1);
                        fence_after();
#pragma unroll
                        for (int k = half * (kTile / 32); k < (half + 1) * (kTile / 32); ++k)
                            mma_ts(o_at, p_at + k * 8, v_low + k * (2048 >> 4), kDescHigh, o_desc, add || k > 0);
                    }
                    p_round ^= 1u << wg;
                };
                // The query warp says what comes: the walk stays out of this thread's registers.
                for (uint32_t item = 0;; ++item) {
                    wait_bar(ctl, &ctl.q_full, item & 1);
                    fence_after();
                    const int n = ctl.item_tiles[item & 1];
                    const bool wide = ctl.item_wide[item & 1];
                    if (n == 0 || aborted(ctl)) break;
                    // Scores of the first tile (two tiles) ahead of the loop.
                    for (int t = 0; t < (wide ? 2 : min(n, 2)); ++t) {
                        if (t == 0 || !wide) ready(seq);
                        fence_after();
                        score(t, wide ? t : 0, seq);
                        if (t == 1 || !wide) mma_commit(&ctl.empty[seq % kStages]), ++seq;
                    }
                    for (int t = 0; t < n; ++t) {
                        // Wide: both halves use this tile's values and the next one's keys.  Else: one half, and the keys after next.
                        const bool more = t + (wide ? 1 : 2) < n;
                        ready(seq);
                        if (wide && more) ready(seq + 1);
                        fence_after();
#pragma unroll 1
                        for (int wg = wide ? 0 : t & 1; wg < (wide ? 2 : (t & 1) + 1); ++wg) {
                            output(wg, seq, t >= (wide ? 1 : 2));
                            if (!more) mma_commit(&ctl.o_full[wg]);
                            if (!wide || wg == 1) mma_commit(&ctl.empty[seq % kStages]);
                            if (more) {
                                if (!wide) {
                                    ready(seq + 1);
                                    fence_after();
                                }
                                score(wg, wide ? wg : 0, seq + 1);
                                if (!wide || wg == 1) mma_commit(&ctl.empty[(seq + 1) % kStages]);
                            }
                        }
                        seq += more ? 2 : 1;
                    }
                }
                if (aborted(ctl)) {  // else the softmax warpgroups have waited for all of them
                    mma_commit(&ctl.drained);
                    drain(&ctl.drained, 0);
                }
            }
            __syncwarp();
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 224;");
        Walk walk;
        walk.start(p, start, end - begin);
        // ---- softmax warpgroups -------------------------------------------------------------------
        const int wg = warp >> 2, row = threadIdx.x & 127;
        const uint32_t lane_base = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16);
        const uint32_t s_addr = lane_base + wg * kTile, o_addr = lane_base + 2 * kTile + wg * D;
        uint32_t seq = 0, s_round = 0, o_round = 0, item = 0;
        for (; walk.valid(p); walk.next(p), ++item) {
            // A warpgroup without a tile in this item has nothing else to wait for: it must not release the next item's queries
            // before the other one is done with this item's.
            if (!aborted(ctl)) wait_bar(ctl, &ctl.q_full, item & 1);
            const Range& r = walk.range;
            const bool wide = walk.shape.wide;
            const int t0 = walk.tile0(), n = walk.tile1() - t0;
            const int32_t q_first = a.query_start[walk.s];
            const int32_t row_token = row * p.group_inv >> 16;
            const int32_t token = r.first + (wide ? wg * p.tile_tokens : 0) + row_token;
            const bool live = row_token < p.tile_tokens && token < r.end;
            const bool warp_live = __any_sync(0xffffffffu, live);
            const int32_t pos = live ? walk.shape.past + token : -1;
            // Positions of this warpgroup's rows: a tile they all see needs no mask.
            const int32_t wg_first = r.first + (wide ? wg * p.tile_tokens : 0), wg_end = min(r.end, wg_first + p.tile_tokens);
            const int32_t wg_min = walk.shape.past + wg_first, wg_max = walk.shape.past + wg_end - 1;
            float ref = -INFINITY, sum = 0.f;
            const int mine = __any_sync(0xffffffffu, aborted(ctl)) ? 0 : wide ? n : (n + 1 - wg) / 2;
            for (int i = 0; i < mine; ++i) {
                const int t = wide ? i : 2 * i + wg;
                const int32_t key0 = r.tile(t0 + t) * kTile;
                const bool seen_by_item = key0 + kTile - 1 <= r.pmin && (a.window == 0 || key0 > r.pmax - a.window || key0 + kTile <= a.sinks);
                const bool seen = key0 + kTile - 1 <= wg_min && (a.window == 0 || key0 > wg_max - a.window || key0 + kTile <= a.sinks);
                wait_bar(ctl, &ctl.s_full[wg], s_round & 1);
                ++s_round;
                fence_after();
                if (!seen_by_item) {
                    const uint32_t v_at = seq + (wide ? 2 * t + 1 : min(n, 2) + t + min(t, max(n - 2, 0)));
                    wait_bar(ctl, &ctl.full[v_at % kStages], (v_at / kStages) & 1);
                    if (clean_values<T, D>(ring + (v_at % kStages) * L::kTileBytes, key0, r, a.window, a.sinks, row)) ctl.poison = 1;
                    fence_async_smem();
                }
                uint32_t x[kTile];
                float shift = 0.f;
                if (warp_live) {
#pragma unroll
                    for (int c = 0; c < kTile; c += 32) tmem_ld32(s_addr + c, x + c);
                    wait_ld();
                    if (p.negate) {
#pragma unroll
                        for (int c = 0; c < kTile; ++c) x[c] ^= p.negate;
                    }
                    if (!seen) {
                        // Visible columns, 32 to a word: up to the row's position, and behind its window's start or among the sinks.
                        auto upto = [](int32_t last) { return last < 0 ? 0u : last >= 31 ? 0xffffffffu : (2u << last) - 1u; };
                        const int32_t hi = pos - key0;
                        const int32_t lo = a.window > 0 ? static_cast<int32_t>(max(static_cast<int64_t>(-1), pos - a.window - key0)) : -1;
                        const int32_t sk = a.window > 0 ? static_cast<int32_t>(min(max(a.sinks - key0, static_cast<int64_t>(0)), static_cast<int64_t>(kTile))) : 0;
#pragma unroll
                        for (int g = 0; g < kTile; g += 32) {
                            const uint32_t visible = upto(hi - g) & (~upto(lo - g) | upto(sk - 1 - g));
#pragma unroll
                            for (int c = 0; c < 32; ++c)
                                if (!((visible >> c) & 1)) x[g + c] = 0xff800000u;
                        }
                    }
                    float m[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                    for (int c = 0; c < kTile; c += 8)
#pragma unroll
                        for (int j = 0; j < 4; ++j) m[j] = fmaxf(fmaxf(m[j], __uint_as_float(x[c + 2 * j])), __uint_as_float(x[c + 2 * j + 1]));
                    const float top = fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3])) * p.scale2 - Kind<T>::bias;
                    const bool raise = top > ref + Kind<T>::grow || (ref == -INFINITY && top > -INFINITY);
                    if (__any_sync(0xffffffffu, raise)) {
                        const float factor = raise ? (ref == -INFINITY ? 0.f : ptx::ex2(ref - top)) : 1.f;
                        if (raise) ref = top;
                        sum *= factor;
                        if (i > 0) {
#pragma unroll 1
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
                    shift = ref == -INFINITY ? 0.f : -ref;
                }
                // Weights, half a tile at a time: the second product starts on the first half.
                const uint64_t scale_2 = ptx::pack2(p.scale2, p.scale2), shift_2 = ptx::pack2(shift, shift);
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    if (warp_live) {
                        uint64_t s0 = 0, s1 = 0;
                        uint32_t w[32];
#pragma unroll
                        for (int c = 0; c < 64; c += 4) {
                            float e0, e1, e2, e3;
                            ptx::unpack2(ptx::fma2(ptx::pack2(__uint_as_float(x[64 * half + c]), __uint_as_float(x[64 * half + c + 1])), scale_2, shift_2), e0, e1);
                            ptx::unpack2(ptx::fma2(ptx::pack2(__uint_as_float(x[64 * half + c + 2]), __uint_as_float(x[64 * half + c + 3])), scale_2, shift_2), e2, e3);
                            e0 = ptx::ex2(e0), e1 = ptx::ex2(e1), e2 = ptx::ex2(e2), e3 = ptx::ex2(e3);
                            s0 = ptx::add2(s0, ptx::pack2(e0, e1)), s1 = ptx::add2(s1, ptx::pack2(e2, e3));
                            w[c / 2] = pack_pair(e0, e1, T{}), w[c / 2 + 1] = pack_pair(e2, e3, T{});
                        }
                        tmem_st32(s_addr + 32 * half, w);
                        float a0, a1;
                        ptx::unpack2(ptx::add2(s0, s1), a0, a1);
                        sum += a0 + a1;
                        wait_st();
                    }
                    fence_before();
                    __syncwarp();
                    if (lane == 0) ptx::mbar_arrive(ptx::smem_addr(&ctl.p_full[wg][half]));
                }
            }
            seq += 2 * n;
            if (mine > 0) {
                wait_bar(ctl, &ctl.o_full[wg], o_round & 1);
                ++o_round;
                fence_after();
            }
            __syncwarp();
            // The space of Q is free now (outputs were committed after every score product that reads it): one half takes the
            // second half of a one-tile item, element by row in float32, half of the columns at a time, the other the
            // finished rows on their way out, so that the stores are whole lines.
            const bool merge = !wide && n > 1, writes = (wide || wg == 0) && warp_live, whole = walk.whole();
            float* exchange = reinterpret_cast<float*>(tiles_smem + (q_smem - ptx::smem_addr(tiles_smem)));
            const uint32_t stage = q_smem + (wide ? wg : 1) * L::kTileBytes;
            const int64_t slot = static_cast<int64_t>(blockIdx.x) * 2 + (walk.st0 == 0 ? 1 : 0);
            if (merge) {
                if (wg == 1) ctl.ref[row] = ref, ctl.sum[row] = sum;
                ptx::named_sync(1, 256);  // the other half's score products are done, too
            }
            float mine_w = 1.f, other_w = 0.f;
            if (merge && wg == 0) {
                const float ref1 = ctl.ref[row], sum1 = ctl.sum[row];
                const float best = fmaxf(ref, ref1);
                if (best > -INFINITY) {
                    mine_w = ptx::ex2(ref - best), other_w = ptx::ex2(ref1 - best);
                    sum = sum * mine_w + sum1 * other_w;
                    ref = best;
                }
            }
            const float inv = sum != 0.f || whole ? 1.f / sum : 0.f;  // a part may see none of a row's keys; a whole row only with scores of -inf: NaN
            mine_w *= inv, other_w *= inv;
            constexpr int kPart = D / 2;
#pragma unroll 1
            for (int c0 = 0; c0 < D; c0 += kPart) {
                if (merge) {
                    if (wg == 1 && warp_live) {
                        uint32_t o[kPart];
#pragma unroll
                        for (int c = 0; c < kPart; c += 32) tmem_ld32(o_addr + c0 + c, o + c);
                        wait_ld();
#pragma unroll
                        for (int c = 0; c < kPart; ++c) exchange[c * kTile + row] = __uint_as_float(o[c]);
                    }
                    ptx::named_sync(1, 256);
                }
                if (writes) {
                    uint32_t o[kPart];
#pragma unroll
                    for (int c = 0; c < kPart; c += 32) tmem_ld32(o_addr + c0 + c, o + c);
                    wait_ld();
#pragma unroll
                    for (int c = 0; c < kPart; ++c) {
                        if (c % 8 == 0) asm volatile("" ::: "memory");  // few loads ahead: all of them would not fit the registers
                        o[c] = __float_as_uint(__uint_as_float(o[c]) * mine_w + (merge ? exchange[c * kTile + row] * other_w : 0.f));
                    }
                    if (whole) {
#pragma unroll
                        for (int j = 0; j < kPart / 8; ++j) {
                            uint32_t w[4];
#pragma unroll
                            for (int i = 0; i < 4; ++i) w[i] = pack_pair(__uint_as_float(o[8 * j + 2 * i]), __uint_as_float(o[8 * j + 2 * i + 1]), T{});
                            const int c = c0 / 8 + j;
                            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(stage + row * (D * 2) + ((c ^ (row & 7)) << 4)), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]) : "memory");
                        }
                    } else if (live) {
                        float4* dst = reinterpret_cast<float4*>(p.parts) + (slot * (D / 4) + c0 / 4) * 256 + wg * kTile + row;
#pragma unroll
                        for (int j = 0; j < kPart / 4; ++j)
                            dst[j * 256] = make_float4(__uint_as_float(o[4 * j]), __uint_as_float(o[4 * j + 1]), __uint_as_float(o[4 * j + 2]), __uint_as_float(o[4 * j + 3]));
                    }
                }
                if (merge) ptx::named_sync(1, 256);
            }
            if (writes) {
                if (live) {
                    const float lse2 = sum != 0.f ? ref + log2f(sum) : -INFINITY;
                    if (!whole) p.part_lse[slot * 256 + wg * kTile + row] = lse2;
                    else if (a.lse != nullptr) a.lse[static_cast<int64_t>(q_first + token) * a.heads + walk.head * p.group + row - row_token * p.group] = lse2 * 0.6931471805599453f;
                }
                if (whole) {
                    __syncwarp();
                    constexpr int kCols = D / 8, kRows = 32 / kCols;
                    const int c = lane % kCols;
#pragma unroll 4
                    for (int r0 = lane / kCols; r0 < 32; r0 += kRows) {
                        const int rr = (warp & 3) * 32 + r0, tok = rr * p.group_inv >> 16;
                        const int32_t to = wg_first + tok;
                        uint4 y;
                        asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(y.x), "=r"(y.y), "=r"(y.z), "=r"(y.w) : "r"(stage + rr * (D * 2) + ((c ^ (rr & 7)) << 4)));
                        if (tok < p.tile_tokens && to < r.end)
                            reinterpret_cast<uint4*>(static_cast<T*>(a.out) + (static_cast<int64_t>(q_first + to) * a.heads + walk.head * p.group + rr - tok * p.group) * D)[c] = y;
                    }
                }
            }
            fence_async_smem();  // the next queries come into this space by TMA
            fence_before();
            __syncwarp();
            if (lane == 0) ptx::mbar_arrive(ptx::smem_addr(&ctl.q_free));
        }
    }
    __syncthreads();
    fence_after();
    if (threadIdx.x == 0) p.flags[blockIdx.x] = ctl.poison | (ctl.abort << 1) | (ctl.broken << 2);
    if (warp == kMmaWarp) tmem_free(tmem, 512);
}

constexpr int kFinishThreads = 256;

// After the tiles: joins the parts of divided items (the CTA in whose part an item ends owns it), computes
// flagged items again row by row, writes every sequence's status and clears the rows of failed ones.
template <typename T, int D>
__global__ void __launch_bounds__(kFinishThreads) attend_finish_kernel(const Params p) {
    __shared__ LocateSpace<kFinishThreads> located;
    __shared__ float qs[kFinishThreads / 32][256];  // also clear_rows' bitmap
    static_assert(sizeof qs >= kClaimWords * sizeof(uint32_t), "space of the bitmap");
    const AttendParams& a = p.a;
    const int c = blockIdx.x, ctas = gridDim.x, warp = threadIdx.x >> 5;
    locate<kFinishThreads>(p, located, c, ctas);  // of the call's inputs alone: may run before the tiles are done
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int64_t total = located.start.total;
    int flagged = 0;
    for (int i = threadIdx.x; i < ctas; i += kFinishThreads) flagged |= p.flags[i];
    const bool broken = __syncthreads_or(flagged & 4) != 0;

    // A sequence's status but for waits that ran out: whether its lengths fit, its rows are its own, and all pages that they see
    // lie in the cache.  All threads of the block take part.
    auto failed = [&](int s) -> int {
        if (!lengths_fit(a, s)) return BMS_STATUS_BAD_LENGTH;
        const int32_t n = a.query_start[s + 1] - a.query_start[s], len = a.seq_lens[s];
        if (n == 0) return 0;
        if (broken && shares_rows(a, s)) return BMS_STATUS_BAD_LENGTH;
        const int64_t low = a.window > 0 ? max(static_cast<int64_t>(0), len - n + 1 - a.window) : 0;
        int bad = 0;
        for (int32_t i = threadIdx.x; i <= (len - 1) / a.page_size; i += kFinishThreads) {
            const int64_t key = static_cast<int64_t>(i) * a.page_size;
            if (key + a.page_size <= low && key >= a.sinks) continue;
            const int32_t pg = a.table[static_cast<int64_t>(s) * a.width + i];
            bad |= pg < 0 || pg >= a.pages;
        }
        return __syncthreads_or(bad) ? BMS_STATUS_BAD_PAGE : 0;
    };

    const int64_t begin = part_begin(total, c, ctas), end = part_begin(total, c + 1, ctas);
    const int abort = __syncthreads_or(flagged & 2);
    Walk walk;
    walk.start(p, located.start, end - begin);
    // After a wait that ran out every sequence fails: its rows are cleared below, by other blocks than would write them here.
    for (bool first = true; !abort && walk.valid(p); walk.next(p), first = false) {
        if (!first && (p.flags[c] & 3) == 0) break;                     // later items that end here are whole
        if (walk.st1 != walk.range.steps) break;                  // ends in a later part
        const int64_t item_begin = end - walk.left - walk.at + kItemCost;  // of the item's first step
        if (walk.st0 == 0 && (p.flags[c] & 3) == 0) continue;           // whole and clean
        int from = c;
        while (from > 0 && part_begin(total, from, ctas) > item_begin) --from;
        int poison = 0;
        for (int i = from; i <= c; ++i) poison |= p.flags[i] & 1;
        if (walk.st0 == 0 && !poison) continue;
        if (failed(walk.s)) continue;
        const int32_t q_first = a.query_start[walk.s];
        const int tokens = walk.range.end - walk.range.first;
        if (poison) {
            for (int i = blockIdx.y * (kFinishThreads / 32) + warp; i < tokens * p.group; i += gridDim.y * (kFinishThreads / 32))
                attend_row<T>(a, walk.s, q_first + walk.range.first + i / p.group, walk.head * p.group + i % p.group, qs[warp]);
            continue;
        }
        const int rows = tokens * p.group;
        for (int i = blockIdx.y * kFinishThreads + threadIdx.x; i < rows * (D / 8); i += gridDim.y * kFinishThreads) {
            const int v = i / rows, rr = i - v * rows;
            const int tok = rr / p.group, j = rr % p.group;
            const int tile = tok / p.tile_tokens;
            const int local = tile * kTile + (tok - tile * p.tile_tokens) * p.group + j;
            auto slot = [&](int cta) { return static_cast<int64_t>(cta) * 2 + (cta == from ? 1 : 0); };
            float best = -INFINITY;
            for (int k = from; k <= c; ++k) best = fmaxf(best, p.part_lse[slot(k) * 256 + local]);
            float o[8] = {}, sum = 0.f;
#pragma unroll 2
            for (int k = from; k <= c; ++k) {
                const float lse = p.part_lse[slot(k) * 256 + local];
                // A part whose rows saw nothing weighs 0; NaN passes on.
                const float w = lse == -INFINITY ? 0.f : exp2f(lse - best);
                const float4* src = reinterpret_cast<const float4*>(p.parts) + (slot(k) * (D / 4) + 2 * v) * 256 + local;
                const float4 x = src[0], y = src[256];
                o[0] += w * x.x, o[1] += w * x.y, o[2] += w * x.z, o[3] += w * x.w;
                o[4] += w * y.x, o[5] += w * y.y, o[6] += w * y.z, o[7] += w * y.w;
                sum += w;
            }
            const float inv = 1.f / sum;
            const int64_t out_row = static_cast<int64_t>(q_first + walk.range.first + tok) * a.heads + walk.head * p.group + j;
            reinterpret_cast<uint4*>(static_cast<T*>(a.out) + out_row * D)[v] =
                make_uint4(pack_pair(o[0] * inv, o[1] * inv, T{}), pack_pair(o[2] * inv, o[3] * inv, T{}), pack_pair(o[4] * inv, o[5] * inv, T{}), pack_pair(o[6] * inv, o[7] * inv, T{}));
            if (v == 0 && a.lse != nullptr) a.lse[out_row] = (best + log2f(sum)) * 0.6931471805599453f;
        }
    }
    if (blockIdx.y != 0) return;
    for (int s = c; s < a.seqs; s += ctas) {
        int code = failed(s);
        if (code == 0 && abort) code = BMS_STATUS_TIMEOUT;
        if (threadIdx.x == 0) a.status[s] = code;
        if (code != 0) clear_rows<T>(a, s, broken, reinterpret_cast<uint32_t*>(qs));
    }
}

}  // namespace tc
}  // namespace bms
