// paged_chunk.cu -- paged attention of chunks of new tokens (and of single
// tokens beside them) on the 5th-generation tensor cores.
//
// The g q heads of a KV head share its keys, so a 128-row tile of S = Q K^T holds
// TQ = 128 / g tokens with all their g heads (row = token * g + head): 16 tokens
// of 8 heads fill the tile that one head of 128 tokens would.  A block is one or
// two such tiles of one KV head of one sequence; its keys come in tiles of 128
// rows, gathered page by page by TMA.  Per CTA:
//   warps 0-3, 4-7  softmax: thread = row = TMEM lane
//   warp 8          work list, TMA of Q and K;  warp 11  TMA of V
//   warps 9, 10     MMA issue for each group
//   TMEM            S0, S1 (P over the columns it came from), O0, O1
// Each group's S is two halves of 64 keys that go their own way: while the group
// takes the softmax of one, the products of the other (P V, then the next tile's
// Q K^T into the same columns) run, so neither waits out the other's latency.
// Two-tile blocks: each softmax group has its own rows, K and V tiles serve
// both, and one group's softmax runs while the other's products do.  One-tile
// blocks (few new tokens): the groups take alternate key tiles of the same rows
// and their (max, sum, O) are joined at the end.
//
// Compute-bound for two-tile blocks (at hd 128 2,560 cycles of tensor work per key
// tile and SM, 2,048 of exponentials), HBM-bound for one-tile blocks.
//
// Work split: the blocks' costs are known to every CTA from the lengths.  Either
// whole blocks are handed out, longest of each sequence first, by a counter; or,
// where blocks are too few or too uneven, all their tiles are concatenated and cut
// into equal slices, the parts of a cut block going to the workspace for a merge
// kernel.
//
// Measured, hd 128: two chunks of 1,024 tokens over 19,000 rows of 8 KV heads,
// bf16, 32 q heads 710 to 750 us (650 GFLOP: 0.52 to 0.56 of the burst rate, 0.62
// to 0.67 of what a plain bf16 product holds under the same power cap); a prompt of 2,048
// 49 us (0.42); 24 single tokens and chunks of 291, 337 and 413 tokens over up to
// 4,000 rows of 4 KV heads 76 us.  A two-tile key tile takes 3,400 to 3,900 cycles:
// the softmax of a half (its exponentials alone 512 on the SM's four units, with the
// rest of its instructions some 800) and the round trip of its products (issue,
// commit, wait: 550) follow one another within a group, and two groups cover
// each other only in part.
#include <algorithm>
#include <cmath>
#include <mutex>
#include <type_traits>

#include <cuda.h>

#include "paged_common.cuh"
#include "tcgen05.cuh"

namespace picoattn {

namespace {

constexpr int BM = 128, BN = 128, BH = BN / 2;
constexpr int kThreads = 384;
constexpr int kPlan = 32;          // runs of sequences whose costs are added up, a lane each
constexpr int kMaxCtas = 160;
// Costs, in units of a quarter of a two-tile block's key tile (some 900 cycles):
constexpr int kItemCost = 4;       // of a block, whatever its tiles
constexpr int kMinCost = 8;        // least per CTA of a slice (40 new over 3,000 rows of 4 x 128: 26 us; 16: 31, 4: 29)
// What cutting blocks costs: their epilogues, the parts written and read again, the merge.  With 16 a prompt of
// 2,048 (longest block 68, mean 66) stays at 49 us, but one of 600 over 100 goes from 19 to 21 and 24 tokens beside
// three chunks from 76 to 92; with 8 the prompt takes 75.
constexpr int kSliceOverhead = 32;
// A cut this near to a block's end moves there (200 new over 3,000 rows of 4 x 128: 38 us without, 28; two such and
// two single tokens of 4 x 64: 36, with 16 37).
constexpr int kMostMoved = 8;
constexpr int kPartRows = 2 * BM;
constexpr int kRing = 4;           // stages of 64 keys, K and V each
constexpr float kNone = -1e30f;    // running maximum before any key
constexpr float kStaleSum = 32768.0f;
// Of weights (weight_lift): 64 keys at their maximum sum to 2^13, which leaves the maximum room to grow by 2^2 and more
// (as much again as most of the 64 lie below it) before a half is done again; fp16 weights vanish below 2^-32 of the largest.
constexpr int kWeightLift = 7;

struct ChunkMeta {  // the cut block whose first part a CTA holds (nt 0: none)
    int b, h, blk, nt, slices;
    long long start, cost;  // its first cost unit; all blocks' units
};

struct ChunkArgs {
    PagedAttnArgs a;
    int tq;              // tokens per tile
    int single;          // whole blocks, at most one per CTA: no counter, nothing to merge
    int* counter;        // next whole block; zero between calls
    ChunkMeta* meta;     // [grid]
    float2* part_ml;     // [2 * grid][256]
    float* part_o;       // [2 * grid][256][hd]
};

struct Item {
    int b, h, tok0, ntok;  // first row of q and tokens of the block
    int pos0;              // position of its first token
    int j0, j1;            // key tiles
    int slot;              // partial slot, -1: whole
    int len;               // rows of the sequence
    int poison;            // a page that does not exist was met
};

// The key tiles of an item that softmax group w works on: all of a two-tile
// block's that its rows see, every other one of a one-tile block's.
__device__ __forceinline__ int own_tiles(const Item& it, int w, int tq) {
    if (it.ntok <= tq) return (it.j1 - it.j0 + 1 - w) / 2;
    return w ? it.j1 - it.j0 : max(0, min(it.j1, (it.pos0 + tq + BN - 1) / BN) - it.j0);
}

// ---- the work list --------------------------------------------------------------

struct Blocks {
    int n, len, t0, per, count;  // new tokens, rows, first token row, tokens per block, blocks
    int tq;
    __device__ __forceinline__ int ntok(int i) const { return min(per, n - i * per); }
    __device__ __forceinline__ int tiles(int i) const { return (len - n + min(n, (i + 1) * per) + BN - 1) / BN; }
    // cost of a key tile: a two-tile block's takes some 3,500 cycles, a one-tile block's 2,600
    __device__ __forceinline__ int cost(int i) const { return tiles(i) * unit(i) + kItemCost; }
    __device__ __forceinline__ int unit(int i) const { return ntok(i) > tq ? 4 : 3; }
};

__device__ __forceinline__ Blocks seq_blocks(const ChunkArgs& c, int b) {
    const SeqSpan sp = seq_span(c.a.b, b);
    Blocks x;
    x.n = sp.ok ? sp.n : 0;
    x.len = sp.len, x.t0 = sp.t0, x.tq = c.tq, x.per = 2 * c.tq;
    x.count = (x.n + x.per - 1) / x.per;
    return x;
}

// One head's cost: 4 * tiles * blocks, in 32 bits for 10^6 tokens of a sequence and more.
__device__ __forceinline__ int head_cost(const Blocks& x) {
    int s = 0;
    for (int i = 0; i < x.count; i++) s += x.cost(i);
    return s;
}
// The same by a whole warp.
__device__ __forceinline__ int head_cost_warp(const Blocks& x, int lane) {
    int s = 0;
    for (int i = lane; i < x.count; i += 32) s += x.cost(i);
    return __reduce_add_sync(0xffffffffu, s);
}

struct Plan {
    long long first_cost[kPlan + 1];  // of each run of sequences
    int first_item[kPlan + 1];
};

// The plan, by one warp: a run of `per` sequences a lane, or, for a few
// sequences, one a lane with its blocks spread over the lanes.  Returns the CTAs
// that share the cut-up list, 0: whole blocks (whose list needs no costs).
// Every CTA makes it for itself and comes to the same result.  This is the first
// thing a call does, from cold instruction caches, so it is kept short.
__device__ __forceinline__ int make_plan(const ChunkArgs& c, Plan* plan, int per, int grid, int lane) {
    long long cost = 0;
    int items = 0, most = 0;
    if (c.a.b.n_seqs <= 4) {
        for (int b = 0; b < c.a.b.n_seqs; b++) {
            const Blocks x = seq_blocks(c, b);
            const int s = head_cost_warp(x, lane);
            if (lane == b) {
                cost = (long long)s * c.a.hkv;
                items = x.count * c.a.hkv;
                most = x.count ? x.tiles(x.count - 1) * 4 + kItemCost : 0;
            }
        }
    } else {
        for (int b = lane * per; b < min((lane + 1) * per, c.a.b.n_seqs); b++) {
            const Blocks x = seq_blocks(c, b);
            cost += (long long)head_cost(x) * c.a.hkv;
            items += x.count * c.a.hkv;
            if (x.count) most = max(most, x.tiles(x.count - 1) * 4 + kItemCost);
        }
    }
    float all = (float)cost;
#pragma unroll 1
    for (int o = 1; o < 32; o <<= 1) {
        all += __shfl_xor_sync(0xffffffffu, all, o);
    }
    const int longest = __reduce_max_sync(0xffffffffu, most), blocks = __reduce_add_sync(0xffffffffu, items);
    // whole blocks end when the longest does, or, dealt out one by one, some 15% after the mean
    const float n = fminf((float)grid, all * (1.0f / kMinCost)), mean = all / fmaxf(n, 1.0f);
    const float whole = fmaxf((float)longest, blocks <= grid ? 0.f : 1.15f * mean);
    if (c.single || mean + kSliceOverhead >= whole) {
#pragma unroll 1
        for (int o = 1; o < 32; o <<= 1) {
            const int io = __shfl_up_sync(0xffffffffu, items, o);
            if (lane >= o) items += io;
        }
        if (lane == 0) plan->first_item[0] = 0;
        plan->first_item[lane + 1] = items;
        __syncwarp();
        return 0;
    }
#pragma unroll 1
    for (int o = 1; o < 32; o <<= 1) {
        const long long co = __shfl_up_sync(0xffffffffu, cost, o);
        if (lane >= o) cost += co;
    }
    if (lane == 0) plan->first_cost[0] = 0;
    plan->first_cost[lane + 1] = cost;
    cost = __shfl_sync(0xffffffffu, cost, 31);
    __syncwarp();
    const int slices = (int)min((long long)grid, (cost + kMinCost - 1) / kMinCost);
    const int over = slices % blocks;
    return over * 8 <= slices && over < slices ? slices - over : slices;  // blocks alike are cut alike, at their ends
}

__device__ __forceinline__ long long slice_first(long long i, long long cost, int n) {
    return quotient(i * cost, n);
}

// A cut this near to a block's ends moves there: less than half a slice, so that no two cuts meet.
__device__ __forceinline__ int most_moved(long long cost, int n) { return (int)min((long long)kMostMoved, quotient(cost, n) / 2); }
// A part's first (or end) tile for a slice that begins (ends) at cost unit x of a block from `start`.
__device__ __forceinline__ int tile_at(long long x, long long start, int unit, int nt, int most) {
    start += kItemCost;
    const long long end = start + (long long)nt * unit;
    if (x >= end) return nt;  // a block may be shorter than `most`
    if (x <= start + most) return 0;
    if (x >= end - most) return nt;
    return (int)quotient(x - start + unit - 1, unit);
}

// Where a CTA is in its work (the producer warp, the same in every lane).
struct Walk {
    int b, h, blk, per_head;  // sequence, head and block; one head's cost
    long long at, end;        // cost units of the slice still to do
    long long base, start;    // first unit of the sequence, of the block
    Blocks x;
    bool open;                // b .. start are set
    int taken;                // whole blocks so far
    int most;                 // most_moved
};

// The slice's first cost unit -> its sequence, head and block.
__device__ __forceinline__ void walk_find(const ChunkArgs& c, Walk& wk, int lane) {
    const int hkv = c.a.hkv;
    for (;; wk.b++) {
        wk.x = seq_blocks(c, wk.b);
        wk.per_head = head_cost_warp(wk.x, lane);
        if (wk.at < wk.base + (long long)wk.per_head * hkv) break;
        wk.base += (long long)wk.per_head * hkv;
    }
    wk.h = (int)quotient(wk.at - wk.base, wk.per_head);
    wk.start = wk.base + (long long)wk.h * wk.per_head;
    const int rest = (int)(wk.at - wk.start);
    int before = 0;  // cost of the head's blocks before the 32 looked at
    for (int i0 = 0;; i0 += 32) {
        const int i = i0 + lane, cost = i < wk.x.count ? wk.x.cost(i) : 0;
        int upto = cost;
#pragma unroll 1
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += v;
        }
        const unsigned past = __ballot_sync(0xffffffffu, rest < before + upto);
        if (past) {
            const int l = __ffs(past) - 1;
            wk.blk = i0 + l;
            wk.start += before + __shfl_sync(0xffffffffu, upto - cost, l);
            break;
        }
        before += __shfl_sync(0xffffffffu, upto, 31);
    }
    wk.open = true;
}

// The next item of a CTA; false: none.
__device__ __forceinline__ bool next_item(const ChunkArgs& c, const Plan* plan, Walk& wk, int slices, int per, Item& it,
                                          int lane) {
    const int hkv = c.a.hkv;
    it.poison = 0;
    if (!slices) {  // whole blocks: the CTA's own first one, then by the counter
        int idx = blockIdx.x;
        if (wk.taken++) {
            if (c.single) return false;
            if (lane == 0) idx = (int)gridDim.x + atomicAdd(c.counter, 1);
            idx = __shfl_sync(0xffffffffu, idx, 0);
        }
        if (idx >= plan->first_item[kPlan]) return false;
        const int run = __popc(__ballot_sync(0xffffffffu, plan->first_item[lane + 1] <= idx));
        int rest = idx - plan->first_item[run], b = run * per;
        Blocks x = seq_blocks(c, b);
        while (rest >= x.count * hkv) {
            rest -= x.count * hkv;
            x = seq_blocks(c, ++b);
        }
        const int r = (int)((unsigned)rest / (unsigned)hkv), i = x.count - 1 - r;  // a sequence's longest first
        it.b = b, it.h = rest - r * hkv;
        it.tok0 = x.t0 + i * x.per, it.ntok = x.ntok(i), it.pos0 = x.len - x.n + i * x.per;
        it.j0 = 0, it.j1 = x.tiles(i), it.slot = -1, it.len = x.len;
        return true;
    }
    while (wk.at < wk.end) {
        if (!wk.open) walk_find(c, wk, lane);
        const int nt = wk.x.tiles(wk.blk), u = wk.x.unit(wk.blk);
        const int j0 = tile_at(wk.at, wk.start, u, nt, wk.most), j1 = tile_at(wk.end, wk.start, u, nt, wk.most);
        if (j0 < j1) {
            it.b = wk.b, it.h = wk.h;
            it.tok0 = wk.x.t0 + wk.blk * wk.x.per, it.ntok = wk.x.ntok(wk.blk);
            it.pos0 = wk.x.len - wk.x.n + wk.blk * wk.x.per;
            it.j0 = j0, it.j1 = j1, it.len = wk.x.len;
            it.slot = j0 == 0 && j1 == nt ? -1 : 2 * (int)blockIdx.x + (j0 == 0 ? 1 : 0);
            if (j0 == 0 && j1 < nt && lane == 0)
                c.meta[blockIdx.x] = {wk.b, wk.h, wk.blk, nt, slices, wk.start, plan->first_cost[kPlan]};
        }
        // step to the next block
        wk.at = wk.start + nt * u + kItemCost;
        if (wk.blk + 1 < wk.x.count) {
            wk.start = wk.at;
            wk.blk++;
        } else if (wk.h + 1 < hkv) {
            wk.h++;
            wk.blk = 0;
            wk.start = wk.at;
        } else {
            wk.base += (long long)wk.per_head * hkv;
            wk.b++;
            wk.open = false;
        }
        if (j0 < j1) return true;
    }
    return false;
}

// ---- one key tile of the online softmax ------------------------------------------

template <class T>
struct Pair16;
template <>
struct Pair16<__half> {
    using V = __half2;
    static __device__ __forceinline__ V cvt(float a, float b) { return __floats2half2_rn(a, b); }
};
template <>
struct Pair16<__nv_bfloat16> {
    using V = __nv_bfloat162;
    static __device__ __forceinline__ V cvt(float a, float b) { return __floats2bfloat162_rn(a, b); }
};

// S (64 fp32 columns at tS, unscaled) -> P = 2^(scale S - m) in 16 bits over its
// first 32 columns; m (log2 units) and the row sum l updated, O (HD columns at tO)
// rescaled when m grows.  lim: keys visible to the row counted from the first;
// mask: some row of the warp does not see all 64.  The maximum is stale by
// design: p is taken against the running one in the same pass that reads S, and
// kept unless the sum passes 2^15 (so that every p is in range in 16 bits); then
// the keys are done again with their own maximum.  wait_prev_pv()
// returns when the group's products so far are in O.
template <class T, int HD, class WaitPrevPV>
__device__ __forceinline__ void softmax_half(uint32_t tS, uint32_t tO, bool first, int lim, bool mask, float scale,
                                             float& m, float& l, WaitPrevPV wait_prev_pv) {
    using P2 = Pair16<T>;
    constexpr float lift = weight_lift<T>(kWeightLift);
    const uint64_t sc2 = f2_pack(scale, scale);
    uint32_t pk[BH / 2], sr[2][32];
    // p of the keys against m into pk; returns their sum
    auto p_pass = [&] {
        uint64_t s2[4] = {0ull, 0ull, 0ull, 0ull};
        const uint64_t nm2 = f2_pack(-m, -m);
#pragma unroll
        for (int c = 0; c < 2; c++) {
            if (c == 1) tmem_ld_wait();
            if (mask) {
#pragma unroll
                for (int e = 0; e < 32; e++)
                    if (c * 32 + e >= lim) sr[c][e] = __float_as_uint(-INFINITY);
            }
#pragma unroll
            for (int e = 0; e < 16; e++) {
                float d0, d1;
                f2_unpack(f2_fma(f2_pack(__uint_as_float(sr[c][2 * e]), __uint_as_float(sr[c][2 * e + 1])), sc2, nm2), d0,
                          d1);
                const float p0 = ex2(d0), p1 = ex2(d1);
                s2[e & 3] = f2_add(s2[e & 3], f2_pack(p0, p1));
                const typename P2::V h = P2::cvt(p0, p1);
                pk[c * 16 + e] = *reinterpret_cast<const uint32_t*>(&h);
            }
        }
        float a0, a1;
        f2_unpack(f2_add(f2_add(s2[0], s2[1]), f2_add(s2[2], s2[3])), a0, a1);
        return a0 + a1;
    };
    tmem_ld32(tS, sr[0]);
    tmem_ld_wait();
    tmem_ld32(tS + 32, sr[1]);
    if (first) {  // start from the maximum of the first 32 keys, less the lift
        float m0 = -INFINITY;
#pragma unroll
        for (int e = 0; e < 32; e++)
            if (!mask || e < lim) m0 = fmaxf(m0, __uint_as_float(sr[0][e]));
        m = fmaxf(m0 * scale - lift, kNone);
    }
    float sum = p_pass();
    if (__any_sync(0xffffffffu, !(sum <= kStaleSum))) {
        tmem_ld32(tS, sr[0]);
        tmem_ld32(tS + 32, sr[1]);
        tmem_ld_wait();
        float mx = -INFINITY;
#pragma unroll
        for (int c = 0; c < 2; c++)
#pragma unroll
            for (int e = 0; e < 32; e++)
                if (!mask || c * 32 + e < lim) mx = fmaxf(mx, __uint_as_float(sr[c][e]));
        const float m_new = fmaxf(mx * scale - lift, first ? kNone : m);
        if (!first) {
            const float corr = ex2(m - m_new);
            wait_prev_pv();
            tc_fence_after();
#pragma unroll 1
            for (int c = 0; c < HD / 32; c++) {
                uint32_t o[32];
                tmem_ld32(tO + c * 32, o);
                tmem_ld_wait();
#pragma unroll
                for (int e = 0; e < 32; e++) o[e] = __float_as_uint(__uint_as_float(o[e]) * corr);
                tmem_st32(tO + c * 32, o);
            }
            tmem_st_wait();
            l *= corr;
        }
        m = m_new;
        sum = p_pass();
    }
    tmem_st32(tS, pk);
    l += sum;
    tmem_st_wait();
}

template <int HD>
struct Smem {
    static constexpr int kBox = BM * 128;            // 128 rows x 64 columns of 16 bits
    static constexpr int kTile = (HD / 64) * kBox;
    static constexpr int kHalf = (HD / 64) * BH * 128;  // a ring stage: 64 keys, HD / 64 boxes of 8 KB
    static constexpr int kHBox = BH * 128;
    static constexpr int kQ = 0;
    static constexpr int kK = 2 * kTile;
    static constexpr int kV = kK + kRing * kHalf;
    static constexpr int kStage = kV + kRing * kHalf;   // 16 KB per softmax group
    static constexpr int kPlanAt = kStage + 8 * 4096;
    static constexpr int kBars = (kPlanAt + (int)sizeof(Plan) + 15) / 16 * 16;
    static constexpr int kItems = kBars + 40 * 8;
    static constexpr int kEnd = kItems + 2 * (int)sizeof(Item) + 16;
    static constexpr int kDyn = kEnd + 1024;         // slack to align the base
    static_assert(kDyn <= 227 * 1024, "one CTA per SM");
};

// The pages of an item's key tiles into a ring of half tiles (64 rows x HD as
// HD / 64 boxes of 128-byte rows), by one warp: a lane per box and page.  t: half
// tiles that the ring has seen, counted up.  False: a wait ran out.
template <int HD>
__device__ __forceinline__ bool load_tiles(const PagedAttnArgs& a, const CUtensorMap& map, const Item& item, int* poison,
                                           uint8_t* ring, uint64_t* full, uint64_t* empty, int& t, unsigned int* status, int lane) {
    using L = Smem<HD>;
    const int rows = min(a.b.page_size, BH), boxes = BH / rows;  // rows of a box, boxes of a half's column group
    const int col = lane / boxes, box = lane % boxes;
    const bool mine = col < HD / 64;
    const int b = item.b, h = item.h, len = item.len, last = 2 * item.j1;
    const int* table = a.b.page_table + (size_t)b * a.b.page_cols;
    auto page_of = [&](int y) {  // of this lane's box of half tile y; -1: none, -2: no such page
        const int r = y * BH + box * rows;
        if (!mine || y >= last || r >= len) return -1;
        const int p = table[r >> a.b.page_shift];
        return p < 0 || p >= a.b.n_pages ? -2 : p;
    };
    int page = page_of(2 * item.j0);
    for (int y = 2 * item.j0; y < last; y++, t++) {
        const int next = page_of(y + 1), s = t % kRing, use = t / kRing;
        const int r = y * BH + box * rows;
        const int at = (max(page, 0) * a.hkv + h) * a.b.page_size + (r & (a.b.page_size - 1));
        if (__any_sync(0xffffffffu, page == -2) && lane == 0) {
            atomicOr(status, PICOATTN_DEV_BAD_PAGE);
            *poison = 1;
        }
        const uint32_t n = __popc(__ballot_sync(0xffffffffu, page != -1));
        if (use > 0 && !__all_sync(0xffffffffu, mbar_wait(&empty[s], (uint32_t)((use - 1) & 1), status))) return false;
        if (lane == 0) mbar_arrive_expect_tx(&full[s], n * (uint32_t)rows * 128u);
        __syncwarp();
        if (page != -1)
            tma_load_2d(ring + s * L::kHalf + col * L::kHBox + box * rows * 128, &map, 64 * col, at, &full[s]);
        page = next;
    }
    return true;
}

// The copies still on their way into the ring: what a copy warp ends with, as whoever was to wait for them may have given up.
__device__ __forceinline__ void settle_ring(uint64_t* full, int t) {
    for (int c = max(0, t - kRing); c < t; c++) mbar_settle(&full[c % kRing], (uint32_t)((c / kRing) & 1));
}

// ---- output ------------------------------------------------------------------------

// 128 bytes of every row of a warp (lane = row, 32 words w) to dst + off(row):
// through a 4 KB shared stage, 16-byte unit u of row r at u ^ (r & 7), so that
// eight lanes write a row's 128 bytes together.  off < 0: the row is not stored.
__device__ __forceinline__ void store_rows(const uint32_t (&w)[32], uint4* stage, uint8_t* dst, long long off, int lane) {
    __syncwarp();
#pragma unroll
    for (int u = 0; u < 8; u++)
        stage[lane * 8 + (u ^ (lane & 7))] = make_uint4(w[4 * u], w[4 * u + 1], w[4 * u + 2], w[4 * u + 3]);
    __syncwarp();
    // all reads before the first store: the compiler cannot tell the two apart
    uint4 v[8];
    long long o[8];
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const int row = 4 * i + (lane >> 3), u = lane & 7;
        v[i] = stage[row * 8 + (u ^ (row & 7))];
        o[i] = __shfl_sync(0xffffffffu, off, row);
    }
#pragma unroll
    for (int i = 0; i < 8; i++)
        if (o[i] >= 0) *reinterpret_cast<uint4*>(dst + o[i] + 16 * (lane & 7)) = v[i];
}

// ---- the kernel --------------------------------------------------------------------

template <class T, int HD>
__global__ void __launch_bounds__(kThreads, 1)
    paged_chunk_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                       const __grid_constant__ CUtensorMap tmV, const __grid_constant__ CUtensorMap tmO,
                       const __grid_constant__ CUtensorMap tmP, const ChunkArgs c) {
    using L = Smem<HD>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    const PagedAttnArgs& a = c.a;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::kBars);
    uint64_t* item_full = bars + 0;     // [2]
    uint64_t* item_empty = bars + 2;    // [2]
    uint64_t* q_full = bars + 4;
    uint64_t* q_empty = bars + 5;
    uint64_t* s_full = bars + 6;        // [group][half]
    uint64_t* p_full = bars + 10;       // [group][half]
    uint64_t* pv_done = bars + 14;      // [group][half]
    uint64_t* o_free = bars + 18;       // [2] per group
    uint64_t* k_full = bars + 20;       // [kRing], each
    uint64_t* k_empty = k_full + kRing;
    uint64_t* v_full = k_empty + kRing;
    uint64_t* v_empty = v_full + kRing;
    uint64_t* mma_item = v_empty + kRing;  // both issuing warps are through with an item
    uint64_t* joined = mma_item + 1;       // group 1's (max, sum) of a one-tile block is there
    uint64_t* settle = joined + 1;         // [2] giving up: an issuing warp's products
    Plan* plan = reinterpret_cast<Plan*>(smem + L::kPlanAt);
    Item* items = reinterpret_cast<Item*>(smem + L::kItems);
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(items + 2);
    unsigned int* status = a.b.status;

    pdl_trigger();
    if (tid == 0) {
        for (int i = 0; i < 2; i++) {
            mbar_init(&item_full[i], 1), mbar_init(&item_empty[i], 5);
            mbar_init(&o_free[i], 4);
        }
        for (int i = 0; i < 4; i++) mbar_init(&s_full[i], 1), mbar_init(&p_full[i], 4), mbar_init(&pv_done[i], 1);
        for (int i = 0; i < kRing; i++) {
            mbar_init(&k_full[i], 1), mbar_init(&k_empty[i], 2);
            mbar_init(&v_full[i], 1), mbar_init(&v_empty[i], 2);
        }
        mbar_init(mma_item, 2);
        mbar_init(joined, 4);
        mbar_init(&settle[0], 1), mbar_init(&settle[1], 1);
        mbar_init(q_full, 1);
        mbar_init(q_empty, 2);
        fence_mbar_init();
        prefetch_tmap(&tmQ);
        prefetch_tmap(&tmK);
        prefetch_tmap(&tmV);
    }
    if (warp == 9) tmem_alloc(tmem_slot, 512);
    if (c.tq * a.g < BM) {  // rows that no load of Q writes
        for (int i = tid; i < 2 * L::kTile / 16; i += kThreads)
            reinterpret_cast<uint4*>(smem + L::kQ)[i] = make_uint4(0, 0, 0, 0);
        fence_proxy_async_shared();
    }
    pdl_wait();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    const float scale = 1.4426950408889634f / sqrtf((float)HD);
    const int g = a.g, tq = c.tq;

    if (warp == 8) {
        // ---------------- work list, TMA of Q and K ----------------
        const int per = (a.b.n_seqs + kPlan - 1) / kPlan;
        const int slices = make_plan(c, plan, per, gridDim.x, lane);
        if (lane == 0) c.meta[blockIdx.x].nt = 0;
        Walk wk{};
        if ((int)blockIdx.x < slices) {
            const long long cost = plan->first_cost[kPlan];
            wk.at = slice_first(blockIdx.x, cost, slices);
            wk.end = slice_first(blockIdx.x + 1, cost, slices);
            wk.most = most_moved(cost, slices);
            const int run = __popc(__ballot_sync(0xffffffffu, plan->first_cost[lane + 1] <= wk.at));
            wk.b = run * per;
            wk.base = plan->first_cost[run];
        }
        int t = 0, loads = 0;  // half tiles of K; Q loads
        bool ok = true;
        for (int k = 0; ok; k++) {
            const int slot = k & 1;
            if (k >= 2) ok = __all_sync(0xffffffffu, mbar_wait(&item_empty[slot], (uint32_t)(((k >> 1) - 1) & 1), status));
            if (!ok) break;
            Item it;
            if (!next_item(c, plan, wk, slices, per, it, lane)) it.b = -1;
            if (lane == 0) {
                items[slot] = it;  // the other lanes go by their own copy
                mbar_arrive(&item_full[slot]);
            }
            if (it.b < 0) break;
            const bool two = it.ntok > tq;
            if (k >= 1) ok = __all_sync(0xffffffffu, mbar_wait(q_empty, (uint32_t)((k - 1) & 1), status));
            if (!ok) break;
            if (lane == 0) {
                mbar_arrive_expect_tx(q_full, (two ? 2u : 1u) * (HD / 64) * (uint32_t)(tq * g) * 128u);
                for (int w = 0; w < (two ? 2 : 1); w++)
                    for (int x = 0; x < HD / 64; x++)
                        tma_load_3d(smem + L::kQ + w * L::kTile + x * L::kBox, &tmQ, 64 * x, it.h * g, it.tok0 + w * tq,
                                    q_full);
            }
            loads++;
            ok = load_tiles<HD>(a, tmK, it, &items[slot].poison, smem + L::kK, k_full, k_empty, t, status, lane);
        }
        if (loads) mbar_settle(q_full, (uint32_t)((loads - 1) & 1));
        settle_ring(k_full, t);
    } else if (warp == 11) {
        // ---------------- TMA of V ----------------
        int t = 0;
        bool ok = true;
        for (int k = 0; ok; k++) {
            const int slot = k & 1;
            ok = __all_sync(0xffffffffu, mbar_wait(&item_full[slot], (uint32_t)((k >> 1) & 1), status));
            if (!ok) break;
            const Item it = items[slot];
            if (it.b >= 0) ok = load_tiles<HD>(a, tmV, it, &items[slot].poison, smem + L::kV, v_full, v_empty, t, status, lane);
            __syncwarp();
            if (lane == 0) mbar_arrive(&item_empty[slot]);
            if (it.b < 0) break;
        }
        settle_ring(v_full, t);
    } else if (warp >= 8) {
        // ---------------- MMA issue: one warp per softmax group ----------------
        // Each waits for what is ready early (V, the next K) while its group is still
        // busy, so that only P stands between a softmax and its products.
        const int w = warp - 9;
        constexpr uint32_t kBf16 = std::is_same<T, __half>::value ? 0u : (1u << 7) | (1u << 10);
        constexpr uint32_t idesc_qk = idesc_f16_f32(BM, BH, false, false) | kBf16;
        constexpr uint32_t idesc_pv = idesc_f16_f32(BM, HD, false, true) | kBf16;
        const uint32_t tS = tmem + w * 128, tO = tmem + 256 + w * 128;
        const uint64_t dq = smem_desc_sw128(smem_u32(smem + L::kQ), 16, 1024);
        const uint64_t dk = smem_desc_sw128(smem_u32(smem + L::kK), 16, 1024);
        const uint64_t dv = smem_desc_sw128(smem_u32(smem + L::kV), L::kHBox, 1024);
        // half y of S from Q tile qt and half tile c of the ring; `last`: the block's last of this
        // group.  A ring stage is free after two arrivals: one of each group, or both of the only
        // group that uses it (`alone`)
        auto qk = [&](int qt, int c, int y, bool alone, bool last) {
            if (elect_one()) {
                const uint64_t qd = desc_advance(dq, qt * L::kTile), kd = desc_advance(dk, (c % kRing) * L::kHalf);
#pragma unroll
                for (int kk = 0; kk < HD / 16; kk++)
                    umma_ss(tS + y * BH, desc_advance(qd, (kk >> 2) * L::kBox + (kk & 3) * 32),
                            desc_advance(kd, (kk >> 2) * L::kHBox + (kk & 3) * 32), idesc_qk, kk > 0 ? 1u : 0u);
                umma_commit(&s_full[2 * w + y]);
                umma_commit(&k_empty[c % kRing]);
                if (alone) umma_commit(&k_empty[c % kRing]);
                if (last) umma_commit(q_empty);
            }
            __syncwarp();
        };
        auto pv = [&](int c, int y, bool alone, bool first) {
            if (elect_one()) {
                const uint64_t vd = desc_advance(dv, (c % kRing) * L::kHalf);
#pragma unroll
                for (int kk = 0; kk < BH / 16; kk++)
                    umma_ts(tO, tS + y * BH + kk * 8, desc_advance(vd, kk * 16 * 128), idesc_pv,
                            (!first || kk > 0) ? 1u : 0u);
                umma_commit(&pv_done[2 * w + y]);
                umma_commit(&v_empty[c % kRing]);
                if (alone) umma_commit(&v_empty[c % kRing]);
            }
            __syncwarp();
        };
        bool ok = true;  // no wait has run out; the same in every lane
        auto wait = [&](uint64_t* bar, int phase) {
            if (ok) ok = __all_sync(0xffffffffu, mbar_wait(bar, (uint32_t)(phase & 1), status));
        };
        int t = 0, mine = 0, uses = 0;  // half tiles of the CTA; tiles of this group; blocks this group worked on
        for (int k = 0; ok; k++) {
            const int slot = k & 1;
            wait(&item_full[slot], k >> 1);
            if (!ok) break;
            const Item it = items[slot];
            __syncwarp();
            if (lane == 0) mbar_arrive(&item_empty[slot]);
            if (it.b < 0) break;
            const int n = it.j1 - it.j0;
            const bool two = it.ntok > tq;
            // this group's tiles j0 + i step, i < own, and from which tile on they are its alone
            // (group 0's keys may end before a two-tile block's)
            const int qt = two ? w : 0, step = two ? 1 : 2, j0 = two ? 0 : w;
            const int own = own_tiles(it, w, tq), solo = two ? (w ? own_tiles(it, 0, tq) : n) : 0;
            wait(q_full, k);
            if (own > 0) {
#pragma unroll
                for (int y = 0; y < 2; y++) {
                    const int c = t + 2 * j0 + y;
                    wait(&k_full[c % kRing], c / kRing);
                    if (!ok) break;
                    tc_fence_after();
                    qk(qt, c, y, j0 >= solo, own == 1 && y == 1);
                }
            } else if (lane == 0) {
                mbar_arrive(q_empty);
            }
            for (int i = 0; i < own && ok; i++, mine++) {
                const int j = j0 + i * step;
                const bool more = i + 1 < own;
#pragma unroll
                for (int y = 0; y < 2; y++) {
                    const int c = t + 2 * j + y, cn = c + 2 * step;
                    if (i == 0 && y == 0 && uses > 0) wait(&o_free[w], uses - 1);
                    // all at once: a probe of a finished phase costs some 110 cycles, and the tensor
                    // pipe may stand still meanwhile
                    const bool now = mbar_test(&v_full[c % kRing], (uint32_t)((c / kRing) & 1)) &
                                     (!(more && two) || mbar_test(&k_full[cn % kRing], (uint32_t)((cn / kRing) & 1))) &
                                     mbar_test(&p_full[2 * w + y], (uint32_t)(mine & 1));
                    if (!__all_sync(0xffffffffu, now)) {
                        wait(&v_full[c % kRing], c / kRing);
                        if (more && two) wait(&k_full[cn % kRing], cn / kRing);
                        wait(&p_full[2 * w + y], mine);
                    }
                    if (!ok) break;
                    tc_fence_after();
                    pv(c, y, j >= solo, i == 0 && y == 0);
                    if (more) {
                        if (!two) {
                            wait(&k_full[cn % kRing], cn / kRing);
                            if (!ok) break;
                            tc_fence_after();
                        }
                        qk(qt, cn, y, j + step >= solo, i + 2 == own && y == 1);
                    }
                }
            }
            t += 2 * n;
            if (own > 0) uses++;
            // The two go on to the next item together.  A wait by parity must find its phase or
            // the one before it current, and a group has not looked at the stages that the other
            // one used alone: here the other has seen all of them full, and none of the next
            // item's can be given back before both have been here.
            if (lane == 0) mbar_arrive(mma_item);
            wait(mma_item, k);
        }
        if (!ok) {  // products in flight end before the TMEM and the stages they read are given up
            if (elect_one()) umma_commit(&settle[w]);
            __syncwarp();
            mbar_settle(&settle[w], 0);
        }
    } else {
        // ---------------- softmax ----------------
        // rows of sequences outside the host's bounds
        for (int b = blockIdx.x; b < a.b.n_seqs; b += gridDim.x) {
            const SeqSpan sp = seq_span(a.b, b);
            if (sp.ok) continue;
            if (tid == 0) atomicOr(status, PICOATTN_DEV_BAD_POS);
            const RowRange rows = rows_inside(a.b, b);
            const long long n = (long long)(rows.end - rows.first) * a.hq * HD;
            for (long long i = tid; i < n; i += 256) {
                const size_t at = (size_t)rows.first * a.hq * HD + i;
                if (a.out_dtype == PICOATTN_DTYPE_F32) static_cast<float*>(a.out)[at] = __int_as_float(0x7fc00000);
                else static_cast<T*>(a.out)[at] = Elem<T>::round(__int_as_float(0x7fc00000));
            }
        }
        const int w = warp >> 2, r = tid & 127;
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t tS = tmem + w * 128 + lanes, tO = tmem + 256 + w * 128 + lanes;
        uint4* gstage = reinterpret_cast<uint4*>(smem + L::kStage + w * 4 * 4096);  // 128 rows of 128 bytes
        float2* xs = reinterpret_cast<float2*>(smem + L::kStage + 4 * 4096);  // group 1's (max, sum), one-tile blocks
        const int rt = r / g, rh = r - rt * g;  // the row's token in its tile, and head
        int t = 0, mine = 0, joins = 0;  // half tiles of the CTA, key tiles of this group, one-tile blocks joined
        bool ok = true;                  // no wait of this thread has run out: then nothing more is stored
        for (int k = 0;; k++) {
            const int slot = k & 1;
            if (ok) ok = mbar_wait(&item_full[slot], (uint32_t)((k >> 1) & 1), status);
            // the group goes on together, with an item that all of it has, or not at all
            if (!named_bar_all(1 + w, 128, ok)) break;
            const Item it = items[slot];
            if (it.b < 0) break;
            const bool two = it.ntok > tq;
            const int n = it.j1 - it.j0;
            const int tok = (two ? w * tq : 0) + rt;
            const bool valid = rt < tq && tok < it.ntok;
            const int lim = valid ? it.pos0 + tok + 1 : 0;  // keys the row sees
            // the fewest and most keys that valid rows of this warp see (rows are token-major)
            const bool live = __any_sync(0xffffffffu, valid);
            const int lim_lo = __reduce_min_sync(0xffffffffu, valid ? lim : 0x7fffffff);
            const int n_own = own_tiles(it, w, tq);
            float m = kNone, l = 0.f;
            for (int i = 0; i < n_own; i++, mine++) {
                const int j = two ? i : 2 * i + w, base = (it.j0 + j) * BN;
#pragma unroll 1
                for (int y = 0; y < 2; y++) {
                    if (ok) ok = mbar_wait(&s_full[2 * w + y], (uint32_t)(mine & 1), status);
                    tc_fence_after();
                    const int hb = base + y * BH;
                    // the products before this half's: the other half's of this tile, or of the one before
                    if (live)
                        softmax_half<T, HD>(tS + y * BH, tO, i == 0 && y == 0, lim - hb, hb + BH > lim_lo, scale, m, l,
                                            [&] { if (ok) ok = mbar_wait(&pv_done[2 * w + (y ^ 1)], (uint32_t)((mine + y + 1) & 1), status); });
                    if (hb + BH > it.len) {
                        // rows past the sequence hold anything: their V must not meet the zero weights as a NaN
                        const int cc = t + 2 * j + y, s = cc % kRing;
                        if (ok) ok = mbar_wait(&v_full[s], (uint32_t)((cc / kRing) & 1), status);
                        for (int e = r; e < BH * 8 * (HD / 64); e += 128) {
                            const int row = (e >> 3) & (BH - 1), x = e >> 9;
                            if (hb + row >= it.len)
                                *reinterpret_cast<uint4*>(smem + L::kV + s * L::kHalf + x * L::kHBox + row * 128 +
                                                          (e & 7) * 16) = make_uint4(0, 0, 0, 0);
                        }
                        fence_proxy_async_shared();
                    }
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&p_full[2 * w + y]);
                }
            }
            t += 2 * n;
            // the items' last tile has been read: its poison flag is final
            if (n_own > 0 && *reinterpret_cast<volatile int*>(&items[slot].poison)) l = __int_as_float(0x7fc00000);
            named_bar_sync(1 + w, 128);  // every warp of the group has read the item
            if (r == 0) mbar_arrive(&item_empty[slot]);
            if (n_own > 0) {
                for (int y = 0; y < 2; y++)
                    if (ok) ok = mbar_wait(&pv_done[2 * w + y], (uint32_t)((mine - 1) & 1), status);
                tc_fence_after();
            }
            const bool join = !two && n > 1;
            if (!two && w == 1) {  // hand over to group 0
                if (join) {
                    if (r == 0) bulk_wait_read_all();
                    named_bar_sync(2, 128);  // the stage, where xs lies, has been read
                    xs[r] = make_float2(m, l);
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(joined);
                }
                continue;
            }
            float w0 = 1.f, w1 = 0.f;
            if (join) {
                if (ok) ok = mbar_wait(joined, (uint32_t)(joins & 1), status);
                joins++;
                tc_fence_after();
                const float2 o = xs[r];
                const float M = fmaxf(m, o.x);
                w0 = ex2(m - M), w1 = ex2(o.x - M);
                l = l * w0 + o.y * w1;
                m = M;
            }
            const bool part = it.slot >= 0;
            if (!part) {
                const float inv = 1.0f / l;
                w0 *= inv, w1 *= inv;
            }
            // 32 columns of the row's O, weighted
            auto load = [&](int col, float (&o)[32]) {
                if (n_own == 0) {
#pragma unroll
                    for (int e = 0; e < 32; e++) o[e] = 0.f;
                    return;
                }
                tmem_ld32(tO + col, reinterpret_cast<uint32_t (&)[32]>(o));
                tmem_ld_wait();
#pragma unroll
                for (int e = 0; e < 32; e++) o[e] *= w0;
                if (join) {
                    uint32_t y[32];
                    tmem_ld32(tO + 128 + col, y);
                    tmem_ld_wait();
#pragma unroll
                    for (int e = 0; e < 32; e++) o[e] = __fmaf_rn(__uint_as_float(y[e]), w1, o[e]);
                }
            };
            auto release = [&] {  // O is in registers: the next block's products may overwrite it
                tc_fence_before();
                __syncwarp();
                if (lane == 0) {
                    if (n_own > 0) mbar_arrive(&o_free[w]);
                    if (join) mbar_arrive(&o_free[1]);
                }
            };
            const int row = w * BM + r;  // of the block's two tiles (one-tile blocks: w is 0)
            if (part && valid && ok) c.part_ml[(size_t)it.slot * kPartRows + row] = make_float2(m, l);
            const bool f32 = part || a.out_dtype == PICOATTN_DTYPE_F32;
            // A tile whose rows are all valid, or any part (its other rows are scratch), leaves by
            // one TMA store per 128 bytes of its rows, from a swizzled stage of the group; the rows
            // of a ragged tile by per-row stores.  (The SM's store path takes some 2,000 cycles
            // for 64 columns of a tile by per-row stores.)
            const bool bulk = part || it.ntok >= (w + 1) * tq;
            const long long orow = ((long long)(it.tok0 + tok) * a.hq + it.h * g + rh) * HD;
            const int step = f32 ? 32 : 64;
            if (r == 0) bulk_wait_read_all();  // the stage's last store
#pragma unroll 1
            for (int col = 0; col < HD; col += step) {
                uint32_t x[32];
                if (f32) {
                    float o[32];
                    load(col, o);
#pragma unroll
                    for (int e = 0; e < 32; e++) x[e] = __float_as_uint(o[e]);
                } else {
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        float o[32];
                        load(col + 32 * h, o);
#pragma unroll
                        for (int e = 0; e < 16; e++) x[16 * h + e] = Elem<T>::pack2(o[2 * e], o[2 * e + 1]);
                    }
                }
                if (col + step == HD) release();
                if (bulk) {
                    named_bar_sync(1 + w, 128);  // the stage is free
#pragma unroll
                    for (int u = 0; u < 8; u++)
                        gstage[r * 8 + (u ^ (r & 7))] = make_uint4(x[4 * u], x[4 * u + 1], x[4 * u + 2], x[4 * u + 3]);
                    fence_proxy_async_shared();
                    named_bar_sync(1 + w, 128);
                    if (r == 0 && ok) {
                        if (part) tma_store_2d(&tmP, gstage, col, it.slot * kPartRows + w * BM);
                        else tma_store_3d(&tmO, gstage, col, it.h * g, it.tok0 + w * tq);
                        bulk_commit_group();
                        if (col + step < HD) bulk_wait_read_all();
                    }
                } else {
                    if (col == 0) named_bar_sync(1 + w, 128);
                    store_rows(x, gstage + (warp & 3) * 256, static_cast<uint8_t*>(a.out) + col * (f32 ? 4 : 2),
                               valid && ok ? orow * (f32 ? 4 : 2) : -1, lane);
                }
            }
        }
        if (r == 0) bulk_wait_all();
    }
    __syncthreads();
    if (warp == 9) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

// Joins the parts of the blocks that slices cut: block (CTA that holds a cut
// block's first part, row group), thread (row, four columns).  Also sets the
// work counter back.
constexpr int kMergeRows = 32, kMergeBlocks = kPartRows / kMergeRows, kMergeThreads = 256;

template <class T, int HD>
__global__ void __launch_bounds__(kMergeThreads) paged_chunk_merge_kernel(ChunkArgs c) {
    constexpr int C4 = HD / 4, RB = kMergeThreads / C4;
    static_assert(kMaxCtas <= kMergeThreads, "a thread per part");
    __shared__ float2 ml_s[kMaxCtas * kMergeRows];
    __shared__ float inv_s[kMergeRows];
    pdl_trigger();
    pdl_wait();
    const PagedAttnArgs& a = c.a;
    if (blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0) *c.counter = 0;
    const ChunkMeta mt = c.meta[blockIdx.x];
    if (mt.nt == 0) return;
    const Blocks x = seq_blocks(c, mt.b);
    const int unit = x.unit(mt.blk);
    // the parts are those of this CTA and the ones after it, as the attention kernel cut them
    const int i = blockIdx.x + threadIdx.x;
    const int most = most_moved(mt.cost, mt.slices);
    const bool has = i < mt.slices && tile_at(slice_first(i, mt.cost, mt.slices), mt.start, unit, mt.nt, most) <
                                          tile_at(slice_first(i + 1, mt.cost, mt.slices), mt.start, unit, mt.nt, most);
    const int parts = __syncthreads_count(has);
    auto slot = [&](int p) { return (size_t)(2 * (blockIdx.x + p) + (p == 0 ? 1 : 0)) * kPartRows; };
    // (max, sum) of the parts of this block's rows -> their weights
    const int row0 = blockIdx.y * kMergeRows, ntok = x.ntok(mt.blk);
    const int last = (ntok > c.tq ? BM : 0) + ((ntok > c.tq ? ntok - c.tq : ntok) * a.g) - 1;  // valid row
    if (row0 > last) return;
    for (int i = threadIdx.x; i < parts * kMergeRows; i += kMergeThreads)
        ml_s[i] = __ldcg(c.part_ml + slot(i / kMergeRows) + row0 + i % kMergeRows);
    __syncthreads();
    {
        constexpr int kSub = kMergeThreads / kMergeRows;  // threads of a row, side by side
        const int row = threadIdx.x / kSub, sub = threadIdx.x % kSub;
        float M = -INFINITY, L = 0.f;
        for (int p = sub; p < parts; p += kSub) M = fmaxf(M, ml_s[p * kMergeRows + row].x);
        for (int o = 1; o < kSub; o <<= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
        for (int p = sub; p < parts; p += kSub) {
            float2& v = ml_s[p * kMergeRows + row];
            v.x = ex2(v.x - M);
            L += v.y * v.x;
        }
        for (int o = 1; o < kSub; o <<= 1) L += __shfl_xor_sync(0xffffffffu, L, o);
        if (sub == 0) inv_s[row] = 1.0f / L;
    }
    __syncthreads();
    constexpr int NR = kMergeRows / RB;
    const int c4 = threadIdx.x % C4, r0 = threadIdx.x / C4;
    float4 acc[NR];
#pragma unroll
    for (int i = 0; i < NR; i++) acc[i] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int p = 0; p < parts; p++) {
        const float4* o = reinterpret_cast<const float4*>(c.part_o + (slot(p) + row0) * HD) + c4;
#pragma unroll
        for (int i = 0; i < NR; i++) {
            const int r = r0 + i * RB;
            const float4 v = __ldcg(o + (size_t)r * C4);
            const float w = ml_s[p * kMergeRows + r].x;
            acc[i].x += v.x * w, acc[i].y += v.y * w, acc[i].z += v.z * w, acc[i].w += v.w * w;
        }
    }
#pragma unroll
    for (int i = 0; i < NR; i++) {
        const int row = row0 + r0 + i * RB;
        const int rt = (row % BM) / a.g, rh = row % BM - rt * a.g, tok = row / BM * c.tq + rt;
        if (rt >= c.tq || tok >= ntok) continue;
        const float inv = inv_s[r0 + i * RB];
        const size_t at = ((size_t)(x.t0 + mt.blk * x.per + tok) * a.hq + mt.h * a.g + rh) * HD + 4 * c4;
        acc[i].x *= inv, acc[i].y *= inv, acc[i].z *= inv, acc[i].w *= inv;
        if (a.out_dtype == PICOATTN_DTYPE_F32)
            *reinterpret_cast<float4*>(static_cast<float*>(a.out) + at) = acc[i];
        else
            *reinterpret_cast<uint2*>(static_cast<T*>(a.out) + at) =
                make_uint2(Elem<T>::pack2(acc[i].x, acc[i].y), Elem<T>::pack2(acc[i].z, acc[i].w));
    }
}

// ---- host -----------------------------------------------------------------------------

typedef CUresult (*EncodeTiled)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiled encoder() {
    static const EncodeTiled fn = [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult q;
        const bool ok = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
                        q == cudaDriverEntryPointSuccess;
        return ok ? reinterpret_cast<EncodeTiled>(p) : nullptr;
    }();
    return fn;
}

// Boxes of 128-byte rows, 128-byte swizzle.
bool make_map(CUtensorMap* m, int dtype, const void* base, int rank, const cuuint64_t* dims, const cuuint64_t* strides,
              const cuuint32_t* box) {
    const EncodeTiled fn = encoder();
    const cuuint32_t one[3] = {1, 1, 1};
    const CUtensorMapDataType t = dtype == PICOATTN_DTYPE_F32   ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                  : dtype == PICOATTN_DTYPE_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                                                : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
    return fn && fn(m, t, (cuuint32_t)rank, const_cast<void*>(base), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
                    CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                    CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

constexpr size_t kMetaBytes = (kMaxCtas * sizeof(ChunkMeta) + 255) / 256 * 256;
constexpr size_t kMlBytes = 2 * (size_t)kMaxCtas * kPartRows * 8;

template <class T, int HD>
cudaError_t launch_types(const PagedAttnArgs& a, cudaStream_t stream) {
    using L = Smem<HD>;
    static PerDeviceOnce setup;
    cudaError_t e = setup.run([] {
        return cudaFuncSetAttribute(paged_chunk_kernel<T, HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, L::kDyn);
    });
    if (e != cudaSuccess) return e;
    ChunkArgs c{};
    c.a = a;
    c.tq = BM / a.g;
    c.counter = &reinterpret_cast<WsHeader*>(a.b.status)->paged_work;
    c.meta = reinterpret_cast<ChunkMeta*>(a.ws);
    c.part_ml = reinterpret_cast<float2*>(a.ws + kMetaBytes);
    c.part_o = reinterpret_cast<float*>(a.ws + kMetaBytes + kMlBytes);
    CUtensorMap mq, mk, mv, mo, mp;
    const cuuint64_t qd[3] = {HD, (cuuint64_t)a.hq, (cuuint64_t)a.b.n_tok}, qs[2] = {HD * 2, (cuuint64_t)a.qs * 2};
    const cuuint32_t qb[3] = {64, (cuuint32_t)a.g, (cuuint32_t)c.tq};
    const cuuint64_t kd[2] = {HD, (cuuint64_t)a.b.n_pages * a.hkv * a.b.page_size}, ks[1] = {HD * 2};
    const cuuint32_t kb[2] = {64, (cuuint32_t)std::min(a.b.page_size, BH)};
    const size_t es = a.out_dtype == PICOATTN_DTYPE_F32 ? 4 : 2;
    const cuuint64_t os[2] = {HD * es, (cuuint64_t)a.hq * HD * es};
    const cuuint32_t ob[3] = {(cuuint32_t)(128 / es), (cuuint32_t)a.g, (cuuint32_t)c.tq};
    const cuuint64_t pd[2] = {HD, 2 * (cuuint64_t)kMaxCtas * kPartRows}, ps[1] = {HD * 4};
    const cuuint32_t pb[2] = {32, BM};
    if (!make_map(&mq, a.dtype, a.q, 3, qd, qs, qb) || !make_map(&mk, a.dtype, a.k_pool, 2, kd, ks, kb) ||
        !make_map(&mv, a.dtype, a.v_pool, 2, kd, ks, kb) || !make_map(&mo, a.out_dtype, a.out, 3, qd, os, ob) ||
        !make_map(&mp, PICOATTN_DTYPE_F32, c.part_o, 2, pd, ps, pb))
        return cudaErrorInvalidValue;
    const long long blocks = (long long)a.b.n_seqs * a.hkv * ((a.b.max_new + 2 * c.tq - 1) / (2 * c.tq));
    const long long tiles = (a.b.max_len + BN - 1) / BN;  // a slice has at least kMinCost units, a whole block a CTA
    const int ctas = std::min(device_sm_count(), kMaxCtas);
    // make_plan hands out whole blocks then, whatever the lengths
    c.single = blocks <= ctas && tiles * 4 + kItemCost <= kSliceOverhead;
    const int grid = (int)std::min<long long>(ctas, c.single ? blocks : blocks * tiles);
    e = launch_pdl(paged_chunk_kernel<T, HD>, dim3(grid), dim3(kThreads), (size_t)L::kDyn, stream, mq, mk, mv, mo, mp, c);
    if (e != cudaSuccess || c.single) return e;
    return launch_pdl(paged_chunk_merge_kernel<T, HD>, dim3(grid, kMergeBlocks), dim3(kMergeThreads), 0, stream, c);
}

}  // namespace

size_t paged_chunk_bytes(int hd) { return kMetaBytes + kMlBytes + 2 * (size_t)kMaxCtas * kPartRows * 4 * hd; }

cudaError_t launch_paged_chunk(const PagedAttnArgs& a, cudaStream_t stream) {
    if (a.dtype == PICOATTN_DTYPE_F16)
        return a.hd == 64 ? launch_types<__half, 64>(a, stream) : launch_types<__half, 128>(a, stream);
    return a.hd == 64 ? launch_types<__nv_bfloat16, 64>(a, stream) : launch_types<__nv_bfloat16, 128>(a, stream);
}

}  // namespace picoattn
