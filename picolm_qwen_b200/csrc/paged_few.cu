// paged_few.cu -- paged attention of sequences with few query rows (new tokens x q
// heads of a KV head): single tokens and drafts, up to 32 rows.
//
// Bound by HBM: each K and V row is read once for all the q heads and new tokens
// that share it, 64 flop or more per two bytes.  A stream is the rows of one KV head
// of one sequence; all streams are concatenated in units of 16 rows and cut into
// equal slices, one per CTA, so every CTA moves the same bytes whatever the mix of
// lengths (a cut near a stream's end moves there).  A producer warp copies tiles of
// 64 or 128 rows into a ring (bulk copies of at most 16 rows: inside a page); for
// each 16 query rows four warps take 16 keys of a tile each: S = Q K^T by m16n8k16
// products (the query rows are the M side), online softmax in fp32 registers in the
// log2 domain, O += P V.  The four warps' (max, sum, O) are joined in shared memory
// at the end of a stream's part; a stream inside one slice is written as output, the
// parts of others go to the workspace and a merge kernel joins them.
//
// Measured, f16: one token of 64 sequences of 1,025 to 8,193 rows of 4 x 128 106 us
// (5.6 TB/s), three of one sequence of 131,072 rows of 8 x 128 91 us (5.9 TB/s, 0.91
// of the copy rate); one token over 512 rows of 4 x 64 6.5 us.  What is left of the
// batch's time over its bytes: the plan and first loads (2 us), a CTA's second part
// (1.7 us), the merge kernel and the tail of the slices (3 to 4 us).
#include <algorithm>
#include <cmath>

#include "paged_common.cuh"

namespace picoattn {

namespace {

constexpr int kUnit = 16;      // cache rows per unit
constexpr int kKeyWarps = 4;   // warps that share the keys of a tile
constexpr int kMostRows = 32;
constexpr long long kTwoGroupBytes = 128ll << 20;
constexpr int kMaxParts = 512;  // most CTAs of the attention kernel
constexpr int kSlots = kMaxParts * kMostRows;  // partial rows in the workspace: two parts of each CTA
constexpr int kSnapBytes = 64 << 10;
constexpr int kMinUnits = 4;   // least units per CTA: a slice shorter than a tile gains nothing

// MT: groups of 16 query rows.  One: two CTAs per SM with a ring of three stages;
// two: one CTA with a ring of six.
template <int HD, int MT>
struct Few {
    static constexpr int kRows = 16 * MT;
    static constexpr int kWarps = kKeyWarps * MT;         // compute warps
    static constexpr int kThreads = 32 * (kWarps + 1);
    static constexpr int kCtas = MT == 1 ? 2 : 1;         // per SM
    // Two CTAs have three warps on a quarter SM: 144 registers leave room there for a warp of the merge kernel, which
    // then starts while they finish (two sequences of 5,000 rows of 4 x 64: 12.8 us, with 152 registers 14.3).  At hd 128
    // its 72 registers would fit too, but 144 spill (two sequences of
    // 16,000 rows of 8 x 128: 36.5 us against 34.1).
    static constexpr int kRegs = HD == 64 ? 144 : 168;
    static constexpr int kMaxCtas = MT == 1 ? kMaxParts : kMaxParts / 2;
    static constexpr int kStages = MT == 1 ? 3 : 6;
    static constexpr int T = 8192 / HD;        // cache rows per tile: 16 KB of K
    static constexpr int GR = T / 8;           // a tile is 8 groups of GR rows, each padded by 16 bytes
    static constexpr int ROW = HD * 2;
    static constexpr int GS = GR * ROW + 16;   // group stride: 8 rows of a product, one per group, on 8 bank quads
    static constexpr int TILE = 8 * GS;
    static constexpr int RG = T / 16;          // 16-key groups per tile
    static constexpr int off_ml = 256;         // [kWarps][16] (max, sum)
    static constexpr int off_join = (off_ml + 8 * kWarps * 16 + 15) / 16 * 16;
    static constexpr int JS = 36;              // floats per row of the join buffer (32 columns, padded)
    static constexpr int off_tiles = (off_join + 4 * kWarps * 16 * JS + 127) / 128 * 128;
    static constexpr int bytes = off_tiles + kStages * 2 * TILE;
    static_assert(kCtas * (bytes + 1024) <= 228 * 1024, "CTAs per SM");
};

struct FewArgs {
    PagedAttnArgs a;
    int4* cut;          // streams for the merge kernel: (stream, its first CTA, its parts)
    float2* part_ml;    // [2 * grid][rows]
    float* part_o;      // [2 * grid][rows][hd]
    int by_cta;         // `cut` has an entry for each CTA (the stream that begins there and goes on), else for each stream
};

__device__ __forceinline__ long long seq_units(const SeqSpan& s, int hkv) {
    return s.ok && s.n > 0 ? (long long)hkv * ((s.len + kUnit - 1) / kUnit) : 0;
}
// CTAs in use, and the units [first(i), first(i + 1)) of CTA i
__device__ __forceinline__ int ctas_used(long long units, int grid) {
    return (int)min((long long)grid, (units + kMinUnits - 1) >> 2);
    static_assert(kMinUnits == 4, "a shift");
}
__device__ __forceinline__ long long first_unit(long long i, long long units, int ctas) { return quotient(i * units, ctas); }
__device__ __forceinline__ int cta_of(long long unit, long long units, int ctas) {
    int i = (int)quotient(unit * ctas, units);
    while (i + 1 < ctas && first_unit(i + 1, units, ctas) <= unit) i++;
    while (i > 0 && first_unit(i, units, ctas) > unit) i--;
    return i;
}
// A cut this near to a stream's end moves there: a second part costs a CTA 1.7 us
// (its Q rows, the join), 64 KB more of the cache up to 1 us.  Less than half a
// slice, so that no two cuts meet.
template <int HD>
__device__ __forceinline__ int most_moved(long long units, int ctas) {
    return (int)min((long long)(kSnapBytes / (kUnit * 4 * HD)), quotient(units, ctas) / 2);
}
struct Cut {
    int b;                // the sequence
    long long from, at;   // its first unit, the cut's
};
__device__ __forceinline__ long long moved(long long cut, long long s0, long long s1, int most) {
    return cut - s0 <= most ? s0 : (s1 - cut <= most ? s1 : cut);
}

template <class T>
__device__ __forceinline__ void mma16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (std::is_same<T, __half>::value) {
        mma_16816(d, a, b0, b1);
    } else {
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
            "{%0,%1,%2,%3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    }
}

// Four output columns of a row, in the output's type.
template <class T>
__device__ __forceinline__ void store_out4(const PagedAttnArgs& a, size_t at, const float4& v) {
    if (a.out_dtype == PICOATTN_DTYPE_F32)
        *reinterpret_cast<float4*>(static_cast<float*>(a.out) + at) = v;
    else
        *reinterpret_cast<uint2*>(static_cast<T*>(a.out) + at) =
            make_uint2(Elem<T>::pack2(v.x, v.y), Elem<T>::pack2(v.z, v.w));
}

// Calls fn(b, span, head, u0, u1, units of the stream) for each part of the
// units [c0, c1), in order; b0: a sequence at or before the first, whose units
// begin at `base`.
template <class F>
__device__ __forceinline__ void for_each_part(const PagedAttnArgs& a, int b0, long long base, long long c0, long long c1,
                                              F&& fn) {
    for (int b = b0; b < a.b.n_seqs && base < c1; b++) {
        const SeqSpan sp = seq_span(a.b, b);
        const long long n = seq_units(sp, a.hkv);
        if (base + n > c0) {
            const int per_head = (sp.len + kUnit - 1) / kUnit;
            long long at = max(base, c0);
            const long long end = min(base + n, c1);
            while (at < end) {
                const int h = (int)quotient(at - base, per_head);
                const int u0 = (int)(at - base - (long long)h * per_head);
                const int u1 = (int)min((long long)per_head, u0 + (end - at));
                fn(b, sp, h, u0, u1, per_head);
                at += u1 - u0;
            }
        }
        base += n;
    }
}

// NaN into the rows of KV head h of a sequence outside the host's bounds (as far
// as they lie in out).
template <class T, int HD>
__device__ __forceinline__ void nan_rows(const PagedAttnArgs& a, int b, int h, int tid, int threads) {
    constexpr int C4 = HD / 4;
    const RowRange rows = rows_inside(a.b, b);
    const float nan = __int_as_float(0x7fc00000);
    const long long n = (long long)(rows.end - rows.first) * a.g * C4;
    for (long long i = tid; i < n; i += threads) {
        const long long x = i / C4;
        store_out4<T>(a, ((size_t)(rows.first + x / a.g) * a.hq + (size_t)h * a.g + x % a.g) * HD + 4 * (i % C4),
                      make_float4(nan, nan, nan, nan));
    }
}

template <class T, int HD, int MT, bool kWhole>
__global__ void __maxnreg__((Few<HD, MT>::kRegs)) paged_few_kernel(FewArgs fa) {
    using F = Few<HD, MT>;
    constexpr int kRows = F::kRows, kWarps = F::kWarps, kThreads = F::kThreads, kStages = F::kStages;
    extern __shared__ __align__(128) uint8_t smem[];
    const PagedAttnArgs& a = fa.a;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    uint64_t* full = reinterpret_cast<uint64_t*>(smem);
    uint64_t* empty = full + kStages;
    int* poison = reinterpret_cast<int*>(empty + kStages);  // [kStages] the tile read a page that does not exist
    int* gave_up = reinterpret_cast<int*>(smem + 124);      // a wait of a compute warp has run out: nothing more is stored
    long long* warp_tot = reinterpret_cast<long long*>(smem + 176);  // [kWarps + 1]
    Cut* cuts = reinterpret_cast<Cut*>(smem + 128);  // [2]
    float2* ml = reinterpret_cast<float2*>(smem + F::off_ml);
    float* join = reinterpret_cast<float*>(smem + F::off_join);
    uint8_t* tiles = smem + F::off_tiles;

    pdl_trigger();
    if (tid == 0) {
        for (int s = 0; s < kStages; s++) mbar_init(&full[s], 1), mbar_init(&empty[s], kWarps);
        *gave_up = 0;
        fence_mbar_init();
    }
    pdl_wait();
    int b0;
    long long base, c0, c1;
    if constexpr (kWhole) {  // a stream per CTA
        b0 = (int)(blockIdx.x / (unsigned)a.hkv);
        const int h = (int)blockIdx.x - b0 * a.hkv;
        const SeqSpan sp = seq_span(a.b, b0);
        if (!sp.ok) {
            if (h == 0 && tid == 0) atomicOr(a.b.status, PICOATTN_DEV_BAD_POS);
            nan_rows<T, HD>(a, b0, h, tid, kThreads);
        }
        if (!sp.ok || sp.n == 0) return;
        const int per_head = (sp.len + kUnit - 1) / kUnit;
        base = 0, c0 = (long long)h * per_head, c1 = c0 + per_head;
        __syncthreads();  // the barriers
    } else {
        // the units of each thread's sequences, and of those before them
        const int per = (a.b.n_seqs + kThreads - 1) / kThreads;
        const int lo = min(tid * per, a.b.n_seqs), hi = min(lo + per, a.b.n_seqs);
        long long mine = 0;
        bool bad = false;
        for (int b = lo; b < hi; b++) {
            const SeqSpan sp = seq_span(a.b, b);
            bad |= !sp.ok;
            mine += seq_units(sp, a.hkv);
        }
        long long incl = mine;
        for (int o = 1; o < 32; o <<= 1) {
            const long long v = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += v;
        }
        if (lane == 31) warp_tot[warp] = incl;
        if (tid == 0 && fa.by_cta) fa.cut[blockIdx.x] = make_int4(-1, 0, 0, 0);
        bad = __syncthreads_or(bad);
        long long first = incl - mine, units = 0;
        for (int w = 0; w <= kWarps; w++) {
            units += warp_tot[w];
            if (w < warp) first += warp_tot[w];
        }
        const int ctas = ctas_used(units, gridDim.x);
        if ((int)blockIdx.x < ctas) {
            const int most = most_moved<HD>(units, ctas);
            const long long begin = first_unit(blockIdx.x, units, ctas);
            // the thread that has a cut's sequence finds the sequence, its first unit, and where the cut goes
            for (int e = 0; e < 2; e++) {
                const long long cut = e ? first_unit(blockIdx.x + 1, units, ctas) : begin;
                if (cut < first || cut >= first + mine) continue;
                long long from = first;
                for (int b = lo; b < hi; b++) {
                    const SeqSpan sp = seq_span(a.b, b);
                    const long long n = seq_units(sp, a.hkv);
                    if (from + n > cut) {
                        const int per_head = (sp.len + kUnit - 1) / kUnit, h = (int)quotient(cut - from, per_head);
                        const long long s0 = from + (long long)h * per_head, s1 = s0 + per_head;
                        const long long at = moved(cut, s0, s1, most);
                        cuts[e] = {b, from, at};
                        if (e == 1 && at > s0 && at < s1 && begin - s0 <= most) {
                            // the stream begins here and goes on, to the CTA of its last unit, or where that one's first
                            // cut moves to the stream's end the one before
                            int last = cta_of(s1 - 1, units, ctas);
                            if (last > (int)blockIdx.x + 1 && s1 - first_unit(last, units, ctas) <= most) last--;
                            const int stream = b * a.hkv + h;
                            fa.cut[fa.by_cta ? (int)blockIdx.x : stream] =
                                make_int4(stream, blockIdx.x, last - (int)blockIdx.x + 1, 0);
                        }
                        break;
                    }
                    from += n;
                }
            }
        }
        if (bad) {  // each CTA its share of the sequences
            if (blockIdx.x == 0 && tid == 0) atomicOr(a.b.status, PICOATTN_DEV_BAD_POS);
            for (int b = blockIdx.x; b < a.b.n_seqs; b += gridDim.x)
                if (!seq_span(a.b, b).ok)
                    for (int h = 0; h < a.hkv; h++) nan_rows<T, HD>(a, b, h, tid, kThreads);
        }
        __syncthreads();
        if ((int)blockIdx.x >= ctas) return;
        b0 = cuts[0].b, base = cuts[0].from, c0 = cuts[0].at;
        c1 = (int)blockIdx.x + 1 < ctas ? cuts[1].at : units;
    }

    if (warp == kWarps) {
        // ---------------- producer: lanes 0-7 the K groups, 8-15 the V groups ----------------
        int t = 0;
        bool ok = true;  // no wait has run out: then nothing more is copied
        const uint8_t* pool = static_cast<const uint8_t*>(lane & 8 ? a.v_pool : a.k_pool);
        for_each_part(a, b0, base, c0, c1, [&](int b, const SeqSpan& sp, int h, int u0, int u1, int stream_units) {
            if (!kWhole && lane == 0 && !fa.by_cta && u0 == 0 && u1 == stream_units)
                fa.cut[b * a.hkv + h] = make_int4(0, 0, 1, 0);  // not cut; written whatever runs out: the merge goes by it
            if (!ok) return;
            const int r1 = min(u1 * kUnit, sp.len);
            const int* table = a.b.page_table + (size_t)b * a.b.page_cols;
            for (int row0 = u0 * kUnit; row0 < r1; row0 += F::T, t++) {
                const int s = t % kStages;
                const int g0 = row0 + F::GR * (lane & 7);
                const bool copy = lane < 16 && g0 < r1;
                const int page = copy ? table[g0 >> a.b.page_shift] : 0;
                const bool bad = page < 0 || page >= a.b.n_pages;
                const int any_bad = __any_sync(0xffffffffu, bad);
                const uint32_t bytes = __popc(__ballot_sync(0xffffffffu, copy)) * (uint32_t)(F::GR * F::ROW);
                if (t >= kStages) {  // its last tile there (a warp that gave up may give it back before), and given back
                    const uint32_t last = (uint32_t)((t / kStages - 1) & 1);
                    ok = __all_sync(0xffffffffu, mbar_wait(&full[s], last, a.b.status) &&
                                                     mbar_wait(&empty[s], last, a.b.status));
                    if (!ok) return;
                }
                if (lane == 0) {
                    if (any_bad) atomicOr(a.b.status, PICOATTN_DEV_BAD_PAGE);
                    poison[s] = any_bad;
                    mbar_arrive_expect_tx(&full[s], bytes);
                }
                __syncwarp();
                if (copy) {
                    const size_t row = ((size_t)(bad ? 0 : page) * a.hkv + h) * a.b.page_size + (g0 & (a.b.page_size - 1));
                    bulk_g2s(tiles + (s * 2 + (lane >> 3)) * F::TILE + (lane & 7) * F::GS, pool + row * F::ROW,
                             F::GR * F::ROW, &full[s]);
                }
            }
        });
        // the compute warps may have given up on copies still on their way: they land before the CTA ends
        if (lane == 0)
            for (int c = max(0, t - kStages); c < t; c++) mbar_settle(&full[c % kStages], (uint32_t)((c / kStages) & 1));
        return;
    }

    // ---------------- compute warps ----------------
    const int gid = lane >> 2, tig = lane & 3, kw = warp % kKeyWarps, mt = warp / kKeyWarps;
    // ldmatrix rows (matrix lane >> 3, its row lane & 7 = tile group): K (keys 0-7 | dims 0-7, keys 0-7 | dims 8-15,
    // keys 8-15 | ..), V transposed (keys 0-7 | dims 0-7, keys 8-15 | dims 0-7, ..); key 8j + q of 16-key group rg is
    // tile row GR q + 2 rg + j
    const uint32_t k_lane = (uint32_t)((lane & 7) * F::GS + (lane >> 4) * F::ROW + ((lane >> 3) & 1) * 16);
    const uint32_t v_lane = (uint32_t)((lane & 7) * F::GS + ((lane >> 3) & 1) * F::ROW + (lane >> 4) * 16);
    const uint32_t tiles_u32 = smem_u32(tiles);
    const float scale = 1.4426950408889634f / sqrtf((float)HD);
    // weights of up to 2^15 of fp16's 2^16 (weight_lift): below 2^-40 of the largest they vanish
    constexpr float lift = weight_lift<T>(15);
    int t = 0;
    for_each_part(a, b0, base, c0, c1, [&](int b, const SeqSpan& sp, int h, int u0, int u1, int stream_units) {
        const int rows = sp.n * a.g;  // <= kRows
        uint32_t qa[HD / 16][4];
        int lim[2];  // keys below it are visible to the lane's rows gid, gid + 8
#pragma unroll
        for (int half = 0; half < 2; half++) {
            const int r = 16 * mt + gid + 8 * half;
            const int i = r / a.g;
            lim[half] = sp.len - sp.n + i + 1;
            const uint32_t* src = reinterpret_cast<const uint32_t*>(
                static_cast<const T*>(a.q) + (sp.t0 + i) * a.qs + (size_t)(h * a.g + r - i * a.g) * HD + 2 * tig);
#pragma unroll
            for (int kk = 0; kk < HD / 16; kk++) {
                qa[kk][half] = r < rows ? src[8 * kk] : 0u;
                qa[kk][2 + half] = r < rows ? src[8 * kk + 4] : 0u;
            }
        }
        float m[2] = {-1e30f, -1e30f}, l[2] = {0.f, 0.f};
        float o[HD / 8][4];
#pragma unroll
        for (int i = 0; i < HD / 8; i++) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
        const int r1 = min(u1 * kUnit, sp.len);
        for (int row0 = u0 * kUnit; row0 < r1; row0 += F::T, t++) {
            const int s = t % kStages;
            // a wait that ran out is noted and the warp goes on, over whatever the stage holds (to leave here, with a vote
            // and a flag in a register, costs 2 to 4%)
            if (!mbar_wait(&full[s], (uint32_t)((t / kStages) & 1), a.b.status)) *gave_up = 1;
            const uint32_t kbase = tiles_u32 + (uint32_t)(s * 2 * F::TILE), vbase = kbase + F::TILE;
            const int valid = r1 - row0;
            if (poison[s]) l[0] = l[1] = __int_as_float(0x7fc00000);
            const bool mask = row0 + F::T > sp.len - sp.n + 1 || valid < F::T;
            const int lim0 = min(lim[0] - row0, valid), lim1 = min(lim[1] - row0, valid);
#pragma unroll
            for (int rg = kw; rg < F::RG; rg += kKeyWarps) {
                if (2 * rg >= valid) continue;
                if (valid < F::T) {
                    // rows past the part hold anything: their V must not meet the zero weights as a NaN.  This warp
                    // alone reads the rows of its key groups, or with the same warps of the other query rows, which
                    // write the same zeros
                    for (int e = lane; e < 16 * (F::ROW / 16); e += 32) {
                        const int key = e / (F::ROW / 16), q = key & 7, u = 2 * rg + (key >> 3);
                        if (F::GR * q + u >= valid)
                            *reinterpret_cast<uint4*>(tiles + (s * 2 + 1) * F::TILE + q * F::GS + u * F::ROW +
                                                      (e % (F::ROW / 16)) * 16) = make_uint4(0, 0, 0, 0);
                    }
                    fence_proxy_async_shared();  // before the ring's next copy into these rows
                    __syncwarp();
                }
                const uint32_t goff = (uint32_t)(2 * rg * F::ROW);
                float sc[2][4];
#pragma unroll
                for (int j = 0; j < 2; j++) sc[j][0] = sc[j][1] = sc[j][2] = sc[j][3] = 0.f;
#pragma unroll
                for (int kk = 0; kk < HD / 16; kk++) {
                    uint32_t bk[4];
                    ldsm_x4(bk, kbase + goff + k_lane + (uint32_t)kk * 32u);
                    mma16<T>(sc[0], qa[kk], bk[0], bk[1]);
                    mma16<T>(sc[1], qa[kk], bk[2], bk[3]);
                }
#pragma unroll
                for (int j = 0; j < 2; j++)
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        sc[j][e] *= scale;
                        if (mask && F::GR * (2 * tig + (e & 1)) + 2 * rg + j >= (e < 2 ? lim0 : lim1))
                            sc[j][e] = -INFINITY;
                    }
                float mx0 = fmaxf(fmaxf(sc[0][0], sc[0][1]), fmaxf(sc[1][0], sc[1][1]));
                float mx1 = fmaxf(fmaxf(sc[0][2], sc[0][3]), fmaxf(sc[1][2], sc[1][3]));
                mx0 = fmaxf(mx0, __shfl_xor_sync(0xffffffffu, mx0, 1));
                mx0 = fmaxf(mx0, __shfl_xor_sync(0xffffffffu, mx0, 2));
                mx1 = fmaxf(mx1, __shfl_xor_sync(0xffffffffu, mx1, 1));
                mx1 = fmaxf(mx1, __shfl_xor_sync(0xffffffffu, mx1, 2));
                const float mn0 = fmaxf(m[0], mx0 - lift), mn1 = fmaxf(m[1], mx1 - lift);
                const float f0 = ex2(m[0] - mn0), f1 = ex2(m[1] - mn1);
                m[0] = mn0;
                m[1] = mn1;
                float p[2][4];
#pragma unroll
                for (int j = 0; j < 2; j++) {
                    p[j][0] = ex2(sc[j][0] - mn0);
                    p[j][1] = ex2(sc[j][1] - mn0);
                    p[j][2] = ex2(sc[j][2] - mn1);
                    p[j][3] = ex2(sc[j][3] - mn1);
                }
                l[0] = l[0] * f0 + ((p[0][0] + p[0][1]) + (p[1][0] + p[1][1]));
                l[1] = l[1] * f1 + ((p[0][2] + p[0][3]) + (p[1][2] + p[1][3]));
                if (__any_sync(0xffffffffu, f0 != 1.f || f1 != 1.f)) {
#pragma unroll
                    for (int i = 0; i < HD / 8; i++) {
                        o[i][0] *= f0, o[i][1] *= f0;
                        o[i][2] *= f1, o[i][3] *= f1;
                    }
                }
                const uint32_t pa[4] = {Elem<T>::pack2(p[0][0], p[0][1]), Elem<T>::pack2(p[0][2], p[0][3]),
                                        Elem<T>::pack2(p[1][0], p[1][1]), Elem<T>::pack2(p[1][2], p[1][3])};
#pragma unroll
                for (int dt = 0; dt < HD / 16; dt++) {
                    uint32_t bv[4];
                    ldsm_x4_t(bv, vbase + goff + v_lane + (uint32_t)dt * 32u);
                    mma16<T>(o[2 * dt], pa, bv[0], bv[1]);
                    mma16<T>(o[2 * dt + 1], pa, bv[2], bv[3]);
                }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&empty[s]);
        }

        // join the key warps' (max, sum, O): thread (row tid / 8, four columns)
#pragma unroll
        for (int half = 0; half < 2; half++) {
            l[half] += __shfl_xor_sync(0xffffffffu, l[half], 1);
            l[half] += __shfl_xor_sync(0xffffffffu, l[half], 2);
            if (tig == 0) ml[warp * 16 + gid + 8 * half] = make_float2(m[half], l[half]);
        }
        named_bar_sync(1, 32 * kWarps);
        // the same for all: who sets it for the next part has been through all of this one's barriers
        const bool store = *gave_up == 0;
        float wgt[2];
#pragma unroll
        for (int half = 0; half < 2; half++) {
            const float2* x = ml + mt * kKeyWarps * 16 + gid + 8 * half;
            float M = x[0].x;
#pragma unroll
            for (int w = 1; w < kKeyWarps; w++) M = fmaxf(M, x[w * 16].x);
            wgt[half] = ex2(m[half] - M);
        }
        const int jr = tid >> 3, jc = (tid & 7) * 4;
        const int jw = (jr >> 4) * kKeyWarps * 16 + (jr & 15);  // the row in its first key warp's 16
        float M = ml[jw].x, Ls = 0.f;
#pragma unroll
        for (int w = 1; w < kKeyWarps; w++) M = fmaxf(M, ml[jw + w * 16].x);
#pragma unroll
        for (int w = 0; w < kKeyWarps; w++) Ls += ml[jw + w * 16].y * ex2(ml[jw + w * 16].x - M);
        const bool whole = kWhole || (u0 == 0 && u1 == stream_units);
        const size_t slot = 2 * (size_t)blockIdx.x + (u0 == 0 ? 1 : 0);
        const int ji = jr / a.g;
        const size_t orow = ((size_t)(sp.t0 + ji) * a.hq + (size_t)(h * a.g + jr - ji * a.g)) * HD;
        if (!whole && (tid & 7) == 0 && jr < rows)
            fa.part_ml[slot * kRows + jr] = make_float2(M, store ? Ls : __int_as_float(0x7fc00000));
#pragma unroll
        for (int c = 0; c < HD / 32; c++) {
#pragma unroll
            for (int i = 0; i < 4; i++) {
                float* d = join + (warp * 16 + gid) * F::JS + 8 * i + 2 * tig;
                *reinterpret_cast<float2*>(d) = make_float2(o[4 * c + i][0] * wgt[0], o[4 * c + i][1] * wgt[0]);
                *reinterpret_cast<float2*>(d + 8 * F::JS) = make_float2(o[4 * c + i][2] * wgt[1], o[4 * c + i][3] * wgt[1]);
            }
            named_bar_sync(1, 32 * kWarps);
            if (jr < rows && store) {
                float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                for (int w = 0; w < kKeyWarps; w++) {
                    const float4 x = *reinterpret_cast<const float4*>(join + (jw + w * 16) * F::JS + jc);
                    v.x += x.x, v.y += x.y, v.z += x.z, v.w += x.w;
                }
                if (whole) {
                    const float inv = 1.0f / Ls;
                    store_out4<T>(a, orow + 32 * c + jc, make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv));
                } else {
                    *reinterpret_cast<float4*>(fa.part_o + (slot * kRows + jr) * HD + 32 * c + jc) = v;
                }
            }
            named_bar_sync(1, 32 * kWarps);
        }
    });
}

// out = sum_p 2^(m_p - M) o_p / sum_p 2^(m_p - M) l_p over the parts of one
// query row of a stream cut across CTAs; block (row, stream or the
// CTA where it begins), thread (part
// group, four columns).  All loads of a row's first parts are in flight at
// once: the merge is one round trip to L2.
constexpr int kMergeThreads = 128;

template <class T, int HD>
__global__ void __launch_bounds__(kMergeThreads) paged_few_merge_kernel(FewArgs fa, int rows) {
    constexpr int C4 = HD / 4, NG = kMergeThreads / C4, RPT = 40 / NG;
    __shared__ float w_s[kMaxParts], red[kMergeThreads / 32][2];
    __shared__ float4 acc_s[kMergeThreads];
    pdl_trigger();
    pdl_wait();
    const PagedAttnArgs& a = fa.a;
    const int tid = threadIdx.x, c4 = tid % C4, grp = tid / C4;
    const int r = blockIdx.x;
    const int4 cut = __ldcg(fa.cut + blockIdx.y);
    if (fa.by_cta && cut.x < 0) return;
    const int stream = fa.by_cta ? cut.x : (int)blockIdx.y;
    const int b = stream / a.hkv, h = stream - b * a.hkv;
    const SeqSpan sp = seq_span(a.b, b);
    if (!sp.ok || r >= sp.n * a.g) return;  // a stream without keys has no entry
    const int lo = cut.y, parts = cut.z;
    if (parts == 1) return;  // written by the attention kernel
    auto slot = [&](int p) -> size_t {  // the first part begins its stream, the others are their CTA's first
        const bool begins = p == 0;
        return ((size_t)(lo + p) * 2 + (begins ? 1 : 0)) * rows + r;
    };
    float4 v[RPT];
#pragma unroll
    for (int i = 0; i < RPT; i++) {
        const int p = grp + i * NG;
        if (p < parts) v[i] = __ldcg(reinterpret_cast<const float4*>(fa.part_o + slot(p) * HD) + c4);
    }
    float M = -INFINITY;
    float2 x[kMaxParts / kMergeThreads];
#pragma unroll
    for (int i = 0; i < kMaxParts / kMergeThreads; i++) {
        const int p = tid + i * kMergeThreads;
        x[i] = p < parts ? __ldcg(fa.part_ml + slot(p)) : make_float2(-INFINITY, 0.f);
        M = fmaxf(M, x[i].x);
    }
    for (int o = 16; o; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
    if ((tid & 31) == 0) red[tid >> 5][0] = M;
    __syncthreads();
    for (int w = 0; w < kMergeThreads / 32; w++) M = fmaxf(M, red[w][0]);
    float L = 0.f;
#pragma unroll
    for (int i = 0; i < kMaxParts / kMergeThreads; i++) {
        const int p = tid + i * kMergeThreads;
        if (p < parts) {
            const float w = ex2(x[i].x - M);
            w_s[p] = w;
            L += w * x[i].y;
        }
    }
    for (int o = 16; o; o >>= 1) L += __shfl_xor_sync(0xffffffffu, L, o);
    if ((tid & 31) == 0) red[tid >> 5][1] = L;
    __syncthreads();
    L = 0.f;
    for (int w = 0; w < kMergeThreads / 32; w++) L += red[w][1];
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    auto add = [&](int p, const float4& y) {
        const float w = w_s[p];
        acc.x += w * y.x, acc.y += w * y.y, acc.z += w * y.z, acc.w += w * y.w;
    };
#pragma unroll
    for (int i = 0; i < RPT; i++)
        if (grp + i * NG < parts) add(grp + i * NG, v[i]);
    for (int p = grp + RPT * NG; p < parts; p += NG)
        add(p, __ldcg(reinterpret_cast<const float4*>(fa.part_o + slot(p) * HD) + c4));
    acc_s[tid] = acc;
    __syncthreads();
    if (grp == 0) {
        for (int g = 1; g < NG; g++) {
            const float4 y = acc_s[g * C4 + c4];
            acc.x += y.x, acc.y += y.y, acc.z += y.z, acc.w += y.w;
        }
        const float inv = 1.0f / L;
        const int i = r / a.g;
        store_out4<T>(a, ((size_t)(sp.t0 + i) * a.hq + (size_t)(h * a.g + r - i * a.g)) * HD + 4 * c4,
                      make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv));
    }
}

// Short sequences: a stream per CTA, nothing merged.  An SM takes in 65 KB a
// microsecond, the merge kernel and a stream's second part cost 3 to 4: up to
// 256 KB a stream (bf16, 4 x 64: 300 rows 6.1 us against 8.8, 800 rows 9.0 both,
// 1,500 rows 13.3 against 9.0), and up to 512 KB where the streams are many
// enough to keep the memory busy (64 of 700 rows of 8 x 128, 4 rows each: 32 us
// against 40; at 1,000 rows 128 streams 19.3 against 22.6, 400 streams 43 both).
// More would gain where all lengths are alike, but the longest decides here.
bool whole_streams(const PagedAttnArgs& a) {
    const long long bytes = (long long)a.b.max_len * a.hd * 4;
    return bytes <= (256 << 10) ||
           (bytes <= (512 << 10) && (long long)a.b.n_seqs * a.hkv * 3 >= 2 * device_sm_count());
}

template <class T, int HD, int MT>
cudaError_t launch_rows(const PagedAttnArgs& a, cudaStream_t stream) {
    using F = Few<HD, MT>;
    static PerDeviceOnce setup;
    cudaError_t e = setup.run([] {
        const cudaError_t w = cudaFuncSetAttribute(paged_few_kernel<T, HD, MT, true>,
                                                   cudaFuncAttributeMaxDynamicSharedMemorySize, F::bytes);
        return w != cudaSuccess ? w
                                : cudaFuncSetAttribute(paged_few_kernel<T, HD, MT, false>,
                                                       cudaFuncAttributeMaxDynamicSharedMemorySize, F::bytes);
    });
    if (e != cudaSuccess) return e;
    FewArgs fa{};
    fa.a = a;
    if (whole_streams(a))
        return launch_pdl(paged_few_kernel<T, HD, MT, true>, dim3(a.b.n_seqs * a.hkv), dim3(F::kThreads),
                          (size_t)F::bytes, stream, fa);
    const long long units = (long long)a.b.n_seqs * a.hkv * ((a.b.max_len + kUnit - 1) / kUnit);
    const int grid = (int)std::min<long long>(std::min(F::kCtas * device_sm_count(), F::kMaxCtas),
                                              (units + kMinUnits - 1) / kMinUnits);
    static_assert(2 * F::kMaxCtas * F::kRows <= kSlots, "workspace");
    fa.part_ml = reinterpret_cast<float2*>(a.ws);
    fa.part_o = reinterpret_cast<float*>(a.ws + (size_t)kSlots * 8);
    fa.cut = reinterpret_cast<int4*>(a.ws + (size_t)kSlots * (8 + 4 * HD));
    // at most one stream begins in a CTA and goes on in the next: with many streams (512 of 16 rows: 8,192 blocks,
    // most of them with nothing to do) the merge goes by those
    fa.by_cta = (long long)a.b.n_seqs * a.hkv > grid;
    e = launch_pdl(paged_few_kernel<T, HD, MT, false>, dim3(grid), dim3(F::kThreads), (size_t)F::bytes, stream, fa);
    if (e != cudaSuccess) return e;
    return launch_pdl(paged_few_merge_kernel<T, HD>, dim3(a.b.max_new * a.g, fa.by_cta ? grid : a.b.n_seqs * a.hkv),
                      dim3(kMergeThreads), 0, stream, fa, F::kRows);
}

template <class T, int HD>
cudaError_t launch_types(const PagedAttnArgs& a, cudaStream_t stream) {
    const int rows = a.b.max_new * a.g;
    return rows <= 16 ? launch_rows<T, HD, 1>(a, stream) : launch_rows<T, HD, 2>(a, stream);
}

}  // namespace

// Up to 16 rows this kernel reads the cache at the memory's rate.  A second group
// of 16 rows doubles the products and the softmax per byte: 4.0 TB/s at hd 64, 4.8
// to 5.8 at hd 128, where the chunk kernel gets to 4.0 and 6.3.  But this one starts
// sooner, so it takes what is short: 24 rows over 2,000 keys of 4 x 64 12.2 us
// against 18.8, 28 rows over 9 sequences of 3,500 of 4 x 128 26 against 30; over 32
// of 4,000 (260 MB) 63 against 55.  Four groups (35 rows and up) were slower on the
// whole: 18 against 13 us for one sequence of 300, 53 against 30 for 9 of 3,500 (17
// warps leave 96 registers each).
bool paged_few_fits(const PagedAttnArgs& a) {
    const long long rows = (long long)a.b.max_new * a.g, streams = (long long)a.b.n_seqs * a.hkv;
    return rows <= 16 || (rows <= kMostRows && streams <= kTwoGroupBytes / ((long long)a.b.max_len * a.hd * 4));
}

size_t paged_few_bytes(int hd) {
    return align_up((size_t)kSlots * (8 + 4 * hd) + (size_t)kMaxParts * 16, 256);
}

cudaError_t launch_paged_few(const PagedAttnArgs& a, cudaStream_t stream) {
    if (a.dtype == PICOATTN_DTYPE_F16)
        return a.hd == 64 ? launch_types<__half, 64>(a, stream) : launch_types<__half, 128>(a, stream);
    return a.hd == 64 ? launch_types<__nv_bfloat16, 64>(a, stream) : launch_types<__nv_bfloat16, 128>(a, stream);
}

}  // namespace picoattn
