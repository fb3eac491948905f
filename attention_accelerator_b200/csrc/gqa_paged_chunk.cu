// gqa_paged_chunk.cu -- any number of queries a sequence over the paged 8-bit
// cache, on the fifth-generation tensor cores.
//
// Work.  A unit is 64 consecutive queries of one sequence and one KV head: 256
// rows (query, Q head), two M = 128 tiles.  Its keys are those that any of its
// rows sees, in tiles of 128 on a grid of absolute positions.  plan_units_kernel
// (one CTA) finds every unit's keys from the lengths and masks in device memory,
// sums the tiles, and says where each CTA of paged_chunk_kernel begins: all tiles
// of all units in order are dealt out at even cost, so that causal
// prompts, ragged batches and one long context alike fill the GPU.  A unit that
// crosses shares leaves FP32 partial rows; its last CTA merges them in order.
//
// Precision.  Codes become FP16 exactly for S = Q K^T; Q is rotated in FP32,
// divided by a power of two that brings the row's largest below 1, and rounded to
// FP16 (2^-11 of a term: three more bits than the BF16 it came as).  K's scale
// multiplies the FP32 scores.  V's codes are exact too: its scale joins the weights,
// 2^(z + log2(V scale) - m), which round to FP16, and O accumulates in FP32 in TMEM:
// together a few 2^-11 of the sum of |weight * value|, and 2^-31 of the row's largest
// weight times scale for each key, for an output that is rounded to 2^-8.
//
// Warps (one CTA per SM):
//   0-3, 4-7   softmax of M tile 0, 1: a thread a row.  Per unit, 4 lanes rotate one
//              query's 4 head rows (16 pairs each) into the swizzled A operand.  Per
//              tile: maximum of the S row from TMEM (per 16 keys, then times their
//              page's scale), weights back over S as FP16 (the A operand of O += P V).
//              The reference m moves only when a maximum passes it by 2^8; then O is
//              rescaled in TMEM, which the in-order tensor pipe leaves still.
//   8-11       conversion: 16 KB of codes (TMA, 128-byte swizzle) to 32 KB of FP16 in
//              the K-major (K) and MN-major (V) operand layout, which are the same
//              bytes: rows of 64 dims, two blocks, 128-byte swizzle.
//   12         MMA issuer: S0 S1 | PV0 S0' PV1 S1' | ..., so that one M tile's products
//              run while the other's softmax does.
//   13         loader: table entries, scales, TMA.
//   14         zeros of units whose rows see nothing.
//
// Bound, for long contexts, by a tile's chain: the softmax of 2 x 128 rows (about
// 2300 cycles), the conversion of K and V (1350 each) and the products (2000)
// overlap to a period of 4500 cycles; the tensor pipe is 43 % busy.  For short
// ones, by the 25 to 28 thousand cycles a unit costs beside its tiles; for a dozen
// queries, by the same chain with most rows empty.  Measured (B200, e4m3):
// 16 x 128 queries on 8192 keys 294 us (928 TFLOP/s, 57 % of the cuBLAS rate;
// 336 us under the power limit), one prompt of 8192 564 us (977 TFLOP/s), 48 x 5
// queries on up to 8191 keys 214 us (int8, 409 MB; 122 in gqa_paged_few.cu).  V's scale
// multiplied into its codes in the conversion took 308 us.  Each of these took longer
// when it was tried: Q prepared by the conversion warps (371 us, spills), two passes
// over S at fewer registers (354), tanh as a polynomial up to 1 instead of 1/2 (355
// against 300, capped prompts), both M tiles on alternate tiles of few queries (281
// against 237, and 9 % off the rest).
#include "gqa_internal.h"
#include "gqa_paged.cuh"
#include "gqa_paged_internal.h"
#include "gqa_paged_units.cuh"
#include "gqa_tcgen05.cuh"

namespace gqa {

namespace {

constexpr int kTile = 128;                 // keys
constexpr int kTileShift = kChunkTileShift;
constexpr int kTokens = kChunkTokens;      // queries of a unit
constexpr int kRowsM = 128;                // rows of an M tile
constexpr int kRawBytes = kTile * kHeadDim;          // K or V codes of a tile
constexpr int kBlockBytes = kTile * 128;             // 128 rows x 64 dims of FP16
constexpr int kHalfTileBytes = 2 * kBlockBytes;      // K or V of a tile in FP16; an M tile of Q
constexpr int kRaw = 3;                    // ring slots of codes
constexpr int kConv = 3;                   // ring slots of FP16
constexpr int kScaleSlots = 4;             // tiles whose scales are in flight
constexpr int kConvWarp = 8, kMmaWarp = 12, kLoadWarp = 13;
constexpr int kThreads = 16 * 32;
// Registers: launched with 128 a thread; each group of four warps takes its share.
constexpr int kLaunchRegs = 128, kSoftmaxRegs = 184, kConvRegs = 80, kRestRegs = 56;
static_assert(2 * kSoftmaxRegs + kConvRegs + kRestRegs <= 4 * kLaunchRegs, "of what the CTA was launched with");
constexpr uint32_t kTmemCols = 512;
constexpr uint32_t kColS = 0, kColO = 256;  // two of 128 columns each; P over the first 64 of its S
constexpr float kHeadroom = 8.f;   // log2 by which a maximum may pass the reference
constexpr float kLift = 7.f;       // weights are 2^(7 ..): up to 2^15, and FP16's 2^-24 is 2^-31 of the reference

constexpr int kSlotFloats = kRowsM * 2 * (kHeadDim + 2);  // a partial: acc [32][256] float4, (m, l) [256]

// kind::f16 with FP16 A and B, FP32 accumulators, M = 128, N = 128.
constexpr uint32_t kIdescS = (1u << 4) | ((128u >> 3) << 17) | ((128u >> 4) << 24);
constexpr uint32_t kIdescO = kIdescS | (1u << 16);  // B (V) MN-major

struct TileScales {
    float k[8];                 // of each 16 keys: K's scale (NaN where V's is no number)
    float v_log2[8], v_inv[8];  // and V's, as VLog2 has it
    uint32_t v_some;            // bits: V is not zeros
    uint32_t pad[7];
};

struct alignas(16) Shared {
    uint64_t raw_full[kRaw], raw_empty[kRaw], conv_full[kConv], conv_empty[kConv];
    uint64_t q_full[2], s_full[2], p_full[2], pv_done[2], group[2];
    uint64_t drain;  // products in flight when the issuer gives up
    TileScales scales[kScaleSlots];
    uint64_t step[kPairs];  // turns per position of each pair
    int64_t cuts[kMaxCtas + 1];
    uint32_t tmem;
    int last[2];
};

struct alignas(64) ChunkPagedArgs {
    CUtensorMap kmap, vmap;  // (128, page_len, heads, pages) bytes, box (128, page_len, 1, 1)
    PagedCall p;
    RopeSteps rope;
    uint32_t* status;
    const Meta* meta;
    const Unit* units;
    const int32_t* starts;  // [ctas] unit in which each share begins
    const int64_t* cuts;    // [ctas + 1] tiles (of all units and heads, in order) where the shares begin
    uint32_t* arrivals;     // [units][heads][2]
    float* partials;        // [ctas][2][kSlotFloats]
};

struct PlanUnitsArgs {
    PagedCall p;
    UnitShape first, other;
};

// ---------------------------------------------------------------------------
// Planning: units of every sequence, the keys each sees, running sums, shares.
// ---------------------------------------------------------------------------
constexpr int kPlanThreads = 1024;

// Exclusive running sums over the CTA of two values a thread; `all` gets the totals.
__device__ __forceinline__ longlong2 scan_exclusive(longlong2 v, longlong2* warp_sum, longlong2* all) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    longlong2 incl = v;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const long long x = __shfl_up_sync(0xffffffffu, incl.x, d), y = __shfl_up_sync(0xffffffffu, incl.y, d);
        if (lane >= d) {
            incl.x += x;
            incl.y += y;
        }
    }
    __syncthreads();
    if (lane == 31) warp_sum[warp] = incl;
    __syncthreads();
    longlong2 mine = warp_sum[lane], base = make_longlong2(0, 0);
    *all = mine;
#pragma unroll
    for (int d = 16; d; d >>= 1) {
        all->x += __shfl_xor_sync(0xffffffffu, all->x, d);
        all->y += __shfl_xor_sync(0xffffffffu, all->y, d);
    }
    if (lane >= warp) mine = make_longlong2(0, 0);
    base = mine;
#pragma unroll
    for (int d = 16; d; d >>= 1) {
        base.x += __shfl_xor_sync(0xffffffffu, base.x, d);
        base.y += __shfl_xor_sync(0xffffffffu, base.y, d);
    }
    return make_longlong2(base.x + incl.x - v.x, base.y + incl.y - v.y);
}

// False where a call cut into the chunked kernel's units would cost less (kChoice).
template <bool kFew, bool kChoice>
__device__ __forceinline__ bool plan_units(const PagedCall& p, const UnitShape& a, int32_t* offset, longlong2* warp_sum,
                                           unsigned long long* chunked) {
    constexpr int kQueries = kFew ? kFewTokens : kChunkTokens, kShift = kFew ? kFewTileShift : kChunkTileShift;
    constexpr int kCost = kFew ? kFewUnitCost : kChunkUnitCost;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, batch = p.batch;
    unsigned long long as_chunks = 0;  // cost, in the chunked kernel's tiles
    // Rows of sequence b, kept within the call's whatever the device's numbers say.
    auto rows_of = [&](int b, int& row0) {
        row0 = min(max(p.first_query[b], 0), p.rows);
        return max(0, min(p.first_query[b + 1], p.rows) - row0);
    };
    const int per = (batch + kPlanThreads - 1) / kPlanThreads;
    const int b0 = min(batch, tid * per), b1 = min(batch, b0 + per);
    longlong2 sum = make_longlong2(0, 0), all;
    for (int b = b0; b < b1; ++b) {
        int row0;
        sum.x += (rows_of(b, row0) + kQueries - 1) / kQueries;
    }
    int64_t at = scan_exclusive(sum, warp_sum, &all).x;
    for (int b = b0; b < b1; ++b) {
        int row0;
        offset[b] = (int)at;
        at += (rows_of(b, row0) + kQueries - 1) / kQueries;
    }
    const int units = (int)min((int64_t)all.x, (int64_t)a.max_units);
    __syncthreads();
    // A warp a unit: the keys that any of its rows sees.
    for (int u = warp; u < units; u += kPlanThreads / 32) {
        int lo_b = 0, hi_b = batch;
        while (hi_b - lo_b > 1) {
            const int mid = (lo_b + hi_b) >> 1;
            if (offset[mid] <= u) lo_b = mid; else hi_b = mid;
        }
        const int b = lo_b;  // (of sequences that share an offset the last: the one with rows)
        int row0;
        const int rows = rows_of(b, row0), skip = (u - offset[b]) * kQueries;
        const int n = min(kQueries, rows - skip), len = paged_length(p, b);
        const int64_t pos0 = (int64_t)p.seq_lens[b] - rows + skip;
        int lo = 0x7fffffff, hi = 0;
        for (int i = lane; i < n; i += 32) {
            const KeyRange r = paged_range(p, row0 + skip + i, pos0 + i, len);
            if (r.hi > r.lo) {
                lo = min(lo, r.lo);
                hi = max(hi, r.hi);
            }
        }
        lo = __reduce_min_sync(0xffffffffu, lo);
        hi = __reduce_max_sync(0xffffffffu, hi);
        if (lane == 0) {
            Unit x;
            x.b = b;
            x.row0 = row0 + skip;
            x.n = n;
            x.pos0 = (int)pos0;
            x.lo = lo;
            x.hi = hi;
            x.tile0 = hi > 0 ? lo >> kShift : 0;
            x.tiles = hi > 0 ? ((hi + (1 << kShift) - 1) >> kShift) - x.tile0 : 0;
            x.first = x.cell = 0;
            a.to.units[u] = x;
            // A unit of the chunked kernel that begins here sees much what this one does.
            if (kChoice && x.tiles && skip / kChunkTokens * kChunkTokens + kQueries > skip)
                as_chunks += (x.tiles >> (kChunkTileShift - kShift)) + 1 + kChunkUnitCost;
        }
    }
    if (kChoice && lane == 0 && as_chunks) atomicAdd(chunked, as_chunks);
    __syncthreads();
    const int heads = p.c.kv_heads;
    const int uper = (units + kPlanThreads - 1) / kPlanThreads;
    const int u0 = min(units, tid * uper), u1 = min(units, u0 + uper);
    // Shares are cut evenly in cost: a unit's cells are kCost of its own, then one for each tile.
    sum = make_longlong2(0, 0);
    for (int u = u0; u < u1; ++u) {
        const int tiles = a.to.units[u].tiles;
        sum.x += tiles;
        sum.y += tiles ? tiles + kCost : 0;
    }
    longlong2 here = scan_exclusive(sum, warp_sum, &all);
    const int64_t total = all.x * heads, cost = all.y * heads;
    if (kChoice && all.y > kChunkTileCost * (int64_t)*chunked) return false;
    for (int u = u0; u < u1; ++u) {
        const int tiles = a.to.units[u].tiles;
        a.to.units[u].first = here.x;
        a.to.units[u].cell = here.y;
        here.x += tiles;
        here.y += tiles ? tiles + kCost : 0;
    }
    __syncthreads();
    // Shares longer than kCost: each has a tile.
    const int64_t G = min((int64_t)a.ctas, cost / (kCost + 1));
    if (tid <= G) {
        int64_t cut = total;
        if (tid < G) {
            const int64_t c = cost * tid / G;
            int lo = 0, hi = units;  // (of units that share a cell the last: the one with tiles)
            while (hi - lo > 1) {
                const int mid = (lo + hi) >> 1;
                if (a.to.units[mid].cell * heads <= c) lo = mid; else hi = mid;
            }
            const Unit x = a.to.units[lo];
            const int64_t each = x.tiles + kCost, off = c - x.cell * heads, h = off / each, t = off - h * each - kCost;
            a.to.starts[tid] = lo;
            cut = x.first * heads + h * x.tiles + (t > 0 ? t : 0);
        }
        a.to.cuts[tid] = cut;
    }
    const int counters = a.counters ? a.counters : units * heads * 2;
    for (int i = tid; i < counters; i += kPlanThreads) a.to.arrivals[i] = 0;
    if (tid == 0) *a.to.meta = Meta{total, (int32_t)G, units};
    return true;
}

template <bool kFew, bool kChoice>
__global__ void __launch_bounds__(kPlanThreads) plan_units_kernel(const __grid_constant__ PlanUnitsArgs a) {
    extern __shared__ int32_t offset[];  // first unit of each sequence
    __shared__ longlong2 warp_sum[kPlanThreads / 32];
    __shared__ unsigned long long chunked;
    if (kChoice && threadIdx.x == 0) chunked = 0;
    dependency_wait();
    allow_dependents();
    if (kChoice) __syncthreads();
    const bool first = plan_units<kFew, kChoice>(a.p, a.first, offset, warp_sum, &chunked);
    if constexpr (kChoice) {
        if (!first) {
            __syncthreads();
            plan_units<false, false>(a.p, a.other, offset, warp_sum, &chunked);
        }
        if (threadIdx.x == 0) *(first ? a.other.to.meta : a.first.to.meta) = Meta{0, 0, 0};
    }
}

__device__ __forceinline__ void tma_load_page(void* dst, const CUtensorMap* map, int head, int page, uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes "
        "[%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(smem_addr(dst)),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(0), "r"(0), "r"(head), "r"(page), "r"(smem_addr(bar))
        : "memory");
}

// V's operand.  A NaN code would reach, times a weight of zero, the rows that do not
// see its key: the maximum with -448 makes it a number.
template <int kCode>
__device__ __forceinline__ uint32_t numbers(uint32_t a) {
    if constexpr (kCode == GQA_CODE_E4M3) {
        const __half2 v = __hmax2(*reinterpret_cast<const __half2*>(&a), __half2half2(__ushort_as_half(0xdf00)));
        return *reinterpret_cast<const uint32_t*>(&v);
    }
    return a;
}

// tanh(x) / x = sum of kTanh[i] x^2i for |x| <= 1/2, within 2^-15 of it (a quarter of
// what a weight's rounding to FP16 moves at a score of 4): interpolated at the
// Chebyshev points of x^2.
__device__ constexpr float kTanh[3] = {0.99997777f, -0.33170217f, 0.11525216f};

// The larger magnitude of two BF16 codes, as FP32 bits (which order as integers).
__device__ __forceinline__ uint32_t magnitudes(uint32_t w) { return max(w << 16 & 0x7fffffffu, w & 0x7fff0000u); }

// The row of a softmax thread.
struct Row {
    float factor;      // scores of the row: S * page scale * factor, in log2 units (or over the cap)
    float cap2;        // cap * log2(e)
    float slope;       // times log2(e)
    int lo, hi, pos;   // visible keys, position
};

template <int kRegs>
__device__ __forceinline__ void take_registers() {
    if constexpr (kRegs > kLaunchRegs)
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegs));
    else
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegs));
}

template <int kCode, bool kCap, bool kBias>
__global__ void __launch_bounds__(kThreads, 1) paged_chunk_kernel(const __grid_constant__ ChunkPagedArgs a) {
    extern __shared__ uint8_t raw_smem[];
    uint8_t* smem = raw_smem + ((1024u - (smem_addr(raw_smem) & 1023u)) & 1023u);
    uint8_t* q_smem = smem;                                // two M tiles
    uint8_t* conv = q_smem + 2 * kHalfTileBytes;           // kConv slots of FP16
    uint8_t* raw = conv + kConv * kHalfTileBytes;          // kRaw slots of codes
    Shared& s = *reinterpret_cast<Shared*>(raw + kRaw * kRawBytes);
    const PagedCall& p = a.p;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

    if (tid == 0) {
        for (int i = 0; i < kRaw; ++i) {
            mbar_init(&s.raw_full[i], 1);
            mbar_init(&s.raw_empty[i], 4);
        }
        for (int i = 0; i < kConv; ++i) {
            mbar_init(&s.conv_full[i], 4);
            mbar_init(&s.conv_empty[i], 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&s.q_full[i], kRowsM);
            mbar_init(&s.s_full[i], 1);
            mbar_init(&s.p_full[i], kRowsM);
            mbar_init(&s.pv_done[i], 1);
            mbar_init(&s.group[i], kRowsM);
        }
        mbar_init(&s.drain, 1);
        fence_barrier_init();
    }
    dependency_wait();
    allow_dependents();
    const Meta meta = *a.meta;
    if (meta.units == 0) return;  // cut for the few-query kernel, or no rows
    if (tid < kPairs) s.step[tid] = a.rope.step[tid];
    if (tid <= meta.ctas) s.cuts[tid] = a.cuts[tid];
    if (warp == kMmaWarp) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&s.tmem)),
                     "r"(kTmemCols)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
        if (lane == 0) {
            prefetch_tensormap(&a.kmap);
            prefetch_tensormap(&a.vmap);
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = s.tmem;
    Walk walk;
    walk.start(a, meta);
    bool ok = true;

    if (warp < kConvWarp) {
        // ============================ softmax ============================
        take_registers<kSoftmaxRegs>();
        const int m = warp >> 2, r = tid & (kRowsM - 1);  // M tile, row: query 32 m + r / 4, head r % 4
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t t_s = tmem + kColS + m * 128 + lanes, t_o = tmem + kColO + m * 128 + lanes;
        uint8_t* q_tile = q_smem + m * kHalfTileBytes;
        int seen = 0;     // tiles of this M tile so far (phases of s_full)
        int pieces = 0;   // of this M tile (phases of pv_done)
        int syncs = 0;    // phases of group
        int slot = 0;     // scales of the piece's first tile
        int row_unit = -1;
        Row row;
        row.cap2 = p.cap * 1.4426950408889634f;
        auto group_sync = [&] {
            mbar_arrive(&s.group[m]);
            if (ok) ok = warp_wait(&s.group[m], syncs & 1);
            ++syncs;
        };
        while (walk.n > 0) {
            const Unit& un = walk.unit;
            const int token = 32 * m + (r >> 2), head = r & 3;
            const bool active = un.n > 32 * m, real = token < un.n;
            if (active && ok) {
                const int64_t pos = (int64_t)un.pos0 + token;
                if (walk.u != row_unit) {  // (the heads of a unit follow one another)
                    row_unit = walk.u;
                    row.pos = (int)pos;
                    row.lo = 0;
                    row.hi = 0x7fffffff;  // rows of no query: nothing to mask, nothing written
                    if (real) {
                        const KeyRange range = paged_range(p, un.row0 + token, pos, paged_length(p, un.b));
                        row.lo = range.lo;
                        row.hi = range.hi;
                    }
                }
                row.slope = kBias ? p.slopes[walk.h * kGroup + head] * 1.4426950408889634f : 0.f;
                row.factor = 0.f;
                // ---- Q: 16 pairs of this lane's query, 4 heads ----
                {
                    const int q4 = lane & 3;
                    // The scale's sign goes into Q, so that a row's factor is not negative (nor are the pages' scales)
                    // and the largest of 16 products is the largest of their scores.
                    const float unit = fabsf(kCap ? p.scale / p.cap : p.scale * 1.4426950408889634f);
                    const int sign = __float_as_int(p.scale) & (int)0x80000000;
                    const uint4 none = make_uint4(0u, 0u, 0u, 0u);
                    const uint4* q = reinterpret_cast<const uint4*>(
                        p.q + (int64_t)(un.row0 + token) * p.q_row_stride + walk.h * kGroup * p.q_head_stride + 16 * q4);
                    uint4 w[kGroup][4];  // pairs 0-7 and 8-15: first, then second elements
#pragma unroll
                    for (int hq = 0; hq < kGroup; ++hq)
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            w[hq][i] = real ? q[hq * (p.q_head_stride / 8) + (i & 1) + 8 * (i >> 1)] : none;
                    float down[kGroup];
#pragma unroll
                    for (int hq = 0; hq < kGroup; ++hq) {
                        // A power of two above the row's largest: a rotated pair passes it by no more than sqrt(2).
                        uint32_t top = 0;
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            top = max(top, max(max(magnitudes(w[hq][i].x), magnitudes(w[hq][i].y)),
                                               max(magnitudes(w[hq][i].z), magnitudes(w[hq][i].w))));
                        top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
                        top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
                        const int e = min(253, max(1, (int)(top >> 23) + 1));
                        if (hq == head)
                            row.factor = top < 0x7f800000u ? unit * __int_as_float(e << 23) : __int_as_float(0x7fffffff);
                        down[hq] = __int_as_float((254 - e) << 23 | sign);
                    }
#pragma unroll
                    for (int c = 0; c < 2; ++c) {  // 8 pairs: 16 bytes of each block
                        float2 f[8];
#pragma unroll
                        for (int i = 0; i < 8; ++i)
                            f[i] = p.q_rotated ? make_float2(1.f, 0.f) : rope_factor_fast(s.step[16 * q4 + 8 * c + i], pos);
#pragma unroll
                        for (int hq = 0; hq < kGroup; ++hq) {
                            const uint4 u4 = w[hq][c], v4 = w[hq][c + 2];
                            const uint32_t uw[4] = {u4.x, u4.y, u4.z, u4.w}, vw[4] = {v4.x, v4.y, v4.z, v4.w};
                            uint32_t x[4], y[4];
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                const float2 u = bf16x2_to_float2(uw[i]), v = bf16x2_to_float2(vw[i]);
                                const float2 f0 = f[2 * i], f1 = f[2 * i + 1];
                                x[i] = pack_half2((u.x * f0.x - v.x * f0.y) * down[hq], (u.y * f1.x - v.y * f1.y) * down[hq]);
                                y[i] = pack_half2((u.x * f0.y + v.x * f0.x) * down[hq], (u.y * f1.y + v.y * f1.x) * down[hq]);
                            }
                            const int qr = (r & ~3) + hq;  // row of the M tile
                            uint8_t* to = q_tile + qr * 128 + (((2 * q4 + c) ^ (qr & 7)) << 4);
                            *reinterpret_cast<uint4*>(to) = make_uint4(x[0], x[1], x[2], x[3]);
                            *reinterpret_cast<uint4*>(to + kBlockBytes) = make_uint4(y[0], y[1], y[2], y[3]);
                        }
                    }
                    fence_proxy_async_smem();
                    mbar_arrive(&s.q_full[m]);
                }
                float ref = -INFINITY;   // weights for O are 2^(z + log2(V scale) - ref)
                float l = 0.f;           // their sum without that scale, times kWeightUnit
                for (int j = 0; j < walk.n; ++j) {
                    if (!warp_wait(&s.s_full[m], (seen + j) & 1)) {
                        ok = false;
                        break;
                    }
                    tc_fence_after();
                    const TileScales& sc = s.scales[(slot + j) & (kScaleSlots - 1)];
                    const int k0 = (un.tile0 + walk.j + j) << kTileShift;
                    const bool edge = __any_sync(0xffffffffu, row.lo > k0 || row.hi < k0 + kTile);
                    // The row's 128 scores, in the reference's units once kCap or kBias needs them so.
                    float z[kTile];
#pragma unroll
                    for (int c = 0; c < 4; ++c) tmem_ld32(t_s + 32 * c, reinterpret_cast<uint32_t(&)[32]>(z[32 * c]));
                    float f[8];
#pragma unroll
                    for (int i = 0; i < 8; ++i) f[i] = row.factor * sc.k[i];
                    tmem_wait_ld();
                    if constexpr (kCap) {
                        // cap tanh(x) as a polynomial up to |x| = 1/2, on the FMA pipe: the MUFU is busy with the
                        // weights.  A tile with a score past half the cap takes the other way, through TMEM.
                        const float2 c0 = make_float2(kTanh[0] * row.cap2, kTanh[0] * row.cap2),
                                     c1 = make_float2(kTanh[1] * row.cap2, kTanh[1] * row.cap2),
                                     c2 = make_float2(kTanh[2] * row.cap2, kTanh[2] * row.cap2);
                        float most = 0.f;
#pragma unroll
                        for (int e = 0; e < kTile; e += 2) {
                            const float2 x = __fmul2_rn(make_float2(z[e], z[e + 1]), make_float2(f[e >> 4], f[e >> 4]));
                            const float2 t = __fmul2_rn(x, x);
                            most = fmaxf(fmaxf(most, t.x), t.y);
                            const float2 y = __fmul2_rn(x, __ffma2_rn(__ffma2_rn(c2, t, c1), t, c0));
                            z[e] = y.x;
                            z[e + 1] = y.y;
                        }
                        if (__any_sync(0xffffffffu, most > kTanhNear)) {
#pragma unroll 1
                            for (int i = 0; i < 8; ++i) {
                                uint32_t v[16];
                                tmem_ld16(t_s + 16 * i, v);
                                const float g = row.factor * sc.k[i];
                                tmem_wait_ld();
#pragma unroll
                                for (int e = 0; e < 16; ++e) {
                                    const float x = __uint_as_float(v[e]) * g, t = x * x;
                                    v[e] = __float_as_uint(row.cap2 * (t > kTanhNear ? tanh_far(x) : tanh_near(x, t)));
                                }
                                tmem_st16(t_s + 16 * i, v);
                            }
                            tmem_wait_st();
#pragma unroll
                            for (int c = 0; c < 4; ++c)
                                tmem_ld32(t_s + 32 * c, reinterpret_cast<uint32_t(&)[32]>(z[32 * c]));
                            tmem_wait_ld();
                        }
                    }
                    if constexpr (kBias) {
                        const float ahead = (float)(k0 - row.pos);
#pragma unroll
                        for (int e = 0; e < kTile; ++e) {
                            if constexpr (!kCap) z[e] *= f[e >> 4];
                            z[e] = fmaf(-row.slope, fabsf(ahead + (float)e), z[e]);
                        }
                    }
                    if (edge) {
                        if constexpr (!kCap && !kBias) {  // scaled before the mask: -inf times a scale of 0 is none
#pragma unroll
                            for (int e = 0; e < kTile; ++e) z[e] *= f[e >> 4];
#pragma unroll
                            for (int i = 0; i < 8; ++i) f[i] = 1.f;
                        }
                        // Visible keys of the tile as bits: from row.lo - k0 on, below row.hi - k0.
#pragma unroll
                        for (int c = 0; c < 4; ++c) {
                            const int from = min(32, max(0, row.lo - k0 - 32 * c)), to = min(32, max(0, row.hi - k0 - 32 * c));
                            const uint32_t seen_bits = __funnelshift_lc(0xffffffffu, 0u, to) & ~__funnelshift_lc(0xffffffffu, 0u, from);
#pragma unroll
                            for (int e = 0; e < 32; ++e)
                                if (!(seen_bits & (1u << e))) z[32 * c + e] = -INFINITY;
                        }
                    }
                    float mx = -INFINITY;
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        // The largest of 16 keys, then their factor: it is not negative.
                        float top = fmaxf(z[16 * i], z[16 * i + 1]);
#pragma unroll
                        for (int e = 2; e < 16; e += 2) top = fmaxf(fmaxf(top, z[16 * i + e]), z[16 * i + e + 1]);
                        mx = fmaxf(mx, kCap || kBias ? top + sc.v_log2[i] : fmaf(top, f[i], sc.v_log2[i]));
                    }
                    // The reference moves when the maximum passes it by 2^kHeadroom (at once from nothing).
                    const float want = mx - kLift;
                    const bool move = want > ref + kHeadroom || (ref == -INFINITY && want > ref);
                    const float to = move ? want : ref;
                    if (__any_sync(0xffffffffu, move)) {
                        const float alpha = move ? fast_exp2(ref - to) : 1.f;
                        l *= alpha;
                        ref = to;
                        if (j > 0) {
#pragma unroll 1
                            for (int c = 0; c < 4; ++c) {
                                uint32_t o[32];
                                tmem_ld32(t_o + 32 * c, o);
                                tmem_wait_ld();
#pragma unroll
                                for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
                                tmem_st32(t_o + 32 * c, o);
                            }
                        }
                    }
                    const float use = ref == -INFINITY ? 0.f : ref;
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        uint32_t w[16];
#pragma unroll
                        for (int half = 0; half < 2; ++half) {  // 16 keys of one page
                            const int i = 2 * c + half;
                            const float off = sc.v_log2[i] - use;
                            float2 sum = make_float2(0.f, 0.f);
#pragma unroll
                            for (int e = 0; e < 16; e += 2) {
                                float2 x = make_float2(z[16 * i + e], z[16 * i + e + 1]);
                                if constexpr (kCap || kBias)
                                    x = __fadd2_rn(x, make_float2(off, off));
                                else
                                    x = __ffma2_rn(x, make_float2(f[i], f[i]), make_float2(off, off));
                                x = make_float2(fast_exp2(x.x), fast_exp2(x.y));
                                sum = __fadd2_rn(sum, x);
                                w[8 * half + (e >> 1)] = pack_half2(x.x, x.y);
                            }
                            l = fmaf(sum.x + sum.y, sc.v_inv[i], l);
                        }
                        tmem_st16(t_s + 16 * c, w);  // over columns that were read
                    }
                    tmem_wait_st();
                    tc_fence_before();
                    mbar_arrive(&s.p_full[m]);
                }
                // ---- the piece's rows ----
                if (ok) ok = warp_wait(&s.pv_done[m], pieces & 1);
                tc_fence_after();
                __nv_bfloat16* out = p.out + (int64_t)(un.row0 + token) * p.out_row_stride +
                                     (walk.h * kGroup + head) * p.out_head_stride;
                auto write = [&](int c, const float (&x)[32]) {
#pragma unroll
                    for (int e = 0; e < 32; e += 8) {
                        uint4 w;
                        uint32_t* wp = &w.x;
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const __nv_bfloat162 v = __floats2bfloat162_rn(x[e + 2 * i], x[e + 2 * i + 1]);
                            wp[i] = *reinterpret_cast<const uint32_t*>(&v);
                        }
                        *reinterpret_cast<uint4*>(out + 32 * c + e) = w;
                    }
                };
                if (walk.n == un.tiles) {
                    const float f = l == 0.f ? 0.f : kWeightUnit / l;  // a row that sees nothing is 0
                    float x[kHeadDim];
#pragma unroll
                    for (int c = 0; c < 4; ++c) tmem_ld32(t_o + 32 * c, reinterpret_cast<uint32_t(&)[32]>(x[32 * c]));
                    tmem_wait_ld();
#pragma unroll
                    for (int e = 0; e < kHeadDim; ++e) x[e] *= f;
                    if (real)
#pragma unroll
                        for (int c = 0; c < 4; ++c) write(c, reinterpret_cast<const float(&)[32]>(x[32 * c]));
                } else {
                    // A piece of a unit: its slots as in decode_paged (a share's first piece 0, its last 1).
                    const int64_t first = walk.unit_first(a);
                    auto share_of = [&](int64_t tile) {  // the last cut at or before it
                        int lo = 0, hi = meta.ctas;
                        while (hi - lo > 1) {
                            const int mid = (lo + hi) >> 1;
                            if (s.cuts[mid] <= tile) lo = mid; else hi = mid;
                        }
                        return lo;
                    };
                    const int c0 = share_of(first), parts = share_of(first + un.tiles - 1) - c0 + 1;
                    const int second = s.cuts[c0] < first ? 1 : 0;
                    auto part = [&](int c) {
                        return a.partials + (int64_t)((c0 + c) * 2 + (c ? 0 : second)) * kSlotFloats;
                    };
                    const int prow = m * kRowsM + r;
                    {
                        float* mine = part((int)blockIdx.x - c0);
                        float x[kHeadDim];
#pragma unroll
                        for (int c = 0; c < 4; ++c) tmem_ld32(t_o + 32 * c, reinterpret_cast<uint32_t(&)[32]>(x[32 * c]));
                        tmem_wait_ld();
                        if (real)
#pragma unroll
                            for (int e = 0; e < kHeadDim / 4; ++e)
                                reinterpret_cast<float4*>(mine)[e * 2 * kRowsM + prow] =
                                    make_float4(x[4 * e], x[4 * e + 1], x[4 * e + 2], x[4 * e + 3]);
                        if (real)
                            reinterpret_cast<float2*>(mine + 2 * kRowsM * kHeadDim)[prow] = make_float2(ref, l);
                    }
                    group_sync();
                    if (r == 0) {
                        uint32_t* count = a.arrivals + ((int64_t)walk.u * p.c.kv_heads + walk.h) * 2 + m;
                        uint32_t before;
                        asm volatile("atom.add.acq_rel.gpu.global.u32 %0, [%1], 1;"
                                     : "=r"(before)
                                     : "l"(count)
                                     : "memory");
                        s.last[m] = before == (uint32_t)(parts - 1);
                    }
                    group_sync();
                    if (ok && s.last[m] && real) {
                        // The first few parts' (m, l) stay in registers; 16 loads of a row in flight.
                        constexpr int kKept = 4;
                        auto ml = [&](int c) {
                            return __ldcg(reinterpret_cast<const float2*>(part(c) + 2 * kRowsM * kHeadDim) + prow);
                        };
                        float2 kept[kKept];
#pragma unroll
                        for (int i = 0; i < kKept; ++i) kept[i] = i < parts ? ml(i) : make_float2(-INFINITY, 0.f);
                        float M = fmaxf(fmaxf(kept[0].x, kept[1].x), fmaxf(kept[2].x, kept[3].x)), L = 0.f;
                        for (int c = kKept; c < parts; ++c) M = fmaxf(M, ml(c).x);
                        const float mu = M == -INFINITY ? 0.f : M;
#pragma unroll
                        for (int i = 0; i < kKept; ++i) {
                            kept[i].x = fast_exp2(kept[i].x - mu);
                            L = fmaf(kept[i].x, kept[i].y, L);
                        }
                        for (int c = kKept; c < parts; ++c) {
                            const float2 v = ml(c);
                            L = fmaf(fast_exp2(v.x - mu), v.y, L);
                        }
                        const float inv = L == 0.f ? 0.f : kWeightUnit / L;
#pragma unroll 1
                        for (int half = 0; half < 2; ++half) {
                            float x[64];
#pragma unroll
                            for (int e = 0; e < 64; ++e) x[e] = 0.f;
#pragma unroll 1
                            for (int c = 0; c < parts; ++c) {
                                const float4* at = reinterpret_cast<const float4*>(part(c)) + half * 16 * 2 * kRowsM + prow;
                                float4 v[16];
#pragma unroll
                                for (int e = 0; e < 16; ++e) v[e] = __ldcg(at + e * 2 * kRowsM);
                                const float f = inv * (c == 0 ? kept[0].x : c == 1 ? kept[1].x : c == 2 ? kept[2].x
                                                       : c == 3 ? kept[3].x : fast_exp2(ml(c).x - mu));
#pragma unroll
                                for (int e = 0; e < 16; ++e) {
                                    x[4 * e] = fmaf(f, v[e].x, x[4 * e]);
                                    x[4 * e + 1] = fmaf(f, v[e].y, x[4 * e + 1]);
                                    x[4 * e + 2] = fmaf(f, v[e].z, x[4 * e + 2]);
                                    x[4 * e + 3] = fmaf(f, v[e].w, x[4 * e + 3]);
                                }
                            }
                            write(2 * half, reinterpret_cast<const float(&)[32]>(x[0]));
                            write(2 * half + 1, reinterpret_cast<const float(&)[32]>(x[32]));
                        }
                    }
                }
                tc_fence_before();  // the next unit's products overwrite O after this thread's next arrival
                seen += walk.n;
                ++pieces;
            }
            slot = (slot + walk.n) & (kScaleSlots - 1);
            if (!ok || !walk.next(a)) break;
        }
    } else if (warp < kMmaWarp) {
        // ============================ conversion ============================
        take_registers<kConvRegs>();
        const int cw = warp - kConvWarp, t = lane & 3;
        // This lane's rows: row0 + 8 i.  Eight lanes that access shared memory together take chunks 0-3
        // of two rows whose numbers differ in bits 0 and 2: with the swizzle, all eight 16-byte columns
        // of the codes' rows and of the operand's.
        const int row0 = 32 * cw + ((lane >> 3) ^ (lane & 4 ? 5 : 0));
        int item = 0;  // K and V of the tiles in turn
        int rs = 0, rphase = 0, cs = 0, cphase = 0, tile_count = 0;
        while (walk.n > 0 && ok) {
            for (int j = 0; j < walk.n && ok; ++j, ++tile_count) {
                const TileScales& sc = s.scales[tile_count & (kScaleSlots - 1)];
                const int k0 = (walk.unit.tile0 + walk.j + j) << kTileShift;
                const int klo = walk.unit.lo - k0, khi = walk.unit.hi - k0;
#pragma unroll 1
                for (int kv = 0; kv < 2; ++kv, ++item) {
                    ok = mbar_wait(&s.raw_full[rs], rphase) && (item < kConv || mbar_wait(&s.conv_empty[cs], cphase ^ 1));
                    ok = __all_sync(0xffffffffu, ok);
                    if (!ok) break;
                    const uint8_t* src = raw + rs * kRawBytes;
                    uint8_t* dst = conv + cs * kHalfTileBytes;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int row = row0 + 8 * i, sw = row & 7;
                        // Where no row sees the key, its codes may be anything.
                        const bool gone = kv && (row < klo || row >= khi || !(sc.v_some >> (2 * cw + (i >> 1)) & 1));
#pragma unroll
                        for (int half = 0; half < 2; ++half) {
                            const int c = 4 * half + t;  // dims 16 c .. 16 c + 15: block `half`
                            const uint4 x = lds128(src + row * kHeadDim + ((c ^ sw) << 4));
                            uint32_t w[8];
                            to_half4<kCode>(x.x, w[0], w[1]);
                            to_half4<kCode>(x.y, w[2], w[3]);
                            to_half4<kCode>(x.z, w[4], w[5]);
                            to_half4<kCode>(x.w, w[6], w[7]);
                            if (kv) {
#pragma unroll
                                for (int e = 0; e < 8; ++e) w[e] = gone ? 0u : numbers<kCode>(w[e]);
                            }
                            uint8_t* at = dst + half * kBlockBytes + row * 128;
                            *reinterpret_cast<uint4*>(at + (((2 * t) ^ sw) << 4)) = make_uint4(w[0], w[1], w[2], w[3]);
                            *reinterpret_cast<uint4*>(at + (((2 * t + 1) ^ sw) << 4)) =
                                make_uint4(w[4], w[5], w[6], w[7]);
                        }
                    }
                    fence_proxy_async_smem();
                    __syncwarp();
                    if (lane == 0) {
                        mbar_arrive(&s.conv_full[cs]);
                        mbar_arrive(&s.raw_empty[rs]);
                    }
                    if (++rs == kRaw) {
                        rs = 0;
                        rphase ^= 1;
                    }
                    if (++cs == kConv) {
                        cs = 0;
                        cphase ^= 1;
                    }
                }
            }
            if (!ok || !walk.next(a)) break;
        }
    } else {
    take_registers<kRestRegs>();
    if (warp == kMmaWarp) {
        // ============================ MMA issuer ============================
        {
            const uint32_t leader = elect_lane();  // (the waits and the walk are the whole warp's)
            int cs = 0, cphase = 0;   // next slot of FP16
            int seen[2] = {0, 0}, pieces[2] = {0, 0};
            auto advance = [&] {
                if (++cs == kConv) {
                    cs = 0;
                    cphase ^= 1;
                }
            };
            const uint32_t cols = uniform(tmem);
            auto issue_s = [&](int m, int slot) {
                const uint64_t kd = smem_desc_sw128(smem_addr(conv + slot * kHalfTileBytes), 16, 1024);
                const uint64_t qd = smem_desc_sw128(smem_addr(q_smem + m * kHalfTileBytes), 16, 1024);
#pragma unroll
                for (int kk = 0; kk < 8; ++kk) {
                    const uint32_t off = ((kk >> 2) * kBlockBytes + (kk & 3) * 32) >> 4;  // (in units of 16 bytes)
                    mma_ss_by(leader, cols + kColS + m * 128, qd + off, kd + off, kIdescS, kk != 0);
                }
                tc_commit_by(leader, &s.s_full[m]);
            };
            while (uniform(walk.n) > 0 && ok) {
                const int ms = uniform(walk.unit.n) > 32 ? 2 : 1, n = uniform(walk.n);
                // S of the first tile.
                ok = warp_wait(&s.conv_full[cs], cphase);
                for (int m = 0; m < ms && ok; ++m) {
                    ok = warp_wait(&s.q_full[m], pieces[m] & 1);
                    if (!ok) break;
                    tc_fence_after();
                    issue_s(m, cs);
                }
                if (!ok) break;
                tc_commit_by(leader, &s.conv_empty[cs]);
                advance();
                for (int j = 0; j < n && ok; ++j) {
                    const int vs = cs, vphase = cphase;
                    advance();
                    const bool more = j + 1 < n;
                    const int ks = cs, kphase = cphase;
                    for (int m = 0; m < ms; ++m) {
                        ok = warp_wait(&s.p_full[m], seen[m] & 1) && (m || warp_wait(&s.conv_full[vs], vphase));
                        if (!ok) break;
                        ++seen[m];
                        tc_fence_after();
                        const uint64_t vd = smem_desc_sw128(smem_addr(conv + vs * kHalfTileBytes), kBlockBytes, 1024);
#pragma unroll
                        for (int kk = 0; kk < 8; ++kk)
                            mma_ts_by(leader, cols + kColO + m * 128, cols + kColS + m * 128 + 8 * kk, vd + kk * (16 * 128 >> 4),
                                   kIdescO, (j > 0 || kk > 0) ? 1u : 0u);
                        if (m == ms - 1) tc_commit_by(leader, &s.conv_empty[vs]);
                        if (more) {
                            if (m == 0) ok = warp_wait(&s.conv_full[ks], kphase);
                            if (!ok) break;
                            tc_fence_after();
                            issue_s(m, ks);
                            if (m == ms - 1) tc_commit_by(leader, &s.conv_empty[ks]);
                        } else {
                            tc_commit_by(leader, &s.pv_done[m]);
                        }
                    }
                    if (more) advance();
                }
                for (int m = 0; m < ms; ++m) ++pieces[m];
                if (!ok || !uniform(walk.next(a))) break;
            }
            if (!ok) {  // shared memory and TMEM are given back with no product under way
                tc_commit_by(leader, &s.drain);
                warp_wait(&s.drain, 0);
            }
        }
    } else if (warp == kLoadWarp) {
        // ============================ loader ============================
        const int shift = p.c.page_shift, per_tile = kTile >> shift;  // pages of a tile
        const int box_bytes = p.c.page_len * kHeadDim;
        int rs = 0, rphase = 0, tile_count = 0, item = 0;
        while (walk.n > 0 && ok) {
            const int32_t* table = p.block_table + walk.unit.b * p.table_stride;
            const int64_t lo = walk.unit.lo, hi = walk.unit.hi;
            // Lane's page of tile j (-1: no visible key, not loaded).
            auto entry = [&](int j) {
                const int64_t key = ((int64_t)(walk.unit.tile0 + walk.j + j) << kTileShift) + ((int64_t)lane << shift);
                if (lane >= per_tile || j >= walk.n || key >= hi || key + p.c.page_len <= lo) return -1;
                const int page = table[key >> shift];
                return page >= 0 && page < p.c.pages ? page : p.c.pages;  // out of the map: TMA fills zeros
            };
            auto scale = [&](const float* at, int page) {
                return page >= 0 && page < p.c.pages ? at[page * p.c.scale_page_stride + walk.h] : 0.f;
            };
            int page = entry(0), page1 = entry(1);
            float ks = scale(p.c.k_scale, page), vs = scale(p.c.v_scale, page);
            for (int j = 0; j < walk.n; ++j, ++tile_count) {
                const int page2 = entry(j + 2);
                const float ks1 = scale(p.c.k_scale, page1), vs1 = scale(p.c.v_scale, page1);
                const uint32_t boxes = __popc(__ballot_sync(0xffffffffu, page >= 0));
                for (int kv = 0; kv < 2; ++kv, ++item) {
                    if (item >= kRaw) ok = __all_sync(0xffffffffu, mbar_wait(&s.raw_empty[rs], rphase ^ 1));
                    if (!ok) break;
                    if (kv == 0) {
                        // Scales of the tile, a lane 16 keys.
                        const int from = (lane & 7) >> (shift - 4);
                        const float kg = __shfl_sync(0xffffffffu, ks, from), vg = __shfl_sync(0xffffffffu, vs, from);
                        const bool fine = fabsf(vg) <= 3.402823466e38f;
                        const VLog2 v = v_log2_of(vg);
                        const uint32_t some = __ballot_sync(0xffffffffu, lane < 8 && v.some);
                        TileScales& sc = s.scales[tile_count & (kScaleSlots - 1)];
                        if (lane == 0) sc.v_some = some;
                        if (lane < 8) {
                            sc.k[lane] = fine ? kg : __int_as_float(0x7fffffff);
                            sc.v_log2[lane] = v.log2;
                            sc.v_inv[lane] = v.inv;
                        }
                        __syncwarp();
                    }
                    if (lane == 0) mbar_arrive_expect_tx(&s.raw_full[rs], boxes * box_bytes);
                    __syncwarp();
                    if (page >= 0)
                        tma_load_page(raw + rs * kRawBytes + lane * box_bytes, kv ? &a.vmap : &a.kmap, walk.h, page,
                                      &s.raw_full[rs]);
                    if (++rs == kRaw) {
                        rs = 0;
                        rphase ^= 1;
                    }
                }
                if (!ok) break;
                page = page1;
                page1 = page2;
                ks = ks1;
                vs = vs1;
            }
            if (!ok || !walk.next(a)) break;
        }
        if (!ok)  // do not leave while copies into this CTA's shared memory are in flight
            for (int i = 1; i <= kRaw && i <= item; ++i) {
                const int at = rs - i;
                mbar_wait(&s.raw_full[at < 0 ? at + kRaw : at], at < 0 ? rphase ^ 1 : rphase);
            }
    } else if (warp == kLoadWarp + 1) {
        // ============================ rows that see nothing ============================
        for (int u = blockIdx.x; u < meta.units; u += gridDim.x) {
            const Unit un = a.units[u];
            if (un.tiles > 0) continue;
            const int per_row = p.c.kv_heads * kGroup;
            for (int i = 0; i < un.n * per_row; ++i)
                *reinterpret_cast<uint2*>(p.out + (int64_t)(un.row0 + i / per_row) * p.out_row_stride +
                                          (i % per_row) * p.out_head_stride + 4 * lane) = make_uint2(0u, 0u);
        }
    }
    }
    if (!ok && lane == 0) atomicOr(a.status, kDevStatusTimeout);

    tc_fence_before();
    __syncthreads();
    if (warp == kMmaWarp) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols) : "memory");
    }
}

constexpr int kSmemBytes =
    1024 + 2 * kHalfTileBytes + kConv * kHalfTileBytes + kRaw * kRawBytes + (int)sizeof(Shared);
static_assert(kSmemBytes <= 227 * 1024, "shared memory of one CTA");

using Kernel = void (*)(ChunkPagedArgs);

Kernel kernel_for(int code, bool cap, bool bias) {
    if (code == GQA_CODE_INT8) {
        if (cap) return bias ? paged_chunk_kernel<0, true, true> : paged_chunk_kernel<0, true, false>;
        return bias ? paged_chunk_kernel<0, false, true> : paged_chunk_kernel<0, false, false>;
    }
    if (cap) return bias ? paged_chunk_kernel<1, true, true> : paged_chunk_kernel<1, true, false>;
    return bias ? paged_chunk_kernel<1, false, true> : paged_chunk_kernel<1, false, false>;
}

UnitRegions regions(int batch, int rows, int heads, int sms) {
    const size_t units = (size_t)rows / kTokens + batch;
    return unit_regions(kPagedPartialsOffset, batch, rows, kTokens, units * heads * 2, sms,
                        (size_t)sms * 2 * kSlotFloats * sizeof(float));
}

}  // namespace

cudaError_t launch_plan_units(const PagedCall& call, const UnitShape& first, const UnitShape* other, cudaStream_t stream) {
    const PlanUnitsArgs a{call, first, other ? *other : first};
    const auto kernel = other       ? plan_units_kernel<true, true>
                        : first.few ? plan_units_kernel<true, false>
                                    : plan_units_kernel<false, false>;
    return launch_dependent(kernel, 1, kPlanThreads, call.batch * sizeof(int32_t), stream, a);
}

int paged_chunk_tile() { return kTile; }

size_t paged_chunk_workspace(int batch, int rows, int heads, int sms) { return regions(batch, rows, heads, sms).end; }

cudaError_t paged_chunk_prepare() {
    for (int i = 0; i < 8; ++i) {
        // The register shares are of kLaunchRegs a thread: with fewer at launch the kernel would wait for good.
        cudaFuncAttributes at;
        cudaError_t e = cudaFuncGetAttributes(&at, kernel_for(i & 1, i & 2, i & 4));
        if (e != cudaSuccess) return e;
        if (at.numRegs != kLaunchRegs) return cudaErrorInvalidConfiguration;
        e = cudaFuncSetAttribute(kernel_for(i & 1, i & 2, i & 4),
                                                   cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemBytes);
        if (e != cudaSuccess) return e;
    }
    return cudaSuccess;
}

UnitShape paged_chunk_shape(const PagedCall& call, int sms, uint8_t* ws) {
    return unit_shape(regions(call.batch, call.rows, call.c.kv_heads, sms), ws, call.rows / kTokens + call.batch,
                      sms < kMaxCtas ? sms : kMaxCtas, 0, false);
}

cudaError_t launch_paged_chunk(const PagedCall& call, const RopeSteps& rope, int code, const CUtensorMap& kmap,
                               const CUtensorMap& vmap, const UnitShape& shape, uint32_t* status, cudaStream_t stream) {
    const UnitPlan& pl = shape.to;
    const ChunkPagedArgs a{kmap, vmap, call, rope, status, pl.meta, pl.units, pl.starts, pl.cuts, pl.arrivals,
                           shape.partials};
    return launch_dependent(kernel_for(code, call.cap > 0.f, call.slopes != nullptr), shape.ctas, kThreads, kSmemBytes,
                            stream, a);
}

}  // namespace gqa
