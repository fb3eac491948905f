// gqa_paged_decode.cu -- one token a sequence over the paged 8-bit cache.
//
//   out[h] = sum_p softmax_p(z)[p] V[p],  z[p] = scale * (Q[h] . K[p]) * k_scale[page of p],
// capped, biased and masked as gqa_b200.h says, in one pass over the visible keys
// with a running maximum and sum a warp.
//
// Work.  A unit is one (sequence, KV head); its visible keys are cut into tiles
// of 32 on a grid of absolute positions.  All tiles of all units, in order, are
// dealt out evenly: CTA i of G (one per SM) takes tiles [T i / G, T (i + 1) / G),
// whatever the lengths -- which only the GPU knows, so every CTA first sums the
// sequences' tiles itself.  A unit inside one CTA's share is written out by it; a
// unit that crosses shares leaves FP32 partial rows (at most two per CTA), and
// the last of its CTAs to finish merges them in CTA order, so that results do not
// depend on which one that is.
//
// A CTA is 8 consumer warps, 2 loader warps, a query warp and 4 finisher warps.
//   loader   four tiles at a time, every second four each: the block-table
//            entries and scales of their pages (two pages a tile at most), then
//            a TMA box per page of K and of V (32 rows of 128 codes in all,
//            128-byte swizzle) into a ring of 8 KB stages, 24 deep, and the
//            pages' scales beside them.  Pages with no visible key are not
//            loaded.  A stage belongs to one loader and one consumer warp, so
//            that no one waits for a phase that another has passed.
//   query    per unit, the 4 Q rows rotated in FP32, divided by a power of two
//            that brings the row's largest below 1, and split into two FP16
//            parts (22 bits): 8 columns, the N of an m16n8k16 product.
//   consumer takes whole tiles, the ring's every 8th.  The M of its products is
//            the keys: S^T = K Q^T, 16 keys x (4 heads x {high, low}), 8 products
//            deep; codes become FP16 exactly, so a score carries FP32's error
//            only.  Softmax runs in the result's layout (lane: 2 keys of one
//            head) without a shuffle but for the maximum.  The weights, times
//            their page's V scale (its power of two joins the score, against the
//            row's largest such sum), split into two FP16 parts again, and movmatrix turns them into the other product's
//            operand: O^T = V^T P^T, M 16 dims, whose operand lanes build from
//            the 16-byte pieces of 4 keys by byte permutes.
//   finisher one a Q head: joins the consumers' rows of a unit and writes it, or
//            its partial, while the consumers are at the next unit.
// Why mma.sync and not tcgen05: with 4 queries a KV head there is nothing to
// amortise a 16-bit copy of K and V in shared memory over; here a code goes from
// its 8-bit stage through registers into the product once.
//
// Bound by HBM for long contexts, by the chain length -> table entry -> page ->
// product -> merge for short ones.  Measured (B200, in a replayed graph): 64 ragged
// sequences, 586 MB, e4m3 98 us (6.0 TB/s, 91 % of the copy rate; 104 us as a call),
// int8 103; 148 of 4096 keys 190 us (6.5 TB/s); one of 131072 keys 50 us (5.4 TB/s),
// of 4096 11.5 us, of 30 5.1 us.  32 sequences read 294.8 MB of DRAM, the codes and no
// more, at 17 % of the tensor pipe and 45 % of the issue slots.  Tiles of 64 keys, half as
// many, left the ring too coarse for the short shares (one of 131072: 53 us); one
// loader warp needed 700 cycles a tile, more than the consumers; 10 to 13 consumer
// warps do not fit the registers.
#include "gqa_internal.h"
#include "gqa_paged.cuh"
#include "gqa_paged_internal.h"

#include <cstring>

namespace gqa {

namespace {

constexpr int kWarps = 8;                      // consumer warps
constexpr int kBurst = 4;                      // tiles that the loader handles at once
constexpr int kFinishers = kGroup;              // finisher warps, one a Q head
constexpr int kLoaders = 2;                    // loader warps
constexpr int kLoaderWarp = kWarps, kQueryWarp = kLoaderWarp + kLoaders, kFinishWarp = kQueryWarp + 1;
constexpr int kThreads = (kFinishWarp + kFinishers) * 32;
constexpr int kTile = 32;                      // keys
constexpr int kTileShift = 5;
constexpr int kSteps = kTile / 16;             // of 16 keys
constexpr int kHalfBytes = kTile * kHeadDim;   // K or V of a tile
constexpr int kStageBytes = 2 * kHalfBytes;
constexpr int kMaxStages = 3 * kWarps;
constexpr int kPagesPerTile = kTile / kPagedMinPage;
static_assert(kSteps == 2 && kPagesPerTile == 2, "scales of two pages a tile");
constexpr float kLift = 12.f;                  // weights up to 2^13: FP16's subnormal step, 2^-24, is 2^-36 of the largest

// Shared memory behind the ring (bytes).
constexpr int kRowF = kHeadDim + 4;  // padded partial row
struct alignas(16) Slot {            // one unit's queries (two slots)
    __half q[2 * kGroup][kHeadDim];  // row 2 head: high parts, 2 head + 1: low parts
    float factor[kGroup];            // scale * log2(e) (or / cap) * the row's power of two
    float slope[kGroup];             // times log2(e)
    int lo, hi, m, pad;
};
struct alignas(16) Shared {
    uint64_t full[kMaxStages], empty[kMaxStages], qfull[2], qempty[2], rfull, rempty;
    Slot slot[2];
    float4 scales[kMaxStages];  // K of the tile's two pages (NaN where V's is no number), V's exponents
    float4 v_rest[kMaxStages];  // V's fractions and inverses, as VScale has them
    struct {  // what the consumer warps make of a piece
        float acc[kWarps][kGroup][kRowF];
        float m[kWarps][kGroup], l[kWarps][kGroup];
    } result;
    int sum[kThreads / 32];
};

struct alignas(64) DecodePagedArgs {
    CUtensorMap kmap, vmap;  // (128, page_len, heads, pages) bytes, box (128, min(page_len, 32), 1, 1)
    PagedCall p;
    RopeSteps rope;
    uint32_t* status;
    uint32_t* arrivals;  // [batch * Q heads], zero between calls
    float* partials;     // [grid][2][4][132]
    int stages;
};

// The sequences' visible keys, lo[b] <= p < hi[b], and the running sum of their
// tiles (per head), in shared memory.
struct TileIndex {
    const int *first, *lo, *hi;
    int batch, heads;
};

// A CTA's walk through its share of the tiles, one unit's piece at a time.
struct Walk {
    int64_t x, end;      // next tile, end of the share
    int b, h;            // unit
    int tile, n;         // absolute first tile and tiles of the piece
    int64_t unit_first;  // the unit's first tile in the whole order
    int unit_tiles;
    __device__ __forceinline__ void start(const TileIndex& t, int64_t x0, int64_t x1) {
        x = x0;
        end = x1;
        n = 0;
        if (x >= end) return;
        int lo = 0, hi = t.batch;
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if ((int64_t)t.first[mid] * t.heads <= x) lo = mid; else hi = mid;
        }
        b = lo;
        unit_tiles = t.first[b + 1] - t.first[b];
        const int64_t rem = x - (int64_t)t.first[b] * t.heads;
        h = (int)(rem / unit_tiles);
        place(t);
    }
    __device__ __forceinline__ void place(const TileIndex& t) {
        unit_first = (int64_t)t.first[b] * t.heads + (int64_t)h * unit_tiles;
        const int j = (int)(x - unit_first);
        tile = (t.lo[b] >> kTileShift) + j;
        n = (int)min((int64_t)(unit_tiles - j), end - x);
    }
    // To the next piece; false at the share's end.
    __device__ __forceinline__ bool next(const TileIndex& t) {
        x += n;
        if (x >= end) return false;
        if (++h == t.heads) {
            h = 0;
            do ++b;
            while (t.first[b + 1] == t.first[b]);
            unit_tiles = t.first[b + 1] - t.first[b];
        }
        place(t);
        return true;
    }
};

// Running state of a consumer warp for the current unit.  Lane (g, t) = (lane / 4,
// lane % 4): head t's maximum of z + V's exponent, the sum of weights (over this
// lane's keys only, without V's scale, times kWeightUnit), and O for head t, dims 16 g
// + 2 i (o[i][0] high parts, [1] low) and + 1 ([2], [3]).
struct State {
    float o[8][4];
    float m, l;
};

template <int kCode, bool kCap, bool kBias>
__device__ __forceinline__ void consume_tile(State& st, const uint8_t* stage, const float4& scales,
                                             const float4& v_rest, const uint32_t (&qf)[16], float factor, float slope, float cap2,
                                             int key0, int lo, int hi, int m_pos, int page_shift, int lane) {
    const int g = lane >> 2, t = lane & 3;
    // Step i (16 keys) lies in page i >> sh of the tile.
    const int sh = min(page_shift, kTileShift) - 4;
    const float4 sc = scales;
    float z[kSteps][2];
    {
        const uint8_t* k = stage + g * kHeadDim;
        const int c0 = ((2 * t) ^ g) << 4, c1 = ((2 * t + 1) ^ g) << 4;
#pragma unroll
        for (int i = 0; i < kSteps; ++i) {
            float s[4] = {0.f, 0.f, 0.f, 0.f};
            const uint4 a = lds128(k + (16 * i) * kHeadDim + c0), b = lds128(k + (16 * i + 8) * kHeadDim + c0);
            const uint4 c = lds128(k + (16 * i) * kHeadDim + c1), d = lds128(k + (16 * i + 8) * kHeadDim + c1);
            const uint32_t up[8] = {a.x, a.y, a.z, a.w, c.x, c.y, c.z, c.w};
            const uint32_t dn[8] = {b.x, b.y, b.z, b.w, d.x, d.y, d.z, d.w};
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                uint32_t a0, a1, a2, a3;
                to_half4<kCode>(up[e], a0, a2);
                to_half4<kCode>(dn[e], a1, a3);
                mma_16x8x16(s, a0, a1, a2, a3, qf[2 * e], qf[2 * e + 1]);
            }
            const float f = factor * (i >> sh ? sc.y : sc.x);
            const float ve = kCap ? 0.f : i >> sh ? sc.w : sc.z;
            z[i][0] = fmaf(s[0] + s[1], f, ve);
            z[i][1] = fmaf(s[2] + s[3], f, ve);
        }
    }
    if constexpr (kCap) {
        cap_scores(reinterpret_cast<float(&)[2 * kSteps]>(z), cap2);
#pragma unroll
        for (int i = 0; i < kSteps; ++i)
#pragma unroll
            for (int e = 0; e < 2; ++e) z[i][e] += i >> sh ? sc.w : sc.z;
    }
    if constexpr (kBias) {
#pragma unroll
        for (int i = 0; i < kSteps; ++i)
#pragma unroll
            for (int e = 0; e < 2; ++e)
                z[i][e] = fmaf(-slope, fabsf((float)(m_pos - (key0 + 16 * i + 8 * e + g))), z[i][e]);
    }
    const bool edge = key0 < lo || key0 + kTile > hi;  // of the whole warp
    if (edge) {
#pragma unroll
        for (int i = 0; i < kSteps; ++i)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int key = key0 + 16 * i + 8 * e + g;
                if (key < lo || key >= hi) z[i][e] = -INFINITY;
            }
    }
    float mx = fmaxf(z[0][0], z[0][1]);
#pragma unroll
    for (int i = 1; i < kSteps; ++i) mx = fmaxf(mx, fmaxf(z[i][0], z[i][1]));
#pragma unroll
    for (int d = 4; d < 32; d <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, d));
    const float m_new = fmaxf(st.m, mx);
    const float m_use = m_new == -INFINITY ? 0.f : m_new;
    if (__any_sync(0xffffffffu, m_new != st.m)) {
        const float alpha = fast_exp2(st.m - m_use);
        st.l *= alpha;
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) st.o[i][e] *= alpha;
        st.m = m_new;
    }
    const float m_low = m_use - kLift;
    const uint8_t* v = stage + kHalfBytes;
    const int r0 = 2 * t * kHeadDim + ((g ^ (2 * t)) << 4), r1 = (2 * t + 1) * kHeadDim + ((g ^ (2 * t + 1)) << 4);
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
        const float r = i >> sh ? v_rest.y : v_rest.x, inv = i >> sh ? v_rest.w : v_rest.z;
        float w[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const float p = fast_exp2(z[i][e] - m_low);
            st.l = fmaf(p, inv, st.l);
            w[e] = p * r;
        }
        const float h0 = __half2float(__float2half_rn(w[0])), h1 = __half2float(__float2half_rn(w[1]));
        const uint32_t b0 = transpose_8x8(pack_half2(h0, w[0] - h0));
        const uint32_t b1 = transpose_8x8(pack_half2(h1, w[1] - h1));
        const uint8_t* vi = v + 16 * i * kHeadDim;
        uint4 x0 = lds128(vi + r0), x1 = lds128(vi + r1);
        uint4 x2 = lds128(vi + 8 * kHeadDim + r0), x3 = lds128(vi + 8 * kHeadDim + r1);
        if (kCode == GQA_CODE_E4M3 && edge) {  // codes of keys out of sight may be NaN
            const int key = key0 + 16 * i + 2 * t;
            const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
            if (key < lo || key >= hi) x0 = zero;
            if (key + 1 < lo || key + 1 >= hi) x1 = zero;
            if (key + 8 < lo || key + 8 >= hi) x2 = zero;
            if (key + 9 < lo || key + 9 >= hi) x3 = zero;
        }
        const uint32_t w0[4] = {x0.x, x0.y, x0.z, x0.w}, w1[4] = {x1.x, x1.y, x1.z, x1.w};
        const uint32_t w2[4] = {x2.x, x2.y, x2.z, x2.w}, w3[4] = {x3.x, x3.y, x3.z, x3.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            uint32_t a0, a1, a2, a3;
            to_half4<kCode>(__byte_perm(w0[j], w1[j], 0x5140), a0, a1);
            to_half4<kCode>(__byte_perm(w2[j], w3[j], 0x5140), a2, a3);
            mma_16x8x16(st.o[2 * j], a0, a1, a2, a3, b0, b1);
            to_half4<kCode>(__byte_perm(w0[j], w1[j], 0x7362), a0, a1);
            to_half4<kCode>(__byte_perm(w2[j], w3[j], 0x7362), a2, a3);
            mma_16x8x16(st.o[2 * j + 1], a0, a1, a2, a3, b0, b1);
        }
    }
}

template <int kCode, bool kCap, bool kBias>
__global__ void __launch_bounds__(kThreads, 1) paged_decode_kernel(const __grid_constant__ DecodePagedArgs a) {
    extern __shared__ uint8_t raw[];
    uint8_t* ring = raw + ((1024u - (smem_addr(raw) & 1023u)) & 1023u);  // 128-byte swizzle atoms
    Shared& s = *reinterpret_cast<Shared*>(ring + a.stages * kStageBytes);
    int* first = reinterpret_cast<int*>(&s + 1);
    int* los = first + (a.p.batch + 1);
    int* his = los + a.p.batch;
    const PagedCall& p = a.p;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int batch = p.batch, heads = p.c.kv_heads, stages = a.stages;

    if (tid == 0) {
        for (int i = 0; i < stages; ++i) {
            mbar_init(&s.full[i], 1);
            mbar_init(&s.empty[i], 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&s.qfull[i], 1);
            mbar_init(&s.qempty[i], kWarps);
        }
        mbar_init(&s.rfull, kWarps);
        mbar_init(&s.rempty, kFinishers);
        fence_barrier_init();
        prefetch_tensormap(&a.kmap);
        prefetch_tensormap(&a.vmap);
    }
    dependency_wait();
    allow_dependents();
    // Tiles of every sequence and their running sum.
    {
        const int per = (batch + kThreads - 1) / kThreads;
        const int b0 = min(batch, tid * per), b1 = min(batch, b0 + per);
        int sum = 0;
        for (int b = b0; b < b1; ++b) {
            const int64_t m = p.query_positions ? p.query_positions[b] : (int64_t)p.seq_lens[b] - 1;
            const KeyRange r = paged_range(p, b, m, paged_length(p, b));
            const int n = r.hi > r.lo ? ((r.hi + kTile - 1) >> kTileShift) - (r.lo >> kTileShift) : 0;
            los[b] = r.lo;
            his[b] = r.hi;
            first[b] = n;
            sum += n;
        }
        int incl = sum;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int x = __shfl_up_sync(0xffffffffu, incl, d);
            if (lane >= d) incl += x;
        }
        if (lane == 31) s.sum[warp] = incl;
        __syncthreads();
        int at = incl - sum;
        for (int w = 0; w < warp; ++w) at += s.sum[w];
        for (int b = b0; b < b1; ++b) {
            const int n = first[b];
            first[b] = at;
            at += n;
        }
        if (b0 < batch && b1 == batch) first[batch] = at;
        __syncthreads();
    }
    const TileIndex index{first, los, his, batch, heads};
    const int64_t total = (int64_t)first[batch] * heads;
    const int64_t G = min((int64_t)gridDim.x, total), me = blockIdx.x;  // CTAs with a share: one tile at least
    Walk walk;
    walk.start(index, me < G ? total * me / G : 0, me < G ? total * (me + 1) / G : 0);

    if (warp >= kLoaderWarp && warp < kQueryWarp) {
        // ============================ loader ============================
        // What a loader warp does per tile takes longer than the tile needs to arrive
        // (about 700 cycles for one tile at a time, 355 in bursts, of which the copies'
        // issue is the most; 8 KB arrive in 355), so each works on kBurst tiles at once,
        // a tile a lane, and each group of kBurst stages has one of the warps.
        const uint64_t policy = l2_evict_first_policy();
        const int shift = p.c.page_shift;
        const bool two = shift < kTileShift;  // two pages a tile (16 tokens each)
        const int box_bytes = min(p.c.page_len, kTile) * kHeadDim;
        int stg = 0, round = 0;  // next stage, times round the ring
        bool ok = true;
        while (walk.n > 0 && ok) {
            const int64_t lo = los[walk.b], hi = his[walk.b];
            const int32_t* row = p.block_table + walk.b * p.table_stride;
            // Lane's tile of a batch of 32: its pages (-1: no visible key, not loaded) and their scales.
            struct Pages {
                int a, b;
            };
            auto entry = [&](int64_t key) {
                if (key >= hi || key + min(p.c.page_len, kTile) <= lo) return -1;
                const int page = row[key >> shift];
                return page >= 0 && page < p.c.pages ? page : p.c.pages;  // out of the map: TMA fills zeros
            };
            auto pages = [&](int j) {
                const int64_t key = (int64_t)(walk.tile + j + lane) << kTileShift;
                return Pages{entry(key), two ? entry(key + kPagedMinPage) : -1};
            };
            auto scale = [&](const float* at, int page) {
                return page >= 0 && page < p.c.pages ? at[page * p.c.scale_page_stride + walk.h] : 0.f;
            };
            auto scales = [&](Pages g) {
                float4 f = make_float4(scale(p.c.k_scale, g.a), 0.f, scale(p.c.v_scale, g.a), 0.f);
                if (two) {
                    f.y = scale(p.c.k_scale, g.b);
                    f.w = scale(p.c.v_scale, g.b);
                }
                return f;
            };
            // Each step a batch ahead of the next (entries two batches ahead of their
            // use, scales one), so that no load is waited for but a piece's first.
            Pages now = pages(0), next = pages(32), later{-1, -1};
            float4 f_now, f_next;
            for (int j0 = 0; j0 < walk.n && ok; j0 += 32) {
                if (j0 > 0) {
                    now = next;
                    f_now = f_next;
                    next = later;
                    f_next = scales(next);
                    later = pages(j0 + 64);
                }
                const int batch_n = min(32, walk.n - j0);
                for (int k0 = 0, n; k0 < batch_n; k0 += n) {
                    n = min(kBurst - stg % kBurst, batch_n - k0);  // to the end of the group
                    const bool mine = stg / kBurst % kLoaders == warp - kLoaderWarp && lane >= k0 && lane < k0 + n;
                    const int to = stg + lane - k0;
                    if (mine && round > 0) ok = mbar_wait(&s.empty[to], (round - 1) & 1);
                    ok = __all_sync(0xffffffffu, ok);
                    if (!ok) break;
                    if (j0 + k0 == 0) {  // a piece's first scales: on their way while its first copies are issued
                        f_now = scales(now);
                        f_next = scales(next);
                        later = pages(64);
                    }
                    if (mine) {
                        uint8_t* dst = ring + to * kStageBytes;
                        const int prow = two ? 0 : ((walk.tile + j0 + lane) * kTile) & (p.c.page_len - 1);
                        if (now.a >= 0) {
                            tma_load_page(dst, &a.kmap, prow, walk.h, now.a, &s.full[to], policy);
                            tma_load_page(dst + kHalfBytes, &a.vmap, prow, walk.h, now.a, &s.full[to], policy);
                        }
                        if (now.b >= 0) {
                            tma_load_page(dst + box_bytes, &a.kmap, 0, walk.h, now.b, &s.full[to], policy);
                            tma_load_page(dst + kHalfBytes + box_bytes, &a.vmap, 0, walk.h, now.b, &s.full[to], policy);
                        }
                        const VScale va = v_scale_of(f_now.z), vb = v_scale_of(f_now.w);
                        const float nan = __int_as_float(0x7fffffff);
                        s.scales[to] = make_float4(fabsf(f_now.z) <= 3.402823466e38f ? f_now.x : nan,
                                                   fabsf(f_now.w) <= 3.402823466e38f ? f_now.y : nan, va.exponent,
                                                   vb.exponent);
                        s.v_rest[to] = make_float4(va.fraction, vb.fraction, va.inv, vb.inv);
                        mbar_arrive_expect_tx(&s.full[to], 2 * ((now.a >= 0) + (now.b >= 0)) * box_bytes);
                    }
                    stg += n;
                    if (stg == stages) {
                        stg = 0;
                        ++round;
                    }
                }
            }
            if (!walk.next(index)) break;
        }
        if (!ok) {
            if (lane == 0) atomicOr(a.status, kDevStatusTimeout);
            // Do not leave while copies into this CTA's shared memory are in flight.
            for (int i = 0; i < stages; ++i) {
                const int filled = i < stg ? round + 1 : round;  // times stage i was, its own group's
                if (i / kBurst % kLoaders == warp - kLoaderWarp && filled > 0) mbar_wait(&s.full[i], (filled - 1) & 1);
            }
        }
        return;
    }
    if (warp == kQueryWarp) {
        // ============================ queries ============================
        int n = 0;
        const uint64_t step0 = a.rope.step[2 * lane], step1 = a.rope.step[2 * lane + 1];
        while (walk.n > 0) {
            const int sl = n & 1;
            if (n >= 2 && !warp_wait(&s.qempty[sl], ((n >> 1) - 1) & 1)) {
                if (lane == 0) atomicOr(a.status, kDevStatusTimeout);
                break;
            }
            __syncwarp();
            Slot& slot = s.slot[sl];
            // Every load first.
            const __nv_bfloat16* q = p.q + walk.b * p.q_row_stride + walk.h * kGroup * p.q_head_stride + 2 * lane;
            uint32_t xw[kGroup], yw[kGroup];
#pragma unroll
            for (int hq = 0; hq < kGroup; ++hq) {
                xw[hq] = *reinterpret_cast<const uint32_t*>(q + hq * p.q_head_stride);
                yw[hq] = *reinterpret_cast<const uint32_t*>(q + hq * p.q_head_stride + kPairs);
            }
            const int64_t m = p.query_positions ? p.query_positions[walk.b] : (int64_t)p.seq_lens[walk.b] - 1;
            float slope = 0.f;
            if (kBias && lane < kGroup) slope = p.slopes[walk.h * kGroup + lane] * 1.4426950408889634f;
            float2 f0 = make_float2(1.f, 0.f), f1 = f0;
            if (!p.q_rotated) {
                f0 = rope_factor(step0, m);
                f1 = rope_factor(step1, m);
            }
            float v[kGroup][4], most[kGroup];
            bool fine[kGroup];
#pragma unroll
            for (int hq = 0; hq < kGroup; ++hq) {
                const float2 x = bf16x2_to_float2(xw[hq]), y = bf16x2_to_float2(yw[hq]);
                v[hq][0] = x.x * f0.x - y.x * f0.y;
                v[hq][1] = x.y * f1.x - y.y * f1.y;
                v[hq][2] = x.x * f0.y + y.x * f0.x;
                v[hq][3] = x.y * f1.y + y.y * f1.x;
                most[hq] = fmaxf(fmaxf(fabsf(v[hq][0]), fabsf(v[hq][1])), fmaxf(fabsf(v[hq][2]), fabsf(v[hq][3])));
                fine[hq] = __all_sync(0xffffffffu, most[hq] <= 3.402823466e38f && v[hq][0] == v[hq][0] &&
                                                       v[hq][1] == v[hq][1] && v[hq][2] == v[hq][2] &&
                                                       v[hq][3] == v[hq][3]);
            }
            // (Magnitudes are non-negative: their bits order as integers.)
#pragma unroll
            for (int hq = 0; hq < kGroup; ++hq)
                most[hq] = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(most[hq])));
#pragma unroll
            for (int hq = 0; hq < kGroup; ++hq) {
                // 2^e just above the largest (2^-126 at least), e <= 127 so that its inverse is a normal number.
                const int e = min(253, max(1, (__float_as_int(most[hq]) >> 23) + 1));
                const float up = __int_as_float(e << 23), down = __int_as_float((254 - e) << 23);
                float hp[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    v[hq][i] *= down;
                    hp[i] = __half2float(__float2half_rn(v[hq][i]));
                }
                *reinterpret_cast<uint32_t*>(&slot.q[2 * hq][2 * lane]) = pack_half2(hp[0], hp[1]);
                *reinterpret_cast<uint32_t*>(&slot.q[2 * hq][kPairs + 2 * lane]) = pack_half2(hp[2], hp[3]);
                *reinterpret_cast<uint32_t*>(&slot.q[2 * hq + 1][2 * lane]) =
                    pack_half2(v[hq][0] - hp[0], v[hq][1] - hp[1]);
                *reinterpret_cast<uint32_t*>(&slot.q[2 * hq + 1][kPairs + 2 * lane]) =
                    pack_half2(v[hq][2] - hp[2], v[hq][3] - hp[3]);
                if (lane == hq) {
                    const float unit = kCap ? p.scale / p.cap : p.scale * 1.4426950408889634f;
                    slot.factor[hq] = fine[hq] ? unit * up : __int_as_float(0x7fffffff);
                    slot.slope[hq] = slope;
                }
            }
            const KeyRange r{los[walk.b], his[walk.b]};
            if (lane == 0) {
                slot.lo = r.lo;
                slot.hi = r.hi;
                slot.m = (int)max(m, -(int64_t)(1 << 30));  // (distances stay 32-bit)
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&s.qfull[sl]);
            ++n;
            if (!walk.next(index)) break;
        }
        return;
    }

    if (warp >= kFinishWarp) {
        // ============================ finishers ============================
        // A warp a head: the consumers' parts of a piece to an output row, or, for a
        // piece of a unit, to a partial row -- while the consumers go on.
        const int hq = warp - kFinishWarp;
        // Sequences that see nothing.
        for (int b = blockIdx.x; b < batch; b += gridDim.x) {
            if (first[b + 1] != first[b]) continue;
            for (int h = 0; h < heads; ++h)
                *reinterpret_cast<uint2*>(p.out + b * p.out_row_stride + (h * kGroup + hq) * p.out_head_stride +
                                          4 * lane) = make_uint2(0u, 0u);
        }
        bool ok = true;  // after a wait that timed out: no more waits, but the counters are kept
        for (int n = 0; walk.n > 0; ++n) {
            if (ok) ok = mbar_wait(&s.rfull, n & 1);
            __syncwarp();
            const auto& r = s.result;
            float M = -INFINITY, L = 0.f;
            float4 A = make_float4(0.f, 0.f, 0.f, 0.f);
            auto add = [&](float f, float l, float4 x) {
                L = fmaf(f, l, L);
                A.x = fmaf(f, x.x, A.x);
                A.y = fmaf(f, x.y, A.y);
                A.z = fmaf(f, x.z, A.z);
                A.w = fmaf(f, x.w, A.w);
            };
#pragma unroll
            for (int w = 0; w < kWarps; ++w) M = fmaxf(M, r.m[w][hq]);
            const float Mu = M == -INFINITY ? 0.f : M;
#pragma unroll
            for (int w = 0; w < kWarps; ++w)
                add(fast_exp2(r.m[w][hq] - Mu), r.l[w][hq], *reinterpret_cast<const float4*>(&r.acc[w][hq][4 * lane]));
            __syncwarp();
            if (lane == 0) mbar_arrive(&s.rempty);
            bool done = walk.n == walk.unit_tiles;
            if (!done) {
                // A piece of a unit: store it, and the unit's last CTA merges all.
                // Tile x lies in the share of CTA ceil((x + 1) G / T) - 1.  A share's
                // first piece goes to its slot 0; its last, if another one, to slot 1:
                // only the unit's first CTA can have begun before it.
                const int c0 = (int)(((walk.unit_first + 1) * G + total - 1) / total) - 1;
                const int pieces = (int)(((walk.unit_first + walk.unit_tiles) * G + total - 1) / total) - c0;
                const int second = total * c0 / G < walk.unit_first ? 1 : 0;
                auto piece = [&](int c) {
                    return a.partials + (((c0 + c) * 2 + (c ? 0 : second)) * kGroup + hq) * kPartialFloats;
                };
                float* mine = piece((int)me - c0);
                *reinterpret_cast<float4*>(mine + 4 * lane) = A;
                if (lane == 0) *reinterpret_cast<float2*>(mine + kHeadDim) = make_float2(M, L);
                __syncwarp();
                uint32_t before = 0;
                if (lane == 0) {
                    // Releases the warp's row and acquires the others'.
                    uint32_t* count = a.arrivals + (walk.b * heads + walk.h) * kGroup + hq;
                    asm volatile("atom.add.acq_rel.gpu.global.u32 %0, [%1], 1;" : "=r"(before) : "l"(count) : "memory");
                    if (before == (uint32_t)(pieces - 1)) *count = 0;
                }
                done = __shfl_sync(0xffffffffu, before, 0) == (uint32_t)(pieces - 1);
                if (done) {
                    constexpr int kAtOnce = 10;
                    M = -INFINITY;
                    L = 0.f;
                    A = make_float4(0.f, 0.f, 0.f, 0.f);
                    for (int c = 0; c < pieces; c += kAtOnce) {
                        float4 v[kAtOnce];
                        float2 ml[kAtOnce];
                        float now = M;
#pragma unroll
                        for (int e = 0; e < kAtOnce; ++e) {
                            const float* x = piece(min(c + e, pieces - 1));
                            ml[e] = __ldcg(reinterpret_cast<const float2*>(x + kHeadDim));
                            v[e] = __ldcg(reinterpret_cast<const float4*>(x + 4 * lane));
                        }
#pragma unroll
                        for (int e = 0; e < kAtOnce; ++e) now = fmaxf(now, ml[e].x);
                        const float use = now == -INFINITY ? 0.f : now;
                        const float f0 = fast_exp2(M - use);
                        M = now;
                        L *= f0;
                        A = make_float4(A.x * f0, A.y * f0, A.z * f0, A.w * f0);
#pragma unroll
                        for (int e = 0; e < kAtOnce; ++e)
                            if (c + e < pieces) add(fast_exp2(ml[e].x - use), ml[e].y, v[e]);
                    }
                }
            }
            if (done) {
                const __nv_bfloat162 x = __floats2bfloat162_rn(A.x / L, A.y / L), y = __floats2bfloat162_rn(A.z / L, A.w / L);
                *reinterpret_cast<uint2*>(p.out + walk.b * p.out_row_stride + (walk.h * kGroup + hq) * p.out_head_stride +
                                          4 * lane) =
                    make_uint2(*reinterpret_cast<const uint32_t*>(&x), *reinterpret_cast<const uint32_t*>(&y));
            }
            if (!walk.next(index)) break;
        }
        if (!ok) atomicOr(a.status, kDevStatusTimeout);  // (any lane's)
        return;
    }

    // ============================ consumers ============================
    const int g = lane >> 2, t = lane & 3;
    int mine = warp;           // this warp's next tile, counted from the piece's first
    int stg = warp, phase = 0; // its stage
    bool ok = true;  // after a wait that timed out: no more waits, but every barrier is kept
    for (int n = 0; walk.n > 0; ++n) {
        const int sl = n & 1;
        if (ok) ok = mbar_wait(&s.qfull[sl], (n >> 1) & 1);
        const Slot& slot = s.slot[sl];
        uint32_t qf[16];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint4 w = lds128(&slot.q[g][32 * t + 8 * i]);
            qf[4 * i] = w.x;
            qf[4 * i + 1] = w.y;
            qf[4 * i + 2] = w.z;
            qf[4 * i + 3] = w.w;
        }
        const float factor = slot.factor[t], slope = slot.slope[t];
        const int lo = slot.lo, hi = slot.hi, m_pos = slot.m;
        __syncwarp();
        if (lane == 0) mbar_arrive(&s.qempty[sl]);

        State st;
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) st.o[i][e] = 0.f;
        st.m = -INFINITY;
        st.l = 0.f;
        // This warp's tiles: every kWarps-th of the CTA's.
        for (; mine < walk.n; mine += kWarps) {
            const int j = mine;
            if (ok) ok = mbar_wait(&s.full[stg], phase);
            consume_tile<kCode, kCap, kBias>(st, ring + stg * kStageBytes, s.scales[stg], s.v_rest[stg], qf, factor, slope,
                                             p.cap * 1.4426950408889634f, (walk.tile + j) * kTile, lo, hi, m_pos,
                                             p.c.page_shift, lane);
            __syncwarp();
            if (lane == 0) mbar_arrive(&s.empty[stg]);
            stg += kWarps;
            if (stg >= stages) {
                stg -= stages;
                phase ^= 1;
            }
        }
        mine -= walk.n;

        // This warp's part of the piece, for the finishers.
        float l = st.l;
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) l += __shfl_xor_sync(0xffffffffu, l, d);
        if (ok && n >= 1) ok = mbar_wait(&s.rempty, (n - 1) & 1);
        auto& r = s.result;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            *reinterpret_cast<float4*>(&r.acc[warp][t][16 * g + 4 * i]) =
                make_float4((st.o[2 * i][0] + st.o[2 * i][1]) * kWeightUnit, (st.o[2 * i][2] + st.o[2 * i][3]) * kWeightUnit,
                            (st.o[2 * i + 1][0] + st.o[2 * i + 1][1]) * kWeightUnit,
                            (st.o[2 * i + 1][2] + st.o[2 * i + 1][3]) * kWeightUnit);
        if (g == 0) {
            r.m[warp][t] = st.m;
            r.l[warp][t] = l;
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&s.rfull);
        if (!walk.next(index)) break;
    }
    if (!ok) atomicOr(a.status, kDevStatusTimeout);
}

// A wait by parity is sound only for the phase after the last one that the same
// warp saw complete, so each stage has one consumer warp and one loader warp: the
// ring is a whole number of stages for each consumer warp, and of loader groups.
int decode_stages(int batch) {
    static_assert(227 * 1024 - 1024 - (int64_t)sizeof(Shared) - (3 * GQA_PAGED_MAX_BATCH + 1) * 4 >=
                      (int64_t)kStageBytes * kWarps,
                  "a stage for every consumer warp");
    static_assert(kWarps % kBurst == 0 && kMaxStages % kWarps == 0, "whole groups");
    const int64_t room = 227 * 1024 - 1024 - (int64_t)sizeof(Shared) - (3 * (int64_t)batch + 1) * 4;
    const int64_t n = room / kStageBytes;
    return (int)(n < kMaxStages ? n : kMaxStages) / kWarps * kWarps;
}

using Kernel = void (*)(DecodePagedArgs);

Kernel kernel_for(int code, bool cap, bool bias) {
    if (code == GQA_CODE_INT8) {
        if (cap) return bias ? paged_decode_kernel<0, true, true> : paged_decode_kernel<0, true, false>;
        return bias ? paged_decode_kernel<0, false, true> : paged_decode_kernel<0, false, false>;
    }
    if (cap) return bias ? paged_decode_kernel<1, true, true> : paged_decode_kernel<1, true, false>;
    return bias ? paged_decode_kernel<1, false, true> : paged_decode_kernel<1, false, false>;
}

}  // namespace

int paged_decode_tile() { return kTile; }

// The counters come first, as many as any call can have: a region that moved with
// the batch would meet another call's partial rows.
size_t paged_decode_workspace(int sms) {
    return kPagedPartialsOffset + (size_t)sms * 2 * kGroup * kPartialFloats * sizeof(float);
}

cudaError_t launch_paged_decode(const PagedCall& call, const RopeSteps& rope, int code, const CUtensorMap& kmap,
                                const CUtensorMap& vmap, int sms, uint8_t* ws, cudaStream_t stream) {
    DecodePagedArgs a;
    a.kmap = kmap;
    a.vmap = vmap;
    a.p = call;
    a.rope = rope;
    a.status = reinterpret_cast<uint32_t*>(ws);
    a.arrivals = reinterpret_cast<uint32_t*>(ws + kPagedArrivalsOffset);
    a.partials = reinterpret_cast<float*>(ws + kPagedPartialsOffset);
    a.stages = decode_stages(call.batch);
    const size_t smem = 1024 + (size_t)a.stages * kStageBytes + sizeof(Shared) + (3 * (size_t)call.batch + 1) * 4;
    return launch_dependent(kernel_for(code, call.cap > 0.f, call.slopes != nullptr), sms, kThreads, smem, stream, a);
}

cudaError_t paged_decode_prepare() {
    for (int i = 0; i < 8; ++i) {
        const cudaError_t e = cudaFuncSetAttribute(kernel_for(i & 1, i & 2, i & 4),
                                                   cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024);
        if (e != cudaSuccess) return e;
    }
    return cudaSuccess;
}

}  // namespace gqa
