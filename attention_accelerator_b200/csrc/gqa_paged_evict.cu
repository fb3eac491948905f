// gqa_paged_evict.cu -- eviction from the paged 8-bit cache: the choice of the rows that
// stay, by their accumulated attention weight, and the move of those that fill the holes.
#include "gqa_internal.h"
#include "gqa_paged.cuh"
#include "gqa_paged_internal.h"

#include <algorithm>

namespace gqa {

namespace {

// ---------------------------------------------------------------------------
// The choice.
//
// A cluster of 1 to 8 CTAs a (request, KV head), each with a stretch of its rows.  A
// row's rank is that of a 32-bit number: the bits of its weight, which order as the
// weights do (they are not negative), and above them whether it is spared; the
// numbers are computed once and kept in shared memory.  Passes over histograms, from
// the top bits down (11, 11 and 10; 4 times 8 for short requests, whose time is the
// bins'), find the number of the last row that stays and how many rows of that very
// number stay.  Two more count, a warp a stretch of rows, a lane four rows, what is equal
// to it and then the holes below `keep` and the rows past it that stay; the last lists
// both in order, and they are paired off.  One more CTA gives the pages back.
//
// Bound by the chain of loads, votes and barriers between the passes, not by the 8 bytes
// a row: 64 requests of 1025 rows and 8 heads 11.3 us in tables of up to 2048 rows, 15.7 in
// tables of up to 8192 and 23.6 of 32768 (the shape goes by the table, and a block there has
// its SM to itself), 8 of up to 32768 26 us (64 clusters of 4), one of 131072 28 us, 64 of up
// to 8192 35 us (replayed graph).
// ---------------------------------------------------------------------------
constexpr int kMaxCluster = 8;
constexpr int kMaxRows = 48 * 1024;  // of a CTA in shared memory; numbers of rows past that are computed again

struct EvictPlanArgs {
    KeyWeightsView w;
    const int32_t *lens, *keep;
    const int32_t* block_table;
    int64_t table_stride;
    int32_t* free_pages;
    const int32_t* n_free;
    int32_t *take, *lens_out, *evicted_out, *n_free_out, *counts;
    uint32_t* ticket;
    int32_t* lists;  // [requests * heads][2][max_keep]: holes and rows that fill them
    int requests, heads, table_width, free_capacity, page_shift, max_keep, sinks, recent;
    int held_rows;   // of a CTA in shared memory
    bool vectors;    // weights and positions of a head are 16-byte aligned
    bool in_place;   // lens_out, evicted_out or n_free_out may be what is read
};

struct Cut {
    int len, keep;  // rows held and rows that stay (keep == len: left as it is)
};
__device__ __forceinline__ Cut cut_of(const EvictPlanArgs& a, int r) {
    const int len = a.lens[r], keep = min(a.keep[r], a.max_keep);
    return Cut{len, keep > 0 && keep < len ? keep : len};
}

__device__ __forceinline__ uint32_t rank_of(const EvictPlanArgs& a, float weight, int position, int64_t recent_from) {
    const uint32_t bits = __float_as_uint(weight);
    const uint32_t w = weight != weight ? 0x7fffffffu : bits & 0x80000000u ? 0u : bits;
    return w | (position < a.sinks || position >= recent_from ? 0x80000000u : 0u);
}

// The sum over a warp, and of the lanes before.
__device__ __forceinline__ int warp_before(int v) {
    const int lane = threadIdx.x & 31;
    int incl = v;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, incl, d);
        if (lane >= d) incl += x;
    }
    return incl - v;
}

template <int kThreads>
struct Radix {
    static constexpr int kBits = kThreads == 128 ? 8 : 11, kPasses = kThreads == 128 ? 4 : 3, kBins = 1 << kBits;
    static __device__ __forceinline__ constexpr int shift(int pass) { return pass + 1 == kPasses ? 0 : 32 - kBits * (pass + 1); }
    static __device__ __forceinline__ constexpr uint32_t mask(int pass) {
        return pass + 1 == kPasses ? (1u << (32 - kBits * (kPasses - 1))) - 1 : (1u << kBits) - 1;
    }
};

// A sum past 32 bits in shared memory.  (64-bit atomics there are loops: the choice of 64 requests took 14.4 us with
// them, of 64 in tables of 32768 rows 35 instead of 23.)
struct WideSum {
    uint32_t low, high;  // of the terms' lower 16 bits and of the others
    __device__ __forceinline__ void clear() { low = high = 0; }
    __device__ __forceinline__ void add(int64_t x) {  // x >= 0, below 2^39
        if (x == 0) return;
        atomicAdd(&low, (uint32_t)x & 0xffffu);
        if (x >> 16) atomicAdd(&high, (uint32_t)(x >> 16));
    }
    __device__ __forceinline__ int64_t value() const { return ((int64_t)high << 16) + low; }
};

template <int kThreads>
struct alignas(16) PlanShared {
    int hist[Radix<kThreads>::kPasses][Radix<kThreads>::kBins];
    int warp_sum[32];
    int2 warp_marks[32];
    int equal;            // rows of the last one's number in this CTA
    int2 marks;           // holes, and rows that fill them, in this CTA
    uint32_t bin, left;
    WideSum give, rows;  // of all requests: a table may name more than 2^31 rows
    int cuts;
    bool last;
};

// Values in the shared memory of a CTA of the cluster.  (Volatile, but not ordered with other memory: several are
// on their way at once, behind the cluster's barrier.)
__device__ __forceinline__ int of_rank(const int& x, uint32_t rank) {
    int v;
    asm volatile("ld.shared::cluster.b32 %0, [%1];" : "=r"(v) : "r"(cluster_map(&x, rank)));
    return v;
}
__device__ __forceinline__ int2 of_rank(const int2& x, uint32_t rank) {
    int2 v;
    asm volatile("ld.shared::cluster.v2.b32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(cluster_map(&x, rank)));
    return v;
}
__device__ __forceinline__ int4 of_rank(const int4& x, uint32_t rank) {
    int4 v;
    asm volatile("ld.shared::cluster.v4.b32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                 : "r"(cluster_map(&x, rank)));
    return v;
}

template <int kThreads, bool kCluster>
__device__ __forceinline__ void choose(const EvictPlanArgs& a, PlanShared<kThreads>& s, uint32_t* ranks, int unit, const Cut& cut,
                                       int evicted, uint32_t rank, uint32_t ctas) {
    using R = Radix<kThreads>;
    constexpr int kWarps = kThreads / 32, kStep = 128 * kWarps;  // four rows a lane
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const float* weight = a.w.weight + (int64_t)unit * a.w.capacity;
    const int32_t* position = a.w.position + (int64_t)unit * a.w.capacity;
    const int64_t recent_from = (int64_t)cut.len + min(max(evicted, 0), 1 << 30) - a.recent;
    const int keep = cut.keep;
    // This CTA's rows: whole steps of 128 for each of its warps.
    const int each = ((cut.len + (int)ctas - 1) / (int)ctas + kStep - 1) / kStep * kStep;
    const int row0 = (int)min((int64_t)cut.len, (int64_t)each * rank), n = min(each, cut.len - row0);
    auto number = [&](int i) { return rank_of(a, weight[i], position[i], recent_from); };
    // Rows i to i + 3 of this CTA (0 past its last).
    auto four = [&](int i) {
        if (i < a.held_rows) return *reinterpret_cast<const uint4*>(ranks + i);
        uint4 x;
        x.x = i < n ? number(row0 + i) : 0u;
        x.y = i + 1 < n ? number(row0 + i + 1) : 0u;
        x.z = i + 2 < n ? number(row0 + i + 2) : 0u;
        x.w = i + 3 < n ? number(row0 + i + 3) : 0u;
        return x;
    };
    auto all_arrive = [&] {
        if constexpr (kCluster) cluster_sync_all(); else __syncthreads();
    };

    for (int i = tid; i < R::kPasses * R::kBins; i += kThreads) s.hist[0][i] = 0;
    __syncthreads();
    auto count_four = [&](int* hist, const uint32_t (&bin)[4], const bool (&in)[4]) {
        // A warp whose rows all have the same counts them as one.
        const uint32_t first = __shfl_sync(0xffffffffu, bin[0], 0);
        bool same = true;
#pragma unroll
        for (int e = 0; e < 4; ++e) same &= in[e] && bin[e] == first;
        if (__all_sync(0xffffffffu, same)) {
            if (lane == 0) atomicAdd(&hist[first], 128);
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (in[e]) atomicAdd(&hist[bin[e]], 1);
        }
    };
    // The numbers, and the first histogram: four steps of the CTA's rows at a time, every load first.
    {
        constexpr int kAtOnce = 4;
        const int room = (int)min(a.w.capacity - row0, (int64_t)each);  // rows that may be read
        for (int i0 = 0; i0 < n; i0 += kStep * kAtOnce) {
            float4 w[kAtOnce];
            int4 p[kAtOnce];
#pragma unroll
            for (int e = 0; e < kAtOnce; ++e) {
                const int i = i0 + e * kStep + 4 * tid;
                w[e] = make_float4(0.f, 0.f, 0.f, 0.f);
                p[e] = make_int4(0, 0, 0, 0);
                if (i >= n) continue;
                if (a.vectors && i + 4 <= room) {
                    w[e] = *reinterpret_cast<const float4*>(weight + row0 + i);
                    p[e] = *reinterpret_cast<const int4*>(position + row0 + i);
                } else {
                    float* we = &w[e].x;
                    int* pe = &p[e].x;
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        if (i + k < n) {
                            we[k] = weight[row0 + i + k];
                            pe[k] = position[row0 + i + k];
                        }
                }
            }
#pragma unroll
            for (int e = 0; e < kAtOnce; ++e) {
                const int i = i0 + e * kStep + 4 * tid;
                if (i0 + e * kStep >= n) break;
                const float we[4] = {w[e].x, w[e].y, w[e].z, w[e].w};
                const int pe[4] = {p[e].x, p[e].y, p[e].z, p[e].w};
                uint32_t x[4], bin[4];
                bool in[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    in[k] = i + k < n;
                    x[k] = in[k] ? rank_of(a, we[k], pe[k], recent_from) : 0u;
                    bin[k] = x[k] >> R::shift(0);
                }
                if (i < a.held_rows) *reinterpret_cast<uint4*>(ranks + i) = make_uint4(x[0], x[1], x[2], x[3]);
                count_four(s.hist[0], bin, in);
            }
        }
    }
    uint32_t found = 0, known = 0;   // the number's upper bits, and which these are
    uint32_t left = (uint32_t)keep;  // rows that stay among those which agree with it so far
#pragma unroll
    for (int pass = 0; pass < R::kPasses; ++pass) {
        const int shift = R::shift(pass);
        const uint32_t mask = R::mask(pass);
        int* hist = s.hist[pass];
        if (pass > 0)
            for (int i0 = 0; i0 < n; i0 += kStep) {
                const int i = i0 + 4 * tid;
                const uint4 x = four(i);
                const uint32_t xs[4] = {x.x, x.y, x.z, x.w};
                uint32_t bin[4];
                bool in[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    in[e] = i + e < n && (xs[e] & known) == found;
                    bin[e] = xs[e] >> shift & mask;
                }
                if (__any_sync(0xffffffffu, in[0] || in[1] || in[2] || in[3])) count_four(hist, bin, in);
            }
        all_arrive();
        // From the highest bin down: the one in which the count passes what is left.
        constexpr int kOf = R::kBins / kThreads;
        int count[kOf], sum = 0;
        if constexpr (kCluster) {
            static_assert(!kCluster || kOf == 4, "a vector of bins a thread");
            int4 of[kMaxCluster];
#pragma unroll
            for (uint32_t c = 0; c < kMaxCluster; ++c)
                of[c] = c < ctas ? of_rank(*reinterpret_cast<const int4*>(&hist[R::kBins - 4 * (tid + 1)]), c)
                                 : make_int4(0, 0, 0, 0);
            int4 all = of[0];
#pragma unroll
            for (uint32_t c = 1; c < kMaxCluster; ++c)
                all = make_int4(all.x + of[c].x, all.y + of[c].y, all.z + of[c].z, all.w + of[c].w);
            count[0] = all.w;
            count[1] = all.z;
            count[2] = all.y;
            count[3] = all.x;
        } else {
#pragma unroll
            for (int i = 0; i < kOf; ++i) count[i] = hist[R::kBins - 1 - (tid * kOf + i)];
        }
#pragma unroll
        for (int i = 0; i < kOf; ++i) sum += count[i];
        const int in_warp = warp_before(sum);
        if (lane == 31) s.warp_sum[warp] = in_warp + sum;
        __syncthreads();
        uint32_t before = (uint32_t)(in_warp + __reduce_add_sync(0xffffffffu, lane < warp ? s.warp_sum[lane] : 0));
#pragma unroll
        for (int i = 0; i < kOf; ++i) {
            if (before < left && left <= before + count[i]) {
                s.bin = (uint32_t)(R::kBins - 1 - (tid * kOf + i));
                s.left = left - before;
            }
            before += count[i];
        }
        __syncthreads();
        found |= s.bin << shift;
        known |= mask << shift;
        left = s.left;
    }
    // A warp's stretch of the CTA's rows.
    const int per_warp = each / kWarps, w0 = warp * per_warp, w1 = min(n, w0 + per_warp);
    // Rows of the very number before this warp's.
    int equal = 0;
    for (int i = w0 + 4 * lane; i < w1; i += 128) {
        const uint4 x = four(i);
        equal += (x.x == found) + (i + 1 < w1 && x.y == found) + (i + 2 < w1 && x.z == found) + (i + 3 < w1 && x.w == found);
    }
    equal = __reduce_add_sync(0xffffffffu, equal);
    if (lane == 0) s.warp_sum[warp] = equal;
    __syncthreads();
    const int of_warp = lane < kWarps ? s.warp_sum[lane] : 0;
    if (warp == 0) {
        const int all = __reduce_add_sync(0xffffffffu, of_warp);
        if (lane == 0) s.equal = all;
    }
    int tie = __reduce_add_sync(0xffffffffu, lane < warp ? of_warp : 0);
    if constexpr (kCluster) {
        cluster_sync_all();
        tie += __reduce_add_sync(0xffffffffu, lane < (int)rank ? of_rank(s.equal, min((uint32_t)lane, ctas - 1)) : 0);
    }
    const int tie0 = tie;
    // Which of rows i to i + 3 (of this CTA; a lane's, by whole warps) are holes or fill one, as bits; ties are counted in order.
    auto marks_of = [&](int i) {
        const uint4 x = i < w1 ? four(i) : make_uint4(0u, 0u, 0u, 0u);
        const uint32_t xs[4] = {x.x, x.y, x.z, x.w};
        uint32_t same = 0, stays = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            same |= (i + e < w1 && xs[e] == found) << e;
            stays |= (xs[e] > found) << e;
        }
        if (__any_sync(0xffffffffu, same)) {
            const int mine = __popc(same);
            int at = tie + warp_before(mine);
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (same >> e & 1) stays |= ((uint32_t)at++ < left) << e;
            tie += __reduce_add_sync(0xffffffffu, mine);
        }
        const uint32_t low = (1u << min(4, max(0, keep - row0 - i))) - 1, rows = (1u << min(4, max(0, w1 - i))) - 1;
        return ((stays & ~low) | (~stays & low)) & rows;
    };
    auto low_of = [&](int i) { return (1u << min(4, max(0, keep - row0 - i))) - 1; };  // rows below keep
    int2 marks = make_int2(0, 0);
    for (int i0 = w0; i0 < w1; i0 += 128) {
        const uint32_t m = marks_of(i0 + 4 * lane), low = low_of(i0 + 4 * lane);
        marks.x += __popc(m & low);
        marks.y += __popc(m & ~low);
    }
    marks = make_int2(__reduce_add_sync(0xffffffffu, marks.x), __reduce_add_sync(0xffffffffu, marks.y));
    if (lane == 0) s.warp_marks[warp] = marks;
    __syncthreads();
    const int2 wm = lane < kWarps ? s.warp_marks[lane] : make_int2(0, 0);
    int2 all = make_int2(__reduce_add_sync(0xffffffffu, wm.x), __reduce_add_sync(0xffffffffu, wm.y));
    int at_hole = __reduce_add_sync(0xffffffffu, lane < warp ? wm.x : 0);
    int at_fill = __reduce_add_sync(0xffffffffu, lane < warp ? wm.y : 0);
    if constexpr (kCluster) {
        if (tid == 0) s.marks = all;
        cluster_sync_all();
        const int2 x = lane < (int)ctas ? of_rank(s.marks, (uint32_t)lane) : make_int2(0, 0);
        all.x = __reduce_add_sync(0xffffffffu, x.x);
        at_hole += __reduce_add_sync(0xffffffffu, lane < (int)rank ? x.x : 0);
        at_fill += __reduce_add_sync(0xffffffffu, lane < (int)rank ? x.y : 0);
    }
    int32_t* holes = a.lists + (int64_t)unit * 2 * a.max_keep;
    int32_t* fills = holes + a.max_keep;
    int32_t* take = a.take + (int64_t)unit * a.max_keep;
    tie = tie0;
    for (int i0 = w0; i0 < w1; i0 += 128) {
        const int i = i0 + 4 * lane;
        const uint32_t m = marks_of(i), low = low_of(i);
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (low >> e & 1 && i + e < w1) take[row0 + i + e] = -1;
        if (!__any_sync(0xffffffffu, m)) continue;
        const int both = __popc(m & low) | __popc(m & ~low) << 16, before = warp_before(both);  // (128 of each at most)
        int hole = at_hole + (before & 0xffff), fill = at_fill + (before >> 16);
        const int all_of = __reduce_add_sync(0xffffffffu, both);
        at_hole += all_of & 0xffff;
        at_fill += all_of >> 16;
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (m >> e & 1) {
                if (low >> e & 1) holes[hole++] = row0 + i + e; else fills[fill++] = row0 + i + e;
            }
    }
    for (int i = keep + (int)rank * kThreads + tid; i < a.max_keep; i += (int)ctas * kThreads) take[i] = -1;
    if constexpr (kCluster) __threadfence();
    all_arrive();
    for (int i = (int)rank * kThreads + tid; i < all.x; i += (int)ctas * kThreads) take[__ldcg(holes + i)] = __ldcg(fills + i);
}

template <int kThreads, bool kCluster>
__global__ void __launch_bounds__(kThreads) plan_eviction_kernel(const __grid_constant__ EvictPlanArgs a) {
    extern __shared__ uint32_t ranks[];
    __shared__ PlanShared<kThreads> s;
    const int tid = threadIdx.x, n = a.requests;
    uint32_t rank = 0, ctas = 1;
    if constexpr (kCluster) {
        asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
        asm("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(ctas));
    }
    const int unit = blockIdx.x / ctas;
    const int page_mask = (1 << a.page_shift) - 1;
    auto pages_of = [&](int len) { return (int)(((int64_t)len + page_mask) >> a.page_shift); };
    if (tid == 0) {
        s.give.clear();
        s.rows.clear();
        s.cuts = 0;
    }
    // Every load that waits for nothing first.
    const int n_free = *a.n_free, mine = min(unit / a.heads, n - 1), evicted = a.w.evicted[mine];
    const Cut cut = cut_of(a, mine);
    __syncthreads();
    // All or nothing: every CTA looks at all requests.
    const int per = (n + kThreads - 1) / kThreads, r0 = min(n, tid * per), r1 = min(n, r0 + per);
    bool bad = false;
    int64_t give = 0;
    for (int r = r0; r < r1; ++r) {
        const Cut c = cut_of(a, r);
        bad |= c.len < 0 || pages_of(c.len) > a.table_width || c.len > a.w.capacity;
        if (!bad) give += pages_of(c.len) - pages_of(c.keep);
    }
    s.give.add(give);
    bad = __syncthreads_or(bad);
    const int64_t given = s.give.value();
    const bool ok = !bad && n_free >= 0 && n_free + given <= a.free_capacity;

    if (unit < n * a.heads) {
        if (ok && cut.keep < cut.len) {
            choose<kThreads, kCluster>(a, s, ranks, unit, cut, evicted, rank, ctas);
        } else {
            int32_t* take = a.take + (int64_t)unit * a.max_keep;
            for (int i = (int)rank * kThreads + tid; i < a.max_keep; i += (int)ctas * kThreads) take[i] = -1;
        }
    } else if (rank == 0) {
        // As many requests at a time as there are threads: each thread its own one's first pages, the warps in turn
        // what is left of the others.
        constexpr int kOwn = 2;
        const int lane = tid & 31, warp = tid >> 5;
        int *at_of = s.hist[0], *from_of = at_of + kThreads, *left_of = from_of + kThreads;
        static_assert(Radix<kThreads>::kBins * Radix<kThreads>::kPasses >= 3 * kThreads, "room in the histograms' place");
        int base = n_free, cuts = 0;
        int64_t rows = 0;
        for (int c0 = 0; c0 < n && ok; c0 += kThreads) {
            const int r = c0 + tid;
            const Cut c = r < n ? cut_of(a, r) : Cut{0, 0};
            cuts += c.keep < c.len;
            rows += c.len - c.keep;
            const int from = pages_of(c.keep), n_pages = pages_of(c.len) - from, in_warp = warp_before(n_pages);
            __syncthreads();  // (the warps have read the last requests' numbers)
            if (lane == 31) s.warp_sum[warp] = in_warp + n_pages;
            __syncthreads();
            int at = base + in_warp, all = 0;
            for (int w = 0; w < kThreads / 32; ++w) {
                const int x = s.warp_sum[w];
                all += x;
                if (w < warp) at += x;
            }
            base += all;
            const int32_t* row = a.block_table + r * a.table_stride + from;
            int own[kOwn];
#pragma unroll
            for (int j = 0; j < kOwn; ++j) own[j] = j < n_pages ? __ldg(row + j) : 0;
#pragma unroll
            for (int j = 0; j < kOwn; ++j)
                if (j < n_pages) a.free_pages[at + j] = own[j];
            at_of[tid] = at;
            from_of[tid] = from;
            left_of[tid] = n_pages;
            if (!__syncthreads_or(n_pages > kOwn)) continue;
            for (int i = warp; i < min(kThreads, n - c0); i += kThreads / 32) {
                const int32_t* of = a.block_table + (c0 + i) * a.table_stride + from_of[i];
                int32_t* to = a.free_pages + at_of[i];
                const int end = left_of[i];
                constexpr int kAtOnce = 4;
                for (int j0 = kOwn + lane; j0 < end; j0 += 32 * kAtOnce) {
                    int32_t page[kAtOnce];
#pragma unroll
                    for (int e = 0; e < kAtOnce; ++e) page[e] = j0 + 32 * e < end ? __ldg(of + j0 + 32 * e) : 0;
#pragma unroll
                    for (int e = 0; e < kAtOnce; ++e)
                        if (j0 + 32 * e < end) to[j0 + 32 * e] = page[e];
                }
            }
        }
        if (cuts) atomicAdd(&s.cuts, cuts);
        s.rows.add(rows);
        __syncthreads();
        if (tid == 0) {
            a.counts[0] = s.cuts;
            a.counts[1] = (int)min(s.rows.value(), (int64_t)0x7fffffff);
            a.counts[2] = ok ? (int)given : 0;
            a.counts[3] = ok ? GQA_OK : GQA_ERR_PAGES;
        }
    }
    // Every CTA has read lens, evicted and n_free once all have arrived here: the outputs may be these.
    bool last = unit == n * a.heads && rank == 0;
    if (a.in_place) {
        __syncthreads();
        if (tid == 0) {
            __threadfence();
            s.last = atomicAdd(a.ticket, 1u) == gridDim.x - 1;
            __threadfence();
            if (s.last) *a.ticket = 0;
        }
        __syncthreads();
        last = s.last;
    }
    if constexpr (kCluster) cluster_sync_all();  // none leaves while another reads its counts
    if (!last) return;
    for (int r = tid; r < n; r += kThreads) {
        const Cut c = cut_of(a, r);
        const int evicted = a.w.evicted[r];
        a.lens_out[r] = ok ? c.keep : c.len;
        a.evicted_out[r] = ok ? evicted + (c.len - c.keep) : evicted;
    }
    if (tid == 0) *a.n_free_out = ok ? n_free + (int)given : n_free;
}

// ---------------------------------------------------------------------------
// The move.
//
// A warp 32 rows of a block (page and head, of K or of V) that rows move into, eight
// warps a CTA: what moves in stays in registers between its largest magnitude and its
// new codes; where the block's scale grew the other rows' codes are rounded again.
// Rows come from past the new length and go below it, so that blocks are independent
// -- but for the page in which the new length ends, which rows leave and enter: the
// blocks of these pages are a launch of their own, behind the others.
//
// Bound by the latency of take -> table -> codes and scale -> store: 8 prompts of up to
// 16384 rows to 2000 (57 MB) 20.7 us in pages of 32, 21 of 64, 26 of 128 (int8); 64
// requests of 272 rows to 257 11.8 us, two launches.
// ---------------------------------------------------------------------------
struct EvictArgs {
    PagedCacheView c;
    KeyWeightsView w;
    const int32_t* block_table;
    int64_t table_stride;
    const int32_t *lens, *take;
    int table_width, max_keep;
    bool last_pages;
};

// A block's scale from the largest magnitude of what moves in (FP32 bits, and what rounding to them took):
// their sum over qmax, rounded once, so that a row of the largest code and the block's own scale leaves it.
__device__ __forceinline__ BlockScale moved_scale(uint32_t top, float rest, float qmax, float old) {
    if (top >= 0x7f800000u) return BlockScale{__int_as_float(0x7fffffff), 0.f, false};
    const float most = __uint_as_float(top), y = __fdiv_rn(most, qmax);
    const float mine = fmaxf(__fmaf_rn(__fadd_rn(__fmaf_rn(-y, qmax, most), rest), 1.f / qmax, y), kMinBlockScale);
    const float value = mine > old ? mine : old;
    return BlockScale{value, value == value ? __frcp_rn(value) : 0.f, mine > old};
}

// s / scale in two parts: c times both, added in one step, is c s / scale rounded to FP32 but for the last
// thousandth of a unit.  The scales of a block and of what moves into it are often in the ratio of two codes, so
// that the quotient lies half way between two others: products rounded one after the other would take either
// (e4m3 values 0.0044 of their norm from the rounded ones instead of 0.0017).
struct Ratio {
    float hi, lo;
};
__device__ __forceinline__ Ratio ratio_of(float s, const BlockScale& scale) {
    const float hi = __fmul_rn(s, scale.inv);
    return Ratio{hi, __fmul_rn(__fmaf_rn(-hi, scale.value, s), scale.inv)};
}
__device__ __forceinline__ float times(float c, const Ratio& r) { return __fmaf_rn(c, r.hi, __fmul_rn(c, r.lo)); }

// Four codes of a word as values.
template <int kCode>
__device__ __forceinline__ void values4(uint32_t w, float (&x)[4]) {
    if constexpr (kCode == GQA_CODE_INT8) {
        const uint32_t u = w ^ 0x80808080u;  // 2^23 + (c + 128) as FP32
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = __uint_as_float(__byte_perm(u, 0x4b000000u, 0x7440 + e)) - 8388736.f;
    } else {
        uint32_t lo, hi;
        to_half4<kCode>(w, lo, hi);
        const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&lo));
        const float2 b = __half22float2(*reinterpret_cast<const __half2*>(&hi));
        x[0] = a.x;
        x[1] = a.y;
        x[2] = b.x;
        x[3] = b.y;
    }
}

constexpr int kEvictWarps = 8, kWarpRows = 32, kHeldRows = kWarpRows / 4;  // (rows of a lane)

template <int kCode>
__global__ void __launch_bounds__(32 * kEvictWarps, 4) evict_kernel(const __grid_constant__ EvictArgs a) {
    __shared__ int2 s_moves[kEvictWarps][kWarpRows];
    __shared__ uint2 s_top[kEvictWarps];
    dependency_wait();
    allow_dependents();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, r = blockIdx.y, sub = lane >> 3, chunk = lane & 7;
    const int shift = a.c.page_shift, page_len = a.c.page_len;
    // Warps of a block, and this one's head and rows.
    const int split = max(1, page_len / kWarpRows), group = warp / split, row0 = (warp - group * split) * kWarpRows;
    const int h = (blockIdx.z >> 1) * (kEvictWarps / split) + group;
    const bool is_k = (blockIdx.z & 1) == 0;
    if (h >= a.c.kv_heads) return;
    // Length, page and rows are asked for together where the column is known before the length.
    const int len = a.lens[r], end = len >> shift;
    const int column = a.last_pages ? max(end, 0) : blockIdx.x;
    if (a.last_pages && (len <= 0 || column >= a.table_width || (len & (page_len - 1)) == 0)) return;
    const int32_t* table = a.block_table + r * a.table_stride;
    const int page = table[column];
    const int64_t unit = (int64_t)r * a.c.kv_heads + h;
    const int32_t* take = a.take + unit * a.max_keep;
    int2* moves = s_moves[warp];  // (row of this page, row of the request)
    uint32_t moved;
    {
        const int row = row0 + lane;
        const int64_t to = ((int64_t)column << shift) + row;
        int from = -1;
        if (row < page_len && to < a.max_keep) from = take[to];
        if (len <= 0 || (!a.last_pages && column >= end) || page < 0 || page >= a.c.pages || to >= len) from = -1;
        if (from < len || from >= (int64_t)a.table_width << shift) from = -1;
        moved = __ballot_sync(0xffffffffu, from >= 0);
        if (from >= 0) moves[__popc(moved & ((1u << lane) - 1))] = make_int2(row, from);
    }
    const int n = __popc(moved);
    // The block's warps go on together, if a row moves into any of them.
    if (!(split > 1 ? named_barrier_or(1 + group, 32 * split, n > 0) : n > 0)) return;
    __syncwarp();
    if (is_k && lane < n) {
        const int64_t to = unit * a.w.capacity + ((int64_t)column << shift) + moves[lane].x;
        const int64_t from = unit * a.w.capacity + moves[lane].y;
        if (moves[lane].y < a.w.capacity) {
            a.w.weight[to] = a.w.weight[from];
            a.w.position[to] = a.w.position[from];
        }
    }
    uint8_t* codes = (is_k ? a.c.k : a.c.v) + h * a.c.head_stride + 16 * chunk;
    float* scales = (is_k ? a.c.k_scale : a.c.v_scale) + h;
    const float qmax = kCode == GQA_CODE_INT8 ? 127.f : 448.f;
    const float old = scales[page * a.c.scale_page_stride];
    // Move i's codes (16 a lane) and scale; a page outside the cache is zeros.
    struct Row {
        uint4 w;
        float scale;
    };
    auto load = [&](int i) {
        const int from = moves[i].y, at = table[from >> shift];
        if (at < 0 || at >= a.c.pages) return Row{make_uint4(0u, 0u, 0u, 0u), 0.f};
        return Row{*reinterpret_cast<const uint4*>(codes + at * a.c.page_stride +
                                                   (from & (page_len - 1)) * a.c.row_stride),
                   scales[at * a.c.scale_page_stride]};
    };
    float most = 0.f, most_rest = 0.f;  // the largest magnitude, and what rounding it to FP32 took
    bool fine = true;
    auto measure = [&](const Row& x) {
        const uint32_t ws[4] = {x.w.x, x.w.y, x.w.z, x.w.w};
        __half2 top = __half2half2(__ushort_as_half(0));
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            uint32_t lo, hi;
            to_half4<kCode>(ws[i], lo, hi);
            top = __hmax2(top, __habs2(*reinterpret_cast<const __half2*>(&lo)));
            top = __hmax2(top, __habs2(*reinterpret_cast<const __half2*>(&hi)));
        }
        const float m = __half2float(__hmax(__low2half(top), __high2half(top)));
        const float v = __fmul_rn(m, x.scale);
        if (v > most) {
            most = v;
            most_rest = __fmaf_rn(m, x.scale, -v);
        }
        fine &= x.scale <= 3.402823466e38f;  // (a block of NaN scale)
    };
    Row held[kHeldRows];
#pragma unroll
    for (int i = 0; i < kHeldRows; ++i) {
        held[i].scale = 0.f;
        if (4 * i + sub < n) held[i] = load(4 * i + sub);
    }
#pragma unroll
    for (int i = 0; i < kHeldRows; ++i)
        if (4 * i + sub < n) measure(held[i]);
    uint32_t top = __reduce_max_sync(0xffffffffu, fine ? __float_as_uint(most) : 0x7f800000u);
    if (__float_as_uint(most) != top) most_rest = -INFINITY;
#pragma unroll
    for (int d = 16; d; d >>= 1) most_rest = fmaxf(most_rest, __shfl_xor_sync(0xffffffffu, most_rest, d));
    if (split > 1) {
        if (lane == 0) s_top[warp] = make_uint2(top, __float_as_uint(most_rest));
        // (Also: every warp of the block has read its rows, wherever they come from, and the old scale.)
        named_barrier_sync(1 + group, 32 * split);
        for (int w = group * split; w < (group + 1) * split; ++w) {
            const uint2 x = s_top[w];
            if (x.x > top || (x.x == top && __uint_as_float(x.y) > most_rest)) {
                top = x.x;
                most_rest = __uint_as_float(x.y);
            }
        }
    }
    const BlockScale scale = moved_scale(top, most_rest, qmax, old);
    const bool number = scale.value == scale.value;
    auto codes16 = [&](const uint4& w, float s) {
        if (!number) return make_uint4(0u, 0u, 0u, 0u);
        if (s == scale.value) return w;
        const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
        const Ratio ratio = ratio_of(s, scale);
        uint32_t o[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float y[4];
            values4<kCode>(ws[i], y);
#pragma unroll
            for (int e = 0; e < 4; ++e) y[e] = times(y[e], ratio);
            o[i] = value_codes4<kCode>(y[0], y[1], y[2], y[3]);
        }
        return make_uint4(o[0], o[1], o[2], o[3]);
    };
    uint8_t* block = codes + page * a.c.page_stride;
    auto store = [&](int i, const Row& x) {
        *reinterpret_cast<uint4*>(block + moves[i].x * a.c.row_stride) = codes16(x.w, x.scale);
    };
#pragma unroll
    for (int i = 0; i < kHeldRows; ++i)
        if (4 * i + sub < n) store(4 * i + sub, held[i]);
    __syncwarp();  // rows of this very page have been read, and the old scale
    if (scale.grew)
        for (int row = row0 + sub; row < min(page_len, row0 + kWarpRows); row += 4) {
            if (moved >> (row - row0) & 1) continue;
            uint4* at = reinterpret_cast<uint4*>(block + row * a.c.row_stride);
            *at = codes16(*at, old);
        }
    if (lane == 0 && row0 == 0) scales[page * a.c.scale_page_stride] = scale.value;
}

// How many CTAs a (request, head) gets goes by the rows that it may hold (its lengths are in device memory): stretches
// of 4096 and more fill a CTA's time beside what a cluster's barriers cost, as long as there are SMs for them.
template <int kThreads, bool kCluster>
cudaError_t launch_plan(const EvictPlanArgs& a, int ctas, size_t smem, cudaStream_t stream) {
    const auto kernel = plan_eviction_kernel<kThreads, kCluster>;
    // The limit is the kernel's, not the call's: always the same, so that another thread's call does not lower it.
    if (smem > 16 * 1024) {
        const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxRows * (int)sizeof(uint32_t));
        if (e != cudaSuccess) return e;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)((a.requests * a.heads + 1) * ctas));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = (unsigned)ctas;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = kCluster ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, kernel, a);
}

cudaError_t launch_plan_eviction(EvictPlanArgs& a, int sms, cudaStream_t stream) {
    const int64_t most = std::min<int64_t>(a.w.capacity, (int64_t)a.table_width << a.page_shift);
    const int units = a.requests * a.heads;
    int ctas = 1;
    while (ctas < kMaxCluster && most >= 8192 * (int64_t)ctas && units * ctas * 2 <= 2 * sms) ctas *= 2;
    const bool small = most <= 2048;
    const int step = small ? 512 : 2048;  // whole steps of a CTA's warps
    const int64_t rows = ((most + ctas - 1) / ctas + step - 1) / step * step;
    a.held_rows = (int)std::min<int64_t>(rows, kMaxRows);
    const size_t smem = a.held_rows * sizeof(uint32_t);
    if (small) return launch_plan<128, false>(a, 1, smem, stream);
    return ctas > 1 ? launch_plan<512, true>(a, ctas, smem, stream) : launch_plan<512, false>(a, 1, smem, stream);
}

bool aligned4(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 3u) == 0; }

int check_key_weights(const gqa_key_weights* w, KeyWeightsView* v) {
    if (!w || !w->weight || !w->position || !w->evicted) return GQA_ERR_NULL_POINTER;
    if (!aligned4(w->weight) || !aligned4(w->position) || !aligned4(w->evicted)) return GQA_ERR_ALIGNMENT;
    if (w->capacity < 1 || w->capacity > 1 << 30) return GQA_ERR_KV_RANGE;
    *v = KeyWeightsView{w->weight, w->position, w->evicted, w->capacity};
    return check_device_memory({w->weight, w->position, w->evicted});
}

}  // namespace

}  // namespace gqa

using namespace gqa;

extern "C" {

size_t gqa_plan_eviction_workspace_bytes(int requests, int kv_heads, int max_keep) {
    if (requests < 1 || requests > GQA_PAGED_MAX_BATCH || kv_heads < 1 || kv_heads > kNumKVHeads || max_keep < 1 ||
        max_keep > 1 << 30)
        return 0;
    return 256 + (size_t)requests * kv_heads * 2 * max_keep * sizeof(int32_t);
}

int gqa_plan_eviction(const gqa_key_weights* weights, int kv_heads, const int32_t* lens, const int32_t* keep, int requests,
                      const int32_t* block_table, int64_t table_stride, int table_width, int32_t* free_pages,
                      int free_capacity, const int32_t* n_free, int page_len, int max_keep, int sinks, int recent,
                      int32_t* take, int32_t* lens_out, int32_t* evicted_out, int32_t* n_free_out, int32_t* counts,
                      void* workspace, size_t workspace_bytes, void* stream) {
    if (!lens || !keep || !block_table || !free_pages || !n_free || !take || !lens_out || !evicted_out || !n_free_out ||
        !counts)
        return GQA_ERR_NULL_POINTER;
    EvictPlanArgs a;
    int st = check_key_weights(weights, &a.w);
    if (st != GQA_OK) return st;
    if (kv_heads < 1 || kv_heads > kNumKVHeads) return GQA_ERR_KV_HEADS;
    if (requests < 1 || requests > GQA_PAGED_MAX_BATCH || table_width < 1 || free_capacity < 0 || max_keep < 1 ||
        max_keep > 1 << 30 || sinks < 0 || recent < 0 || (requests > 1 && table_stride < table_width))
        return GQA_ERR_BATCH;
    int shift = 4;
    while (shift < 7 && (1 << shift) != page_len) ++shift;
    if ((1 << shift) != page_len) return GQA_ERR_KV_BLOCK_LEN;
    if (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 15u) ||
        workspace_bytes < gqa_plan_eviction_workspace_bytes(requests, kv_heads, max_keep))
        return GQA_ERR_WORKSPACE;
    int sms = 0;
    st = device_sms(&sms);
    if (st != GQA_OK) return st;
    st = check_device_memory({lens, keep, block_table, free_pages, n_free, take, lens_out, evicted_out, n_free_out, counts,
                              workspace});
    if (st != GQA_OK) return st;
    a.lens = lens;
    a.keep = keep;
    a.block_table = block_table;
    a.table_stride = table_stride;
    a.free_pages = free_pages;
    a.n_free = n_free;
    a.take = take;
    a.lens_out = lens_out;
    a.evicted_out = evicted_out;
    a.n_free_out = n_free_out;
    a.counts = counts;
    a.ticket = static_cast<uint32_t*>(workspace) + 1;
    a.lists = static_cast<int32_t*>(workspace) + 64;
    a.requests = requests;
    a.heads = kv_heads;
    a.table_width = table_width;
    a.free_capacity = free_capacity;
    a.page_shift = shift;
    a.max_keep = max_keep;
    a.sinks = sinks;
    a.recent = recent;
    auto overlap = [](const int32_t* x, int64_t nx, const int32_t* y, int64_t ny) { return x < y + ny && y < x + nx; };
    a.in_place = false;
    for (const int32_t* out : {lens_out, evicted_out})
        a.in_place |= overlap(out, requests, lens, requests) || overlap(out, requests, keep, requests) ||
                      overlap(out, requests, weights->evicted, requests) || overlap(out, requests, n_free, 1);
    a.in_place |= overlap(n_free_out, 1, n_free, 1) || overlap(n_free_out, 1, lens, requests) ||
                  overlap(n_free_out, 1, keep, requests) || overlap(n_free_out, 1, weights->evicted, requests);
    a.vectors = weights->capacity % 4 == 0 && !((reinterpret_cast<uintptr_t>(a.w.weight) | reinterpret_cast<uintptr_t>(a.w.position)) & 15u);
    return launch_plan_eviction(a, sms, static_cast<cudaStream_t>(stream)) == cudaSuccess ? GQA_OK : GQA_ERR_CUDA;
}

int gqa_evict_paged(const gqa_paged_cache* cache, const int32_t* block_table, int64_t table_stride, int table_width,
                    const gqa_key_weights* weights, const int32_t* lens, const int32_t* take, int requests, int max_keep,
                    void* stream) {
    if (!cache || !block_table || !lens || !take) return GQA_ERR_NULL_POINTER;
    EvictArgs a;
    int st = check_paged_cache(cache, &a.c);
    if (st != GQA_OK) return st;
    st = check_key_weights(weights, &a.w);
    if (st != GQA_OK) return st;
    if (requests < 1 || requests > GQA_PAGED_MAX_BATCH || table_width < 1 || max_keep < 1 || max_keep > 1 << 30 ||
        (requests > 1 && table_stride < table_width) || (int64_t)table_width * cache->page_len > 1 << 30)
        return GQA_ERR_BATCH;
    int sms = 0;
    st = device_sms(&sms);
    if (st != GQA_OK) return st;
    st = check_device_memory({cache->k, cache->v, cache->k_scale, cache->v_scale, block_table, lens, take});
    if (st != GQA_OK) return st;
    a.block_table = block_table;
    a.table_stride = table_stride;
    a.lens = lens;
    a.take = take;
    a.table_width = table_width;
    a.max_keep = max_keep;
    const int columns = (max_keep + cache->page_len - 1) / cache->page_len;
    const int heads = kEvictWarps / (cache->page_len > kWarpRows ? cache->page_len / kWarpRows : 1);  // of a CTA
    const int groups = (cache->kv_heads + heads - 1) / heads;
    const auto kernel = cache->code == GQA_CODE_INT8 ? evict_kernel<GQA_CODE_INT8> : evict_kernel<GQA_CODE_E4M3>;
    cudaError_t e = cudaSuccess;
    for (int last = 0; last < 2 && e == cudaSuccess; ++last) {
        a.last_pages = last != 0;
        e = launch_dependent(kernel, dim3(last ? 1 : columns < table_width ? columns : table_width, requests, 2 * groups),
                             32 * kEvictWarps, 0, static_cast<cudaStream_t>(stream), a);
    }
    return e == cudaSuccess ? GQA_OK : GQA_ERR_CUDA;
}

}  // extern "C"
