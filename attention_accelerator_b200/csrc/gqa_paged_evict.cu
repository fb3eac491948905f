// gqa_paged_evict.cu -- eviction from the paged 8-bit cache: the choice of the rows that
// stay, by their accumulated attention weight, and the move of those that fill the holes.
#include "gqa_internal.h"
#include "gqa_paged.cuh"
#include "gqa_paged_internal.h"

namespace gqa {

namespace {

// ---------------------------------------------------------------------------
// The choice.
//
// A CTA a (request, KV head).  A row's rank is that of a 32-bit number: the bits of its
// weight, which order as the weights do (they are not negative), and above them whether
// it is spared.  Three passes over histograms of 11, 11 and 10 bits, from the top, find
// the number of the last row that stays and how many rows of that very number stay; one
// more pass, in the order of rows, marks them, counts holes below `keep` and rows that
// stay past it, and pairs them off.  One more CTA gives the pages back.
// ---------------------------------------------------------------------------
constexpr int kThreads = 512, kWarps = kThreads / 32;
constexpr int kEach = 4;  // rows of a thread at a time
constexpr int kBins = 2048;

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
};

struct Cut {
    int len, keep;  // rows held and rows that stay (keep == len: left as it is)
};
__device__ __forceinline__ Cut cut_of(const EvictPlanArgs& a, int r) {
    const int len = a.lens[r], keep = min(a.keep[r], a.max_keep);
    return Cut{len, keep > 0 && keep < len ? keep : len};
}

// The sum over the CTA of values a thread, and of those before it.
struct Sum {
    int before, all;
};
__device__ __forceinline__ Sum block_sum(int v, int* warp_sum) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int incl = v;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, incl, d);
        if (lane >= d) incl += x;
    }
    __syncthreads();
    if (lane == 31) warp_sum[warp] = incl;
    __syncthreads();
    Sum s{incl - v, 0};
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
        const int x = warp_sum[w];
        s.all += x;
        if (w < warp) s.before += x;
    }
    return s;
}

__device__ __forceinline__ uint32_t rank_of(const EvictPlanArgs& a, float weight, int position, int64_t recent_from) {
    const uint32_t bits = __float_as_uint(weight);
    const uint32_t w = weight != weight ? 0x7fffffffu : bits & 0x80000000u ? 0u : bits;
    return w | (position < a.sinks || position >= recent_from ? 0x80000000u : 0u);
}

__device__ void choose(const EvictPlanArgs& a, int r, int h, const Cut& cut, int* hist, int* warp_sum) {
    __shared__ uint32_t s_bin, s_left;
    const int tid = threadIdx.x;
    const int64_t unit = (int64_t)r * a.heads + h;
    const float* weight = a.w.weight + unit * a.w.capacity;
    const int32_t* position = a.w.position + unit * a.w.capacity;
    const int64_t recent_from = (int64_t)cut.len + min(max(a.w.evicted[r], 0), 1 << 30) - a.recent;
    const int len = cut.len, keep = cut.keep;
    auto number = [&](int i) { return rank_of(a, weight[i], position[i], recent_from); };

    uint32_t found = 0, known = 0;  // the number's upper bits, and which these are
    uint32_t left = (uint32_t)keep; // rows that stay among those which agree with it so far
    constexpr int kShift[3] = {21, 10, 0};
#pragma unroll
    for (int pass = 0; pass < 3; ++pass) {
        const int shift = kShift[pass];
        const uint32_t mask = pass == 2 ? 1023u : 2047u;
        for (int i = tid; i < kBins; i += kThreads) hist[i] = 0;
        __syncthreads();
        for (int i = tid; i < len; i += kThreads) {
            const uint32_t x = number(i);
            if ((x & known) == found) atomicAdd(&hist[x >> shift & mask], 1);
        }
        __syncthreads();
        // From the highest bin down: the one in which the count passes what is left.
        constexpr int kOf = kBins / kThreads;
        int count[kOf], sum = 0;
#pragma unroll
        for (int i = 0; i < kOf; ++i) {
            count[i] = hist[kBins - 1 - (tid * kOf + i)];
            sum += count[i];
        }
        uint32_t before = (uint32_t)block_sum(sum, warp_sum).before;
#pragma unroll
        for (int i = 0; i < kOf; ++i) {
            if (before < left && left <= before + count[i]) {
                s_bin = (uint32_t)(kBins - 1 - (tid * kOf + i));
                s_left = left - before;
            }
            before += count[i];
        }
        __syncthreads();
        found |= s_bin << shift;
        known |= mask << shift;
        left = s_left;
    }

    int32_t* holes = a.lists + unit * 2 * a.max_keep;
    int32_t* fills = holes + a.max_keep;
    int32_t* take = a.take + unit * a.max_keep;
    int equal = 0, n_holes = 0, n_fills = 0;  // of all rows before: of the very number, holes, rows that fill them
    for (int i0 = 0; i0 < len; i0 += kThreads * kEach) {
        const int first = i0 + tid * kEach;
        uint32_t x[kEach];
        int same = 0;
#pragma unroll
        for (int e = 0; e < kEach; ++e) {
            x[e] = first + e < len ? number(first + e) : 0u;
            same += first + e < len && x[e] == found;
        }
        const Sum ties = block_sum(same, warp_sum);
        int tie = equal + ties.before;
        equal += ties.all;
        bool mark[kEach];
        int marks = 0;  // holes, and from bit 16 on rows that fill them
        static_assert(kThreads * kEach < 32768, "15 bits of each");
#pragma unroll
        for (int e = 0; e < kEach; ++e) {
            const int i = first + e;
            bool stays = i < len && x[e] > found;
            if (i < len && x[e] == found) stays = (uint32_t)tie++ < left;
            mark[e] = i < len && stays == (i >= keep);
            if (mark[e]) marks += i < keep ? 1 : 1 << 16;
        }
        const Sum both = block_sum(marks, warp_sum);
        int at_hole = n_holes + (both.before & 0xffff), at_fill = n_fills + (both.before >> 16);
        n_holes += both.all & 0xffff;
        n_fills += both.all >> 16;
#pragma unroll
        for (int e = 0; e < kEach; ++e) {
            const int i = first + e;
            if (i < keep) take[i] = -1;
            if (mark[e]) {
                if (i < keep) holes[at_hole++] = i; else fills[at_fill++] = i;
            }
        }
    }
    for (int i = keep + tid; i < a.max_keep; i += kThreads) take[i] = -1;
    __syncthreads();
    for (int i = tid; i < n_holes; i += kThreads) take[holes[i]] = fills[i];
}

__global__ void __launch_bounds__(kThreads) plan_eviction_kernel(const __grid_constant__ EvictPlanArgs a) {
    __shared__ int hist[kBins];
    __shared__ int warp_sum[kWarps];
    __shared__ bool s_last;
    const int tid = threadIdx.x, n = a.requests;
    const int page_mask = (1 << a.page_shift) - 1;
    auto pages_of = [&](int len) { return (int)(((int64_t)len + page_mask) >> a.page_shift); };
    const int n_free = *a.n_free;
    // All or nothing: every CTA looks at all requests.
    const int per = (n + kThreads - 1) / kThreads, r0 = min(n, tid * per), r1 = min(n, r0 + per);
    bool bad = false;
    int give = 0;
    for (int r = r0; r < r1; ++r) {
        const Cut c = cut_of(a, r);
        bad |= c.len < 0 || pages_of(c.len) > a.table_width || c.len > a.w.capacity;
        if (!bad) give += pages_of(c.len) - pages_of(c.keep);
    }
    bad = __syncthreads_or(bad);
    const Sum gives = block_sum(bad ? 0 : give, warp_sum);
    const bool ok = !bad && n_free >= 0 && (int64_t)n_free + gives.all <= a.free_capacity;

    if ((int)blockIdx.x < n * a.heads) {
        const int r = blockIdx.x / a.heads, h = blockIdx.x - r * a.heads;
        const Cut cut = cut_of(a, r);
        if (ok && cut.keep < cut.len) {
            choose(a, r, h, cut, hist, warp_sum);
        } else {
            int32_t* take = a.take + (int64_t)blockIdx.x * a.max_keep;
            for (int i = tid; i < a.max_keep; i += kThreads) take[i] = -1;
        }
    } else {
        int at = gives.before, cuts = 0, rows = 0;
        for (int r = r0; r < r1 && ok; ++r) {
            const Cut c = cut_of(a, r);
            cuts += c.keep < c.len;
            rows += c.len - c.keep;
            const int32_t* row = a.block_table + r * a.table_stride;
            for (int j = pages_of(c.keep); j < pages_of(c.len); ++j) a.free_pages[n_free + at++] = row[j];
        }
        cuts = block_sum(cuts, warp_sum).all;
        rows = block_sum(rows, warp_sum).all;
        if (tid == 0) {
            a.counts[0] = cuts;
            a.counts[1] = rows;
            a.counts[2] = ok ? gives.all : 0;
            a.counts[3] = ok ? GQA_OK : GQA_ERR_PAGES;
        }
    }
    // Every CTA has read lens, evicted and n_free once all have arrived here: the outputs may be these.
    __syncthreads();
    if (tid == 0) {
        __threadfence();
        s_last = atomicAdd(a.ticket, 1u) == gridDim.x - 1;
        __threadfence();
        if (s_last) *a.ticket = 0;
    }
    __syncthreads();
    if (!s_last) return;
    for (int r = tid; r < n; r += kThreads) {
        const Cut c = cut_of(a, r);
        const int evicted = a.w.evicted[r];
        a.lens_out[r] = ok ? c.keep : c.len;
        a.evicted_out[r] = ok ? evicted + (c.len - c.keep) : evicted;
    }
    if (tid == 0) *a.n_free_out = ok ? n_free + gives.all : n_free;
}

// ---------------------------------------------------------------------------
// The move.
//
// A warp a block (page and head, of K or of V) that rows move into: their largest
// magnitude, the block's new scale, their codes, and where the scale grew the other
// rows' codes again.  Rows come from past the new length and go below it, so that
// blocks are independent -- but for the page in which the new length ends, which
// rows leave and enter: the blocks of these pages are a launch of their own, behind
// the others.
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

// c s / scale, rounded to FP32 but for the last half of a thousandth of a unit.  The scales of a block and of
// what moves into it are often in the ratio of two codes, so that the quotient lies half way between two
// others: products rounded one after the other would take either (outputs twice as far from the rounded
// values of e4m3).
__device__ __forceinline__ float over_scale(float c, float s, const BlockScale& scale) {
    const float x = __fmul_rn(c, s), x_rest = __fmaf_rn(c, s, -x);
    const float y = __fmul_rn(x, scale.inv);
    return __fmaf_rn(__fadd_rn(__fmaf_rn(-y, scale.value, x), x_rest), scale.inv, y);
}

constexpr int kHeldRows = 8;  // rows of a lane that stay in registers between the two passes

template <int kCode>
__global__ void __launch_bounds__(256) evict_kernel(const __grid_constant__ EvictArgs a) {
    __shared__ int2 s_moves[kNumKVHeads][kPagedMaxPage];
    dependency_wait();
    allow_dependents();
    const int lane = threadIdx.x & 31, h = threadIdx.x >> 5, r = blockIdx.y, sub = lane >> 3, chunk = lane & 7;
    const bool is_k = blockIdx.z == 0;
    const int shift = a.c.page_shift, page_len = a.c.page_len, len = a.lens[r], end = len >> shift;
    const int column = a.last_pages ? end : blockIdx.x;
    if (len <= 0 || column >= a.table_width || (a.last_pages ? (len & (page_len - 1)) == 0 : column >= end)) return;
    const int32_t* table = a.block_table + r * a.table_stride;
    const int page = table[column];
    if (page < 0 || page >= a.c.pages) return;
    const int64_t unit = (int64_t)r * a.c.kv_heads + h;
    const int32_t* take = a.take + unit * a.max_keep;
    int2* moves = s_moves[h];  // (row of this page, row of the request)
    int n = 0;
    uint32_t moved[kPagedMaxPage / 32];
#pragma unroll
    for (int i = 0; i < kPagedMaxPage / 32; ++i) {
        const int row = 32 * i + lane;
        const int64_t to = ((int64_t)column << shift) + row;
        int from = -1;
        if (row < page_len && to < a.max_keep && to < len) from = take[to];
        if (from < len || from >= (int64_t)a.table_width << shift) from = -1;
        moved[i] = __ballot_sync(0xffffffffu, from >= 0);
        if (from >= 0) moves[n + __popc(moved[i] & ((1u << lane) - 1))] = make_int2(row, from);
        n += __popc(moved[i]);
    }
    if (n == 0) return;
    __syncwarp();
    if (is_k)
        for (int i = lane; i < n; i += 32) {
            const int64_t to = unit * a.w.capacity + ((int64_t)column << shift) + moves[i].x;
            const int64_t from = unit * a.w.capacity + moves[i].y;
            if (moves[i].y < a.w.capacity) {
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
    auto code = [](const uint4& w, int e) {
        const uint32_t x = e < 4 ? w.x : e < 8 ? w.y : e < 12 ? w.z : w.w;
        return code_value<kCode>((uint8_t)(x >> (8 * (e & 3))));
    };
    float most = 0.f, most_rest = 0.f;  // the largest magnitude, and what rounding it to FP32 took
    bool fine = true;
    auto measure = [&](const Row& x) {
        float m = 0.f;
#pragma unroll
        for (int e = 0; e < 16; ++e) m = fmaxf(m, fabsf(code(x.w, e)));
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
    for (int i = 4 * kHeldRows + sub; i < n; i += 4) measure(load(i));
    const uint32_t top = __reduce_max_sync(0xffffffffu, fine ? __float_as_uint(most) : 0x7f800000u);
    if (__float_as_uint(most) != top) most_rest = -INFINITY;
#pragma unroll
    for (int d = 16; d; d >>= 1) most_rest = fmaxf(most_rest, __shfl_xor_sync(0xffffffffu, most_rest, d));
    const BlockScale scale = moved_scale(top, most_rest, qmax, old);
    const bool number = scale.value == scale.value;
    auto codes16 = [&](const uint4& w, float s) {
        uint32_t o[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float y[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) y[e] = number ? over_scale(code(w, 4 * i + e), s, scale) : 0.f;
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
    for (int i = 4 * kHeldRows + sub; i < n; i += 4) store(i, load(i));
    __syncwarp();  // rows of this very page have been read, and the old scale
    if (scale.grew)
        for (int row = sub; row < page_len; row += 4) {
            if (moved[row >> 5] >> (row & 31) & 1) continue;
            uint4* at = reinterpret_cast<uint4*>(block + row * a.c.row_stride);
            *at = codes16(*at, old);
        }
    if (lane == 0) scales[page * a.c.scale_page_stride] = scale.value;
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
    plan_eviction_kernel<<<requests * kv_heads + 1, kThreads, 0, static_cast<cudaStream_t>(stream)>>>(a);
    return cudaGetLastError() == cudaSuccess ? GQA_OK : GQA_ERR_CUDA;
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
    const auto kernel = cache->code == GQA_CODE_INT8 ? evict_kernel<GQA_CODE_INT8> : evict_kernel<GQA_CODE_E4M3>;
    cudaError_t e = cudaSuccess;
    for (int last = 0; last < 2 && e == cudaSuccess; ++last) {
        a.last_pages = last != 0;
        e = launch_dependent(kernel, dim3(last ? 1 : columns < table_width ? columns : table_width, requests, 2),
                             32 * cache->kv_heads, 0, static_cast<cudaStream_t>(stream), a);
    }
    return e == cudaSuccess ? GQA_OK : GQA_ERR_CUDA;
}

}  // extern "C"
