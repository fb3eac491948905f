// gqa_paged.cu -- the paged 8-bit KV cache: argument checks of its C entry
// points, page planning, append (RoPE, quantisation) and read-back kernels.
#include "gqa_paged.cuh"
#include "gqa_internal.h"
#include "gqa_paged_internal.h"
#include "gqa_paged_units.cuh"

#include <cmath>
#include <cstring>

namespace gqa {

namespace {

// ---------------------------------------------------------------------------
// Page planning.
//
// Three running sums over the requests (new tokens, pages needed, pages given
// back) place everything: every CTA computes them all in shared memory -- a few
// KB of reads from L2, cheaper than a second launch or a wait between CTAs --
// and then fills its share of the slots, table entries and stack entries, each
// found by a binary search in the sums.  A popped page comes from the pages
// given back in this very call or from below them on the stack, so no CTA reads
// what another writes.  lens_out and n_free_out may be the inputs: the last CTA
// to have read those writes them.
//
// Bound by latency: two chains of loads, the sums' barriers and the search, 6.5 us
// for 64 requests, 9.7 for 1024 with 66 thousand tokens (1.6 MB), in a replayed graph.
// ---------------------------------------------------------------------------
constexpr int kPlanThreads = 1024;

struct PlanArgs {
    const int32_t *lens, *new_lens;
    int32_t* block_table;
    int64_t table_stride;
    int32_t* free_pages;
    const int32_t* n_free;
    int32_t *lens_out, *n_free_out, *first_token;
    int64_t* slots;
    int32_t *positions, *counts;
    uint32_t* ticket;
    int32_t requests, table_width, free_capacity, page_shift, max_tokens;
};

// Last index r in [0, n) with first[r] <= x (first is non-decreasing, first[0] = 0).
__device__ __forceinline__ int last_at_most(const int32_t* first, int n, int x) {
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (first[mid] <= x) lo = mid; else hi = mid;
    }
    return lo;
}

__global__ void __launch_bounds__(kPlanThreads) plan_pages_kernel(const __grid_constant__ PlanArgs a) {
    extern __shared__ int32_t sums[];  // tokens, needs, gives: [requests + 1] each
    __shared__ long long warp_sum[3][32];
    __shared__ int s_bad;
    __shared__ bool s_last;
    const int n = a.requests, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    int32_t* tokens = sums;
    int32_t* needs = sums + (n + 1);
    int32_t* gives = sums + 2 * (n + 1);
    const int page_mask = (1 << a.page_shift) - 1;
    auto pages_of = [&](long long len) { return (int)((len + page_mask) >> a.page_shift); };
    if (tid == 0) s_bad = 0;
    const int n_free = *a.n_free;
    __syncthreads();

    // Each thread sums a stretch of consecutive requests, then the block scans the stretches.
    const int per = (n + kPlanThreads - 1) / kPlanThreads;
    const int r0 = min(n, tid * per), r1 = min(n, r0 + per);
    long long sum[3] = {0, 0, 0};
    bool bad = false;
    for (int r = r0; r < r1; ++r) {
        const int len = a.lens[r], add = a.new_lens[r];
        bad |= len < 0 || pages_of(len) > a.table_width;
        if (add < 0) {
            sum[2] += pages_of(len);
        } else {
            const long long after = (long long)len + add;
            bad |= after > 0x7FFFFFFF || pages_of(after) > a.table_width;
            sum[0] += add;
            sum[1] += pages_of(after) - pages_of(len);
        }
    }
    long long incl[3] = {sum[0], sum[1], sum[2]};
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
#pragma unroll
        for (int i = 0; i < 3; ++i) {
            const long long x = __shfl_up_sync(0xffffffffu, incl[i], d);
            if (lane >= d) incl[i] += x;
        }
    }
    if (lane == 31)
        for (int i = 0; i < 3; ++i) warp_sum[i][warp] = incl[i];
    if (bad) s_bad = 1;
    __syncthreads();
    long long total[3], base[3];
#pragma unroll
    for (int i = 0; i < 3; ++i) {
        total[i] = warp_sum[i][lane];
        base[i] = lane < warp ? total[i] : 0;
#pragma unroll
        for (int d = 16; d; d >>= 1) {
            total[i] += __shfl_xor_sync(0xffffffffu, total[i], d);
            base[i] += __shfl_xor_sync(0xffffffffu, base[i], d);
        }
    }
    // All or nothing.  (The sums in shared memory are 32-bit: with `ok` they fit.)
    const bool ok = !s_bad && n_free >= 0 && total[0] <= a.max_tokens && n_free + total[2] <= a.free_capacity &&
                    total[1] <= n_free + total[2];
    {
        long long at[3] = {base[0] + incl[0] - sum[0], base[1] + incl[1] - sum[1], base[2] + incl[2] - sum[2]};
        for (int r = r0; r < r1; ++r) {
            const int len = a.lens[r], add = a.new_lens[r];
            tokens[r] = ok ? (int32_t)at[0] : 0;
            needs[r] = (int32_t)at[1];
            gives[r] = (int32_t)at[2];
            if (add < 0) {
                at[2] += pages_of(len);
            } else {
                at[0] += add;
                at[1] += pages_of((long long)len + add) - pages_of(len);
            }
        }
        if (tid == 0) {
            tokens[n] = ok ? (int32_t)total[0] : 0;
            needs[n] = (int32_t)total[1];
            gives[n] = (int32_t)total[2];
        }
    }
    __syncthreads();

    // (Unsigned: max_tokens and the stack may come within a step of 2^31.)
    const uint32_t stride = gridDim.x * kPlanThreads, first = blockIdx.x * kPlanThreads + tid;
    const int n_tokens = tokens[n], n_need = ok ? needs[n] : 0, n_give = ok ? gives[n] : 0;
    for (uint32_t r = first; r <= (uint32_t)n; r += stride) a.first_token[r] = tokens[r];
    // Page given back number i: its request is the last whose sum is at most i
    // and which gives any (requests that give none repeat the next one's sum).
    auto given = [&](int i) {
        const int r = last_at_most(gives, n, i);
        return a.block_table[r * a.table_stride + (i - gives[r])];
    };
    // Page popped number j: the top of the stack with this call's pages pushed on it.
    auto popped = [&](int j) { return j < n_give ? given(n_give - 1 - j) : a.free_pages[n_free - 1 - (j - n_give)]; };
    for (uint32_t t = first; t < (uint32_t)a.max_tokens; t += stride) {
        int64_t slot = -1;
        int pos = -1;
        if (t < (uint32_t)n_tokens) {
            const int r = last_at_most(tokens, n, (int)t);
            const int len = a.lens[r], held = pages_of(len);
            pos = len + ((int)t - tokens[r]);
            const int col = pos >> a.page_shift;
            const int page = col < held ? a.block_table[r * a.table_stride + col] : popped(needs[r] + col - held);
            slot = ((int64_t)page << a.page_shift) + (pos & page_mask);
        }
        a.slots[t] = slot;
        a.positions[t] = pos;
    }
    for (uint32_t j = first; j < (uint32_t)n_need; j += stride) {
        const int r = last_at_most(needs, n, (int)j);
        a.block_table[r * a.table_stride + pages_of(a.lens[r]) + ((int)j - needs[r])] = popped((int)j);
    }
    for (uint32_t i = first; i < (uint32_t)n_give; i += stride) a.free_pages[n_free + (int)i] = given((int)i);
    if (blockIdx.x == 0 && tid == 0) {
        a.counts[0] = n_tokens;
        a.counts[1] = n_need;
        a.counts[2] = n_give;
        a.counts[3] = ok ? GQA_OK : GQA_ERR_PAGES;
    }
    // Every CTA has read lens and n_free once all have arrived here.
    __syncthreads();
    if (tid == 0) {
        bool last = true;
        if (gridDim.x > 1) {
            __threadfence();
            last = atomicAdd(a.ticket, 1u) == gridDim.x - 1;
            __threadfence();
            if (last) *a.ticket = 0;
        }
        s_last = last;
    }
    __syncthreads();
    if (!s_last) return;
    for (int r = tid; r < n; r += kPlanThreads) {
        const int len = a.lens[r], add = a.new_lens[r];
        a.lens_out[r] = !ok ? len : add < 0 ? 0 : len + add;
    }
    if (tid == 0) *a.n_free_out = ok ? n_free + n_give - n_need : n_free;
}

// ---------------------------------------------------------------------------
// Append: RoPE of K, quantisation, and the rescale of a page's earlier codes.
//
// Two kernels: a step's rows, and prompts.  Measured: a step's 64 rows 3.5 us, bound by
// latency (6.0 in pages of 64, 8.9 in pages of 128, where every block's scale grows and
// its rows are rounded again, one after the other); 18000 rows in pages of 32 33 us (111 MB, 3.3 TB/s), of 64, e4m3, 34, of 128
// 40, of 16 39, bound by the latency of a run's steps at 16 warps an SM.  With a head
// after the other in a CTA, a barrier each and the rows in 256-byte pieces, they took 42,
// 45, 60 and 46.
// ---------------------------------------------------------------------------
struct AppendArgs {
    PagedCacheView c;
    const __nv_bfloat16 *k, *v;
    int64_t k_tstride, k_hstride, v_tstride, v_hstride;
    const int64_t* slots;
    const int32_t* positions;
    int n_tokens;
    RopeSteps rope;
};

constexpr int kWindow = 16;  // tokens of a prompt in which a CTA looks for runs
constexpr float kMinBlockScale = 0x1p-100f;  // keeps 1 / scale finite for a block of zeros

template <int kCode>
__device__ __forceinline__ uint2 encode8(const float* x, float inv) {
    return make_uint2(value_codes4<kCode>(__fmul_rn(x[0], inv), __fmul_rn(x[1], inv), __fmul_rn(x[2], inv), __fmul_rn(x[3], inv)),
                      value_codes4<kCode>(__fmul_rn(x[4], inv), __fmul_rn(x[5], inv), __fmul_rn(x[6], inv), __fmul_rn(x[7], inv)));
}

__device__ __forceinline__ void unpack8(uint4 w, float* x) {
    const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = bf16x2_to_float2(ws[i]);
        x[2 * i] = f.x;
        x[2 * i + 1] = f.y;
    }
}

// Rows of the run that starts at token t0: up to the page's end, the call's end or the
// first slot that does not follow.  By a whole warp.
__device__ __forceinline__ int run_length(const AppendArgs& a, int t0, int64_t slot, int room) {
    const int lane = threadIdx.x & 31;
    int len = 0;
    for (int at = 0; at < room; at += 32) {
        const int i = at + lane;
        const bool in = i < room && i < a.n_tokens - t0 && a.slots[t0 + i] == slot + i;
        const unsigned miss = ~__ballot_sync(0xffffffffu, in);
        len += miss ? __ffs(miss) - 1 : 32;
        if (miss) break;
    }
    return len;
}

// A block's scale from the largest magnitude of its new rows (FP32 bits) and the
// scale that its earlier rows have.
struct BlockScale {
    float value, inv;
    bool grew;
};
__device__ __forceinline__ BlockScale block_scale(uint32_t top, float qmax, float old) {
    const float most = top < 0x7f800000u ? __uint_as_float(top) : INFINITY;
    const float mine = most == INFINITY ? __int_as_float(0x7fffffff) : fmaxf(__fdiv_rn(most, qmax), kMinBlockScale);
    const float value = mine > old || mine != mine ? mine : old;
    return BlockScale{value, value == value ? __frcp_rn(value) : 0.f, mine > old};
}

// A lane's dims 0..7 and 64..71 of a row, from `row` on.
template <int kCode>
__device__ __forceinline__ void store_row(uint8_t* row, float* x, const BlockScale& scale) {
    if (!(scale.value == scale.value))
#pragma unroll
        for (int e = 0; e < 16; ++e) x[e] = 0.f;
    *reinterpret_cast<uint2*>(row) = encode8<kCode>(x, scale.inv);
    *reinterpret_cast<uint2*>(row + 64) = encode8<kCode>(x + 8, scale.inv);
}

// The same of an earlier row, whose block's scale was `old`.
template <int kCode>
__device__ __forceinline__ void rescale_row(uint8_t* row, float old, float inv) {
#pragma unroll
    for (int half = 0; half < 2; ++half) {
        uint2* at = reinterpret_cast<uint2*>(row + 64 * half);
        const uint2 w = *at;
        float y[8];
#pragma unroll
        for (int e = 0; e < 8; ++e)
            y[e] = __fmul_rn(code_value<kCode>((uint8_t)((e < 4 ? w.x : w.y) >> (8 * (e & 3)))), old);
        *at = encode8<kCode>(y, inv);
    }
}

// A decode step's rows, one a request or a few: a CTA the run that starts at token
// blockIdx.x, if one does, for one head, 64 threads, so that all CTAs of the step are
// resident at once.  8 threads take a row, each 8 rotate_half pairs, and a thread two
// rows; a run of more than 16 rows is read twice.
template <int kCode>
__global__ void __launch_bounds__(64) append_step_kernel(const __grid_constant__ AppendArgs a) {
    constexpr int kRowsPerPass = 8, kRows = 2, kBlock = kRowsPerPass * kRows;
    __shared__ uint32_t s_max[2];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, t0 = blockIdx.x, head = blockIdx.y;
    const bool is_k = blockIdx.z == 0, turn = is_k && a.positions;
    const int page_len = a.c.page_len, page_mask = page_len - 1;
    const int64_t n_slots = (int64_t)a.c.pages << a.c.page_shift;
    const int64_t tstride = is_k ? a.k_tstride : a.v_tstride, hstride = is_k ? a.k_hstride : a.v_hstride;
    const float qmax = kCode == GQA_CODE_INT8 ? 127.f : 448.f;
    const int chunk = tid & 7, row0 = tid >> 3;

    // A run starts at a slot of the cache whose predecessor is not the token before.
    const int64_t slot = a.slots[t0], before = t0 > 0 ? a.slots[t0 - 1] : -1;
    if (slot < 0 || slot >= n_slots || ((slot & page_mask) && before == slot - 1)) return;
    const int r0 = (int)(slot & page_mask);
    const int len = run_length(a, t0, slot, page_len - r0);
    const int64_t page = slot >> a.c.page_shift;
    // Rows b0 + row0, b0 + row0 + 8 of the run: dims 8 chunk .. and 64 + 8 chunk ..
    uint4 raw[kRows][2];
    float x[kRows][16];
    auto load = [&](int b0) {
        const __nv_bfloat16* src = (is_k ? a.k : a.v) + head * hstride + 8 * chunk;
#pragma unroll
        for (int p = 0; p < kRows; ++p) {
            const int r = b0 + row0 + p * kRowsPerPass;
            if (r >= len) continue;
            const __nv_bfloat16* row = src + (int64_t)(t0 + r) * tstride;
            raw[p][0] = *reinterpret_cast<const uint4*>(row);
            raw[p][1] = *reinterpret_cast<const uint4*>(row + 64);
        }
    };
    // The rows' values, and the largest magnitude, as FP32 bits (which order as integers).
    auto values = [&](int b0, uint32_t top) {
#pragma unroll
        for (int p = 0; p < kRows; ++p) {
            const int r = b0 + row0 + p * kRowsPerPass;
            if (r >= len) continue;
            float2 f[8];
            if (turn) {
                const int pos = a.positions[t0 + r];
#pragma unroll
                for (int e = 0; e < 8; ++e) f[e] = rope_factor_fast(a.rope.step[8 * chunk + e], pos);
            }
            unpack8(raw[p][0], x[p]);
            unpack8(raw[p][1], x[p] + 8);
            if (turn) {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float re = x[p][e], im = x[p][8 + e];
                    x[p][e] = re * f[e].x - im * f[e].y;
                    x[p][8 + e] = re * f[e].y + im * f[e].x;
                }
            }
#pragma unroll
            for (int e = 0; e < 16; ++e) top = max(top, __float_as_uint(x[p][e]) & 0x7fffffffu);
        }
        return top;
    };
    load(0);
    uint8_t* base = (is_k ? a.c.k : a.c.v) + head * a.c.head_stride + page * a.c.page_stride;
    float* scale_at = (is_k ? a.c.k_scale : a.c.v_scale) + head + page * a.c.scale_page_stride;
    const float old = r0 ? *scale_at : 0.f;
    uint32_t top = values(0, 0u);
    for (int b0 = kBlock; b0 < len; b0 += kBlock) {
        load(b0);
        top = values(b0, top);
    }
    top = __reduce_max_sync(0xffffffffu, top);
    if (lane == 0) s_max[warp] = top;
    __syncthreads();  // (and everyone has read the old scale)
    const BlockScale scale = block_scale(max(s_max[0], s_max[1]), qmax, old);
    for (int b0 = 0; b0 < len; b0 += kBlock) {
        if (len > kBlock) {
            load(b0);
            values(b0, 0u);
        }
#pragma unroll
        for (int p = 0; p < kRows; ++p) {
            const int r = b0 + row0 + p * kRowsPerPass;
            if (r < len) store_row<kCode>(base + (r0 + r) * a.c.row_stride + 8 * chunk, x[p], scale);
        }
    }
    if (scale.grew)
        for (int r = row0; r < r0; r += kRowsPerPass) rescale_row<kCode>(base + r * a.c.row_stride + 8 * chunk, old, scale.inv);
    if (tid == 0) *scale_at = scale.value;
}

// Prompts: a warp a head, so that a run's rows are read whole, all heads at once,
// and the maximum over a block needs no barrier.  Lane (sub, chunk) = (lane / 8, lane
// % 8) has rows sub, sub + 4, ... and dims 8 chunk .. and 64 + 8 chunk .. of them; 32
// rows stay in registers as they came (BF16) and are rotated once for the maximum and
// once more for their codes, a longer run's other rows are read again from L2.  The
// rotation factors of the run's rows are in shared memory, one computation for all
// heads.
template <int kCode>
__global__ void __launch_bounds__(256, 2) append_pages_kernel(const __grid_constant__ AppendArgs a) {
    constexpr int kRows = 8, kBlock = 4 * kRows;  // of a lane, of a warp
    extern __shared__ float4 factors[];           // [row][4][chunk]: of pairs 8 chunk + 2 j and the one after
    __shared__ uint64_t steps[kPairs];
    const int tid = threadIdx.x, lane = tid & 31, head = tid >> 5, chunk = lane & 7, sub = lane >> 3;
    const bool is_k = blockIdx.z == 0, turn = is_k && a.positions;
    const int page_len = a.c.page_len, page_mask = page_len - 1;
    const int64_t n_slots = (int64_t)a.c.pages << a.c.page_shift;
    const int64_t tstride = is_k ? a.k_tstride : a.v_tstride, hstride = is_k ? a.k_hstride : a.v_hstride;
    const float qmax = kCode == GQA_CODE_INT8 ? 127.f : 448.f;

    // The tokens of the window that start a run: slots of the cache whose predecessor is not the token before.
    const int w0 = blockIdx.x * kWindow;
    unsigned starts;
    {
        int64_t slot = -1, before = -1;
        if (lane < kWindow && lane < a.n_tokens - w0) {
            const int t = w0 + lane;
            slot = a.slots[t];
            if (t > 0) before = a.slots[t - 1];
        }
        starts = __ballot_sync(0xffffffffu, slot >= 0 && slot < n_slots && ((slot & page_mask) == 0 || before != slot - 1));
    }
    if (!starts) return;
    for (int i = tid; turn && i < kPairs; i += blockDim.x) steps[i] = a.rope.step[i];
    for (; starts; starts &= starts - 1) {
        const int t0 = w0 + __ffs(starts) - 1;
        const int64_t slot = a.slots[t0], page = slot >> a.c.page_shift;
        const int r0 = (int)(slot & page_mask);
        const int len = run_length(a, t0, slot, page_len - r0);
        const __nv_bfloat16* src = (is_k ? a.k : a.v) + head * hstride + 8 * chunk;
        uint4 raw[kRows][2];
        auto load = [&](int b0) {
#pragma unroll
            for (int i = 0; i < kRows; ++i) {
                const int r = b0 + sub + 4 * i;
                if (r >= len) continue;
                const __nv_bfloat16* row = src + (int64_t)(t0 + r) * tstride;
                raw[i][0] = *reinterpret_cast<const uint4*>(row);
                raw[i][1] = *reinterpret_cast<const uint4*>(row + 64);
            }
        };
        load(0);
        if (turn) {
            __syncthreads();  // the steps, and the last run's factors are no longer read
            for (int i = tid; i < len * 32; i += blockDim.x) {
                const int pair = 8 * (i & 7) + 2 * (i >> 3 & 3), pos = a.positions[t0 + (i >> 5)];
                const float2 u = rope_factor_fast(steps[pair], pos), v = rope_factor_fast(steps[pair + 1], pos);
                factors[i] = make_float4(u.x, u.y, v.x, v.y);
            }
            __syncthreads();
        }
        // Row r's values, from its two pieces.
        auto values = [&](int i, int r, float (&x)[16]) {
            unpack8(raw[i][0], x);
            unpack8(raw[i][1], x + 8);
            if (!turn) return;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float4 f = factors[r * 32 + 8 * j + chunk];
                float re = x[2 * j], im = x[8 + 2 * j];
                x[2 * j] = re * f.x - im * f.y;
                x[8 + 2 * j] = re * f.y + im * f.x;
                re = x[2 * j + 1];
                im = x[9 + 2 * j];
                x[2 * j + 1] = re * f.z - im * f.w;
                x[9 + 2 * j] = re * f.w + im * f.z;
            }
        };
        uint8_t* base = (is_k ? a.c.k : a.c.v) + head * a.c.head_stride + page * a.c.page_stride;
        float* scale_at = (is_k ? a.c.k_scale : a.c.v_scale) + head + page * a.c.scale_page_stride;
        const float old = r0 ? *scale_at : 0.f;
        // The largest magnitude, as FP32 bits (which order as integers).
        uint32_t top = 0;
        int b0 = 0;
        for (;;) {
#pragma unroll
            for (int i = 0; i < kRows; ++i) {
                const int r = b0 + sub + 4 * i;
                if (r >= len) continue;
                float x[16];
                values(i, r, x);
#pragma unroll
                for (int e = 0; e < 16; ++e) top = max(top, __float_as_uint(x[e]) & 0x7fffffffu);
            }
            if (b0 + kBlock >= len) break;
            b0 += kBlock;
            load(b0);
        }
        top = __reduce_max_sync(0xffffffffu, top);
        const BlockScale scale = block_scale(top, qmax, old);
        for (;;) {  // from the last rows, which are still here, back
#pragma unroll
            for (int i = 0; i < kRows; ++i) {
                const int r = b0 + sub + 4 * i;
                if (r >= len) continue;
                float x[16];
                values(i, r, x);
                store_row<kCode>(base + (r0 + r) * a.c.row_stride + 8 * chunk, x, scale);
            }
            if (b0 == 0) break;
            b0 -= kBlock;
            load(b0);
        }
        if (scale.grew)
            for (int r = sub; r < r0; r += 4) rescale_row<kCode>(base + r * a.c.row_stride + 8 * chunk, old, scale.inv);
        __syncwarp();  // every lane has read the old scale
        if (lane == 0) *scale_at = scale.value;
    }
}

// Rows back to BF16: a thread 16 codes of one (row, head), of K or V.  18000 rows
// 21 us (111 MB, 5.2 TB/s), 64 rows 4.5 us.
struct ReadArgs {
    PagedCacheView c;
    const int64_t* slots;
    __nv_bfloat16 *out_k, *out_v;
    int n;
};

template <int kCode>
__global__ void __launch_bounds__(256) read_kernel(const __grid_constant__ ReadArgs a) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int chunk = (int)(i & 7);
    const int64_t at = i >> 3, row = at / a.c.kv_heads;
    const int head = (int)(at - row * a.c.kv_heads);
    if (row >= a.n) return;
    const int64_t slot = a.slots[row];
    uint4 o[2] = {make_uint4(0u, 0u, 0u, 0u), make_uint4(0u, 0u, 0u, 0u)};
    if (slot >= 0 && slot < ((int64_t)a.c.pages << a.c.page_shift)) {
        const int64_t page = slot >> a.c.page_shift;
        const uint8_t* codes = (blockIdx.y ? a.c.v : a.c.k) + page * a.c.page_stride +
                               (slot & (a.c.page_len - 1)) * a.c.row_stride + head * a.c.head_stride + 16 * chunk;
        const float s = (blockIdx.y ? a.c.v_scale : a.c.k_scale)[page * a.c.scale_page_stride + head];
        const uint4 w = *reinterpret_cast<const uint4*>(codes);
        const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
        uint32_t* to = &o[0].x;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const uint32_t pair = ws[e >> 1] >> (16 * (e & 1));
            const __nv_bfloat162 v = __floats2bfloat162_rn(code_value<kCode>((uint8_t)pair) * s,
                                                           code_value<kCode>((uint8_t)(pair >> 8)) * s);
            to[e] = *reinterpret_cast<const uint32_t*>(&v);
        }
    }
    uint4* out = reinterpret_cast<uint4*>((blockIdx.y ? a.out_v : a.out_k) + at * kHeadDim + 16 * chunk);
    out[0] = o[0];
    out[1] = o[1];
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// A pure function of theta, kept per thread for the value last asked.
const RopeSteps& rope_steps_of(float theta) {
    static thread_local float last = 0.f;
    static thread_local RopeSteps steps;
    if (last != theta) {
        for (int i = 0; i < kPairs; ++i) steps.step[i] = rope_step(theta, i, kHeadDim);
        last = theta;
    }
    return steps;
}

int check_cache(const gqa_paged_cache* c, PagedCacheView* v) {
    if (!c->k || !c->v || !c->k_scale || !c->v_scale) return GQA_ERR_NULL_POINTER;
    if (c->kv_heads < 1 || c->kv_heads > kNumKVHeads) return GQA_ERR_KV_HEADS;
    if (c->code != GQA_CODE_INT8 && c->code != GQA_CODE_E4M3) return GQA_ERR_FLAGS;
    int shift = 4;
    while (shift < 7 && (1 << shift) != c->page_len) ++shift;
    if ((1 << shift) != c->page_len || c->page_len < kPagedMinPage) return GQA_ERR_KV_BLOCK_LEN;
    if (c->pages < 1) return GQA_ERR_KV_RANGE;
    if (!aligned16(c->k) || !aligned16(c->v) || ((uintptr_t)c->k_scale & 3) || ((uintptr_t)c->v_scale & 3))
        return GQA_ERR_ALIGNMENT;
    // TMA strides: multiples of 16 bytes below 2^40.
    for (const int64_t s : {c->page_stride, c->row_stride, c->head_stride})
        if (s < kHeadDim || s % 16 || s >= (int64_t)1 << 40) return GQA_ERR_ALIGNMENT;
    if (c->scale_page_stride < c->kv_heads) return GQA_ERR_ALIGNMENT;
    v->k = static_cast<uint8_t*>(c->k);
    v->v = static_cast<uint8_t*>(c->v);
    v->k_scale = c->k_scale;
    v->v_scale = c->v_scale;
    v->kv_heads = c->kv_heads;
    v->page_len = c->page_len;
    v->page_shift = shift;
    v->pages = c->pages;
    v->page_stride = c->page_stride;
    v->row_stride = c->row_stride;
    v->head_stride = c->head_stride;
    v->scale_page_stride = c->scale_page_stride;
    return GQA_OK;
}

// Checks both attention calls share; fills `call`.
int check_call(const void* q, void* out, const gqa_paged_cache* c, const gqa_paged_params* p, bool chunked,
               PagedCall* call) {
    if (!q || !out || !c || !p || !p->block_table || !p->seq_lens || (chunked && !p->first_query))
        return GQA_ERR_NULL_POINTER;
    std::memset(call, 0, sizeof(*call));
    const int st = check_cache(c, &call->c);
    if (st != GQA_OK) return st;
    if (p->batch < 1 || p->batch > GQA_PAGED_MAX_BATCH || p->rows < 0 || (!chunked && p->rows != p->batch) ||
        p->table_width < 1 || p->reserved != 0)
        return GQA_ERR_BATCH;
    if (p->batch > 1 && p->table_stride < p->table_width) return GQA_ERR_BATCH;
    if (p->flags & ~GQA_FLAG_Q_ROTATED) return GQA_ERR_FLAGS;
    if (!(p->scale != 0.f) || !std::isfinite(p->scale)) return GQA_ERR_SCALE;
    if (!(p->score_cap >= 0.f) || !std::isfinite(p->score_cap)) return GQA_ERR_SCALE;
    if (!(p->rope_theta > 0.f) || !std::isfinite(p->rope_theta)) return GQA_ERR_ROPE_THETA;
    if (!aligned16(q) || !aligned16(out)) return GQA_ERR_ALIGNMENT;
    for (const int64_t s : {p->q_row_stride, p->q_head_stride, p->out_row_stride, p->out_head_stride})
        if (s < 0 || s % 8) return GQA_ERR_ALIGNMENT;
    call->q = static_cast<const __nv_bfloat16*>(q);
    call->out = static_cast<__nv_bfloat16*>(out);
    call->block_table = p->block_table;
    call->seq_lens = p->seq_lens;
    call->query_positions = chunked ? nullptr : p->query_positions;
    call->first_query = chunked ? p->first_query : nullptr;
    call->doc_starts = p->doc_starts;
    call->prefix_ends = p->prefix_ends;
    call->slopes = p->slopes;
    call->table_stride = p->table_stride;
    call->q_row_stride = p->q_row_stride;
    call->q_head_stride = p->q_head_stride;
    call->out_row_stride = p->out_row_stride;
    call->out_head_stride = p->out_head_stride;
    call->batch = p->batch;
    call->rows = p->rows;
    call->table_width = p->table_width;
    call->scale = p->scale;
    // In FP32 a cap beyond 2^96 leaves the scores as they are and one below 2^-96 makes them 0, within 2^-96; in
    // between the products with it are normal numbers.
    call->cap = p->score_cap > 0x1p96f ? 0.f : p->score_cap > 0.f && p->score_cap < 0x1p-96f ? 0x1p-96f : p->score_cap;
    call->q_rotated = (p->flags & GQA_FLAG_Q_ROTATED) != 0;
    // Key positions, a tile past them, and tile counts are 32-bit.
    if ((int64_t)p->table_width * c->page_len > 1 << 30 ||
        (int64_t)p->batch * p->table_width * (c->page_len / 32 + 1) > 0x7FFFFFFF)
        return GQA_ERR_BATCH;
    return check_device_memory({q, out, c->k, c->v, c->k_scale, c->v_scale, p->block_table, p->seq_lens,
                                call->query_positions, call->first_query, p->doc_starts, p->prefix_ends, p->slopes});
}

int launched() { return cudaGetLastError() == cudaSuccess ? GQA_OK : GQA_ERR_CUDA; }

// A chunked call goes to the kernel for a few queries a sequence (gqa_paged_few.cu)
// where its rows are 6 a sequence or less on average: 48 sequences of 5 queries take
// 117 us there and 214 in the chunked kernel, of 2 85 and 212; 12 a sequence are two
// of its units each and take as long as the one chunk (211 and 215).  One sequence may hold most
// of the rows (a chunk of a prompt among single tokens), which only the GPU knows:
// beyond kFewAlone rows both kernels are launched and the plan hands the call to
// the one it is cheaper for.
constexpr int kFewAverage = 6, kFewAlone = 12;
bool few_queries(int batch, int rows) { return rows <= (int64_t)kFewAverage * batch; }

size_t workspace_of(int batch, int rows, int heads, bool chunked, int sms) {
    if (!chunked) return paged_decode_workspace(sms);
    // Both kernels' regions whichever takes the call: a workspace for the largest call holds every smaller one.
    return paged_few_workspace(batch, rows, heads, sms);
}

int attend(const void* q, void* out, const gqa_paged_cache* cache, const gqa_paged_params* p, void* workspace,
           size_t workspace_bytes, void* stream, bool chunked) {
    PagedCall call;
    int st = check_call(q, out, cache, p, chunked, &call);
    if (st != GQA_OK) return st;
    if (!workspace || !aligned16(workspace)) return GQA_ERR_WORKSPACE;
    int sms = 0;
    st = paged_attention_sms(&sms);
    if (st != GQA_OK) return st;
    if (workspace_bytes < workspace_of(p->batch, p->rows, cache->kv_heads, chunked, sms)) return GQA_ERR_WORKSPACE;
    st = check_device_memory({workspace});
    if (st != GQA_OK) return st;
    if (p->rows == 0) return GQA_OK;
    const RopeSteps& rope = rope_steps_of(p->rope_theta);
    uint8_t* ws = static_cast<uint8_t*>(workspace);
    uint32_t* status = reinterpret_cast<uint32_t*>(ws);
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    CUtensorMap kmap, vmap;
    auto maps = [&](int tile) {
        const int k = paged_map(&kmap, call.c.k, call.c, tile);
        return k != GQA_OK ? k : paged_map(&vmap, call.c.v, call.c, tile);
    };
    cudaError_t e = cudaSuccess;
    if (!chunked) {
        if ((st = maps(paged_decode_tile())) != GQA_OK) return st;
        e = launch_paged_decode(call, rope, cache->code, kmap, vmap, sms, ws, s);
    } else {
        const bool few = few_queries(p->batch, p->rows), many = !few || p->rows > kFewAlone;
        const UnitShape chunk = paged_chunk_shape(call, sms, ws), small = few ? paged_few_shape(call, sms, ws) : chunk;
        e = launch_plan_units(call, small, few && many ? &chunk : nullptr, s);
        if (e == cudaSuccess && few) {
            if ((st = maps(paged_few_tile())) != GQA_OK) return st;
            e = launch_paged_few(call, rope, cache->code, kmap, vmap, small, status, s);
        }
        if (e == cudaSuccess && many) {
            if ((st = maps(paged_chunk_tile())) != GQA_OK) return st;
            e = launch_paged_chunk(call, rope, cache->code, kmap, vmap, chunk, status, s);
        }
    }
    return e == cudaSuccess ? GQA_OK : GQA_ERR_CUDA;
}

}  // namespace

}  // namespace gqa

using namespace gqa;

extern "C" {

int gqa_plan_pages(const int32_t* lens, const int32_t* new_lens, int requests, int32_t* block_table,
                   int64_t table_stride, int table_width, int32_t* free_pages, int free_capacity,
                   const int32_t* n_free, int page_len, int max_tokens, int32_t* lens_out, int32_t* n_free_out,
                   int32_t* first_token, int64_t* slots, int32_t* positions, int32_t* counts, void* workspace,
                   size_t workspace_bytes, void* stream) {
    if (!lens || !new_lens || !block_table || !free_pages || !n_free || !lens_out || !n_free_out || !first_token ||
        !counts || (max_tokens > 0 && (!slots || !positions)))
        return GQA_ERR_NULL_POINTER;
    if (requests < 1 || requests > GQA_PAGED_MAX_BATCH || table_width < 1 || free_capacity < 0 || max_tokens < 0 ||
        (requests > 1 && table_stride < table_width))
        return GQA_ERR_BATCH;
    int shift = 4;
    while (shift < 7 && (1 << shift) != page_len) ++shift;
    if ((1 << shift) != page_len) return GQA_ERR_KV_BLOCK_LEN;
    if (!workspace || !aligned16(workspace) || workspace_bytes < GQA_CHUNKED_WORKSPACE_BYTES) return GQA_ERR_WORKSPACE;
    int sms = 0;
    int st = device_sms(&sms);
    if (st != GQA_OK) return st;
    st = check_device_memory({lens, new_lens, block_table, free_pages, n_free, lens_out, n_free_out, first_token,
                                  slots, positions, counts, workspace});
    if (st != GQA_OK) return st;
    PlanArgs a;
    a.lens = lens;
    a.new_lens = new_lens;
    a.block_table = block_table;
    a.table_stride = table_stride;
    a.free_pages = free_pages;
    a.n_free = n_free;
    a.lens_out = lens_out;
    a.n_free_out = n_free_out;
    a.first_token = first_token;
    a.slots = slots;
    a.positions = positions;
    a.counts = counts;
    a.ticket = static_cast<uint32_t*>(workspace) + 1;
    a.requests = requests;
    a.table_width = table_width;
    a.free_capacity = free_capacity;
    a.page_shift = shift;
    a.max_tokens = max_tokens;
    // The limit is the kernel's, not the call's: always the same, so that another thread's call does not lower it
    // before this one's launch.
    constexpr int kMostSmem = 3 * (GQA_PAGED_MAX_BATCH + 1) * (int)sizeof(int32_t);
    const size_t smem = 3 * (size_t)(requests + 1) * sizeof(int32_t);
    if (smem > 40 * 1024 && cudaFuncSetAttribute(plan_pages_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                 kMostSmem) != cudaSuccess)
        return GQA_ERR_CUDA;
    const int64_t items = max_tokens > requests ? max_tokens : requests;
    int64_t grid = (items + kPlanThreads - 1) / kPlanThreads;
    if (grid > 128) grid = 128;
    plan_pages_kernel<<<(int)grid, kPlanThreads, smem, static_cast<cudaStream_t>(stream)>>>(a);
    return launched();
}

int gqa_append_paged(const void* k, const void* v, int n_tokens, int64_t k_token_stride, int64_t k_head_stride,
                     int64_t v_token_stride, int64_t v_head_stride, const int64_t* slots, const int32_t* positions,
                     float rope_theta, const gqa_paged_cache* cache, void* stream) {
    if (!k || !v || !slots || !cache) return GQA_ERR_NULL_POINTER;
    AppendArgs a;
    int st = check_cache(cache, &a.c);
    if (st != GQA_OK) return st;
    if (n_tokens < 0) return GQA_ERR_BATCH;
    if (!(rope_theta > 0.f) || !std::isfinite(rope_theta)) return GQA_ERR_ROPE_THETA;
    if (!aligned16(k) || !aligned16(v)) return GQA_ERR_ALIGNMENT;
    for (const int64_t s : {k_token_stride, k_head_stride, v_token_stride, v_head_stride})
        if (s < 0 || s % 8) return GQA_ERR_ALIGNMENT;
    int sms = 0;
    st = device_sms(&sms);
    if (st != GQA_OK) return st;
    st = check_device_memory({k, v, slots, positions, cache->k, cache->v, cache->k_scale, cache->v_scale});
    if (st != GQA_OK) return st;
    if (n_tokens == 0) return GQA_OK;
    a.k = static_cast<const __nv_bfloat16*>(k);
    a.v = static_cast<const __nv_bfloat16*>(v);
    a.k_tstride = k_token_stride;
    a.k_hstride = k_head_stride;
    a.v_tstride = v_token_stride;
    a.v_hstride = v_head_stride;
    a.slots = slots;
    a.positions = positions;
    a.n_tokens = n_tokens;
    // A step's rows are runs of one, prompts' runs fill pages, so that a window of 16 tokens begins one at most; the
    // count of rows stands for which it is.  Measured at the change, pages of 64: 1024 runs of one row 24 us as a step
    // (93 with every scale grown), 1025 as prompts, 16 runs after one another in a CTA, 32 us (203), 8192 122 us; 18000
    // rows of prompts in pages of 32 33 us.
    const bool step = n_tokens <= 1024;
    a.rope = rope_steps_of(rope_theta);
    const dim3 grid(step ? n_tokens : (n_tokens - 1) / kWindow + 1, step ? cache->kv_heads : 1, 2);
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    const bool int8 = cache->code == GQA_CODE_INT8;
    if (step) {
        (int8 ? append_step_kernel<GQA_CODE_INT8> : append_step_kernel<GQA_CODE_E4M3>)<<<grid, 64, 0, s>>>(a);
    } else {
        const auto kernel = int8 ? append_pages_kernel<GQA_CODE_INT8> : append_pages_kernel<GQA_CODE_E4M3>;
        const int smem = positions ? cache->page_len * kPairs * (int)sizeof(float2) : 0;
        if (smem > 40 * 1024 &&
            cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess)
            return GQA_ERR_CUDA;
        kernel<<<grid, 32 * cache->kv_heads, smem, s>>>(a);
    }
    return launched();
}

int gqa_read_paged(const gqa_paged_cache* cache, const int64_t* slots, int n, void* out_k, void* out_v, void* stream) {
    if (!cache || !slots || !out_k || !out_v) return GQA_ERR_NULL_POINTER;
    ReadArgs a;
    int st = check_cache(cache, &a.c);
    if (st != GQA_OK) return st;
    if (n < 0) return GQA_ERR_BATCH;
    if (!aligned16(out_k) || !aligned16(out_v)) return GQA_ERR_ALIGNMENT;
    int sms = 0;
    st = device_sms(&sms);
    if (st != GQA_OK) return st;
    st = check_device_memory({cache->k, cache->v, cache->k_scale, cache->v_scale, slots, out_k, out_v});
    if (st != GQA_OK) return st;
    if (n == 0) return GQA_OK;
    a.slots = slots;
    a.out_k = static_cast<__nv_bfloat16*>(out_k);
    a.out_v = static_cast<__nv_bfloat16*>(out_v);
    a.n = n;
    const dim3 grid((unsigned)(((int64_t)n * cache->kv_heads * 8 + 255) / 256), 2);
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (cache->code == GQA_CODE_INT8)
        read_kernel<GQA_CODE_INT8><<<grid, 256, 0, s>>>(a);
    else
        read_kernel<GQA_CODE_E4M3><<<grid, 256, 0, s>>>(a);
    return launched();
}

size_t gqa_paged_workspace_bytes(const gqa_paged_cache* cache, const gqa_paged_params* p) {
    if (!cache || !p || p->batch < 1 || p->batch > GQA_PAGED_MAX_BATCH || p->rows < 0 || cache->kv_heads < 1 ||
        cache->kv_heads > kNumKVHeads)
        return 0;
    int sms = 0;
    if (device_sms(&sms) != GQA_OK) return 0;
    return workspace_of(p->batch, p->rows, cache->kv_heads, p->first_query != nullptr, sms);
}

int gqa_decode_paged(const void* q, void* out, const gqa_paged_cache* cache, const gqa_paged_params* p,
                     void* workspace, size_t workspace_bytes, void* stream) {
    return attend(q, out, cache, p, workspace, workspace_bytes, stream, false);
}

int gqa_decode_paged_chunked(const void* q, void* out, const gqa_paged_cache* cache, const gqa_paged_params* p,
                             void* workspace, size_t workspace_bytes, void* stream) {
    return attend(q, out, cache, p, workspace, workspace_bytes, stream, true);
}

}  // extern "C"
