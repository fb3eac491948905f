// gqa_paged.cuh -- what the paged 8-bit cache's kernels share: the cache and
// call descriptions they take by value, the visible range of a query and the
// conversions between codes and values.
#pragma once

#include "gqa_b200.h"
#include "gqa_device.cuh"

#include <cuda_fp16.h>
#include <cuda_fp8.h>

namespace gqa {

constexpr int kPagedMinPage = 16, kPagedMaxPage = 128;

// Q0.64 turns per position of each rotate_half pair, passed by value.
struct RopeSteps {
    uint64_t step[kPairs];
};

struct PagedCacheView {
    uint8_t *k, *v;
    float *k_scale, *v_scale;
    int32_t kv_heads, page_len, page_shift, pages;
    int64_t page_stride, row_stride, head_stride, scale_page_stride;
};

// One attention call over the cache (gqa_paged_params, checked).
struct PagedCall {
    PagedCacheView c;
    const __nv_bfloat16* q;
    __nv_bfloat16* out;
    const int32_t* block_table;
    const int32_t *seq_lens, *query_positions, *first_query;
    const int32_t *doc_starts, *prefix_ends;
    const float* slopes;
    int64_t table_stride;
    int64_t q_row_stride, q_head_stride, out_row_stride, out_head_stride;
    int32_t batch, rows, table_width;
    float scale, cap;
    int32_t q_rotated;
};

// Keys of sequence b that can be visible at all: its length, cut to what its
// block-table row can name.
__device__ __forceinline__ int paged_length(const PagedCall& a, int b) {
    const int64_t room = (int64_t)a.table_width << a.c.page_shift;
    const int n = a.seq_lens[b];
    return n < 0 ? 0 : (int)(n < room ? n : room);
}

struct KeyRange {
    int lo, hi;  // visible keys lo <= p < hi (none where hi <= lo)
};

// Visible keys of query row `row` at position m of a sequence with `len` keys.
__device__ __forceinline__ KeyRange paged_range(const PagedCall& a, int row, int64_t m, int len) {
    int64_t hi = m + 1;
    if (a.prefix_ends) {
        const int e = a.prefix_ends[row];
        if (e > hi) hi = e;
    }
    if (hi > len) hi = len;
    if (hi < 0) hi = 0;
    int lo = a.doc_starts ? a.doc_starts[row] : 0;
    if (lo < 0) lo = 0;
    return KeyRange{lo, (int)hi};
}

// rope_factor from the top 32 bits of the phase: 2^-32 turns, a 128th of what FP32 leaves of it.
__device__ __forceinline__ float2 rope_factor_fast(uint64_t step, int64_t pos) {
    const int turns = (int)((step * (uint64_t)pos) >> 32);
    float sn, cs;
    sincospif(__int2float_rn(turns) * 0x1p-31f, &sn, &cs);
    return make_float2(cs, sn);
}

// Programmatic dependent launch: a kernel so launched starts before the one in
// front of it in the stream has ended, and touches no memory before the wait.
__device__ __forceinline__ void dependency_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void allow_dependents() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

template <typename Args>
inline cudaError_t launch_dependent(void (*kernel)(Args), int grid, int threads, size_t smem, cudaStream_t stream,
                                    const Args& a) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, a);
}

// Value of one code.
template <int kCode>
__device__ __forceinline__ float code_value(uint8_t c) {
    if constexpr (kCode == GQA_CODE_INT8) {
        return (float)(int8_t)c;
    } else {
        const __half_raw h = __nv_cvt_fp8_to_halfraw(c, __NV_E4M3);
        return __half2float(__half(h));
    }
}

// Codes of 4 values already divided by their scale, first in the low byte: round to
// nearest even.  For int8 the caller keeps |y| below 127.5; the sum with 1.5 * 2^23
// leaves the integer in the low bits.  e4m3 saturates.
template <int kCode>
__device__ __forceinline__ uint32_t value_codes4(float y0, float y1, float y2, float y3) {
    if constexpr (kCode == GQA_CODE_INT8) {
        const uint32_t a = __float_as_uint(__fadd_rn(y0, 12582912.f)), b = __float_as_uint(__fadd_rn(y1, 12582912.f));
        const uint32_t c = __float_as_uint(__fadd_rn(y2, 12582912.f)), d = __float_as_uint(__fadd_rn(y3, 12582912.f));
        return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
    } else {
        const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(y0, y1), __NV_SATFINITE, __NV_E4M3);
        const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(y2, y3), __NV_SATFINITE, __NV_E4M3);
        return lo | hi << 16;
    }
}

// Four codes of a word to two FP16 pairs, exactly.
template <int kCode>
__device__ __forceinline__ void to_half4(uint32_t w, uint32_t& lo, uint32_t& hi) {
    if constexpr (kCode == GQA_CODE_INT8) {
        // 1024 + (c + 128) is the FP16 number 0x6400 | byte; minus 1152 it is c.
        const __half2 bias = __halves2half2(__ushort_as_half(0x6480), __ushort_as_half(0x6480));
        const uint32_t u = w ^ 0x80808080u;
        const uint32_t x = __byte_perm(u, 0x64646464u, 0x4140), y = __byte_perm(u, 0x64646464u, 0x4342);
        const __half2 a = __hsub2(*reinterpret_cast<const __half2*>(&x), bias);
        const __half2 b = __hsub2(*reinterpret_cast<const __half2*>(&y), bias);
        lo = *reinterpret_cast<const uint32_t*>(&a);
        hi = *reinterpret_cast<const uint32_t*>(&b);
    } else {
        asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, a;\n\t"
            "cvt.rn.f16x2.e4m3x2 %1, b;\n\t}"
            : "=r"(lo), "=r"(hi)
            : "r"(w));
    }
}

// V's scales join the weights as exponents: the weights of a row for the product
// with V's codes are 2^(z + log2(V scale) - m), m the row's reference for this sum,
// so that what a row does not see, or gives no weight, takes no bits from what it
// does; their sum, which divides, takes each page's scale out again in FP32 (1 /
// scale is kept as kWeightUnit / scale: up to 2^121, the scale of BF16's largest
// number, no part of it passes FP32's range).  A block of zeros has the smallest
// scale that an append writes, 2^-100, and a page never written one of 0: such
// blocks count as zeros, with 2^-60 in their scale's place, so that their keys'
// weights stay in the sum beside pages of 2^-80 to 2^60.
constexpr float kWeightUnit = 0x1p-12f, kNoVScale = 0x1p-100f;
struct VScale {
    float exponent, fraction;  // of a page's V scale; the fraction in [1, 2), 0 where V is zeros
    float inv;                 // kWeightUnit / 2^exponent
};
__device__ __forceinline__ VScale v_scale_of(float s) {
    const bool some = s > kNoVScale;
    const uint32_t bits = __float_as_uint(some ? fminf(s, 0x1.fffffep121f) : 0x1p-60f);
    const int e = (int)(bits >> 23) - 127;
    return VScale{(float)e, some ? __uint_as_float((bits & 0x7fffffu) | 0x3f800000u) : 0.f,
                  kWeightUnit * __uint_as_float((uint32_t)(127 - e) << 23)};
}
// The fraction joined to the exponent (its logarithm is good to 2^-22 of 1).
struct VLog2 {
    float log2, inv;  // inv: kWeightUnit / scale
    bool some;        // V is not zeros
};
__device__ __forceinline__ VLog2 v_log2_of(float s) {
    const VScale v = v_scale_of(s);
    const bool some = v.fraction > 0.f;
    const float f = some ? v.fraction : 1.f;
    return VLog2{v.exponent + __log2f(f), __fdividef(v.inv, f), some};
}

__device__ __forceinline__ uint32_t pack_half2(float lo, float hi) {
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
}

// tanh, to a few 2^-23 of itself however small it is: a cap far above the scores
// multiplies it back, so that an absolute error would grow with the cap.
// Up to |x| = 1/2 as x times a polynomial in t = x^2, interpolated at the Chebyshev
// points of tanh(x) / x (2^-26 of it); beyond as 1 - 2 / (e^2x + 1).
constexpr float kTanhNear = 0.25f;  // of t
__device__ __forceinline__ float tanh_near(float x, float t) {
    float p = fmaf(0.0171313453f, t, -0.0529842377f);
    p = fmaf(p, t, 0.13324751f);
    p = fmaf(p, t, -0.333330691f);
    return x * fmaf(p, t, 1.f);
}
__device__ __forceinline__ float tanh_far(float x) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(fast_exp2(x * 2.8853900817779268f) + 1.f));
    return fmaf(-2.f, r, 1.f);
}

// cap2 * tanh of a warp's scores, kN a lane (a multiple of the cap in, log2 units out).
template <int kN>
__device__ __forceinline__ void cap_scores(float (&z)[kN], float cap2) {
    float x[kN];
    bool far = false;
#pragma unroll
    for (int i = 0; i < kN; ++i) {
        x[i] = z[i];
        const float t = x[i] * x[i];
        far |= t > kTanhNear;
        z[i] = cap2 * tanh_near(x[i], t);
    }
    if (__any_sync(0xffffffffu, far))
#pragma unroll
        for (int i = 0; i < kN; ++i)
            if (x[i] * x[i] > kTanhNear) z[i] = cap2 * tanh_far(x[i]);
}

// Rows of a page from `row` on (as many as the map's box) of K or V of a head.
__device__ __forceinline__ void tma_load_page(void* dst, const CUtensorMap* map, int row, int head, int page,
                                              uint64_t* bar, uint64_t policy) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.L2::cache_hint "
        "[%0], [%1, {%2, %3, %4, %5}], [%6], %7;" ::"r"(smem_addr(dst)),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(0), "r"(row), "r"(head), "r"(page), "r"(smem_addr(bar)), "l"(policy)
        : "memory");
}

__device__ __forceinline__ void mma_16x8x16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                            uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t transpose_8x8(uint32_t a) {
    uint32_t d;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
    return d;
}

}  // namespace gqa
