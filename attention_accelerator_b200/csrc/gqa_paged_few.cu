// gqa_paged_few.cu -- a few queries a sequence over the paged 8-bit cache: drafted
// tokens to verify, short chunks, steps that mix them with single tokens.
//
// Work.  A unit is 6 consecutive queries of one sequence and one KV head, its keys
// those that any of its queries sees, in tiles of 32 on a grid of absolute
// positions; plan_units_kernel finds them and cuts all tiles into even shares.  A
// unit that crosses shares leaves FP32 partial rows, which its last CTA merges in
// CTA order.
//
// A CTA is 8 consumer warps, 4 finisher warps, 2 loader warps and a query warp (and
// one that writes zeros for units whose rows see nothing): the roles of the one-token
// kernel (gqa_paged_decode.cu), with its products turned the same way, S^T = K Q^T
// and O^T = V^T P^T on m16n8k16.  Where that kernel's 8 columns are 4 heads x {high,
// low parts}, these are 4 heads x 2 queries, and there are three such groups: a
// code is read from shared memory and becomes FP16 once for all 24 rows, whose O
// takes 96 registers of a lane.
//
// Precision.  Q, divided by a power of two that brings the row's largest below 1,
// and the weights, 2^(z + log2(V scale) - m), round to FP16 (2^-11 of a term: three
// bits more than the BF16 that Q came as and the output becomes; 2^-31 of the row's
// largest weight times scale for each key); codes are exact, sums and scores FP32.
//
// Bound by the consumers' instructions: of a tile's 3300 cycles in a warp the products
// with K take 1280, those with V 1120, the softmax 860, with the tensor pipe 28 % busy
// and 2 warps a scheduler (O's registers leave no room for more).  Measured (B200,
// int8, page 64, 48 sequences of up to 8191 keys, 409 MB): 5 queries each 122 us (3.4
// TB/s; the chunked kernel 214), 4 101, 2 89 (4.6 TB/s), 5 of e4m3 116, with cap 132.
// One sequence of 5 queries 32 us, a third of it the merge of its 18 shares.  Masks tested score by
// score, a branch each, took 164 us; two result buffers and a second query warp
// gained nothing (short contexts lost 13 %).
#include "gqa_paged_units.cuh"

namespace gqa {

namespace {

constexpr int kWarps = 8;          // consumer warps
constexpr int kFinishers = kGroup; // one a Q head
constexpr int kLoaders = 2;
constexpr int kBurst = 4;          // tiles that a loader handles at once
constexpr int kFinishWarp = kWarps, kLoaderWarp = kFinishWarp + kFinishers, kQueryWarp = kLoaderWarp + kLoaders;
constexpr int kZeroWarp = kQueryWarp + 1;
constexpr int kThreads = (kZeroWarp + 1) * 32;
// Registers: launched with 128 a thread; each group of four warps takes its share.
constexpr int kLaunchRegs = 128, kConsumerRegs = 192, kRestRegs = 64;
static_assert(kThreads == 512 && 2 * kConsumerRegs + 2 * kRestRegs <= 4 * kLaunchRegs, "of what the CTA was launched with");
constexpr int kTokens = kFewTokens;  // queries of a unit
constexpr int kPairsQ = kTokens / 2;
constexpr int kTileShift = kFewTileShift, kTile = 1 << kTileShift;
constexpr int kSteps = kTile / 16;
constexpr int kHalfBytes = kTile * kHeadDim;
constexpr int kStageBytes = 2 * kHalfBytes;
constexpr int kStages = 2 * kWarps;
constexpr int kRowF = kHeadDim + 4;    // padded row
constexpr int kUnitRows = kTokens * kGroup;
// Weights are lifted by 2^7 and may pass the reference by 2^8: up to 2^15, and FP16's
// 2^-24 is 2^-31 of a weight at the reference.
constexpr float kHeadroom = 8.f, kLift = 7.f;

struct alignas(16) Slot {  // one unit's queries (two slots)
    uint4 q[kPairsQ][4][32];       // the lanes' operands: column 2 head + query % 2, 8 of the lane's 32 dims
    float factor[kPairsQ][8];      // per column: scale * log2(e) (or / cap) * the row's power of two
    float slope[kGroup];           // times log2(e)
    int lo[kTokens], hi[kTokens];  // visible keys of each query
    int lo_most, hi_least, m;      // keys in between are seen by all; position of the first
    int tile, tiles, pairs, last;  // the piece: its first tile, how many, pairs of queries, whether the share ends
    int pad;
};
struct alignas(16) Shared {
    uint64_t full[kStages], empty[kStages], qfull[2], qempty[2], rfull, rempty;
    Slot slot[2];
    float4 scales[kStages];  // K of the tile's two pages (NaN where V's is no number), log2 of V's
    float4 v_inv[kStages];   // V's, as VLog2 has them; 0 where V is zeros, else 1
    struct {  // what the consumer warps make of two queries of a piece
        float acc[kWarps][2 * kGroup][kRowF];
        float m[kWarps][2 * kGroup], l[kWarps][2 * kGroup];
    } result;
    int64_t cuts[kMaxCtas + 1];
};

struct alignas(64) FewPagedArgs {
    CUtensorMap kmap, vmap;  // (128, page_len, heads, pages) bytes, box (128, min(page_len, 32), 1, 1)
    PagedCall p;
    RopeSteps rope;
    uint32_t* status;
    const Meta* meta;
    const Unit* units;
    const int32_t* starts;
    const int64_t* cuts;
    uint32_t* arrivals;  // [ctas][4]: of the unit that begins in a share and goes on in the next, a Q head
    float* partials;     // [ctas][2][24][132]
};

template <int kRegs>
__device__ __forceinline__ void take_registers() {
    if constexpr (kRegs > kLaunchRegs)
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegs));
    else
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegs));
}

// Running state of a consumer warp for the current unit.  Lane (g, t) = (lane / 4,
// lane % 4): head t's reference and sum (over this lane's keys only, times
// kWeightUnit) for each query, and O for head t, dims 16 g + 2 i (o[][i][0] the
// pair's first query, [1] its second) and + 1 ([2], [3]).
struct State {
    float o[kPairsQ][8][4];
    float m[kPairsQ][2], l[kPairsQ][2];
};

// Tiles of a unit with kN pairs of queries.
template <int kCode, bool kCap, bool kBias, int kN>
__device__ __forceinline__ void consume_tile(State& st, const uint8_t* stage, const float4& sc, const float4& vi,
                                             const Slot& slot, float cap2, int key0, int page_shift, int lane) {
    const int g = lane >> 2, t = lane & 3;
    // Step i (16 keys) lies in page i >> sh of the tile.
    const int sh = min(page_shift, kTileShift) - 4;
    float z[kN][kSteps][4];  // [key g or g + 8][query], as the product leaves them
    {
        // Both steps' products side by side: each is a chain of eight.
        const uint8_t* k = stage + g * kHeadDim;
        const int c0 = ((2 * t) ^ g) << 4, c1 = ((2 * t + 1) ^ g) << 4;
#pragma unroll
        for (int n = 0; n < kN; ++n)
#pragma unroll
            for (int i = 0; i < kSteps; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) z[n][i][e] = 0.f;
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            uint4 up[kSteps], dn[kSteps];
#pragma unroll
            for (int i = 0; i < kSteps; ++i) {
                up[i] = lds128(k + (16 * i) * kHeadDim + (half ? c1 : c0));
                dn[i] = lds128(k + (16 * i + 8) * kHeadDim + (half ? c1 : c0));
            }
#pragma unroll
            for (int f = 0; f < 2; ++f) {
                uint4 q[kN];
#pragma unroll
                for (int n = 0; n < kN; ++n) q[n] = lds128(&slot.q[n][2 * half + f][lane]);
#pragma unroll
                for (int e = 0; e < 2; ++e)
#pragma unroll
                    for (int i = 0; i < kSteps; ++i) {
                        uint32_t x[4];
                        to_half4<kCode>(f ? e ? up[i].w : up[i].z : e ? up[i].y : up[i].x, x[0], x[2]);
                        to_half4<kCode>(f ? e ? dn[i].w : dn[i].z : e ? dn[i].y : dn[i].x, x[1], x[3]);
#pragma unroll
                        for (int n = 0; n < kN; ++n)
                            mma_16x8x16(z[n][i], x[0], x[1], x[2], x[3], e ? q[n].z : q[n].x, e ? q[n].w : q[n].y);
                    }
            }
        }
    }
    const bool edge = key0 < slot.lo_most || key0 + kTile > slot.hi_least;  // of the whole warp
#pragma unroll
    for (int n = 0; n < kN; ++n) {
        const float2 factor = *reinterpret_cast<const float2*>(&slot.factor[n][2 * t]);
#pragma unroll
        for (int i = 0; i < kSteps; ++i) {
            const float f = i >> sh ? sc.y : sc.x, f0 = f * factor.x, f1 = f * factor.y;
            const float lv = kCap ? 0.f : i >> sh ? sc.w : sc.z;
#pragma unroll
            for (int e = 0; e < 4; ++e) z[n][i][e] = fmaf(z[n][i][e], e & 1 ? f1 : f0, lv);
        }
        if constexpr (kCap) {
            cap_scores(reinterpret_cast<float(&)[4 * kSteps]>(z[n]), cap2);
#pragma unroll
            for (int i = 0; i < kSteps; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) z[n][i][e] += i >> sh ? sc.w : sc.z;
        }
        if constexpr (kBias) {
#pragma unroll
            for (int i = 0; i < kSteps; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    z[n][i][e] = fmaf(-slot.slope[t],
                                      fabsf((float)(slot.m + 2 * n + (e & 1) - (key0 + 16 * i + 8 * (e >> 1) + g))),
                                      z[n][i][e]);
        }
    }
    if (edge) {  // where a query does not see a key, in one branch of the whole warp
#pragma unroll
        for (int n = 0; n < kN; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int lo = slot.lo[2 * n + e] - key0 - g, hi = slot.hi[2 * n + e] - key0 - g;
#pragma unroll
                for (int i = 0; i < kSteps; ++i)
#pragma unroll
                    for (int u = 0; u < 2; ++u)
                        if (16 * i + 8 * u < lo || 16 * i + 8 * u >= hi) z[n][i][2 * u + e] = -INFINITY;
            }
    }
    float mx[kN][2];  // of this lane's keys
    bool above = false;
#pragma unroll
    for (int n = 0; n < kN; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            mx[n][e] = fmaxf(fmaxf(z[n][0][e], z[n][0][2 + e]), fmaxf(z[n][1][e], z[n][1][2 + e])) - kLift;
            above |= mx[n][e] > st.m[n][e] + kHeadroom;
        }
    // The references move only when a score passes one by kHeadroom.
    if (__any_sync(0xffffffffu, above)) {
#pragma unroll
        for (int n = 0; n < kN; ++n) {
            float f[2];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                float m_new = fmaxf(st.m[n][e], mx[n][e]);
#pragma unroll
                for (int d = 4; d < 32; d <<= 1) m_new = fmaxf(m_new, __shfl_xor_sync(0xffffffffu, m_new, d));
                f[e] = fast_exp2(st.m[n][e] - (m_new == -INFINITY ? 0.f : m_new));
                st.m[n][e] = m_new;
                st.l[n][e] *= f[e];
            }
#pragma unroll
            for (int i = 0; i < 8; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) st.o[n][i][e] *= f[e & 1];
        }
    }
#pragma unroll
    for (int n = 0; n < kN; ++n) {
        const float m0 = st.m[n][0] == -INFINITY ? 0.f : st.m[n][0], m1 = st.m[n][1] == -INFINITY ? 0.f : st.m[n][1];
#pragma unroll
        for (int i = 0; i < kSteps; ++i) {
            const float inv = i >> sh ? vi.y : vi.x, some = i >> sh ? vi.w : vi.z;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float y = fast_exp2(z[n][i][e] - (e & 1 ? m1 : m0));
                st.l[n][e & 1] = fmaf(y, inv, st.l[n][e & 1]);
                z[n][i][e] = y * some;
            }
        }
    }
    uint32_t w[kN][kSteps][2];
#pragma unroll
    for (int n = 0; n < kN; ++n)
#pragma unroll
        for (int i = 0; i < kSteps; ++i)
#pragma unroll
            for (int u = 0; u < 2; ++u) w[n][i][u] = transpose_8x8(pack_half2(z[n][i][2 * u], z[n][i][2 * u + 1]));
    const uint8_t* v = stage + kHalfBytes;
    const int r0 = 2 * t * kHeadDim + ((g ^ (2 * t)) << 4), r1 = (2 * t + 1) * kHeadDim + ((g ^ (2 * t + 1)) << 4);
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
        const uint8_t* vi = v + 16 * i * kHeadDim;
        const uint4 x0 = lds128(vi + r0), x1 = lds128(vi + r1);
        const uint4 x2 = lds128(vi + 8 * kHeadDim + r0), x3 = lds128(vi + 8 * kHeadDim + r1);
        uint32_t w0[4] = {x0.x, x0.y, x0.z, x0.w}, w1[4] = {x1.x, x1.y, x1.z, x1.w};
        uint32_t w2[4] = {x2.x, x2.y, x2.z, x2.w}, w3[4] = {x3.x, x3.y, x3.z, x3.w};
        if (kCode == GQA_CODE_E4M3 && edge) {  // a code that no query sees may be NaN: 0 in its place
            auto number = [](uint32_t& x) { x &= ~__vcmpeq4(x & 0x7f7f7f7fu, 0x7f7f7f7fu); };
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                number(w0[j]);
                number(w1[j]);
                number(w2[j]);
                number(w3[j]);
            }
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const uint32_t sel = j & 1 ? 0x7362 : 0x5140;
            uint32_t a0, a1, a2, a3;
            to_half4<kCode>(__byte_perm(w0[j >> 1], w1[j >> 1], sel), a0, a1);
            to_half4<kCode>(__byte_perm(w2[j >> 1], w3[j >> 1], sel), a2, a3);
#pragma unroll
            for (int n = 0; n < kN; ++n) mma_16x8x16(st.o[n][j], a0, a1, a2, a3, w[n][i][0], w[n][i][1]);
        }
    }
}

template <int kCode, bool kCap, bool kBias>
__global__ void __launch_bounds__(kThreads, 1) paged_few_kernel(const __grid_constant__ FewPagedArgs a) {
    extern __shared__ uint8_t raw[];
    uint8_t* ring = raw + ((1024u - (smem_addr(raw) & 1023u)) & 1023u);  // 128-byte swizzle atoms
    Shared& s = *reinterpret_cast<Shared*>(ring + kStages * kStageBytes);
    const PagedCall& p = a.p;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

    if (tid == 0) {
        for (int i = 0; i < kStages; ++i) {
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
    const Meta meta = *a.meta;
    if (meta.units == 0) return;  // cut for the chunked kernel, or no rows
    if (tid <= meta.ctas) s.cuts[tid] = a.cuts[tid];
    __syncthreads();
    bool ok = true;  // after a wait that timed out: no more waits, but every barrier and counter is kept

    if (warp < kWarps) {
        // ============================ consumers ============================
        take_registers<kConsumerRegs>();
        const int g = lane >> 2, t = lane & 3;
        int mine = warp;            // this warp's next tile, counted from the piece's first
        int stg = warp, phase = 0;  // its stage
        int passes = 0;             // pairs of queries handed over so far
        for (int n = 0; (int)blockIdx.x < meta.ctas; ++n) {
            const int sl = n & 1;
            // One outcome for the warp: a lane that left alone would leave the others in a vote.
            ok = __all_sync(0xffffffffu, ok && mbar_wait(&s.qfull[sl], (n >> 1) & 1));
            if (!ok) break;  // (all that follow give up too)
            const Slot& slot = s.slot[sl];
            const int pairs = slot.pairs, tiles = slot.tiles, tile0 = slot.tile;
            const bool last = slot.last;
            State st;
#pragma unroll
            for (int q = 0; q < kPairsQ; ++q) {
#pragma unroll
                for (int i = 0; i < 8; ++i)
#pragma unroll
                    for (int e = 0; e < 4; ++e) st.o[q][i][e] = 0.f;
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    st.m[q][e] = -INFINITY;
                    st.l[q][e] = 0.f;
                }
            }
            // This warp's tiles: every kWarps-th of the CTA's.
            for (; mine < tiles; mine += kWarps) {
                if (ok) ok = mbar_wait(&s.full[stg], phase);
                const uint8_t* stage = ring + stg * kStageBytes;
                const int key0 = (tile0 + mine) * kTile;
                const float cap2 = p.cap * 1.4426950408889634f;
                const float4 sc = s.scales[stg], vi = s.v_inv[stg];
                if (pairs == 1)
                    consume_tile<kCode, kCap, kBias, 1>(st, stage, sc, vi, slot, cap2, key0, p.c.page_shift, lane);
                else if (pairs == 2)
                    consume_tile<kCode, kCap, kBias, 2>(st, stage, sc, vi, slot, cap2, key0, p.c.page_shift, lane);
                else
                    consume_tile<kCode, kCap, kBias, 3>(st, stage, sc, vi, slot, cap2, key0, p.c.page_shift, lane);
                __syncwarp();
                if (lane == 0) mbar_arrive(&s.empty[stg]);
                stg += kWarps;
                if (stg >= kStages) {
                    stg -= kStages;
                    phase ^= 1;
                }
            }
            mine -= tiles;
            __syncwarp();
            if (lane == 0) mbar_arrive(&s.qempty[sl]);

            // This warp's part of the piece, for the finishers, two queries at a time.
            auto& r = s.result;
#pragma unroll
            for (int q = 0; q < kPairsQ; ++q) {
                if (q >= pairs) break;
                float l[2] = {st.l[q][0], st.l[q][1]};
#pragma unroll
                for (int d = 4; d < 32; d <<= 1) {
                    l[0] += __shfl_xor_sync(0xffffffffu, l[0], d);
                    l[1] += __shfl_xor_sync(0xffffffffu, l[1], d);
                }
                if (ok && passes >= 1) ok = mbar_wait(&s.rempty, (passes - 1) & 1);
#pragma unroll
                for (int e = 0; e < 2; ++e)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        *reinterpret_cast<float4*>(&r.acc[warp][2 * t + e][16 * g + 4 * i]) =
                            make_float4(st.o[q][2 * i][e], st.o[q][2 * i][2 + e], st.o[q][2 * i + 1][e],
                                        st.o[q][2 * i + 1][2 + e]);
                if (g == 0) {
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        r.m[warp][2 * t + e] = st.m[q][e];
                        r.l[warp][2 * t + e] = l[e];
                    }
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(&s.rfull);
                ++passes;
            }
            if (last) break;
        }
    } else if (warp < kLoaderWarp) {
        // ============================ finishers ============================
        // A warp a head: the consumers' parts of a piece to output rows, or, for a
        // piece of a unit, to partial rows -- while the consumers go on.
        take_registers<kRestRegs>();
        Walk walk;
        walk.start(a, meta);
        const int hq = warp - kFinishWarp;
        int passes = 0;
        for (; walk.n > 0;) {
            const Unit& un = walk.unit;
            const int pairs = (un.n + 1) >> 1;
            const bool whole = walk.n == un.tiles;
            const int64_t first = walk.unit_first(a);
            auto share_of = [&](int64_t tile) {  // the last cut at or before it
                int lo = 0, hi = meta.ctas;
                while (hi - lo > 1) {
                    const int mid = (lo + hi) >> 1;
                    if (s.cuts[mid] <= tile) lo = mid; else hi = mid;
                }
                return lo;
            };
            // A share's first piece goes to its slot 0; its last, if another one, to
            // slot 1: only the unit's first CTA can have begun before it.
            int c0 = 0, pieces = 1, second = 0;
            if (!whole) {
                c0 = share_of(first);
                pieces = share_of(first + un.tiles - 1) - c0 + 1;
                second = s.cuts[c0] < first ? 1 : 0;
            }
            auto piece = [&](int c, int q, int e) {
                return a.partials + ((int64_t)(((c0 + c) * 2 + (c ? 0 : second)) * kUnitRows) + (2 * q + e) * kGroup + hq) * kRowF;
            };
            auto write = [&](int q, int e, float4 x, float l) {
                const int token = 2 * q + e;
                if (token >= un.n) return;
                const float inv = l == 0.f ? 0.f : kWeightUnit / l;  // 0 for a row that sees nothing
                const __nv_bfloat162 u = __floats2bfloat162_rn(x.x * inv, x.y * inv), v = __floats2bfloat162_rn(x.z * inv, x.w * inv);
                *reinterpret_cast<uint2*>(p.out + (int64_t)(un.row0 + token) * p.out_row_stride +
                                          (walk.h * kGroup + hq) * p.out_head_stride + 4 * lane) =
                    make_uint2(*reinterpret_cast<const uint32_t*>(&u), *reinterpret_cast<const uint32_t*>(&v));
            };
            for (int q = 0; q < pairs; ++q, ++passes) {
                if (ok) ok = mbar_wait(&s.rfull, passes & 1);
                __syncwarp();
                const auto& r = s.result;
                float M[2], L[2];
                float4 A[2];
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int row = 2 * hq + e;
                    M[e] = -INFINITY;
                    L[e] = 0.f;
                    A[e] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                    for (int w = 0; w < kWarps; ++w) M[e] = fmaxf(M[e], r.m[w][row]);
                    const float mu = M[e] == -INFINITY ? 0.f : M[e];
#pragma unroll
                    for (int w = 0; w < kWarps; ++w) {
                        const float f = fast_exp2(r.m[w][row] - mu);
                        const float4 x = *reinterpret_cast<const float4*>(&r.acc[w][row][4 * lane]);
                        L[e] = fmaf(f, r.l[w][row], L[e]);
                        A[e] = make_float4(fmaf(f, x.x, A[e].x), fmaf(f, x.y, A[e].y), fmaf(f, x.z, A[e].z), fmaf(f, x.w, A[e].w));
                    }
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(&s.rempty);
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    if (whole) {
                        write(q, e, A[e], L[e]);
                    } else {
                        float* mine = piece((int)blockIdx.x - c0, q, e);
                        *reinterpret_cast<float4*>(mine + 4 * lane) = A[e];
                        if (lane == 0) *reinterpret_cast<float2*>(mine + kHeadDim) = make_float2(M[e], L[e]);
                    }
                }
            }
            if (!whole) {
                __syncwarp();
                uint32_t before = 0;
                if (lane == 0)  // releases the warp's rows and acquires the others'
                    asm volatile("atom.add.acq_rel.gpu.global.u32 %0, [%1], 1;"
                                 : "=r"(before)
                                 : "l"(a.arrivals + c0 * kGroup + hq)
                                 : "memory");
                if (__shfl_sync(0xffffffffu, before, 0) == (uint32_t)(pieces - 1)) {
                    constexpr int kAtOnce = 6;
                    for (int token = 0; token < un.n; ++token) {
                        const int q = token >> 1, e = token & 1;
                        float M = -INFINITY, L = 0.f;
                        float4 A = make_float4(0.f, 0.f, 0.f, 0.f);
                        for (int c = 0; c < pieces; c += kAtOnce) {
                            float4 v[kAtOnce];
                            float2 ml[kAtOnce];
                            float now = M;
#pragma unroll
                            for (int i = 0; i < kAtOnce; ++i) {
                                const float* x = piece(min(c + i, pieces - 1), q, e);
                                ml[i] = __ldcg(reinterpret_cast<const float2*>(x + kHeadDim));
                                v[i] = __ldcg(reinterpret_cast<const float4*>(x + 4 * lane));
                            }
#pragma unroll
                            for (int i = 0; i < kAtOnce; ++i) now = fmaxf(now, ml[i].x);
                            const float use = now == -INFINITY ? 0.f : now;
                            const float f0 = fast_exp2(M - use);
                            M = now;
                            L *= f0;
                            A = make_float4(A.x * f0, A.y * f0, A.z * f0, A.w * f0);
#pragma unroll
                            for (int i = 0; i < kAtOnce; ++i)
                                if (c + i < pieces) {
                                    const float f = fast_exp2(ml[i].x - use);
                                    L = fmaf(f, ml[i].y, L);
                                    A = make_float4(fmaf(f, v[i].x, A.x), fmaf(f, v[i].y, A.y), fmaf(f, v[i].z, A.z), fmaf(f, v[i].w, A.w));
                                }
                        }
                        write(q, e, A, L);
                    }
                }
            }
            if (!walk.next(a)) break;
        }
    } else {
        take_registers<kRestRegs>();
        Walk walk;
        walk.start(a, meta);
        if (warp < kQueryWarp) {
            // ============================ loaders ============================
            // kBurst tiles at once, a tile a lane; each group of kBurst stages has one of the warps.
            const uint64_t policy = l2_evict_first_policy();
            const int shift = p.c.page_shift;
            const bool two = shift < kTileShift;  // two pages a tile (16 tokens each)
            const int box_bytes = min(p.c.page_len, kTile) * kHeadDim;
            int stg = 0, round = 0;  // next stage, times round the ring
            while (walk.n > 0 && ok) {
                const int64_t lo = walk.unit.lo, hi = walk.unit.hi;
                const int32_t* row = p.block_table + walk.unit.b * p.table_stride;
                const int tile = walk.unit.tile0 + walk.j;
                struct Pages {
                    int a, b;
                };
                auto entry = [&](int64_t key) {
                    if (key >= hi || key + min(p.c.page_len, kTile) <= lo) return -1;
                    const int page = row[key >> shift];
                    return page >= 0 && page < p.c.pages ? page : p.c.pages;  // out of the map: TMA fills zeros
                };
                // Lane's tile of a batch of 32: its pages (-1: no visible key, not loaded) and their scales.
                auto pages = [&](int j) {
                    const int64_t key = (int64_t)(tile + j + lane) << kTileShift;
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
                // Entries a batch of 32 tiles ahead of their use, scales with the batch before.
                Pages now = pages(0);
                float4 f_now = scales(now);
                for (int j0 = 0; j0 < walk.n && ok; j0 += 32) {
                    const Pages next = pages(j0 + 32);
                    const int batch_n = min(32, walk.n - j0);
                    for (int k0 = 0, n; k0 < batch_n; k0 += n) {
                        n = min(kBurst - stg % kBurst, batch_n - k0);  // to the end of the group
                        const bool mine = stg / kBurst % kLoaders == warp - kLoaderWarp && lane >= k0 && lane < k0 + n;
                        const int to = stg + lane - k0;
                        if (mine && round > 0) ok = mbar_wait(&s.empty[to], (round - 1) & 1);
                        ok = __all_sync(0xffffffffu, ok);
                        if (!ok) break;
                        if (mine) {
                            uint8_t* dst = ring + to * kStageBytes;
                            const int prow = two ? 0 : ((tile + j0 + lane) * kTile) & (p.c.page_len - 1);
                            if (now.a >= 0) {
                                tma_load_page(dst, &a.kmap, prow, walk.h, now.a, &s.full[to], policy);
                                tma_load_page(dst + kHalfBytes, &a.vmap, prow, walk.h, now.a, &s.full[to], policy);
                            }
                            if (now.b >= 0) {
                                tma_load_page(dst + box_bytes, &a.kmap, 0, walk.h, now.b, &s.full[to], policy);
                                tma_load_page(dst + kHalfBytes + box_bytes, &a.vmap, 0, walk.h, now.b, &s.full[to], policy);
                            }
                            const VLog2 va = v_log2_of(f_now.z), vb = v_log2_of(f_now.w);
                            const float nan = __int_as_float(0x7fffffff);
                            s.scales[to] = make_float4(fabsf(f_now.z) <= 3.402823466e38f ? f_now.x : nan,
                                                       fabsf(f_now.w) <= 3.402823466e38f ? f_now.y : nan, va.log2, vb.log2);
                            s.v_inv[to] = make_float4(va.inv, vb.inv, va.some ? 1.f : 0.f, vb.some ? 1.f : 0.f);
                            mbar_arrive_expect_tx(&s.full[to], 2 * ((now.a >= 0) + (now.b >= 0)) * box_bytes);
                        }
                        stg += n;
                        if (stg == kStages) {
                            stg = 0;
                            ++round;
                        }
                    }
                    now = next;
                    f_now = scales(next);
                }
                if (!walk.next(a)) break;
            }
            if (!ok)
                // Do not leave while copies into this CTA's shared memory are in flight.
                for (int i = 0; i < kStages; ++i) {
                    const int filled = i < stg ? round + 1 : round;  // times stage i was, its own group's
                    if (i / kBurst % kLoaders == warp - kLoaderWarp && filled > 0) mbar_wait(&s.full[i], (filled - 1) & 1);
                }
        } else if (warp == kQueryWarp) {
            // ============================ queries ============================
            const uint64_t step0 = a.rope.step[2 * lane], step1 = a.rope.step[2 * lane + 1];
            for (int n = 0; walk.n > 0; ++n) {
                const int sl = n & 1;
                if (n >= 2 && !warp_wait(&s.qempty[sl], ((n >> 1) - 1) & 1)) {
                    ok = false;
                    break;
                }
                __syncwarp();
                Slot& slot = s.slot[sl];
                const Unit& un = walk.unit;
                if (kBias && lane < kGroup) slot.slope[lane] = p.slopes[walk.h * kGroup + lane] * 1.4426950408889634f;
                // A column's dims 2 lane, 2 lane + 1 and 64 above them, to the lanes that hold them.
                auto put = [&](int q, int column, int dim, uint32_t x) {
                    uint32_t* to = reinterpret_cast<uint32_t*>(&slot.q[q][(dim & 31) >> 3][column * 4 + (dim >> 5)]);
                    to[(dim & 7) >> 1] = x;
                };
                int lo_most = 0, hi_least = 0x7fffffff;
                const int len = paged_length(p, un.b);
                for (int token = 0; token < 2 * ((un.n + 1) >> 1); ++token) {
                    const int q = token >> 1, e = token & 1;
                    if (token >= un.n) {  // the second of a pair, not there: it sees what the first sees
                        for (int hq = 0; hq < kGroup; ++hq) {
                            put(q, 2 * hq + e, 2 * lane, 0u);
                            put(q, 2 * hq + e, kPairs + 2 * lane, 0u);
                        }
                        if (lane < kGroup) slot.factor[q][2 * lane + e] = 0.f;
                        if (lane == 0) {
                            slot.lo[token] = slot.lo[token - 1];
                            slot.hi[token] = slot.hi[token - 1];
                        }
                        continue;
                    }
                    const int64_t m = (int64_t)un.pos0 + token;
                    const __nv_bfloat16* at = p.q + (int64_t)(un.row0 + token) * p.q_row_stride +
                                              walk.h * kGroup * p.q_head_stride + 2 * lane;
                    uint32_t xw[kGroup], yw[kGroup];
#pragma unroll
                    for (int hq = 0; hq < kGroup; ++hq) {
                        xw[hq] = *reinterpret_cast<const uint32_t*>(at + hq * p.q_head_stride);
                        yw[hq] = *reinterpret_cast<const uint32_t*>(at + hq * p.q_head_stride + kPairs);
                    }
                    const KeyRange r = paged_range(p, un.row0 + token, m, len);
                    float2 f0 = make_float2(1.f, 0.f), f1 = f0;
                    if (!p.q_rotated) {
                        f0 = rope_factor_fast(step0, m);
                        f1 = rope_factor_fast(step1, m);
                    }
#pragma unroll
                    for (int hq = 0; hq < kGroup; ++hq) {
                        const float2 x = bf16x2_to_float2(xw[hq]), y = bf16x2_to_float2(yw[hq]);
                        const float v0 = x.x * f0.x - y.x * f0.y, v1 = x.y * f1.x - y.y * f1.y;
                        const float v2 = x.x * f0.y + y.x * f0.x, v3 = x.y * f1.y + y.y * f1.x;
                        const float most = fmaxf(fmaxf(fabsf(v0), fabsf(v1)), fmaxf(fabsf(v2), fabsf(v3)));
                        const bool fine = __all_sync(0xffffffffu, most <= 3.402823466e38f && v0 == v0 && v1 == v1 &&
                                                                      v2 == v2 && v3 == v3);
                        // (Magnitudes are non-negative: their bits order as integers.)
                        const uint32_t top = __reduce_max_sync(0xffffffffu, __float_as_uint(most));
                        // 2^e just above the largest (2^-126 at least), e <= 127 so that its inverse is a normal number.
                        const int ex = min(253, max(1, (int)(top >> 23) + 1));
                        const float up = __int_as_float(ex << 23), down = __int_as_float((254 - ex) << 23);
                        put(q, 2 * hq + e, 2 * lane, pack_half2(v0 * down, v1 * down));
                        put(q, 2 * hq + e, kPairs + 2 * lane, pack_half2(v2 * down, v3 * down));
                        const float unit = kCap ? p.scale / p.cap : p.scale * 1.4426950408889634f;
                        if (lane == hq) slot.factor[q][2 * hq + e] = fine ? unit * up : __int_as_float(0x7fffffff);
                    }
                    if (lane == 0) {
                        slot.lo[token] = r.lo;
                        slot.hi[token] = r.hi;
                    }
                    lo_most = max(lo_most, r.lo);
                    hi_least = min(hi_least, r.hi);
                }
                if (lane == 0) {
                    slot.lo_most = lo_most;
                    slot.hi_least = hi_least;
                    slot.m = max(un.pos0, -(1 << 30));  // (distances stay 32-bit)
                    slot.tile = un.tile0 + walk.j;
                    slot.tiles = walk.n;
                    slot.pairs = (un.n + 1) >> 1;
                }
                const bool more = walk.next(a);
                if (lane == 0) slot.last = !more;
                __syncwarp();
                if (lane == 0) mbar_arrive(&s.qfull[sl]);
                if (!more) break;
            }
        } else {
            // Units whose rows see nothing.
            const int per_row = p.c.kv_heads * kGroup;
            for (int u = blockIdx.x; u < meta.units; u += gridDim.x) {
                const Unit un = a.units[u];
                if (un.tiles > 0) continue;
                for (int i = 0; i < un.n * per_row; ++i)
                    *reinterpret_cast<uint2*>(p.out + (int64_t)(un.row0 + i / per_row) * p.out_row_stride +
                                              (i % per_row) * p.out_head_stride + 4 * lane) = make_uint2(0u, 0u);
            }
        }
    }
    if (!ok) atomicOr(a.status, kDevStatusTimeout);  // (any lane's)
}

constexpr int kSmemBytes = 1024 + kStages * kStageBytes + (int)sizeof(Shared);
static_assert(kSmemBytes <= 227 * 1024, "shared memory of one CTA");
static_assert(kWarps % kBurst == 0 && kStages % (kBurst * kLoaders) == 0 && kStages % kWarps == 0,
              "each stage has one loader and one consumer warp");

using Kernel = void (*)(FewPagedArgs);

Kernel kernel_for(int code, bool cap, bool bias) {
    if (code == GQA_CODE_INT8) {
        if (cap) return bias ? paged_few_kernel<0, true, true> : paged_few_kernel<0, true, false>;
        return bias ? paged_few_kernel<0, false, true> : paged_few_kernel<0, false, false>;
    }
    if (cap) return bias ? paged_few_kernel<1, true, true> : paged_few_kernel<1, true, false>;
    return bias ? paged_few_kernel<1, false, true> : paged_few_kernel<1, false, false>;
}

// Behind the chunked kernel's.  Units enough for any split of the rows, so that a call
// with more rows never needs less.
UnitRegions regions(int batch, int rows, int heads, int sms) {
    return unit_regions(paged_chunk_workspace(batch, rows, heads, sms), batch, rows, kTokens, (size_t)sms * kGroup, sms,
                        (size_t)sms * 2 * kUnitRows * kRowF * sizeof(float));
}

}  // namespace

int paged_few_tile() { return kTile; }

size_t paged_few_workspace(int batch, int rows, int heads, int sms) { return regions(batch, rows, heads, sms).end; }

UnitShape paged_few_shape(const PagedCall& call, int sms, uint8_t* ws) {
    const int ctas = sms < kMaxCtas ? sms : kMaxCtas;
    return unit_shape(regions(call.batch, call.rows, call.c.kv_heads, sms), ws, call.rows / kTokens + call.batch, ctas,
                      ctas * kGroup, true);
}

cudaError_t paged_few_prepare() {
    for (int i = 0; i < 8; ++i) {
        // The register shares are of kLaunchRegs a thread: with fewer at launch the kernel would wait for good.
        cudaFuncAttributes at;
        cudaError_t e = cudaFuncGetAttributes(&at, kernel_for(i & 1, i & 2, i & 4));
        if (e != cudaSuccess) return e;
        if (at.numRegs != kLaunchRegs) return cudaErrorInvalidConfiguration;
        e = cudaFuncSetAttribute(kernel_for(i & 1, i & 2, i & 4), cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemBytes);
        if (e != cudaSuccess) return e;
    }
    return cudaSuccess;
}

cudaError_t launch_paged_few(const PagedCall& call, const RopeSteps& rope, int code, const CUtensorMap& kmap,
                             const CUtensorMap& vmap, const UnitShape& shape, uint32_t* status, cudaStream_t stream) {
    const UnitPlan& pl = shape.to;
    const FewPagedArgs a{kmap, vmap, call, rope, status, pl.meta, pl.units, pl.starts, pl.cuts, pl.arrivals, shape.partials};
    return launch_dependent(kernel_for(code, call.cap > 0.f, call.slopes != nullptr), shape.ctas, kThreads, kSmemBytes,
                            stream, a);
}

}  // namespace gqa
