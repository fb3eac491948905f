// gqa_paged_weigh.cu -- the attention weight that keys of the paged 8-bit cache get,
// summed over queries and over the Q heads of a KV head's group.
//
//   weight[b][h][k] += sum over queries i that see k, Q heads g of h:  2^(z_igk - log2 sum_k' 2^z_igk')
//
// One token a sequence: paged_decode_kernel leaves its scores (16 bytes a key and KV
// head) and the rows' sums; score_weights_kernel turns them into weights.
//
// Any number of queries, in four kernels on the fifth-generation tensor cores:
//   weigh_queries_kernel  rotates the queries of a unit (64 consecutive queries of a
//                         sequence, one KV head: 256 rows) and leaves them as two FP16
//                         parts in the operand layout, so that no later pass rotates again.
//   weigh_kernel, rows    S = Q K^T, a thread a row: running maximum and sum over the keys.
//   weigh_kernel, keys    S^T = K Q^T, a thread a key and a quarter of the rows: the sum of
//                         2^(z - row's log2) over the rows needs no exchange between
//                         lanes.  A sequence's only unit adds to the weights at once;
//                         of several each share keeps its own sums, and
//   join_sums_kernel      adds those share by share: no atomics.
// The sums of a row are known only once all its keys were seen, so the product is
// computed twice; keeping it (1 KB a key and KV head for 64 queries) would move eight
// times the bytes that the codes have.
//
// Precision.  The weights are FP32 results: Q, divided by a power of two that brings a
// row's largest below 1, is split into two FP16 parts (22 bits), both products
// accumulate in the same FP32 columns; codes are exact.  Scores past kFar are rounded to
// FP32 before a row's reference is taken from them, and the reference before its sum's
// logarithm: in one step the rounding of a large product would be left in the exponent.
//
// Bound: a tile of 128 keys for a unit takes 2048 cycles of the tensor pipe (two parts of
// Q) and 2048 of the special-function unit in each pass; overlapped they come to 3100
// (rows: S has one place for each M tile, the queries' parts take the other half of TMEM)
// and 3900 (keys).  Measured (B200): the last 64 queries of 8 prompts of up to 16384 keys,
// e4m3, 198 to 222 us (9 + 97 + 115 + 4 one by one), 32 queries 142, 5 queries
// 122; 6 ragged prompts of up to 2051 tokens, every query, int8, cap 50, 328 to 348 us (32 +
// 150 + 165 + 7).  The keys' pass goes unit by unit: with a thread block for each key's
// tile, which needs no joining, a run has few tiles, the queries' 128 KB are loaded for
// each, and the pass took 235 (for one unit a sequence the join costs 2, for two 9 of 348).
// score_weights_kernel: 64 ragged sequences (2.3 M keys and heads, 90 MB, mostly
// from L2) 11 us.
//
// Warps of weigh_kernel (one CTA per SM; shares of even cost, from the lengths in device
// memory, which every CTA sums itself):
//   0-15      sums, four groups of four: a thread a row and half of the tile's keys (rows: two
//             groups each M tile), or a key and a quarter of the columns (keys)
//   16-19     codes to FP16: to the B operand in shared memory (rows), or a thread a key to
//             the A operand in TMEM (keys)
//   20        MMA issuer
//   21, 22    loaders of codes and of queries
//   23        finds the share's runs, ahead of all others
// The A operand is in TMEM in both passes -- the unit's queries, written by the rows'
// threads, or the tile's keys -- because two operands of 128 x 16 in shared memory are
// read at half the rate of the products; so are the operands' other users, 1700 of a
// tile's cycles in all.
#include "gqa_internal.h"
#include "gqa_paged.cuh"
#include "gqa_paged_internal.h"
#include "gqa_tcgen05.cuh"

namespace gqa {

namespace {

// ---------------------------------------------------------------------------
// One token a sequence: scores to weights.
// ---------------------------------------------------------------------------
struct ScoreArgs {
    PagedCall p;
    PagedScores s;
    KeyWeightsView w;
};

constexpr int kScoreThreads = 256, kScoreKeys = 4;  // keys a thread at a time

// From such scores on a row's sum has to stand beside its largest score, not in one number with it: a number of that
// size has no room for the logarithm.
constexpr float kFar = 0x1p10f;

// A row's largest score and log2 of the sum of 2^(score - it), over `len` keys, by the block: for the head `head` of
// the scores.  (Seldom: each block goes through the row.)
__device__ __noinline__ float2 row_of_scores(const float* scores, int head, int len) {
    __shared__ float part[kScoreThreads / 32];
    auto over_block = [&](float v, bool largest) {
        auto join = [&](float x, float y) { return largest ? fmaxf(x, y) : x + y; };
#pragma unroll
        for (int d = 16; d; d >>= 1) v = join(v, __shfl_xor_sync(0xffffffffu, v, d));
        __syncthreads();  // (what stood there has been read)
        if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
        __syncthreads();
        v = part[0];
        for (int w = 1; w < kScoreThreads / 32; ++w) v = join(v, part[w]);
        return v;
    };
    float most = -INFINITY, sum = 0.f;
    for (int64_t k = threadIdx.x; k < len; k += kScoreThreads) most = fmaxf(most, __ldcg(scores + k * kGroup + head));
    most = over_block(most, true);
    for (int64_t k = threadIdx.x; k < len; k += kScoreThreads) sum += fast_exp2(__ldcg(scores + k * kGroup + head) - most);
    return make_float2(most, log2f(over_block(sum, false)));
}

__global__ void __launch_bounds__(kScoreThreads) score_weights_kernel(const __grid_constant__ ScoreArgs a) {
    dependency_wait();
    allow_dependents();
    const int heads = a.p.c.kv_heads, b = blockIdx.x / heads;
    const int len = paged_length(a.p, b), last = a.p.seq_lens[b] - 1;
    if (len == 0) return;
    const int64_t at = (int64_t)blockIdx.x * a.w.capacity;
    const float4* scores = reinterpret_cast<const float4*>(a.s.scores) + (int64_t)blockIdx.x * a.s.keys;
    float4 sum = *reinterpret_cast<const float4*>(a.s.row_log2 + (int64_t)blockIdx.x * kGroup), most = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int g = 0; g < kGroup; ++g) {
        float &log2 = (&sum.x)[g], &top = (&most.x)[g];
        if (fabsf(log2) >= kFar) {
            const float2 row = row_of_scores(reinterpret_cast<const float*>(scores), g, len);
            top = row.x;
            log2 = row.y;
        }
    }
    constexpr int kBlock = kScoreThreads * kScoreKeys;
    for (int64_t k0 = (int64_t)blockIdx.y * kBlock + threadIdx.x; k0 < len; k0 += (int64_t)gridDim.y * kBlock) {
        float4 z[kScoreKeys];
        float old[kScoreKeys];
#pragma unroll
        for (int i = 0; i < kScoreKeys; ++i) {
            const int64_t k = k0 + i * kScoreThreads;
            if (k >= len) break;
            z[i] = __ldcg(scores + k);
            old[i] = k < last ? a.w.weight[at + k] : 0.f;
        }
#pragma unroll
        for (int i = 0; i < kScoreKeys; ++i) {
            const int64_t k = k0 + i * kScoreThreads;
            if (k >= len) break;
            const float w = (fast_exp2((z[i].x - most.x) - sum.x) + fast_exp2((z[i].y - most.y) - sum.y)) +
                            (fast_exp2((z[i].z - most.z) - sum.z) + fast_exp2((z[i].w - most.w) - sum.w));
            a.w.weight[at + k] = old[i] + w;
            if (k == last) a.w.position[at + k] = last + (last > 0 ? paged_evicted(a.p, b) : 0);
        }
    }
    if (last == 0 && blockIdx.x == b * heads && blockIdx.y == 0 && threadIdx.x == 0) a.w.evicted[b] = 0;
}

// ---------------------------------------------------------------------------
// Any number of queries.
// ---------------------------------------------------------------------------
constexpr int kTokens = 64;                        // queries of a unit
constexpr int kRows = kTokens * kGroup;            // its rows
constexpr int kTile = 128, kTileShift = 7;         // keys
constexpr int kRawBytes = kTile * kHeadDim;
constexpr int kBlockBytes = kTile * 128;           // 64 dims of a tile in FP16
constexpr int kTileBytes = 2 * kBlockBytes;
constexpr int kQBlockBytes = kRows * 128;          // 64 dims of a part of the rows
constexpr int kQBytes = 4 * kQBlockBytes;          // [part][64 dims][row]
constexpr int kScaleSlots = 16;
constexpr int kConvWarp = 16, kMmaWarp = 20, kLoadWarp = 21, kQueryWarp = 22, kWalkWarp = 23;
constexpr int kThreads = 24 * 32, kPrepThreads = 8 * 32;
// Registers: launched with 80 a thread; each group of four warps takes its share.
constexpr int kLaunchRegs = 80, kSumRegs = 88, kConvRegs = 64, kRestRegs = 64;
static_assert(4 * kSumRegs + kConvRegs + kRestRegs <= 6 * kLaunchRegs, "of what the CTA was launched with");
// TMEM.  Rows: S of each M tile, then its queries' two parts.  Keys: three S of up to 128 columns, two tiles of keys.
constexpr uint32_t kTmemCols = 512;
constexpr uint32_t kColQ = 256, kColK = 384;
constexpr int kSums = 3;  // S of the keys' pass
constexpr int kParts = 4; // tiles whose quarters' sums wait to be joined
constexpr int kRuns = 4;  // runs found ahead
// What a unit costs beside its tiles when the shares of the rows' pass are cut, in tiles.
constexpr int kUnitCost = 2;
// The rows' reference is the largest of the first keys; a sum of weights past 2^kOverflow moves it.
constexpr float kOverflow = 0x1p90f;
// (kFar: from such references on a score is rounded before they are taken from it.  The test of it costs both passes 2 %:
// a window of 64 queries on 8 x 16384 keys 217 -> 220 us.)

// Shared memory of a pass: rings of codes and of FP16 tiles, or of codes beside the queries.
template <bool kKeys>
struct Rings {
    static constexpr int kRaw = kKeys ? 4 : 3, kConv = kKeys ? 2 : 4;
    static constexpr int kBytes = kRaw * kRawBytes + (kKeys ? kQBytes : kConv * kTileBytes);
};

// kind::f16, FP16 A and B (both K-major), FP32 accumulators, M = 128.
constexpr uint32_t kIdesc = (1u << 4) | ((128u >> 4) << 24);
__device__ __forceinline__ constexpr uint32_t idesc_n(uint32_t n) { return kIdesc | ((n >> 3) << 17); }

// A share's part of one (sequence, head) whose queries are several units: the first
// run's sums and, if there are more runs, those of the others, which all begin at tile 0.
// (sequence, head) + share numbers them: it grows by one at least from each to the next.
struct Piece {
    int64_t cell;    // of the first run's first tile
    int a0, a1, b1;  // tiles of the first run, [a0, a1), and of the others, [0, b1)
};

struct alignas(64) WeighArgs {
    CUtensorMap kmap;  // (128, page_len, heads, pages) bytes, box (128, page_len, 1, 1)
    PagedCall p;
    RopeSteps rope;
    KeyWeightsView w;
    const int32_t* known;
    uint32_t* status;
    uint8_t* queries;    // [units * heads][kQBytes]
    float* factor;       // [units * heads][kRows]: z of a row is its product times the page's scale times this
    float2* row_sums;    // [units * heads][kRows]: reference, and log2 of the sum of 2^(z - reference)
    uint32_t* arrivals;  // [units * heads]
    float2* partials;    // [ctas][2][kRows]: reference and sum
    Piece* pieces;       // [batch * heads + ctas]
    int2* shares_of;     // [batch * heads]: first and last share
    float* sums;         // of pieces: by cell, or two rows a piece (sum_rows)
    int64_t sum_rows;    // floats of such a row; 0: by cell
    int64_t max_cells;
    int max_units;
};

// A sequence's queries and keys.  Queries at negative positions see nothing and are left out.
struct Seq {
    int row0, n, pos0, len;  // first query row, queries, the first one's row of the cache, keys
    int tiles, units, id0;   // tiles of keys, units of queries, number of the first unit in the call
    int c;                   // ceil(pos0 / 64)
    __device__ __forceinline__ Seq() {}
    __device__ __forceinline__ Seq(const PagedCall& p, int b) {
        const int first = min(max(p.first_query[b], 0), p.rows);
        const int all = max(0, min(p.first_query[b + 1], p.rows) - first), keys = max(0, p.seq_lens[b]);
        n = min(all, keys);
        row0 = first + all - n;
        pos0 = keys - n;
        len = paged_length(p, b);
        tiles = (len + kTile - 1) >> kTileShift;
        units = (n + kTokens - 1) / kTokens;
        // A number for each unit that needs no sum over the sequences: it grows by one from unit to unit and by
        // one at least from sequence to sequence.
        id0 = row0 / kTokens + b;
        c = (pos0 + kTokens - 1) / kTokens;
    }
    // Tiles that unit u sees: of the keys up to its last query, ceil((pos0 + 64 (u + 1)) / 128) = floor((c + u + 2) / 2).
    __device__ __forceinline__ int unit_tiles(int u) const {
        return min(tiles, u < units - 1 ? (c + u + 2) >> 1 : (int)(((int64_t)pos0 + n + kTile - 1) >> kTileShift));
    }
    // Cells of units before u, a unit's own cost and one a tile: the sum of floor(i / 2) up to i < k is floor((k - 1)^2 / 4).
    __device__ __forceinline__ int64_t unit_cells(int u) const {
        const int v = min(u, units - 1);
        const int whole = min(v, max(0, 2 * tiles - c - 2));  // units that do not see all tiles
        auto f = [](int64_t k) { return (k - 1) * (k - 1) / 4; };
        int64_t cells = f((int64_t)c + 2 + whole) - f((int64_t)c + 2) + (int64_t)(v - whole) * tiles;
        if (u == units && units > 0) cells += unit_tiles(units - 1);
        return cells + (int64_t)u * kUnitCost;
    }
    __device__ __forceinline__ int64_t cells() const { return units == 0 ? 0 : unit_cells(units); }
};

// A CTA's share, run by run: consecutive tiles for one unit of queries and one head.
struct Walk {
    const PagedCall& p;
    Seq q;
    int b, h, u;             // sequence, head, unit
    int tile0, count;        // of the run
    int64_t cell, base, end; // cell of the run's first tile; of the sequence's first; the share's end
    __device__ __forceinline__ Walk(const PagedCall& call) : p(call) {}

    __device__ __forceinline__ int id() const { return q.id0 + u; }
    __device__ __forceinline__ int queries() const { return min(kTokens, q.n - u * kTokens); }
    __device__ __forceinline__ int pos() const { return q.pos0 + u * kTokens; }
    __device__ __forceinline__ int64_t head_cell() const { return base + h * q.cells(); }  // the head's first cell

    // From cell x (of sequence `seq`, whose first cell is `first`) to `stop`.
    __device__ __forceinline__ void start(int seq, int64_t first, int64_t x, int64_t stop) {
        count = 0;
        end = stop;
        if (x >= stop) return;
        b = seq;
        base = first;
        q = Seq(p, b);
        const int64_t each = q.cells();
        h = (int)((x - base) / each);
        const int64_t rem = x - base - h * each;
        int lo = 0, hi = q.units;  // the last unit at or before the cell
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (q.unit_cells(mid) <= rem) lo = mid; else hi = mid;
        }
        u = lo;
        tile0 = (int)max((int64_t)0, rem - q.unit_cells(u) - kUnitCost);
        run();
    }
    // To the next run; count is 0 at the share's end.
    __device__ __forceinline__ void next() {
        tile0 = 0;
        if (++u == q.units) {
            u = 0;
            if (++h == p.c.kv_heads) {
                h = 0;
                base += q.cells() * p.c.kv_heads;
                do {
                    if (++b >= p.batch || base >= end) {
                        count = 0;
                        return;
                    }
                    q = Seq(p, b);
                } while (q.units == 0);
            }
        }
        run();
    }

private:
    __device__ __forceinline__ void run() {
        cell = head_cell() + q.unit_cells(u) + kUnitCost + tile0;
        count = (int)max((int64_t)0, min((int64_t)(q.unit_tiles(u) - tile0), end - cell));
    }
};

// A run as the warps of a CTA take it.
struct Run {
    int b, h, u, count;       // sequence, head, unit, tiles (0: the share's end)
    int tile0, n, pos, len;   // first tile, queries, the first one's row, keys of the sequence
    int known, evicted;       // keys
    int add_below;            // keys, sums of several units: tiles below it add to what is there (-1: the only unit)
    int64_t out;              // and where tile 0's would be, in floats
    int tiles, c0, parts, second;  // rows: the unit's tiles; its first share, its shares, the first one's slot
    int64_t cell;             // unit and head
};

struct alignas(16) Shared {
    Run runs[kRuns];
    uint64_t run_full[kRuns], run_empty[kRuns];
    uint64_t raw_full[4], raw_empty[4], conv_full[4], conv_empty[4];
    uint64_t q_full[2], q_empty, s_full[4], s_empty[kSums];  // s_full, keys: [half][tile % 2]
    uint64_t part_full[kParts];
    uint64_t drain;  // products in flight when the issuer gives up
    float scales[kScaleSlots][8];
    float4 columns[4][2][kRows / 8];  // keys: factors and -log2 of two columns, of a quarter's run and the next
    float4 far[4][2][kRows / 8];      // and of those past kFar, whose -log2 is 0 there, reference and logarithm
    float part[kParts][3][kTile];     // keys: sums of the quarters but the first
    float2 other[2][2][kTile];        // rows: references and sums of the second half of the keys
    long long warp_sum[kThreads / 32];
    long long start_base;
    int start_b;
    uint32_t tmem;
    int last;
};

// Rotation and split of a unit's queries, and the row's factors.  Lane = (query, 16 pairs).
struct PrepArgs {
    PagedCall p;
    RopeSteps rope;
    const int32_t* known;
    uint8_t* queries;
    float* factor;
    uint32_t* arrivals;
    Piece* pieces;
    int2* shares_of;
    int n_pieces;
};

__device__ __forceinline__ uint32_t bf16_magnitudes(uint32_t w) { return max(w << 16 & 0x7fffffffu, w & 0x7fff0000u); }

// A sequence without rows before these is a new one: nothing was evicted from it.
__device__ __forceinline__ int known_of(const int32_t* known, int b, const Seq& q) { return known ? known[b] : q.pos0; }

__global__ void __launch_bounds__(kPrepThreads, 2) weigh_queries_kernel(const __grid_constant__ PrepArgs a) {
    const PagedCall& p = a.p;
    const int id = blockIdx.x, h = blockIdx.y, tid = threadIdx.x, token = tid >> 2, q4 = tid & 3;
    __shared__ uint64_t step[kPairs];
    if (tid < kPairs) step[tid] = a.rope.step[tid];
    dependency_wait();
    allow_dependents();
    for (int i = (blockIdx.y * gridDim.x + blockIdx.x) * kPrepThreads + tid; i < a.n_pieces;
         i += gridDim.x * gridDim.y * kPrepThreads)
        a.pieces[i] = Piece{0, 0, 0, 0};
    for (int i = (blockIdx.y * gridDim.x + blockIdx.x) * kPrepThreads + tid; i < p.batch * p.c.kv_heads;
         i += gridDim.x * gridDim.y * kPrepThreads)
        a.shares_of[i] = make_int2(0, -1);
    // The last sequence whose first unit has this number or a lower one: a thread a candidate, of stretches and then of
    // the one that it lies in (the numbers grow).
    int lo = 0;
    for (int room = p.batch; room > 1;) {
        const int stride = (room + kPrepThreads - 1) / kPrepThreads, at = lo + tid * stride;
        const int below = __syncthreads_count(tid * stride < room && Seq(p, at).id0 <= id);
        lo += max(0, below - 1) * stride;
        room = min(stride, p.batch - lo);
    }
    const Seq q(p, lo);
    const int u = id - q.id0;
    if (u < 0 || u >= q.units) return;
    const int64_t cell = (int64_t)id * p.c.kv_heads + h;
    if (tid == 0) a.arrivals[cell] = 0;
    __syncthreads();  // (the steps)
    const int n = min(kTokens, q.n - u * kTokens);
    if (token >= ((n + 15) & ~15)) return;  // whole steps of 64 rows are read
    const bool real = token < n;
    const int64_t pos = (int64_t)q.pos0 + u * kTokens + token +
                        (known_of(a.known, lo, q) > 0 ? paged_evicted(p, lo) : 0);
    const float unit = p.cap > 0.f ? p.scale / p.cap : p.scale * 1.4426950408889634f;
    const uint4 none = make_uint4(0u, 0u, 0u, 0u);
    const uint4* src = reinterpret_cast<const uint4*>(p.q + (int64_t)(q.row0 + u * kTokens + token) * p.q_row_stride +
                                                      h * kGroup * p.q_head_stride + 8 * q4);
    // Of a head's pairs 8 q4 to 8 q4 + 7 and those 32 further on, first and then second elements, asked for a head
    // ahead.  (Four lanes write 64 bytes in a row, whole sectors; with 16 pairs in a row a lane, halves of them, the
    // kernel took 44 us instead of 33 for 6700 tokens of 8 heads.)
    auto load = [&](int hq, int i) { return real ? src[hq * (p.q_head_stride / 8) + 4 * i] : none; };
    uint4 next[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) next[i] = load(0, i);
    float2 f[16];
#pragma unroll
    for (int i = 0; i < 16; ++i)
        f[i] = p.q_rotated ? make_float2(1.f, 0.f) : rope_factor(step[8 * q4 + (i & 7) + 4 * (i & 8)], pos);
    uint8_t* out = a.queries + cell * kQBytes;
#pragma unroll 1
    for (int hq = 0; hq < kGroup; ++hq) {
        uint4 w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            w[i] = next[i];
            if (hq + 1 < kGroup) next[i] = load(hq + 1, i);
        }
        // A power of two above the row's largest: a rotated pair passes it by no more than sqrt(2).
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            top = max(top, max(max(bf16_magnitudes(w[i].x), bf16_magnitudes(w[i].y)),
                               max(bf16_magnitudes(w[i].z), bf16_magnitudes(w[i].w))));
        const unsigned quad = 0xfu << (tid & 28);
        top = max(top, __shfl_xor_sync(quad, top, 1));
        top = max(top, __shfl_xor_sync(quad, top, 2));
        const int e = min(253, max(1, (int)(top >> 23) + 1));
        const float down = __int_as_float((254 - e) << 23);
        const int row = token * kGroup + hq;
        if (q4 == 0)
            a.factor[cell * kRows + row] =
                !real ? 0.f : top < 0x7f800000u ? unit * __int_as_float(e << 23) : __int_as_float(0x7fffffff);
#pragma unroll
        for (int c = 0; c < 2; ++c) {  // 8 pairs: 16 bytes of each block of 64 dims, and of each part
            const uint4 u4 = w[c], v4 = w[c + 2];
            const uint32_t uw[4] = {u4.x, u4.y, u4.z, u4.w}, vw[4] = {v4.x, v4.y, v4.z, v4.w};
            uint32_t xh[4], xl[4], yh[4], yl[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float2 s = bf16x2_to_float2(uw[i]), t = bf16x2_to_float2(vw[i]);
                const float2 f0 = f[8 * c + 2 * i], f1 = f[8 * c + 2 * i + 1];
                const float x0 = (s.x * f0.x - t.x * f0.y) * down, x1 = (s.y * f1.x - t.y * f1.y) * down;
                const float y0 = (s.x * f0.y + t.x * f0.x) * down, y1 = (s.y * f1.y + t.y * f1.x) * down;
                const float hx0 = __half2float(__float2half_rn(x0)), hx1 = __half2float(__float2half_rn(x1));
                const float hy0 = __half2float(__float2half_rn(y0)), hy1 = __half2float(__float2half_rn(y1));
                xh[i] = pack_half2(hx0, hx1);
                xl[i] = pack_half2(x0 - hx0, x1 - hx1);
                yh[i] = pack_half2(hy0, hy1);
                yl[i] = pack_half2(y0 - hy0, y1 - hy1);
            }
            uint8_t* to = out + row * 128 + (((q4 + 4 * c) ^ (row & 7)) << 4);
            *reinterpret_cast<uint4*>(to) = make_uint4(xh[0], xh[1], xh[2], xh[3]);
            *reinterpret_cast<uint4*>(to + kQBlockBytes) = make_uint4(yh[0], yh[1], yh[2], yh[3]);
            *reinterpret_cast<uint4*>(to + 2 * kQBlockBytes) = make_uint4(xl[0], xl[1], xl[2], xl[3]);
            *reinterpret_cast<uint4*>(to + 3 * kQBlockBytes) = make_uint4(yl[0], yl[1], yl[2], yl[3]);
        }
    }
}

// cap2 * tanh of a thread's scores (multiples of the cap in, log2 units out), as cap_scores, two at a time.
template <int kN>
__device__ __forceinline__ void cap_pairs(float (&z)[kN], float cap2) {
    auto both = [](float v) { return make_float2(v, v); };
    float x[kN], most = 0.f;
#pragma unroll
    for (int i = 0; i < kN; i += 2) {
        const float2 v = make_float2(z[i], z[i + 1]), t = __fmul2_rn(v, v);
        x[i] = v.x;
        x[i + 1] = v.y;
        most = fmaxf(fmaxf(most, t.x), t.y);
        float2 y = __ffma2_rn(both(kTanh9), t, both(kTanh7));
        y = __ffma2_rn(y, t, both(kTanh5));
        y = __ffma2_rn(y, t, both(kTanh3));
        y = __fmul2_rn(__ffma2_rn(y, t, both(1.f)), __fmul2_rn(v, both(cap2)));
        z[i] = y.x;
        z[i + 1] = y.y;
    }
    if (most > kTanhNear)
#pragma unroll
        for (int i = 0; i < kN; ++i)
            if (x[i] * x[i] > kTanhNear) z[i] = cap2 * tanh_far(x[i]);
    __syncwarp();
}

// Rows of a unit as the MMA takes them: whole steps of 64 columns.
__device__ __forceinline__ int columns_of(int n) { return (n * kGroup + 63) & ~63; }

// A copy that stays in L2 as others do: the unit's tiles are dealt to several CTAs.
__device__ __forceinline__ void bulk_load_queries(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_addr(dst)),
        "l"(src), "r"(bytes), "r"(smem_addr(bar))
        : "memory");
}

template <int kRegs>
__device__ __forceinline__ void take_registers() {
    if constexpr (kRegs > kLaunchRegs)
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegs));
    else
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegs));
}

template <int kCode, bool kCap, bool kKeys>
__global__ void __launch_bounds__(kThreads, 1) weigh_kernel(const __grid_constant__ WeighArgs a) {
    using R = Rings<kKeys>;
    constexpr int kRaw = R::kRaw, kConv = R::kConv;
    extern __shared__ uint8_t raw_smem[];
    uint8_t* smem = raw_smem + ((1024u - (smem_addr(raw_smem) & 1023u)) & 1023u);
    uint8_t* raw = smem;
    uint8_t* conv = raw + kRaw * kRawBytes;    // rows: the tiles in FP16
    uint8_t* q_smem = raw + kRaw * kRawBytes;  // keys: the unit's queries
    Shared& s = *reinterpret_cast<Shared*>(smem + R::kBytes);
    const PagedCall& p = a.p;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, heads = p.c.kv_heads;

    if (tid == 0) {
        for (int i = 0; i < kRaw; ++i) {
            mbar_init(&s.raw_full[i], 1);
            mbar_init(&s.raw_empty[i], 4);
        }
        for (int i = 0; i < kConv; ++i) {
            mbar_init(&s.conv_full[i], 4);
            mbar_init(&s.conv_empty[i], 1);
        }
        for (int i = 0; i < 4; ++i) mbar_init(&s.s_full[i], 1);
        for (int i = 0; i < kSums; ++i) mbar_init(&s.s_empty[i], 8);
        for (int i = 0; i < kParts; ++i) mbar_init(&s.part_full[i], 12);
        for (int i = 0; i < 2; ++i) mbar_init(&s.q_full[i], kKeys ? 1 : 8);
        for (int i = 0; i < kRuns; ++i) {
            mbar_init(&s.run_full[i], 1);
            mbar_init(&s.run_empty[i], kKeys ? kWalkWarp : kWalkWarp - 1);  // all other warps (rows: but the queries' loader)
        }
        mbar_init(&s.q_empty, 1);
        mbar_init(&s.drain, 1);
        fence_barrier_init();
        prefetch_tensormap(&a.kmap);
    }
    if (warp == kMmaWarp) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&s.tmem)),
                     "r"(kTmemCols)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    dependency_wait();
    allow_dependents();
    // Cells of all sequences, and the one that this share begins in.
    int64_t total, from, to;
    int64_t shares;
    {
        const int per = (p.batch + kThreads - 1) / kThreads;
        const int b0 = min(p.batch, tid * per), b1 = min(p.batch, b0 + per);
        long long sum = 0;
        for (int b = b0; b < b1; ++b) sum += Seq(p, b).cells() * heads;
        long long incl = sum;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const long long x = __shfl_up_sync(0xffffffffu, incl, d);
            if (lane >= d) incl += x;
        }
        if (lane == 31) s.warp_sum[warp] = incl;
        __syncthreads();
        long long at = incl - sum;
        total = 0;
        for (int w = 0; w < kThreads / 32; ++w) {
            if (w < warp) at += s.warp_sum[w];
            total += s.warp_sum[w];
        }
        total = min(total, a.max_cells);  // (numbers of first queries that fall: no access leaves the workspace)
        shares = max((int64_t)1, min((int64_t)gridDim.x, total / (kUnitCost + 1)));
        const int64_t me = blockIdx.x;
        from = me < shares ? total * me / shares : total;
        to = me < shares ? total * (me + 1) / shares : total;
        if (from < to && at <= from && from < at + sum)
            for (int b = b0; b < b1; ++b) {
                const int64_t each = Seq(p, b).cells() * heads;
                if (from < at + each) {
                    s.start_b = b;
                    s.start_base = at;
                    break;
                }
                at += each;
            }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = s.tmem;
    bool ok = true;
    // The runs, in the order in which kWalkWarp finds them.  A warp that gave up goes through the others without work;
    // the waits here last longer than all that can be waited for in between.
    int run_i = 0;
    auto next_run = [&](Run& r) {
        const int at = run_i & (kRuns - 1);
        bool got = false;
        for (int i = 0; i < 16 && !got; ++i) got = warp_wait(&s.run_full[at], run_i / kRuns & 1);
        r = s.runs[at];
        if (!got) ok = false;
        return got && r.count > 0;
    };
    auto end_run = [&] {
        __syncwarp();
        if (lane == 0) mbar_arrive(&s.run_empty[run_i & (kRuns - 1)]);
        ++run_i;
    };
    Run run;

    if (warp < kConvWarp) {
        // ============================ sums ============================
        take_registers<kSumRegs>();
        const int g = warp >> 3, part = warp >> 2 & 1, r = tid & (kTile - 1);
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
        const float cap2 = p.cap * 1.4426950408889634f;
        int slot = 0;  // scales of the tile
        auto next_slot = [&] { slot = (slot + 1) & (kScaleSlots - 1); };
        if constexpr (!kKeys) {
            // A thread a row of M tile g and half of a tile's keys; S and queries of the M tile are these eight warps'.
            const uint32_t t_s = tmem + lanes + g * kTile + 64 * part, t_q = tmem + lanes + kColQ + g * kTile + 64 * part;
            int phase = 0, runs = 0;
            for (; next_run(run); end_run()) {
                const int n = run.n, token = 32 * g + (r >> 2);
                const bool active = n > 32 * g, real = token < n;
                const int64_t cell = run.cell;
                const float factor = real ? a.factor[cell * kRows + g * kTile + r] : 0.f;
                const int hi = real ? min(run.pos + token + 1, run.len) : 0x7fffffff;
                float ref = -INFINITY, l = 0.f;
                if (active) {
                    // One part of the row's queries to TMEM (the products that read the last ones were waited for).
                    const uint8_t* src = a.queries + cell * kQBytes + (g * kTile + r) * 128 + 2 * part * kQBlockBytes;
#pragma unroll
                    for (int b = 0; b < 2; ++b) {
                        uint32_t w[32];
#pragma unroll
                        for (int c = 0; c < 8; ++c)
                            reinterpret_cast<uint4*>(w)[c] =
                                real ? *reinterpret_cast<const uint4*>(src + b * kQBlockBytes + ((c ^ (r & 7)) << 4))
                                     : make_uint4(0u, 0u, 0u, 0u);
                        tmem_st32(t_q + 32 * b, w);
                    }
                    tmem_wait_st();
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&s.q_full[g]);
                }
                for (int t = 0; t < run.count; ++t, next_slot()) {
                    if (!active) continue;
                    if (ok) ok = warp_wait(&s.s_full[g], phase);
                    phase ^= 1;
                    tc_fence_after();
                    const int k0 = ((run.tile0 + t) << kTileShift) + 64 * part;
                    const bool masked = __any_sync(0xffffffffu, hi < k0 + 64);
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        const bool edge = kCap ? masked : __any_sync(0xffffffffu, masked || fabsf(ref) >= kFar);  // (or -inf)
                        float z[32];
                        tmem_ld32(t_s + 32 * c, reinterpret_cast<uint32_t(&)[32]>(z));
                        float f0 = factor * s.scales[slot][4 * part + 2 * c], f1 = factor * s.scales[slot][4 * part + 2 * c + 1];
                        tmem_wait_ld();
                        if (c == 1) {
                            tc_fence_before();
                            __syncwarp();
                            if (lane == 0) mbar_arrive(&s.s_empty[g]);
                        }
                        if (kCap || edge) {  // scaled before the mask: -inf times a scale of 0 is none
#pragma unroll
                            for (int e = 0; e < 32; ++e) z[e] *= e < 16 ? f0 : f1;
                            f0 = f1 = 1.f;
                        }
                        if constexpr (kCap) {
                            cap_pairs(reinterpret_cast<float(&)[16]>(z[0]), cap2);
                            cap_pairs(reinterpret_cast<float(&)[16]>(z[16]), cap2);
                        }
                        if (edge) {
                            const int left = hi - k0 - 32 * c;
#pragma unroll
                            for (int e = 0; e < 32; ++e)
                                if (e >= left) z[e] = -INFINITY;
                        }
                        // Sum of 2^(z - ref) over the chunk, z times its factor.
                        auto chunk = [&](float use) {
                            float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
                            for (int e = 0; e < 32; e += 2) {
                                const float f = e < 16 ? f0 : f1;
                                float2 x = make_float2(z[e], z[e + 1]);
                                x = kCap ? __fadd2_rn(x, make_float2(-use, -use))
                                         : __ffma2_rn(x, make_float2(f, f), make_float2(-use, -use));
                                sum[e >> 1 & 1] = __fadd2_rn(sum[e >> 1 & 1], make_float2(fast_exp2(x.x), fast_exp2(x.y)));
                            }
                            return (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
                        };
                        float sum = ref == -INFINITY ? INFINITY : chunk(ref);
                        if (!(sum < kOverflow)) {  // the row's first keys, or larger ones by far
                            float mx = -INFINITY;
#pragma unroll
                            for (int e = 0; e < 32; ++e) {
                                if constexpr (!kCap) z[e] *= e < 16 ? f0 : f1;
                                mx = fmaxf(mx, z[e]);
                            }
                            f0 = f1 = 1.f;
                            const float now = fmaxf(ref, mx);
                            l *= fast_exp2(ref - (now == -INFINITY ? 0.f : now));
                            ref = now;
                            sum = chunk(now == -INFINITY ? 0.f : now);
                        }
                        l += sum;
                        __syncwarp();
                    }
                }
                // ---- the run's rows: both halves of the keys ----
                float2& other = s.other[runs & 1][g][r];
                ++runs;
                if (part) other = make_float2(ref, l);
                named_barrier_sync(2 + g, 2 * kTile);
                if (!part) {
                    const float now = fmaxf(ref, other.x), use = now == -INFINITY ? 0.f : now;
                    l = l * fast_exp2(ref - use) + other.y * fast_exp2(other.x - use);
                    ref = now;
                    float2* out = a.row_sums + cell * kRows + g * kTile + r;
                    auto row_of = [&](float m, float sum) {
                        return !real ? make_float2(INFINITY, 0.f) : sum == 0.f ? make_float2(-INFINITY, 0.f) : make_float2(m, log2f(sum));
                    };
                    if (run.count == run.tiles) {
                        if (active) *out = row_of(ref, l);
                    } else {
                        // A piece of a unit.
                        const int c0 = run.c0, parts = run.parts, second = run.second;
                        auto piece = [&](int c) {
                            return a.partials + (int64_t)((c0 + c) * 2 + (c ? 0 : second)) * kRows + g * kTile + r;
                        };
                        if (active) *piece((int)blockIdx.x - c0) = make_float2(ref, l);
                        named_barrier_sync(1, 2 * kTile);
                        if (tid == 0) {
                            uint32_t before;
                            asm volatile("atom.add.acq_rel.gpu.global.u32 %0, [%1], 1;"
                                         : "=r"(before)
                                         : "l"(a.arrivals + cell)
                                         : "memory");
                            s.last = before == (uint32_t)(parts - 1);
                        }
                        named_barrier_sync(1, 2 * kTile);
                        if (s.last && active) {
                            float M = -INFINITY, L = 0.f;
                            for (int c = 0; c < parts; ++c) {
                                const float2 x = __ldcg(piece(c));
                                const float top = fmaxf(M, x.x), by = top == -INFINITY ? 0.f : top;
                                L = L * fast_exp2(M - by) + x.y * fast_exp2(x.x - by);
                                M = top;
                            }
                            *out = row_of(M, L);
                        }
                        named_barrier_sync(1, 2 * kTile);  // s.last is read
                    }
                }
            }
        } else {
            // A thread a key and a quarter of the columns; S of a tile's halves follow one another.
            // (A half has full barriers of its own: a wait by parity tells only one phase from the next.)
            int buf = g, tiles = 0, runs = 0;
            for (; next_run(run); end_run()) {
                const int half = columns_of(run.n) >> 1, mine = half >> 1, col0 = g * half + part * mine;
                const int64_t cell = run.cell;
                float4 *column = s.columns[2 * g + part][runs & 1], *far_column = s.far[2 * g + part][runs & 1];
                ++runs;
                bool mine_far = false;
                if (r < mine) {
                    const int at = (r >> 1) * 4 + (r & 1);
                    float *to = reinterpret_cast<float*>(column) + at, *far_to = reinterpret_cast<float*>(far_column) + at;
                    const float2 row = a.row_sums[cell * kRows + col0 + r];
                    mine_far = fabsf(row.x) >= kFar && fabsf(row.x) < INFINITY;
                    to[0] = a.factor[cell * kRows + col0 + r];
                    to[2] = mine_far ? 0.f : -(row.x + row.y);
                    far_to[0] = mine_far ? -row.x : 0.f;
                    far_to[2] = mine_far ? -row.y : 0.f;
                }
                const bool far = named_barrier_or(2 + 2 * g + part, kTile, mine_far);
                // The only unit's sums are added to the weights; those of several units are joined behind this kernel.
                const bool only = run.add_below < 0;
                const int known = run.known, len = run.len;
                float* out = only ? a.w.weight + ((int64_t)run.b * heads + run.h) * a.w.capacity : a.sums + run.out;
                int32_t* position = a.w.position + ((int64_t)run.b * heads + run.h) * a.w.capacity;
                for (int t = 0; t < run.count; ++t, ++tiles, next_slot()) {
                    const int tile = run.tile0 + t, key = (tile << kTileShift) + r;
                    const bool held = warp < 4 && (!only || key < len);
                    float weight = 0.f;
                    if (held && (only ? key < known : tile < run.add_below)) weight = out[key];
                    if (ok) ok = warp_wait(&s.s_full[2 * g + (tiles & 1)], (tiles >> 1) & 1);
                    tc_fence_after();
                    // Rows that see the key: from this column on.  (All do that stand 64 rows and more behind it; up to 2^31.)
                    const int from_col = max(key - run.pos, -kTokens) * kGroup - col0;
                    const bool edge = __any_sync(0xffffffffu, from_col > 0);
                    const float ks = s.scales[slot][r >> 4];
                    const uint32_t cols = tmem + lanes + buf * kTile + part * mine;
                    float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
                    for (int c = 0; c < mine >> 4; ++c) {  // 16 columns
                        float v[16];
                        tmem_ld16(cols + 16 * c, reinterpret_cast<uint32_t(&)[16]>(v));
                        tmem_wait_ld();
                        if (c + 1 == mine >> 4) {
                            tc_fence_before();
                            __syncwarp();
                            if (lane == 0) mbar_arrive(&s.s_empty[buf]);
                        }
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            const float4 k = column[8 * c + i];
                            const float2 f = __fmul2_rn(make_float2(k.x, k.y), make_float2(ks, ks));
                            float2 x = make_float2(v[2 * i], v[2 * i + 1]);
                            x = kCap ? __fmul2_rn(x, f) : __ffma2_rn(x, f, make_float2(k.z, k.w));
                            v[2 * i] = x.x;
                            v[2 * i + 1] = x.y;
                        }
                        if constexpr (kCap) {
                            cap_pairs(v, cap2);
#pragma unroll
                            for (int i = 0; i < 8; ++i) {
                                v[2 * i] += column[8 * c + i].z;
                                v[2 * i + 1] += column[8 * c + i].w;
                            }
                        }
                        if (far) {
#pragma unroll
                            for (int i = 0; i < 8; ++i) {
                                const float4 k = far_column[8 * c + i];
                                v[2 * i] = (v[2 * i] + k.x) + k.z;
                                v[2 * i + 1] = (v[2 * i + 1] + k.y) + k.w;
                            }
                        }
                        if (edge) {
                            const int skip = from_col - 16 * c;
#pragma unroll
                            for (int i = 0; i < 16; ++i)
                                if (i < skip) v[i] = -INFINITY;
                        }
#pragma unroll
                        for (int i = 0; i < 16; i += 2)
                            sum[i >> 1 & 1] = __fadd2_rn(sum[i >> 1 & 1], make_float2(fast_exp2(v[i]), fast_exp2(v[i + 1])));
                    }
                    buf += 2;  // (the other half's S lies between)
                    if (buf >= kSums) buf -= kSums;
                    const float total_mine = (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
                    const int ring = tiles & (kParts - 1);
                    if (warp >= 4) {
                        // (The first quarter is at most two tiles behind: S of the third would take the place of one
                        // that it has not read.)
                        s.part[ring][2 * g + part - 1][r] = total_mine;
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&s.part_full[ring]);
                    } else {
                        if (ok) ok = warp_wait(&s.part_full[ring], tiles / kParts & 1);
                        if (held) {
                            out[key] =
                                weight + ((total_mine + s.part[ring][0][r]) + (s.part[ring][1][r] + s.part[ring][2][r]));
                            if (only && key >= known) position[key] = key + run.evicted;
                            if (only && key == 0 && known <= 0 && run.h == 0) a.w.evicted[run.b] = 0;
                        }
                    }
                }
            }
        }
    } else if (warp < kMmaWarp) {
        // ============================ conversion ============================
        take_registers<kConvRegs>();
        const int cw = warp - kConvWarp, t = lane & 3;
        // Rows: as in the chunked attention kernel, eight lanes that access shared memory together have all eight
        // 16-byte columns of the codes' rows and of the operand's.  Keys: a lane a key, whose eight neighbours' rows
        // hold a chunk in eight different columns.
        const int row0 = 32 * cw + ((lane >> 3) ^ (lane & 4 ? 5 : 0)), key = 32 * cw + lane;
        int rs = 0, rphase = 0, cs = 0, cphase = 0, items = 0;
        for (; next_run(run); end_run()) {
            for (int j = 0; j < run.count && ok; ++j, ++items) {
                ok = mbar_wait(&s.raw_full[rs], rphase) && (items < kConv || mbar_wait(&s.conv_empty[cs], cphase ^ 1));
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                const uint8_t* src = raw + rs * kRawBytes;
                if constexpr (kKeys) {
                    tc_fence_after();  // the products that read this tile's place are done
                    const uint32_t to = tmem + ((uint32_t)(32 * cw) << 16) + kColK + cs * 64;
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        uint32_t w[32];
#pragma unroll
                        for (int c = 0; c < 4; ++c) {
                            const uint4 x = lds128(src + key * kHeadDim + (((4 * half + c) ^ (key & 7)) << 4));
                            to_half4<kCode>(x.x, w[8 * c], w[8 * c + 1]);
                            to_half4<kCode>(x.y, w[8 * c + 2], w[8 * c + 3]);
                            to_half4<kCode>(x.z, w[8 * c + 4], w[8 * c + 5]);
                            to_half4<kCode>(x.w, w[8 * c + 6], w[8 * c + 7]);
                        }
                        tmem_st32(to + 32 * half, w);
                    }
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&s.raw_empty[rs]);
                    tmem_wait_st();
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&s.conv_full[cs]);
                } else {
                    uint8_t* dst = conv + cs * kTileBytes;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int row = row0 + 8 * i, sw = row & 7;
#pragma unroll
                        for (int block = 0; block < 2; ++block) {
                            const uint4 x = lds128(src + row * kHeadDim + (((4 * block + t) ^ sw) << 4));
                            uint32_t w[8];
                            to_half4<kCode>(x.x, w[0], w[1]);
                            to_half4<kCode>(x.y, w[2], w[3]);
                            to_half4<kCode>(x.z, w[4], w[5]);
                            to_half4<kCode>(x.w, w[6], w[7]);
                            uint8_t* at = dst + block * kBlockBytes + row * 128;
                            *reinterpret_cast<uint4*>(at + (((2 * t) ^ sw) << 4)) = make_uint4(w[0], w[1], w[2], w[3]);
                            *reinterpret_cast<uint4*>(at + (((2 * t + 1) ^ sw) << 4)) = make_uint4(w[4], w[5], w[6], w[7]);
                        }
                    }
                    fence_proxy_async_smem();
                    __syncwarp();
                    if (lane == 0) {
                        mbar_arrive(&s.conv_full[cs]);
                        mbar_arrive(&s.raw_empty[rs]);
                    }
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
    } else {
    take_registers<kRestRegs>();
    if (warp == kMmaWarp) {
        // ============================ MMA issuer ============================
        const uint32_t leader = elect_lane(), cols = uniform(tmem);
        int cs = 0, cphase = 0, runs = 0;
        int used[2] = {0, 0}, q_runs[2] = {0, 0};  // rows: tiles and runs of each M tile
        int buf = 0, phase = 0, sums = 0, items = 0;  // keys
        auto next_tile = [&] {
            if (++cs == kConv) {
                cs = 0;
                cphase ^= 1;
            }
        };
        for (; next_run(run); end_run()) {
            if (!ok) continue;
            const int n = uniform(run.n), count = uniform(run.count);
            if constexpr (kKeys) {
                const int half = columns_of(n) >> 1;
                const uint32_t idesc = idesc_n(half);
                ok = warp_wait(&s.q_full[0], runs & 1);
                ++runs;
                const uint64_t qd = smem_desc_sw128(smem_addr(q_smem), 16, 1024);
                for (int j = 0; j < count && ok; ++j, ++items) {
                    ok = warp_wait(&s.conv_full[cs], cphase);
                    for (int h = 0; h < 2 && ok; ++h, ++sums) {
                        ok = sums < kSums || warp_wait(&s.s_empty[buf], phase ^ 1);
                        if (!ok) break;
                        tc_fence_after();
#pragma unroll
                        for (int part = 0; part < 2; ++part)
#pragma unroll
                            for (int kk = 0; kk < 8; ++kk)
                                mma_ts_by(leader, cols + buf * kTile, cols + kColK + cs * 64 + 8 * kk,
                                          qd + (((2 * part + (kk >> 2)) * kQBlockBytes + h * half * 128 + (kk & 3) * 32) >> 4),
                                          idesc, part || kk ? 1u : 0u);
                        tc_commit_by(leader, &s.s_full[2 * h + (items & 1)]);
                        if (++buf == kSums) {
                            buf = 0;
                            phase ^= 1;
                        }
                    }
                    if (!ok) break;
                    tc_commit_by(leader, &s.conv_empty[cs]);
                    if (j + 1 == count) tc_commit_by(leader, &s.q_empty);
                    next_tile();
                }
            } else {
                const int products = n <= 32 ? 1 : 2;
                for (int j = 0; j < count && ok; ++j) {
                    ok = warp_wait(&s.conv_full[cs], cphase);
                    const uint64_t kd = smem_desc_sw128(smem_addr(conv + cs * kTileBytes), 16, 1024);
                    for (int m = 0; m < products && ok; ++m) {
                        if (j == 0) {
                            ok = warp_wait(&s.q_full[m], q_runs[m] & 1);
                            ++q_runs[m];
                        }
                        ok = ok && (used[m] == 0 || warp_wait(&s.s_empty[m], (used[m] - 1) & 1));
                        if (!ok) break;
                        ++used[m];
                        tc_fence_after();
#pragma unroll
                        for (int part = 0; part < 2; ++part)
#pragma unroll
                            for (int kk = 0; kk < 8; ++kk)
                                mma_ts_by(leader, cols + m * kTile, cols + kColQ + m * kTile + 64 * part + 8 * kk,
                                          kd + (((kk >> 2) * kBlockBytes + (kk & 3) * 32) >> 4), idesc_n(kTile),
                                          part || kk ? 1u : 0u);
                        tc_commit_by(leader, &s.s_full[m]);
                    }
                    if (!ok) break;
                    tc_commit_by(leader, &s.conv_empty[cs]);
                    next_tile();
                }
            }
        }
        if (!ok) {  // shared memory and TMEM are given back with no product under way
            tc_commit_by(leader, &s.drain);
            warp_wait(&s.drain, 0);
        }
    } else if (warp == kLoadWarp) {
        // ============================ codes ============================
        const int shift = p.c.page_shift, per_tile = kTile >> shift;  // pages of a tile
        const int box_bytes = p.c.page_len * kHeadDim;
        const uint64_t policy = l2_evict_first_policy();
        int rs = 0, rphase = 0, items = 0, slot = 0;
        for (; next_run(run); end_run()) {
            if (!ok) continue;
            const int32_t* table = p.block_table + run.b * p.table_stride;
            const int64_t hi = run.len;
            // Lane's page of tile j of the run (-1: past the sequence's keys, not loaded).
            auto entry = [&](int j) {
                const int64_t key = ((int64_t)(run.tile0 + j) << kTileShift) + ((int64_t)lane << shift);
                if (lane >= per_tile || j >= run.count || key >= hi) return -1;
                const int page = table[key >> shift];
                return page >= 0 && page < p.c.pages ? page : p.c.pages;  // out of the map: TMA fills zeros
            };
            auto scale = [&](int page) {
                return page >= 0 && page < p.c.pages ? p.c.k_scale[page * p.c.scale_page_stride + run.h] : 0.f;
            };
            int page = entry(0), page1 = entry(1);
            float ks = scale(page);
            for (int j = 0; j < run.count; ++j, ++items) {
                const int page2 = entry(j + 2);
                const float ks1 = scale(page1);
                if (items >= kRaw) ok = __all_sync(0xffffffffu, mbar_wait(&s.raw_empty[rs], rphase ^ 1));
                if (!ok) break;
                const float x = __shfl_sync(0xffffffffu, ks, (lane & 7) >> (shift - 4));  // a lane 16 keys
                if (lane < 8) s.scales[slot][lane] = x;
                __syncwarp();
                slot = (slot + 1) & (kScaleSlots - 1);
                const uint32_t boxes = __popc(__ballot_sync(0xffffffffu, page >= 0));
                if (lane == 0) mbar_arrive_expect_tx(&s.raw_full[rs], boxes * box_bytes);
                __syncwarp();
                if (page >= 0)
                    tma_load_page(raw + rs * kRawBytes + lane * box_bytes, &a.kmap, 0, run.h, page, &s.raw_full[rs], policy);
                if (++rs == kRaw) {
                    rs = 0;
                    rphase ^= 1;
                }
                page = page1;
                page1 = page2;
                ks = ks1;
            }
        }
        if (!ok)  // do not leave while copies into this CTA's shared memory are in flight
            for (int i = 1; i <= kRaw && i <= items; ++i) {
                const int at = rs - i;
                mbar_wait(&s.raw_full[at < 0 ? at + kRaw : at], at < 0 ? rphase ^ 1 : rphase);
            }
    } else if (kKeys && warp == kQueryWarp) {
        // ============================ queries ============================
        int runs = 0;
        for (; next_run(run); end_run()) {
            if (!ok) continue;
            if (runs > 0) ok = warp_wait(&s.q_empty, (runs - 1) & 1);
            if (!ok) continue;  // (the last copies have landed: their products were waited for)
            const uint32_t bytes = columns_of(run.n) * 128;
            const uint8_t* src = a.queries + run.cell * kQBytes;
            if (lane == 0) mbar_arrive_expect_tx(&s.q_full[0], 4 * bytes);
            __syncwarp();
            if (lane < 4) bulk_load_queries(q_smem + lane * kQBlockBytes, src + lane * kQBlockBytes, bytes, &s.q_full[0]);
            ++runs;
        }
        if (runs > 0) warp_wait(&s.q_full[0], (runs - 1) & 1);  // no copy in flight when the CTA leaves
    } else if (warp == kWalkWarp && lane == 0) {
        // ============================ runs ============================
        Walk walk(p);
        walk.start(s.start_b, s.start_base, from, to);
        Piece piece;
        int unit = -1;  // (sequence, head) of the piece
        auto share_of = [&](int64_t x) { return (int)(min(((x + 1) * shares + total - 1) / total, shares) - 1); };
        for (int i = 0;; ++i) {
            const int at = i & (kRuns - 1);
            if (i >= kRuns) {
                ok = false;
                for (int k = 0; k < 8 && !ok; ++k) ok = mbar_wait(&s.run_empty[at], (i / kRuns - 1) & 1);
            }
            const bool more = ok && walk.count > 0;
            Run& r = s.runs[at];
            r.count = more ? walk.count : 0;
            if (more) {
                const Seq& q = walk.q;
                r.b = walk.b;
                r.h = walk.h;
                r.u = walk.u;
                r.tile0 = walk.tile0;
                r.n = walk.queries();
                r.pos = walk.pos();
                r.len = q.len;
                r.cell = (int64_t)walk.id() * heads + walk.h;
                if constexpr (kKeys) {
                    r.known = known_of(a.known, walk.b, q);
                    r.evicted = r.known > 0 ? paged_evicted(p, walk.b) : 0;
                    r.add_below = -1;
                    if (q.units > 1) {
                        const int now = walk.b * heads + walk.h;
                        const int64_t at_piece = now + blockIdx.x;
                        const bool first = now != unit;
                        if (first) {
                            unit = now;
                            piece = Piece{walk.cell, walk.tile0, walk.tile0 + walk.count, 0};
                            const int64_t from_cell = walk.head_cell();
                            a.shares_of[now] = make_int2(share_of(from_cell + kUnitCost), share_of(from_cell + q.cells() - 1));
                        }
                        // (The runs behind the first begin at tile 0, each reaching as far as the one before or, the
                        // share's last, less far.)
                        r.add_below = first ? 0 : piece.b1;
                        r.out = a.sum_rows ? (2 * at_piece + (first ? 0 : 1)) * a.sum_rows
                                : first    ? (piece.cell - piece.a0) * kTile
                                           : (piece.cell + piece.a1 - piece.a0) * kTile;
                        if (!first) piece.b1 = max(piece.b1, walk.count);
                        a.pieces[at_piece] = piece;
                    }
                } else {
                    r.tiles = q.unit_tiles(walk.u);
                    if (walk.count != r.tiles) {
                        // A share's first piece goes to its slot 0; its last, if another one, to slot 1: only the
                        // unit's first share can have begun before it.
                        const int64_t first = walk.cell - walk.tile0;  // the cell of the unit's first tile
                        r.c0 = share_of(first);
                        r.parts = share_of(first + r.tiles - 1) - r.c0 + 1;
                        r.second = total * r.c0 / shares < first - kUnitCost ? 1 : 0;
                    }
                }
            }
            mbar_arrive(&s.run_full[at]);
            if (!more) break;
            walk.next();
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

// The sums of sequences with several units, share by share, to the weights.
struct JoinArgs {
    PagedCall p;
    KeyWeightsView w;
    const int32_t* known;
    const Piece* pieces;
    const int2* shares_of;
    const float* sums;
    int64_t sum_rows;
};

constexpr int kJoined = 4;  // shares at a time

__device__ __forceinline__ void join_sums(const JoinArgs& a, int unit) {
    const int heads = a.p.c.kv_heads, b = unit / heads;
    const Seq q(a.p, b);
    if (q.units < 2) return;
    const int known = known_of(a.known, b, q), evicted = known > 0 ? paged_evicted(a.p, b) : 0;
    const int2 shares = a.shares_of[unit];
    const int64_t at = (int64_t)unit * a.w.capacity;
    for (int64_t key = (int64_t)blockIdx.y * kScoreThreads + threadIdx.x; key < q.len; key += (int64_t)gridDim.y * kScoreThreads) {
        const int tile = (int)(key >> kTileShift);
        float w = key < known ? a.w.weight[at + key] : 0.f;
        // (Several shares' loads at a time: 7.3 us for 6 prompts of up to 2051 keys and 8 heads, one by one 10.8.)
        for (int c0 = shares.x; c0 <= shares.y; c0 += kJoined) {
            Piece piece[kJoined];
            float2 part[kJoined];
#pragma unroll
            for (int i = 0; i < kJoined; ++i) {
                piece[i] = Piece{0, 0, 0, 0};
                if (c0 + i <= shares.y) piece[i] = a.pieces[unit + c0 + i];
            }
#pragma unroll
            for (int i = 0; i < kJoined; ++i) {
                const Piece& x = piece[i];
                const int64_t row = 2 * (int64_t)(unit + c0 + i) * a.sum_rows;
                part[i] = make_float2(0.f, 0.f);
                if (tile >= x.a0 && tile < x.a1)
                    part[i].x = __ldcg(a.sums + (a.sum_rows ? row : (x.cell - x.a0) * kTile) + key);
                if (tile < x.b1)
                    part[i].y = __ldcg(a.sums + (a.sum_rows ? row + a.sum_rows : (x.cell + x.a1 - x.a0) * kTile) + key);
            }
#pragma unroll
            for (int i = 0; i < kJoined; ++i) w = (w + part[i].x) + part[i].y;
        }
        a.w.weight[at + key] = w;
        if (key >= known) a.w.position[at + key] = (int)key + evicted;
        if (key == 0 && known <= 0 && unit == b * heads) a.w.evicted[b] = 0;
    }
}

// A block's units are every gridDim.x-th.
__global__ void __launch_bounds__(kScoreThreads) join_sums_kernel(const __grid_constant__ JoinArgs a) {
    dependency_wait();
    allow_dependents();
    const int all = a.p.batch * a.p.c.kv_heads, step = gridDim.x;
    for (int first = blockIdx.x; first < all; first += step * kScoreThreads) {
        const int end = min(all, first + step * kScoreThreads), mine = first + (int)threadIdx.x * step;
        // Where there are many, mostly of one query, the threads look at one each first.
        if (all > step && !__syncthreads_or(mine < end && Seq(a.p, mine / a.p.c.kv_heads).units > 1)) continue;
        for (int unit = first; unit < end; unit += step) join_sums(a, unit);
    }
}

template <bool kKeys>
constexpr int kSmemBytes = 1024 + Rings<kKeys>::kBytes + (int)sizeof(Shared);
static_assert(kSmemBytes<false> <= 227 * 1024 && kSmemBytes<true> <= 227 * 1024, "shared memory of one CTA");

using Kernel = void (*)(WeighArgs);

template <bool kKeys>
Kernel kernel_for(int code, bool cap) {
    if (code == GQA_CODE_INT8) return cap ? weigh_kernel<0, true, kKeys> : weigh_kernel<0, false, kKeys>;
    return cap ? weigh_kernel<1, true, kKeys> : weigh_kernel<1, false, kKeys>;
}

struct Regions {
    size_t partials, pieces, shares_of, arrivals, factor, row_sums, queries, sums, end;
    int64_t sum_rows, max_cells;
    int n_pieces;
};
// Units: their numbers (Seq) are below this.
int units_of(int batch, int rows) { return rows / kTokens + batch + 1; }
// The sums of several units by cell where there are few units, else two rows a piece: the smaller of both.
Regions regions(int batch, int rows, int heads, int64_t keys, int sms) {
    auto up = [](size_t x) { return (x + 255) & ~(size_t)255; };
    const size_t units = (size_t)units_of(batch, rows) * heads;
    Regions r;
    r.partials = up(kPagedPartialsOffset);
    r.n_pieces = batch * heads + sms;
    r.pieces = r.partials + up((size_t)sms * 2 * kRows * sizeof(float2));
    r.shares_of = r.pieces + up((size_t)r.n_pieces * sizeof(Piece));
    r.arrivals = r.shares_of + up((size_t)batch * heads * sizeof(int2));
    r.factor = r.arrivals + up(units * sizeof(uint32_t));
    r.row_sums = r.factor + units * kRows * sizeof(float);
    r.queries = r.row_sums + units * kRows * sizeof(float2);
    r.sums = r.queries + units * kQBytes;
    const size_t tiles = (size_t)((keys + kTile - 1) / kTile);
    const size_t by_cell = units * (tiles + kUnitCost) * kTile, by_row = 2 * (size_t)r.n_pieces * tiles * kTile;
    r.max_cells = (int64_t)(units * (tiles + kUnitCost));
    r.sum_rows = by_row < by_cell ? (int64_t)(tiles * kTile) : 0;
    r.end = r.sums + (rows > kTokens ? (by_row < by_cell ? by_row : by_cell) * sizeof(float) : 0);  // (else one unit each)
    return r;
}

}  // namespace

int paged_weigh_box() { return kTile; }

size_t paged_weigh_workspace(int batch, int rows, int heads, int64_t keys, int sms) {
    return regions(batch, rows, heads, keys, sms).end;
}

cudaError_t paged_weigh_prepare() {
    for (int i = 0; i < 8; ++i) {
        // The register shares are of kLaunchRegs a thread: with fewer at launch the kernel would wait for good.
        cudaFuncAttributes at;
        cudaError_t e = cudaFuncGetAttributes(&at, i & 4 ? kernel_for<true>(i & 1, i & 2) : kernel_for<false>(i & 1, i & 2));
        if (e != cudaSuccess) return e;
        if (at.numRegs != kLaunchRegs) return cudaErrorInvalidConfiguration;
        e = cudaFuncSetAttribute(i & 4 ? kernel_for<true>(i & 1, i & 2) : kernel_for<false>(i & 1, i & 2),
                                                   cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                   i & 4 ? kSmemBytes<true> : kSmemBytes<false>);
        if (e != cudaSuccess) return e;
    }
    return cudaSuccess;
}

cudaError_t launch_score_weights(const PagedCall& call, const PagedScores& scores, const KeyWeightsView& weights, int sms,
                                 cudaStream_t stream) {
    const ScoreArgs a{call, scores, weights};
    const int units = call.batch * call.c.kv_heads;
    const int64_t most = (scores.keys + kScoreThreads * kScoreKeys - 1) / (kScoreThreads * kScoreKeys);
    const int64_t want = ((int64_t)sms * 16 + units - 1) / units;
    return launch_dependent(score_weights_kernel, dim3(units, (unsigned)(want < most ? want : most)), kScoreThreads, 0,
                            stream, a);
}

cudaError_t launch_paged_weigh(const PagedCall& call, const RopeSteps& rope, int code, const CUtensorMap& kmap,
                               const KeyWeightsView& weights, const int32_t* known, int sms, uint8_t* ws,
                               cudaStream_t stream) {
    const int64_t keys = (int64_t)call.table_width << call.c.page_shift;
    const Regions r = regions(call.batch, call.rows, call.c.kv_heads, keys, sms);
    WeighArgs a;
    a.kmap = kmap;
    a.p = call;
    a.rope = rope;
    a.w = weights;
    a.known = known;
    a.status = reinterpret_cast<uint32_t*>(ws);
    a.queries = ws + r.queries;
    a.factor = reinterpret_cast<float*>(ws + r.factor);
    a.row_sums = reinterpret_cast<float2*>(ws + r.row_sums);
    a.arrivals = reinterpret_cast<uint32_t*>(ws + r.arrivals);
    a.partials = reinterpret_cast<float2*>(ws + r.partials);
    a.pieces = reinterpret_cast<Piece*>(ws + r.pieces);
    a.shares_of = reinterpret_cast<int2*>(ws + r.shares_of);
    a.sums = reinterpret_cast<float*>(ws + r.sums);
    a.sum_rows = r.sum_rows;
    a.max_cells = r.max_cells;
    a.max_units = units_of(call.batch, call.rows);
    const PrepArgs prep{call, rope, known, a.queries, a.factor, a.arrivals, a.pieces, a.shares_of, r.n_pieces};
    cudaError_t e = launch_dependent(weigh_queries_kernel, dim3(a.max_units, call.c.kv_heads), kPrepThreads, 0, stream, prep);
    if (e == cudaSuccess)
        e = launch_dependent(kernel_for<false>(code, call.cap > 0.f), dim3(sms), kThreads, kSmemBytes<false>, stream, a);
    if (e == cudaSuccess)
        e = launch_dependent(kernel_for<true>(code, call.cap > 0.f), dim3(sms), kThreads, kSmemBytes<true>, stream, a);
    if (e == cudaSuccess && call.rows > kTokens) {  // a sequence may have several units
        const JoinArgs join{call, weights, known, a.pieces, a.shares_of, a.sums, a.sum_rows};
        const int heads = call.batch * call.c.kv_heads;
        const int64_t most = (keys + kScoreThreads - 1) / kScoreThreads, want = ((int64_t)sms * 8 + heads - 1) / heads;
        e = launch_dependent(join_sums_kernel, dim3(heads < 8 * sms ? heads : 8 * sms, (unsigned)(want < most ? want : most)), kScoreThreads, 0, stream, join);
    }
    return e;
}

}  // namespace gqa
