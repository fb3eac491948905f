// gqa_paged_internal.h -- launch entry points of the paged attention kernels.
#pragma once

#include "gqa_paged.cuh"

namespace gqa {

// The cache a call names, checked.  A status.
int check_paged_cache(const gqa_paged_cache* c, PagedCacheView* v);

// TMA map of K or V codes: (128, page_len, heads, pages) bytes, box (128,
// min(page_len, rows), 1, 1), 128-byte swizzle.  A status.
int paged_map(CUtensorMap* map, const uint8_t* base, const PagedCacheView& c, int rows);

// Workspace of both attention calls: status word, one counter per (sequence, Q
// head) -- zero between calls -- and partial rows.
constexpr size_t kPagedArrivalsOffset = 256;
constexpr size_t kPagedPartialsOffset =
    kPagedArrivalsOffset + (size_t)GQA_PAGED_MAX_BATCH * kNumQHeads * sizeof(uint32_t);

// One token a sequence.
int paged_decode_tile();
size_t paged_decode_workspace(int sms);
// With `scores`, every score and the rows' sums as well (call.evicted says how far the queries
// stand behind their rows).
struct PagedScores {
    float* scores;    // [batch][heads][keys][4], log2 units; null: none
    float* row_log2;  // [batch][Q heads]: log2 of the sum of 2^score
    int64_t keys;
};
cudaError_t launch_paged_decode(const PagedCall& call, const RopeSteps& rope, int code, const CUtensorMap& kmap,
                                const CUtensorMap& vmap, int sms, uint8_t* ws, const PagedScores& scores,
                                cudaStream_t stream);

// The keys' accumulated weights (gqa_key_weights, checked): [batch][heads][capacity].
struct KeyWeightsView {
    float* weight;
    int32_t *position, *evicted;
    int64_t capacity;
};

// Workspace of the one-token call that adds up weights: behind decode_paged's.
struct ScoreRegions {
    size_t row_log2, scores, end;
};
inline ScoreRegions score_regions(int batch, int heads, int64_t keys, int sms) {
    ScoreRegions r;
    r.row_log2 = (paged_decode_workspace(sms) + 255) & ~(size_t)255;
    r.scores = r.row_log2 + (((size_t)batch * heads * kGroup * sizeof(float) + 255) & ~(size_t)255);
    r.end = r.scores + (size_t)batch * heads * keys * kGroup * sizeof(float);
    return r;
}
cudaError_t launch_score_weights(const PagedCall& call, const PagedScores& scores, const KeyWeightsView& weights, int sms,
                                 cudaStream_t stream);

// The weights of any number of queries (gqa_paged_weigh.cu).
int paged_weigh_box();
size_t paged_weigh_workspace(int batch, int rows, int heads, int64_t keys, int sms);
cudaError_t launch_paged_weigh(const PagedCall& call, const RopeSteps& rope, int code, const CUtensorMap& kmap,
                               const KeyWeightsView& weights, const int32_t* known, int sms, uint8_t* ws,
                               cudaStream_t stream);

// Any number of queries a sequence: units and shares, then the kernel for them
// (gqa_paged_units.cuh).
int paged_chunk_tile();
size_t paged_chunk_workspace(int batch, int rows, int heads, int sms);
int paged_few_tile();
size_t paged_few_workspace(int batch, int rows, int heads, int sms);

}  // namespace gqa
