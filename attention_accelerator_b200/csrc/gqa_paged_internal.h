// gqa_paged_internal.h -- launch entry points of the paged attention kernels.
#pragma once

#include "gqa_paged.cuh"

namespace gqa {

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
cudaError_t launch_paged_decode(const PagedCall& call, const RopeSteps& rope, int code, const CUtensorMap& kmap,
                                const CUtensorMap& vmap, int sms, uint8_t* ws, cudaStream_t stream);

// Any number of queries a sequence: units and shares, then the kernel for them
// (gqa_paged_units.cuh).
int paged_chunk_tile();
size_t paged_chunk_workspace(int batch, int rows, int heads, int sms);
int paged_few_tile();
size_t paged_few_workspace(int batch, int rows, int heads, int sms);

}  // namespace gqa
