// gqa_paged_units.cuh -- the units of a call with any number of queries a
// sequence: what plan_units_kernel leaves in the workspace for the kernel behind it.
#pragma once

#include "gqa_paged.cuh"
#include "gqa_paged_internal.h"

namespace gqa {

constexpr int kMaxCtas = 255;

struct Unit {
    int32_t b, row0, n, pos0;     // sequence, first query row, queries, position of the first
    int32_t lo, hi, tiles, tile0; // keys that any row sees, their tiles
    int64_t first, cell;          // tiles and cost of all units before it (per head)
};
struct Meta {
    int64_t total;  // tiles of all units and heads
    int32_t ctas;   // with a share
    int32_t units;
};
struct UnitPlan {
    Meta* meta;
    Unit* units;
    int32_t* starts;     // [ctas] unit in which each share begins
    int64_t* cuts;       // [ctas + 1] tiles (of all units and heads, in order) where the shares begin
    uint32_t* arrivals;  // counters, zeroed
};

// How a kernel wants a call cut, and where it reads that.
struct UnitShape {
    UnitPlan to;
    float* partials;
    int32_t max_units, ctas, counters;  // counters to zero (0: two a unit and head)
    bool few;
};

// Layout in the workspace, from `base` on; everything here is written by each call.
struct UnitRegions {
    size_t meta, starts, cuts, units, arrivals, partials, end;
};
inline UnitRegions unit_regions(size_t base, int batch, int rows, int tokens, size_t counters, int sms, size_t partials) {
    auto up = [](size_t x) { return (x + 255) & ~(size_t)255; };
    UnitRegions r;
    r.meta = base;
    r.starts = base + 256;
    r.cuts = r.starts + up((size_t)sms * sizeof(int32_t));
    r.units = r.cuts + up((size_t)(sms + 1) * sizeof(int64_t));
    r.arrivals = r.units + up(((size_t)rows / tokens + batch) * sizeof(Unit));
    r.partials = r.arrivals + up(counters * sizeof(uint32_t));
    r.end = r.partials + up(partials);
    return r;
}
inline UnitShape unit_shape(const UnitRegions& r, uint8_t* ws, int max_units, int ctas, int counters, bool few) {
    return UnitShape{UnitPlan{reinterpret_cast<Meta*>(ws + r.meta), reinterpret_cast<Unit*>(ws + r.units),
                              reinterpret_cast<int32_t*>(ws + r.starts), reinterpret_cast<int64_t*>(ws + r.cuts),
                              reinterpret_cast<uint32_t*>(ws + r.arrivals)},
                     reinterpret_cast<float*>(ws + r.partials), max_units, ctas, counters, few};
}

// A CTA's walk through its share, one unit's piece at a time.
struct Walk {
    int64_t x, end;
    int u, h, j, n;  // unit, KV head, first tile within the unit and tiles of the piece
    Unit unit;
    template <typename Args>
    __device__ __forceinline__ void start(const Args& a, const Meta& meta) {
        n = 0;
        const int me = blockIdx.x;
        if (me >= meta.ctas) return;
        x = a.cuts[me];
        end = a.cuts[me + 1];
        u = a.starts[me];
        unit = a.units[u];
        const int64_t rem = x - unit.first * a.p.c.kv_heads;
        h = (int)(rem / unit.tiles);
        place(a);
    }
    template <typename Args>
    __device__ __forceinline__ int64_t unit_first(const Args& a) const {
        return unit.first * a.p.c.kv_heads + (int64_t)h * unit.tiles;
    }
    template <typename Args>
    __device__ __forceinline__ void place(const Args& a) {
        j = (int)(x - unit_first(a));
        n = (int)min((int64_t)(unit.tiles - j), end - x);
    }
    template <typename Args>
    __device__ __forceinline__ bool next(const Args& a) {
        x += n;
        if (x >= end) return false;
        if (++h == a.p.c.kv_heads) {
            h = 0;
            do unit = a.units[++u];
            while (unit.tiles == 0);
        }
        place(a);
        return true;
    }
};

// Queries of a unit, keys of a tile (log2) and what a unit costs beside its tiles, in
// tiles: of the chunked kernel (measured: 25 to 28 thousand cycles to a tile's 5) and
// of the one for few queries (48 x 5 drafted tokens: 147 us with 4, 128 with 12, 124
// with 16 or 20).  And a tile of the former in tiles of the latter: 4500 cycles to 540.
constexpr int kChunkTokens = 64, kChunkTileShift = 7, kChunkUnitCost = 5;
constexpr int kFewTokens = 6, kFewTileShift = 5, kFewUnitCost = 20;
constexpr int kChunkTileCost = 8;

// One CTA: the call cut as `first` wants it or, where `other` is given and the
// lengths in device memory make that cheaper, as that; the kernel of the one not
// taken finds no units.
cudaError_t launch_plan_units(const PagedCall& call, const UnitShape& first, const UnitShape* other, cudaStream_t stream);
UnitShape paged_chunk_shape(const PagedCall& call, int sms, uint8_t* ws);
UnitShape paged_few_shape(const PagedCall& call, int sms, uint8_t* ws);
cudaError_t launch_paged_chunk(const PagedCall& call, const RopeSteps& rope, int code, const CUtensorMap& kmap,
                               const CUtensorMap& vmap, const UnitShape& shape, uint32_t* status, cudaStream_t stream);
cudaError_t launch_paged_few(const PagedCall& call, const RopeSteps& rope, int code, const CUtensorMap& kmap,
                             const CUtensorMap& vmap, const UnitShape& shape, uint32_t* status, cudaStream_t stream);

}  // namespace gqa
