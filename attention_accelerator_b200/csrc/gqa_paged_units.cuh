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

// Layout behind the counters that the decode keeps; everything here is written by each call.
struct UnitRegions {
    size_t starts, cuts, units, arrivals, partials, end;
};
inline UnitRegions unit_regions(int batch, int rows, int tokens, size_t counters_a_unit, int sms, size_t partials) {
    auto up = [](size_t x) { return (x + 255) & ~(size_t)255; };
    const size_t units = (size_t)rows / tokens + batch;
    UnitRegions r;
    r.starts = kPagedPartialsOffset + 256;  // (Meta first)
    r.cuts = r.starts + up((size_t)sms * sizeof(int32_t));
    r.units = r.cuts + up((size_t)(sms + 1) * sizeof(int64_t));
    r.arrivals = r.units + up(units * sizeof(Unit));
    r.partials = r.arrivals + up(units * counters_a_unit * sizeof(uint32_t));
    r.end = r.partials + partials;
    return r;
}
inline UnitPlan unit_plan(const UnitRegions& r, uint8_t* ws) {
    return UnitPlan{reinterpret_cast<Meta*>(ws + kPagedPartialsOffset), reinterpret_cast<Unit*>(ws + r.units),
                    reinterpret_cast<int32_t*>(ws + r.starts), reinterpret_cast<int64_t*>(ws + r.cuts),
                    reinterpret_cast<uint32_t*>(ws + r.arrivals)};
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

// One CTA: units of `tokens` queries, their keys in tiles of 2^tile_shift, shares
// of even cost (a unit costs unit_cost tiles beside its own), `counters` zeroed (0:
// two a unit and head).
cudaError_t launch_plan_units(const PagedCall& call, const UnitPlan& to, int tokens, int tile_shift, int unit_cost,
                              int counters, int ctas, cudaStream_t stream);

}  // namespace gqa
