// Products grouped by expert with ragged sizes (nxq_qmatmul_ragged): the table
// of experts, and the plan every kernel of such a call walks.
#pragma once
#include <vector>

#include "nxq_internal.h"

namespace nxq {

constexpr int kMaxExperts = 1024;

// Experts of one projection (the nxq_experts_t handle).
struct ExpertTable {
    int count;
    TiledShape shape;                // of every expert
    std::vector<nxq_weight_t> refs;  // referenced weights
    const uint8_t** dev = nullptr;   // device array: tiled copy of each expert
};

// The plan of a call, written on the device by one CTA from the offsets: the
// experts that have rows, in order, and a running count of their row blocks
// of `blk` rows.  Work tiles (128 weight rows x one row block) are numbered
// expert by expert, inside an expert by weight tile and then by row block, so
// consecutive work tiles read the same weight tile.
struct RaggedEntry {
    int e;     // expert
    int row0;  // first slot
    int rows;  // slots (> 0)
    int blk0;  // row blocks of the entries before
};
struct RaggedPlan {
    int entries;
    int blocks;  // row blocks of all entries
    int pad[2];
    RaggedEntry it[1];
};
inline size_t plan_bytes(int64_t max_entries) { return 16 + (size_t)max_entries * sizeof(RaggedEntry); }

struct RaggedCall {
    const ExpertTable* w;   // (gate) experts
    const ExpertTable* up;  // SwiGLU pairing, or null
    const void* x;
    int x_dtype;
    int64_t X;
    const int32_t* rows;  // or null
    void* y;
    int y_dtype;
    int64_t R;
    const int32_t* offsets;
    cudaStream_t st;
};

// One work tile: weight tile `tile` of entry `i`, rows [row0, row0 + rows).
struct RaggedTile {
    int e, tile, row0, rows;
};
// Work tile g of a plan whose experts have `tiles` weight tiles each.
__device__ __forceinline__ RaggedTile ragged_tile(const RaggedPlan* plan, int blk, int tiles, int64_t g) {
    // The last entry whose first work tile is <= g.
    int lo = 0, hi = plan->entries - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if ((int64_t)plan->it[mid].blk0 * tiles <= g)
            lo = mid;
        else
            hi = mid - 1;
    }
    const RaggedEntry it = plan->it[lo];
    const int nb = (it.rows + blk - 1) / blk;
    const int local = (int)(g - (int64_t)it.blk0 * tiles);
    RaggedTile t;
    t.e = it.e;
    t.tile = local / nb;
    const int b = local - t.tile * nb;
    t.row0 = it.row0 + b * blk;
    t.rows = it.rows - b * blk < blk ? it.rows - b * blk : blk;
    return t;
}

}  // namespace nxq
