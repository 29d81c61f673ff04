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
    int e;              // expert
    int row0;           // first slot
    int rows;           // slots (> 0)
    int blk0;           // row blocks of the entries before
    const uint8_t* w;   // the expert's tiled weight
    const uint8_t* up;  // its up weight (SwiGLU)
};
struct RaggedPlan {
    int entries;
    int blocks;  // row blocks of all entries
    int pad[6];
    RaggedEntry it[1];
};
// At least 32 entries, so that a warp may load the first 32 whatever their number.
inline size_t plan_bytes(int64_t max_entries) {
    return 32 + (size_t)(max_entries < 32 ? 32 : max_entries) * sizeof(RaggedEntry);
}

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

// Row blocks of `blk` slots for n >= 0 slots, any int (n + blk - 1 may pass 2^31).
__host__ __device__ inline int row_blocks(int n, int blk) { return n / blk + (n % blk != 0); }

// One work tile: weight tile `tile` of the expert's weights, slots [row0, row0 +
// rows).
struct RaggedTile {
    const uint8_t *w, *up;
    int tile, row0, rows;
};

// Walks a plan's work tiles in ascending order (experts of `tiles` weight tiles,
// row blocks of at most `blk` slots).  EVEN: an expert's slots are cut into row
// blocks of nearly equal size, a multiple of 16, instead of full ones and a rest
// (with more than 8 blocks the rest is small beside them, and the rounding
// could leave the last block empty).
template <bool EVEN>
struct RaggedWalk {
    const RaggedPlan* plan;
    int blk, tiles, entries, i;
    int64_t first, end;  // work tiles of entry i
    RaggedEntry cur;
    int nb;
    __device__ __forceinline__ void load(int j) {
        i = j;
        const int4* q = reinterpret_cast<const int4*>(&plan->it[j]);
        const int4 v = q[0];
        const longlong2 a = *reinterpret_cast<const longlong2*>(q + 1);
        cur = RaggedEntry{v.x, v.y, v.z, v.w, reinterpret_cast<const uint8_t*>(a.x), reinterpret_cast<const uint8_t*>(a.y)};
        nb = row_blocks(cur.rows, blk);
        first = (int64_t)cur.blk0 * tiles;
        end = first + (int64_t)nb * tiles;
    }
    // Starts at work tile g (one that exists).  By a converged warp, which looks
    // at 32 entries at a time: one round trip to memory for most calls.
    __device__ __forceinline__ void start(const RaggedPlan* p, int blk_, int tiles_, int64_t g) {
        plan = p;
        blk = blk_;
        tiles = tiles_;
        entries = p->entries;
        const int lane = threadIdx.x & 31;
        int lo = 0;
        for (int j0 = 0;; j0 += 32) {  // the last entry whose first work tile is <= g
            const bool in = j0 + lane < entries && (int64_t)p->it[j0 + lane].blk0 * tiles <= g;
            const unsigned m = __ballot_sync(0xFFFFFFFFu, in);
            if (m) lo = j0 + 31 - __clz(m);
            if (m != 0xFFFFFFFFu) break;
        }
        load(lo);
    }
    // Work tile g, not before the last one asked for.
    __device__ __forceinline__ RaggedTile at(int64_t g) {
        while (g >= end && i + 1 < entries) load(i + 1);
        const int local = (int)(g - first);
        RaggedTile t;
        t.w = cur.w;
        t.up = cur.up;
        t.tile = local / nb;
        const int b = local - t.tile * nb;
        int rb = blk;
        if (EVEN && nb <= 8) rb = ((cur.rows + nb - 1) / nb + 15) & ~15;
        t.row0 = cur.row0 + b * rb;
        t.rows = cur.rows - b * rb < rb ? cur.rows - b * rb : rb;
        return t;
    }
};

// Row blocks a plan can have at most.
inline int64_t ragged_max_blocks(int64_t E, int64_t R, int blk) { return (E < R ? E : R) + R / blk; }

// tcgen05 kernel (ragged_gemm.cu): xh [X][K] f16, 16-byte aligned, slot s reads
// row s.  `plan` is made for row blocks of ragged_gemm_blk() slots.
int ragged_gemm_init();
bool ragged_gemm_supported(const TiledShape& s);
int ragged_gemm_blk();
int ragged_gemm(const RaggedCall& c, const void* xh, int64_t X, const RaggedPlan* plan);

// Warp-level kernel for few slots per expert (ragged_mma.cu): xh [X][K] f16,
// 16-byte aligned; slot s reads row rows[s] (rows null: s).  `blk` is the slots
// of a row block (0 from ragged_mma_blk declines); `part` has
// ragged_mma_partials() bytes, `cnt` ragged_mma_workers() counters, zeroed on
// the stream.
int ragged_mma_init();
int ragged_mma_blk(const RaggedCall& c);
int ragged_mma_workers();
size_t ragged_mma_partials();
int ragged_mma(const RaggedCall& c, const __half* xh, int64_t X, const int32_t* rows, const RaggedPlan* plan, float* part,
               unsigned* cnt);

}  // namespace nxq
