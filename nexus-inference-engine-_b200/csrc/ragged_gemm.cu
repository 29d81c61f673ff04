// Tensor-core ragged products on tcgen05 / TMEM: y[s] = x[s] W_e^T for the
// slots of every expert, and the SwiGLU form with a gate and an up product.
//
// A persistent grid of one CTA per SM walks the plan's work tiles (ragged.h): two
// 128-row weight tiles x one row block of up to 128 slots of an expert.  The
// two tiles are neighbours of one weight (plain), or the gate's and the up
// weight's (PAIR); both multiply the same activations, so an SM reads 32 bytes of
// activations and 18 of Q4_K weights per cycle of MMA work, where one tile x
// 256 slots would read 64 and 9.  Roles, per k-step of 128 elements:
//   warp 26      producer: the packed tile-chunks (256 k) by 1-D bulk copies
//   warp 0       producer: the activations of the row block by TMA, as boxes of
//                64 k x 64 slots (128-byte swizzle, no multicast), only as many
//                as the block has slots for
//   warps 2-17   four dequant warpgroups, one per tile and k-step parity: thread
//                r decodes the 128 elements of row r, 64 at a time (the lane
//                decoders of the decode GEMV), and writes them to TMEM, the MMA's
//                A operand; a stage belongs to one warpgroup
//   warps 1, 27  one for each tile: a lane issues tcgen05.mma kind::f16 M=128,
//                K=16 with N = the block's slots rounded up to 16 (a short block
//                costs less), into the tile's 128-column fp32 accumulator
//   warps 18-25  epilogue: tcgen05.ld of the accumulators, conversion (PAIR:
//                silu(gate) * up, so the two products never reach memory), and
//                16-bit outputs through a staging buffer in shared memory: the
//                accumulators are handed back as soon as they are read, and
//                rows leave as 16-byte stores while the next tile's MMAs run
//
// What bounds it is the latency of handing stages on, not the MMAs (16 to 64
// cycles each, two issuing warps): an issuing warp needs some 600 cycles from
// one k-step to the next whatever N is, with its operands there 94 % of the time
// when a k-step had 64 elements.  So a k-step has 128, with one handshake for
// each warpgroup (1 to 4 % in one run; 32768 slots of 64 experts, Q4_K 4096x2048,
// now take 545 to 585 us under the power cap); the issuing loops run warp-wide, half the lanes
// watching the activations and half the A operand, with only the MMA and the
// commits in the elected lane.  Loops are kept short rather than unrolled over
// a chunk: four copies of the decode and of the issue were 12 % slower for few
// slots (1024 slots of 64 experts, Q4_K 4096x2048: 117 us against 104, and 93
// with the slow path of the waits out of line; 91 today, with f16 activations
// and three input sets in turn).  There the bytes are worth 48 us, and neither
// DRAM nor a pipe is full: 2.6 instructions per cycle, the ALU pipe at 55 %.  Blocks of 64 slots, which
// leave TMEM for more A stages, gained 2 to 9 % up to 12 slots per expert and
// lost from 16 on.
//
// An MMA column depends on its own slot's activations only, so what the boxes
// hold behind a block's slots (the next expert's rows, or zeros) reaches no
// stored value.  Every wait is bounded (sm100_ptx.cuh).  Numerics as the dense
// kernels: weights rounded once to f16, f16 activations, fp32 accumulation.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "lane_dq.cuh"
#include "qmm_gemm.h"
#include "ragged.h"
#include "sm100_ptx.cuh"

namespace nxq {

namespace {

constexpr int kDeqGroups = 4;
constexpr int kEpiWarps = 8, kEpiThreads = 32 * kEpiWarps;
constexpr int kWarpProducer = 0, kWarpMma = 1, kWarpDeq0 = 2, kWarpEpi0 = 2 + 4 * kDeqGroups;
constexpr int kWarpWProducer = kWarpEpi0 + kEpiWarps;
constexpr int kWarpMma1 = kWarpWProducer + 1;
constexpr int kThreads = 32 * (kWarpMma1 + 1);
constexpr int kMats = 2;  // weight tiles of a work tile
constexpr int kKS = 64;   // reduction elements of a swizzle atom
constexpr int kHalves = 2;                // swizzle atoms of a k-step
constexpr int kStepsPerChunk = CHUNK_K / (kHalves * kKS);
constexpr int kACols = 32 * kMats;        // TMEM columns of an atom's A, both tiles
constexpr int NT = 128;                   // slots of a work tile
constexpr int kBarBytes = 512;
constexpr uint32_t kTmemCols = 512;
constexpr int kColD = (int)kTmemCols - kMats * NT;  // accumulators: columns kColD + NT mat
constexpr int kStages = kColD / (kHalves * kACols);  // of the TMEM A ring: the columns left
static_assert(kStages == kStepsPerChunk, "a warpgroup's k-step of every chunk has the same stage");
constexpr int kBoxRows = 64;
constexpr int kBoxBytes = kBoxRows * kKS * 2;
constexpr int kXB = kHalves * NT * kKS * 2;     // 32 KB of activations per k-step
constexpr int kStageOut = NT * TILE_ROWS * 2;  // 32 KB: one tile's 16-bit outputs [slot][row]

// Ring depths in shared memory: three k-steps of activations if at least four
// tile-chunks fit beside them (or no more fit beside two), else two; then as many
// tile-chunks as fit, up to six.  An even number: the two tiles' chunks alternate
// in the ring, so each tile keeps its own stages.  With an odd number a stage
// would change hands, and a warpgroup that waits for a phase of its own could
// take the phase before the other tile's for it - copies land in any order.
// Every type has two or three stages per tile but Q8_0 (and NXF INT8), whose
// chunks of 34 KB leave room for one: the next copy starts when the chunk before
// is decoded (64 experts x 16 slots, 4096x2048: 132 us, 67 % of the copy rate; Q4_K
// 91 us, 53 %).
template <int TYPE>
struct Rings {
    static constexpr int WB = lane::Lane<TYPE>::kStage;
    static constexpr int kBudget = 227 * 1024 - 1024 - kBarBytes - kStageOut;
    static constexpr int chunks_beside(int x) {
        const int n = (kBudget - x * kXB) / WB / kMats * kMats;
        return n > 6 ? 6 : n;
    }
    static constexpr int kX = chunks_beside(3) >= 4 || chunks_beside(3) == chunks_beside(2) ? 3 : 2;
    static constexpr int kW = chunks_beside(kX);
    static_assert(kW >= kMats && kW % kMats == 0, "a tile-chunk stage belongs to one tile");
    static_assert((2 * kX + 2 * kW + 2 * kMats * kStages + 2 + kMats) * 8 + 8 <= kBarBytes, "barrier area too small");
    static constexpr size_t smem = 1024 + (size_t)kX * kXB + kStageOut + (size_t)kW * WB + kBarBytes;
};

struct Params {
    TiledShape s;
    int tiles;  // work tiles per row block
    void* y;
    int y_dtype;
    int vec;  // rows of y are 16-byte aligned
    const RaggedPlan* plan;
    DeviceStatus* status;
};

__device__ __forceinline__ uint32_t pack16(bool bf16, float a, float b) {
    if (bf16) {
        const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&v);
    }
    const __half2 v = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&v);
}

// silu(g) * u = (g / 4) / ((1 + exp(-g)) / 4) * u.  The fast division is within 2
// units in the last place for divisors up to 2^126, which the quarter never
// passes while exp(-g) is finite; undivided, it gave 0 for g between -88.7 and
// -87.3.  (The exact division of the other kernels spills registers here and
// takes 8 % longer: 1132 -> 1222 us for 32768 slots of 64 experts, gate and up of
// Q4_K 2048x4096.)
__device__ __forceinline__ float swiglu1(float g, float u) {
    return __fdividef(0.25f * g, fmaf(0.25f, expf(-g), 0.25f)) * u;
}

// A barrier of the epilogue warps that tells whether `ok` holds in all of them.
__device__ __forceinline__ bool epi_all(bool ok) {
    uint32_t r;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "setp.ne.u32 q, %1, 0;\n\t"
        "barrier.cta.red.and.pred p, 1, %2, q;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(r)
        : "r"((uint32_t)ok), "n"(kEpiThreads)
        : "memory");
    return r != 0;
}
__device__ __forceinline__ void epi_sync() { asm volatile("barrier.cta.sync 1, %0;" ::"n"(kEpiThreads) : "memory"); }

// Ring position: stage index and the phase parity of its current use.
struct Ring {
    int i = 0;
    uint32_t ph = 0;
    __device__ __forceinline__ void next(int n) {
        if (++i == n) {
            i = 0;
            ph ^= 1u;
        }
    }
};

// Weight tile `mat` of work tile t: the tile's index, and whether it exists (a
// weight with an odd number of tiles ends with a work tile of one; its second
// half repeats the first and is not stored).
template <bool PAIR>
__device__ __forceinline__ int weight_tile(const RaggedTile& t, int mat, int64_t tiles, bool* exists) {
    if (PAIR) {
        *exists = true;
        return t.tile;
    }
    const int i = 2 * t.tile + mat;
    *exists = i < tiles;
    return *exists ? i : 2 * t.tile;
}

template <int TYPE, bool PAIR>
__global__ void __launch_bounds__(kThreads, 1) ragged_gemm_kernel(const Params p, const __grid_constant__ CUtensorMap xmap) {
    using Rg = Rings<TYPE>;
    constexpr int WB = Rg::WB, kW = Rg::kW, kX = Rg::kX;

    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = smem_raw + ((1024 - (ptx::smem_addr(smem_raw) & 1023)) & 1023);
    uint8_t* xs = smem;
    uint8_t* stg = xs + kX * kXB;
    uint8_t* ws = stg + kStageOut;
    uint64_t* x_full = reinterpret_cast<uint64_t*>(ws + kW * WB);
    uint64_t* x_empty = x_full + kX;
    uint64_t* w_full = x_empty + kX;
    uint64_t* w_empty = w_full + kW;
    uint64_t* a_full = w_empty + kW;
    uint64_t* done = a_full + kMats * kStages;  // [mat][stage]: the MMAs that read the stage's A are
    uint64_t* d_full = done + kMats * kStages;
    uint64_t* d_empty = d_full + 1;
    uint64_t* drain = d_empty + 1;  // [mat]
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + kMats);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const ptx::WaitCtl ctl{abort_flag, p.status};
    if (threadIdx.x == 0) {
        for (int i = 0; i < kX; ++i) {
            ptx::mbar_init(&x_full[i], 1);
            ptx::mbar_init(&x_empty[i], kMats);  // both tiles' MMAs
        }
        for (int i = 0; i < kW; ++i) {
            ptx::mbar_init(&w_full[i], 1);
            ptx::mbar_init(&w_empty[i], 4 * kDeqGroups / kMats);  // the warps that decode a tile-chunk
        }
        for (int i = 0; i < kMats * kStages; ++i) {
            ptx::mbar_init(&a_full[i], 4);  // the warps that write a tile's stage
            ptx::mbar_init(&done[i], 1);
        }
        ptx::mbar_init(d_full, kMats);
        ptx::mbar_init(d_empty, kEpiWarps);
        for (int i = 0; i < kMats; ++i) ptx::mbar_init(&drain[i], 1);
        *abort_flag = 0;
        ptx::fence_mbar_init();
    }
    __syncwarp();
    if (warp == kWarpProducer) {
        ptx::tmem_alloc(tmem_slot, kTmemCols);
        ptx::tmem_relinquish();
    }
    ptx::tc_fence_before();
    __syncthreads();
    ptx::tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    overlap_begin();  // everything above overlaps the plan kernel

    // (A CTA without work tiles walks none and leaves.)
    const int64_t total = (int64_t)p.plan->blocks * p.tiles;
    const int chunks = (int)p.s.chunks;
    const int64_t G = gridDim.x;

    if (warp == kWarpWProducer) {
        RaggedWalk<true> walk;
        walk.start(p.plan, NT, p.tiles, blockIdx.x);
        if (lane == 0) {
            Ring rw;
            uint32_t issued = 0;
            bool ok = true;
            for (int64_t g = blockIdx.x; g < total && ok; g += G) {
                const RaggedTile t = walk.at(g);
                const uint8_t* src[kMats];
#pragma unroll
                for (int mat = 0; mat < kMats; ++mat) {
                    bool exists;
                    const int wt = weight_tile<PAIR>(t, mat, p.s.tiles, &exists);
                    src[mat] = (PAIR && mat ? t.up : t.w) + p.s.chunk_offset(wt, 0);
                }
                for (int c = 0; c < chunks && ok; ++c)
#pragma unroll
                    for (int mat = 0; mat < kMats; ++mat) {
                        ok = ok && ptx::mbar_wait(&w_empty[rw.i], rw.ph ^ 1u, ctl, 41);
                        if (!ok) continue;
                        ptx::mbar_arrive_expect_tx(&w_full[rw.i], WB);
                        ptx::bulk_g2s(ws + rw.i * WB, src[mat] + (int64_t)c * WB, WB, &w_full[rw.i]);
                        rw.next(kW);
                        ++issued;
                    }
            }
            // Do not leave with copies in flight (bounded, ignoring the abort flag).
            for (uint32_t k = issued >= kW ? issued - kW : 0; k < issued; ++k) {
                const long long t0 = clock64();
                while (!ptx::mbar_try_wait(&w_full[k % kW], (k / kW) & 1) && clock64() - t0 < ptx::kWaitCycles) {
                }
            }
        }
    } else if (warp == kWarpProducer) {
        if (lane == 0) ptx::prefetch_tmap(&xmap);
        // The activations were written through the generic proxy; TMA reads them
        // through the async one.
        asm volatile("fence.proxy.async;" ::: "memory");
        Ring rx;
        uint32_t issued = 0;
        bool ok = true;
        RaggedWalk<true> walk;
        walk.start(p.plan, NT, p.tiles, blockIdx.x);
        for (int64_t g = blockIdx.x; g < total && ok; g += G) {
            const RaggedTile t = walk.at(g);
            const int boxes = (t.rows + kBoxRows - 1) / kBoxRows;
            for (int ks = 0; ks < chunks * kStepsPerChunk && ok; ++ks) {
                ok = ptx::warp_mbar_wait(&x_empty[rx.i], rx.ph ^ 1u, ctl, 42);
                if (!ok) break;
                if (lane == 0) ptx::mbar_arrive_expect_tx(&x_full[rx.i], kHalves * boxes * kBoxBytes);
                __syncwarp();
                const int half = lane & 1, box = lane >> 1;
                if (box < boxes)
                    ptx::tma_load_2d(xs + rx.i * kXB + half * (kXB / kHalves) + box * kBoxBytes, &xmap,
                                     (kHalves * ks + half) * kKS, t.row0 + box * kBoxRows, &x_full[rx.i]);
                rx.next(kX);
                ++issued;
            }
        }
        // Do not leave with copies in flight (bounded, ignoring the abort flag).
        for (uint32_t k = issued >= kX ? issued - kX : 0; k < issued; ++k) {
            const long long t0 = clock64();
            while (!ptx::mbar_try_wait(&x_full[k % kX], (k / kX) & 1) && clock64() - t0 < ptx::kWaitCycles) {
            }
        }
    } else if (warp == kWarpMma || warp == kWarpMma1) {
        const int mat = warp == kWarpMma ? 0 : 1;
        uint32_t nt = 0;  // work tiles so far
        bool ok = true;
        Ring rx, ra;
        RaggedWalk<true> walk;
        walk.start(p.plan, NT, p.tiles, blockIdx.x);
        const uint64_t desc0 = ptx::desc_sw128_kmajor(ptx::smem_addr(xs));
        const uint32_t d = tmem + kColD + mat * NT, a = tmem + mat * 32;
        uint64_t* const af = a_full + mat * kStages;
        uint64_t* const dn = done + mat * kStages;
        bool ready = false;
        for (int64_t g = blockIdx.x; g < total && ok; g += G, ++nt) {
            const RaggedTile t = walk.at(g);
            const uint32_t idesc = ptx::idesc_f16_f32(128, (t.rows + 15) & ~15);
            ok = nt == 0 || ptx::warp_mbar_wait(d_empty, (nt - 1) & 1, ctl, 43);
            ptx::tc_fence_after();
            const int steps = chunks * kStepsPerChunk;
            for (int ks = 0; ks < steps && ok; ++ks) {
                if (!__all_sync(0xFFFFFFFFu, ready)) {
                    ok = ptx::warp_mbar_wait(lane < 16 ? &x_full[rx.i] : &af[ra.i], lane < 16 ? rx.ph : ra.ph, ctl, 44);
                    if (!ok) break;
                }
                const int i = ra.i, ix = rx.i;
                rx.next(kX);
                ra.next(kStages);
                // The next k-step's barriers, read while this one's MMAs issue.
                ready = ptx::mbar_test_wait(lane < 16 ? &x_full[rx.i] : &af[ra.i], lane < 16 ? rx.ph : ra.ph);
                ptx::tc_fence_after();
                if (ptx::elect_one()) {
                    const uint32_t ai = a + i * (kHalves * kACols);
                    const uint64_t xi = desc0 + ((uint32_t)(ix * kXB) >> 4);
                    ptx::mma_ts_f16_k64(d, ai, xi, idesc, ks ? 1u : 0u);
                    ptx::mma_ts_f16_k64(d, ai + kACols, xi + ((uint32_t)(kXB / kHalves) >> 4), idesc, 1u);
                    ptx::mma_commit(&dn[i]);
                    ptx::mma_commit(&x_empty[ix]);
                    if (ks == steps - 1) ptx::mma_commit(d_full);
                }
                __syncwarp();
            }
        }
        if (ptx::elect_one()) ptx::mma_commit(&drain[mat]);
        __syncwarp();
        const long long t0 = clock64();
        while (!ptx::mbar_try_wait(&drain[mat], 0) && clock64() - t0 < ptx::kWaitCycles) {
        }
    } else if (warp < kWarpEpi0) {
        // Warpgroup wg decodes k-step wg % 2 of every chunk of tile wg / 2.
        const int wg = (warp - kWarpDeq0) >> 2, quad = warp & 3, r = quad * 32 + lane;
        const int mat = wg >> 1, par = wg & 1;
        Ring rw;
        if (mat) rw.next(kW);
        bool ok = true;
        uint32_t ph = 1u;
        uint64_t* const mine_done = done + mat * kStages + par;
        uint64_t* const mine_full = a_full + mat * kStages + par;
        const uint32_t tbase = tmem + ((uint32_t)(quad * 32) << 16) + mat * 32 + kHalves * par * kACols;
        for (int64_t g = blockIdx.x; g < total && ok; g += G) {
            for (int c = 0; c < chunks && ok; ++c) {
                if (!(ok = ptx::warp_mbar_wait(&w_full[rw.i], rw.ph, ctl, 46))) break;
                const uint8_t* stage = ws + rw.i * WB;
#pragma unroll 1
                for (int h = 0; h < kHalves; ++h) {
                    uint32_t o[32];
                    {
                        lane::Lane<TYPE> L;
                        L.load(stage, r, kHalves * par + h);
#pragma unroll
                        for (int m = 0; m < 8; ++m) {
                            uint32_t q[4];
                            L.pairs(m, q);
#pragma unroll
                            for (int i = 0; i < 4; ++i) o[4 * m + i] = q[i];
                        }
                    }
                    if (h == 0) {
                        if (!(ok = ptx::warp_mbar_wait(mine_done, ph, ctl, 47))) break;
                        ptx::tc_fence_after();
                    }
                    ptx::tmem_st32(tbase + h * kACols, o);
                }
                if (!ok) break;
                ptx::tmem_wait_st();
                ptx::tc_fence_before();
                __syncwarp();
                if (lane == 0) {
                    ptx::mbar_arrive(mine_full);
                    ptx::mbar_arrive(&w_empty[rw.i]);
                }
                ph ^= 1u;
                rw.next(kW);
                rw.next(kW);
            }
        }
    } else {
        // Epilogue: warp (quad, sub) reads TMEM lanes 32 quad .. (its lane
        // quadrant) = weight row n of each tile, and half `sub` of the slots.
        const int ew = warp - kWarpEpi0, quad = warp & 3, r = quad * 32 + lane, sub = ew >> 2;
        constexpr int kHalf = NT / 2;
        const int tid = threadIdx.x - 32 * kWarpEpi0;
        const int64_t N = p.s.N;
        const bool bf = p.y_dtype == NXQ_BF16;
        uint16_t* const out16 = reinterpret_cast<uint16_t*>(stg);  // [slot][row]
        uint32_t nt = 0;
        RaggedWalk<true> walk;
        walk.start(p.plan, NT, p.tiles, blockIdx.x);
        const uint32_t td = tmem + ((uint32_t)(quad * 32) << 16) + kColD + kHalf * sub;
        // Slots kHalf sub + c .. + 15 of a tile's accumulator (PAIR: the outputs).
        auto read16 = [&](int mat, int c, float (&v)[16]) {
            uint32_t a[16];
            ptx::tmem_ld16(td + mat * NT + c, a);
            if constexpr (PAIR) {
                uint32_t u[16];
                ptx::tmem_ld16(td + NT + c, u);
                ptx::tmem_wait_ld();
#pragma unroll
                for (int j = 0; j < 16; ++j) v[j] = swiglu1(__uint_as_float(a[j]), __uint_as_float(u[j]));
            } else {
                ptx::tmem_wait_ld();
#pragma unroll
                for (int j = 0; j < 16; ++j) v[j] = __uint_as_float(a[j]);
            }
        };
        auto put16 = [&](int c, const uint32_t (&q)[8]) {
            uint16_t* d = out16 + (kHalf * sub + c) * TILE_ROWS + r;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                d[(2 * j) * TILE_ROWS] = (uint16_t)(q[j] & 0xFFFFu);
                d[(2 * j + 1) * TILE_ROWS] = (uint16_t)(q[j] >> 16);
            }
        };
        // The staged tile wt (16-bit) to y.
        auto flush = [&](const RaggedTile& t, int wt) {
            const int64_t n0 = (int64_t)wt * TILE_ROWS;
            uint16_t* const y = static_cast<uint16_t*>(p.y);
            for (int i = tid; i < t.rows * 16; i += kEpiThreads) {
                const int s = i >> 4, c = (i & 15) * 8;
                const int64_t at = ((int64_t)t.row0 + s) * N + n0 + c;
                const uint4 q = *reinterpret_cast<const uint4*>(out16 + s * TILE_ROWS + c);
                if (p.vec && n0 + c + 8 <= N) {
                    *reinterpret_cast<uint4*>(y + at) = q;
                } else {
                    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        if (n0 + c + j < N) y[at + j] = (uint16_t)(w[j >> 1] >> (16 * (j & 1)));
                }
            }
        };
        for (int64_t g = blockIdx.x; g < total; g += G, ++nt) {
            const RaggedTile t = walk.at(g);
            bool has1;
            const int wt0 = PAIR ? t.tile : 2 * t.tile, wt1 = weight_tile<PAIR>(t, 1, p.s.tiles, &has1);
            // All epilogue warps go on or give up together; nobody still reads
            // the staging buffer.
            if (!epi_all(ptx::warp_mbar_wait(d_full, nt & 1, ctl, 48))) break;
            ptx::tc_fence_after();
            const int left = t.rows - kHalf * sub;  // slots of this half
            if (p.y_dtype == NXQ_F32) {
#pragma unroll 1
                for (int mat = 0; mat < (PAIR ? 1 : 2); ++mat)
#pragma unroll 1
                    for (int c = 0; c < kHalf && c < left; c += 16) {
                        float v[16];
                        read16(mat, c, v);
                        const int64_t n = (int64_t)(mat ? wt1 : wt0) * TILE_ROWS + r;
                        float* q = static_cast<float*>(p.y) + ((int64_t)t.row0 + kHalf * sub + c) * N + n;
                        if (n < N && (mat == 0 || has1))
#pragma unroll
                            for (int j = 0; j < 16; ++j, q += N)
                                if (c + j < left) *q = v[j];
                        __syncwarp();
                    }
                ptx::tc_fence_before();
                __syncwarp();
                if (lane == 0) ptx::mbar_arrive(d_empty);
                continue;
            }
            // The first tile's (PAIR: the) outputs into the staging buffer, the
            // second tile's into registers; then the accumulators are free.
#pragma unroll 1
            for (int c = 0; c < kHalf && c < left; c += 16) {
                float v[16];
                uint32_t q[8];
                read16(0, c, v);
#pragma unroll
                for (int j = 0; j < 8; ++j) q[j] = pack16(bf, v[2 * j], v[2 * j + 1]);
                put16(c, q);
            }
            // (`hold` is what the plain kernels spill 116 to 128 bytes for, at the 72
            // registers that 896 threads leave; the SwiGLU ones spill none.)
            uint32_t hold[PAIR ? 1 : kHalf / 16][8];
            if constexpr (!PAIR) {
#pragma unroll
                for (int c = 0; c < kHalf / 16; ++c)
                    if (16 * c < left) {
                        float v[16];
                        read16(1, 16 * c, v);
#pragma unroll
                        for (int j = 0; j < 8; ++j) hold[c][j] = pack16(bf, v[2 * j], v[2 * j + 1]);
                    }
            }
            ptx::tc_fence_before();
            __syncwarp();
            if (lane == 0) ptx::mbar_arrive(d_empty);
            epi_sync();
            flush(t, wt0);
            if constexpr (!PAIR) {
                if (has1) {
                    epi_sync();
#pragma unroll
                    for (int c = 0; c < kHalf / 16; ++c)
                        if (16 * c < left) put16(16 * c, hold[c]);
                    epi_sync();
                    flush(t, wt1);
                }
            }
        }
    }

    ptx::tc_fence_before();
    __syncthreads();
    if (warp == kWarpProducer) {
        ptx::tc_fence_after();
        ptx::tmem_dealloc(tmem, kTmemCols);
    }
}

template <int TYPE>
int set_attr() {
    cudaError_t e = cudaFuncSetAttribute(ragged_gemm_kernel<TYPE, false>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         (int)Rings<TYPE>::smem);
    if (e == cudaSuccess)
        e = cudaFuncSetAttribute(ragged_gemm_kernel<TYPE, true>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                 (int)Rings<TYPE>::smem);
    return e == cudaSuccess ? NXQ_OK : cuda_fail(e, "cudaFuncSetAttribute (ragged_gemm)");
}

template <int TYPE>
int launch(const Params& p, const CUtensorMap& tmap, bool pair, unsigned grid, cudaStream_t st) {
    const cudaError_t e = launch_overlapped(pair ? ragged_gemm_kernel<TYPE, true> : ragged_gemm_kernel<TYPE, false>, grid,
                                            kThreads, Rings<TYPE>::smem, st, p, tmap);
    note_launches(1);
    return e == cudaSuccess ? NXQ_OK : cuda_fail(e, "ragged_gemm launch");
}

}  // namespace

int ragged_gemm_init() {
    int rc;
    if ((rc = set_attr<T_Q4_K>()) || (rc = set_attr<T_Q4_0>()) || (rc = set_attr<T_Q8_0>()) ||
        (rc = set_attr<T_Q3_K>()) || (rc = set_attr<T_I4G128>()) || (rc = set_attr<T_Q6_K>()) ||
        (rc = set_attr<T_Q5_K>()) || (rc = set_attr<T_Q4_1>()) || (rc = set_attr<T_Q2_K>()) ||
        (rc = set_attr<T_I4G32>()) || (rc = set_attr<T_I4G64>()) || (rc = set_attr<T_I4G256>()))
        return rc;
    return NXQ_OK;
}

// Where the dense prefill GEMM runs (NXQ_PREFILL_KERNEL=simt turns both off).
bool ragged_gemm_supported(const TiledShape& s) { return gemm_supported(s, 33); }

int ragged_gemm_blk() { return NT; }

int ragged_gemm(const RaggedCall& c, const void* xh, int64_t X, const RaggedPlan* plan) {
    const TiledShape& s = c.w->shape;
    Params p{s, (int)(c.up ? s.tiles : (s.tiles + 1) / 2), c.y, c.y_dtype,
             s.N % 8 == 0 && (uintptr_t)c.y % 16 == 0, plan, context_status()};
    CUtensorMap tmap;
    if (int rc = gemm_activation_map(&tmap, xh, X, s.K, kBoxRows)) return rc;
    const int64_t work = ragged_max_blocks(c.w->count, c.R, NT) * p.tiles;
    const unsigned grid = (unsigned)(work < context_sm_count() ? work : context_sm_count());
    switch (s.type) {
        case T_Q4_K: return launch<T_Q4_K>(p, tmap, c.up != nullptr, grid, c.st);
        case T_Q4_0: return launch<T_Q4_0>(p, tmap, c.up != nullptr, grid, c.st);
        case T_Q8_0:
        case T_NXF_I8: return launch<T_Q8_0>(p, tmap, c.up != nullptr, grid, c.st);
        case T_Q3_K: return launch<T_Q3_K>(p, tmap, c.up != nullptr, grid, c.st);
        case T_I4G128: return launch<T_I4G128>(p, tmap, c.up != nullptr, grid, c.st);
        case T_Q6_K: return launch<T_Q6_K>(p, tmap, c.up != nullptr, grid, c.st);
        case T_Q5_K: return launch<T_Q5_K>(p, tmap, c.up != nullptr, grid, c.st);
        case T_Q4_1: return launch<T_Q4_1>(p, tmap, c.up != nullptr, grid, c.st);
        case T_Q2_K: return launch<T_Q2_K>(p, tmap, c.up != nullptr, grid, c.st);
        case T_I4G32: return launch<T_I4G32>(p, tmap, c.up != nullptr, grid, c.st);
        case T_I4G64: return launch<T_I4G64>(p, tmap, c.up != nullptr, grid, c.st);
        case T_I4G256: return launch<T_I4G256>(p, tmap, c.up != nullptr, grid, c.st);
        default: return NXQ_ERR_UNSUPPORTED;
    }
}

}  // namespace nxq
