// Warp-level tensor-core ragged products for few slots per expert (decode): y[s] =
// x[rows[s]] W_e^T, and the SwiGLU form.
//
// The work is the packed weights of the experts that have slots, streamed once:
// the kernel is bound by HBM and by the instructions that unpack the codes.
// Units are those of the decode GEMV (qmm_mma.cu): one tile-chunk (128 rows x 256
// k, one bulk copy) staged in shared memory, consumed by 8 warps with the
// dequantized weights as the 16-row A operand of mma.sync.m16n8k16 and the
// slots as its 8 columns (lane_dq.cuh).  What differs is where the units come
// from: the experts' sizes are known on the device only, so every worker derives
// its run from the plan (ragged.h).
//
// A worker is a group of 8 consumer warps with a producer warp and a ring of its
// own, two to a CTA and one CTA to an SM.  The U = row blocks x weight tiles x
// chunks units of the whole call are cut into equal runs of consecutive units,
// one per worker, whatever the experts' sizes (a decode step of one sequence
// has 50 to 400 tiles: whole tiles per SM would leave up to half of them idle).
// Inside a run nothing synchronizes the 8 warps: each stores its rows of a
// finished tile and goes on as far as the ring reaches.  (Two groups taking a
// tile's units in turn, as in the decode GEMV, met at a barrier at every tile's
// end: 0.9 us of 8 chunks' 5 us.)  A tile shared by workers b0 .. b1 is finished
// by b0, which holds its first units and reaches it at the end of its run: b0 + 1
// .. b1, which reach it at the start of theirs, store their fp32 partials in the
// call's workspace and count themselves in on b0's counter; b0 waits (bounded)
// and adds the partials in worker order, so the sum does not depend on timing.
// A worker publishes before any wait of its own and waits for later workers only,
// so the waits end in whatever order the CTAs get their SMs.  The bound (2 s by
// default) does count the time in which a later CTA has no SM: beside a kernel of
// another stream that holds SMs for longer, the call ends with NXQ_ERR_TIMEOUT.
//
// Row blocks have up to 8 slots, the columns of one MMA.  Slots behind a block's
// end hold stale activations of the stage's earlier units: an MMA column
// depends on its own slot only, and those columns are not stored.  (Variants
// with blocks of 16 and 32, 2 to 4 MMAs for every decoded fragment, were slower
// up to 8 slots per expert, and the tcgen05 kernel takes over from 6: their rings
// are shallower and every warp reads all activation fragments.)
//
// What bounds it (64 experts of Q4_K 4096x2048, 256 slots, 290 MB in 82 us = 3.5
// TB/s): the instructions of the decode, 387 a warp and unit, issue slots 64 %
// busy, integer pipe 52 %, DRAM 42 %.  A third worker per SM (72 registers)
// changed nothing.
//
// Numerics as the decode GEMV: weights rounded once to f16, f16 activations,
// exact products, fp32 accumulation.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "lane_dq.cuh"
#include "qmm_mma.h"
#include "ragged.h"
#include "sm100_ptx.cuh"

namespace nxq {

namespace {

constexpr int kWarps = 8;                  // of a consumer group
constexpr int kThreads = kWarps * 32;
constexpr int kGroups = 2;                 // workers of a CTA
constexpr int kConsumers = kGroups * kThreads;
constexpr int kMT = 8;                     // slots of a row block: one n8 tile

using lane::Lane;
using lane::mma16816;

template <int TYPE, bool PAIR>
struct Cfg {
    static constexpr int WB = Lane<TYPE>::kStage;
    static constexpr int XB = 8 * 32 * 16;         // pieces (m, lane) of 16 B
    static constexpr int PB = kMT * TILE_ROWS * 4;  // one tile's fp32 partial, [row][slot]
    static constexpr int SETS = PAIR ? 2 : 1;
    static constexpr int S0 = (227 * 1024 - 2048) / (kGroups * (WB + XB));
    static constexpr int S = S0 > 8 ? 8 : S0;  // stages of a worker's ring
    static constexpr int kAll = kConsumers + 32 * kGroups;
    // As in the decode GEMV: two accumulator chains for Q4_K.
    static constexpr int kAccSets = TYPE == T_Q4_K ? 2 : 1;
    static constexpr size_t smem = (size_t)kGroups * S * (WB + XB);
    static_assert(S >= 2, "pipeline too shallow");
};

struct Params {
    const __half* x;
    int64_t X;
    const int32_t* rows;  // or null: slot s reads row s
    void* y;
    int y_dtype;
    int64_t N, K;
    int chunks, tiles;
    const RaggedPlan* plan;
    float* part;    // a partial-sum slot per worker
    unsigned* cnt;  // a counter per worker, zeroed with the plan
    DeviceStatus* status;
};

__device__ __forceinline__ void store_y(void* y, int dt, int64_t i, float v) {
    if (dt == NXQ_F32)
        reinterpret_cast<float*>(y)[i] = v;
    else if (dt == NXQ_F16)
        reinterpret_cast<__half*>(y)[i] = __float2half_rn(v);
    else
        reinterpret_cast<__nv_bfloat16*>(y)[i] = __float2bfloat16_rn(v);
}
// x piece (16 B) by cp.async; src_bytes = 0 fills the piece with zeros.
__device__ __forceinline__ void cp_async16_zfill(void* dst, const void* src, uint32_t src_bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(ptx::smem_addr(dst)), "l"(src), "r"(src_bytes)
                 : "memory");
}
// Arrives (once, counted in the barrier's expected count) on `bar` when all
// cp.async this thread issued so far have landed.
__device__ __forceinline__ void cp_async_arrive(uint64_t* bar) {
    asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(ptx::smem_addr(bar)) : "memory");
}
__device__ __forceinline__ void named_sync(int id, int threads) {
    asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory");
}

template <int TYPE, bool PAIR>
__global__ void __launch_bounds__(Cfg<TYPE, PAIR>::kAll, 1) ragged_mma_kernel(const Params p) {
    using Cf = Cfg<TYPE, PAIR>;
    constexpr int S = Cf::S, WB = Cf::WB, XB = Cf::XB, PB = Cf::PB;
    constexpr int RS = kMT;  // floats per row in a partial
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ uint64_t full_s[kGroups][S];   // unit landed: tile-chunk bytes + one arrival per producer lane + 1
    __shared__ uint64_t empty_s[kGroups][S];  // the worker's 8 warps are done with the stage
    __shared__ int s_abort;
    __shared__ int s_last[kGroups];  // the counts of the tile a worker finishes are in

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const bool producer = warp >= kGroups * kWarps;
    const int gi = producer ? warp - kGroups * kWarps : warp >> 3;  // the CTA's worker
    uint64_t* const full = full_s[gi];
    uint64_t* const empty = empty_s[gi];
    uint8_t* const wst = smem + (size_t)gi * S * (WB + XB);  // S x WB
    uint8_t* const xst = wst + (size_t)S * WB;               // S x XB
    if (producer && lane == 0) {
        for (int st = 0; st < S; ++st) {
            ptx::mbar_init(&full[st], 1 + 32);
            ptx::mbar_init(&empty[st], kWarps);
        }
        s_abort = 0;
        ptx::fence_mbar_init();
    }
    __syncthreads();
    const ptx::WaitCtl ctl{&s_abort, p.status};
    overlap_begin();  // everything above overlaps the plan kernel

    const int Kc = p.chunks, kun = PAIR ? 2 * Kc : Kc;  // units per tile
    const int U = p.plan->blocks * p.tiles * kun;       // checked on the host to fit
    const int G = kGroups * (int)gridDim.x < U ? kGroups * (int)gridDim.x : U;  // workers with units
    const int q = kGroups * blockIdx.x + gi;
    if (kGroups * (int)blockIdx.x >= G) return;  // the whole CTA
    const int ub = U / G, ur = U % G;
    const int g0 = q < G ? q * ub + (q < ur ? q : ur) : U, g1 = q < G ? g0 + ub + (q < ur ? 1 : 0) : U;
    const int n = g1 - g0;

    int w_issued = 0;  // producer lane 0: tile-chunk copies issued
    if (n == 0) {
        // The other worker has the CTA's last units.
    } else if (producer) {
        // ---- producer: lane 0 issues the tile-chunk bulk copies; all lanes copy
        // the x pieces of the block's slots: piece (slot, t4, m) holds the 8
        // elements x[row][k0 + 64 t4 + 8m ..] at index 32 m + 4 slot + t4.  Every
        // lane arrives once per unit on the unit's full barrier, after the stage's
        // previous unit was released.
        const int t4 = (lane >> 3) & 3, m = lane & 7;
        RaggedWalk<false> walk;
        walk.start(p.plan, kMT, p.tiles, g0 / kun);
        const uint8_t *wg = nullptr, *wu = nullptr;
        int row0 = -1, slots = 0;
        int64_t src_row = 0;  // lane l: the source row of slot l (-1: zeros)
        for (int u = 0, t = g0 / kun, c = g0 % kun; u < n; ++u) {
            if (u == 0 || c == 0) {
                const RaggedTile tl = walk.at(t);
                wg = tl.w + (int64_t)tl.tile * Kc * WB;
                if constexpr (PAIR) wu = tl.up + (int64_t)tl.tile * Kc * WB;
                if (tl.row0 != row0) {
                    row0 = tl.row0;
                    slots = tl.rows;
                    src_row = -1;
                    if (lane < slots) {
                        const int s = row0 + lane;
                        src_row = p.rows ? p.rows[s] : s;
                        if (src_row < 0 || src_row >= p.X) {
                            raise_index(p.status, kIndexRow);
                            src_row = -1;
                        }
                    }
                }
            }
            const int stg = u % S;
            if (u >= S && !ptx::warp_mbar_wait(&empty[stg], (uint32_t)(u / S - 1) & 1u, ctl, 51)) break;
            // The activations first: behind a ring full of weight copies they
            // would be what the first units wait for.
            const int cx = PAIR && c >= Kc ? c - Kc : c;
            const int64_t k = (int64_t)cx * CHUNK_K + 64 * t4 + 8 * m;
            uint4* xd = reinterpret_cast<uint4*>(xst + stg * XB) + m * 32 + t4;
#pragma unroll
            for (int j = 0; j < kMT; ++j) {
                const int64_t row = __shfl_sync(0xFFFFFFFFu, src_row, j);
                if (j < slots) {
                    const bool in = row >= 0 && k < p.K;
                    cp_async16_zfill(xd + 4 * j, p.x + (in ? row * p.K + k : 0), in ? 16u : 0u);
                }
            }
            cp_async_arrive(&full[stg]);
            if (lane == 0) {
                ptx::mbar_arrive_expect_tx(&full[stg], WB);
                ptx::bulk_g2s(wst + stg * WB, (PAIR && c >= Kc ? wu : wg) + (int64_t)cx * WB, WB, &full[stg]);
                ++w_issued;
            }
            if (++c == kun) {
                c = 0;
                ++t;
            }
        }
    } else {
        // ---- consumers: the units [cs, ce) that this worker holds of tile t ----
        const int wg = warp & 7, g = lane >> 2, tq = lane & 3;
        const int r0 = 16 * wg + g;  // the fragment rows r0, r0 + 8 of a tile
        bool dead = false;
        RaggedWalk<false> walk;
        walk.start(p.plan, kMT, p.tiles, g0 / kun);
        auto worker_of = [&](int gu) {
            const int big = ur * (ub + 1);
            return gu < big ? gu / (ub + 1) : ur + (gu - big) / ub;
        };
        auto part_of = [&](int b) { return p.part + (size_t)b * (Cf::SETS * PB / 4); };
        for (int t = g0 / kun; t * kun < g1; ++t) {
            const RaggedTile tl = walk.at(t);
            const int cs = g0 > t * kun ? g0 - t * kun : 0;
            const int ce = g1 < (t + 1) * kun ? g1 - t * kun : kun;
            // acc[c0..c3]: c0/c1 = row 16wg+g, slots 2t, 2t+1; c2/c3 = row 16wg+8+g.
            // PAIR: accu/accu2 hold the up projection's sums.
            float acc[4], acc2[4], accu[4], accu2[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[e] = acc2[e] = accu[e] = accu2[e] = 0.0f;
            // Unit c of this tile into the sums A (A2: the second chain).
            auto unit = [&](int c, float(&A)[4], float(&A2)[4]) {
                const int u = t * kun + c - g0, stg = u % S;
                if (!dead && !ptx::warp_mbar_wait(&full[stg], (uint32_t)(u / S) & 1u, ctl, 52)) dead = true;
                if (!dead) {
                    Lane<TYPE> LA, LB;
                    LA.load(wst + stg * WB, 16 * wg + g, tq);
                    LB.load(wst + stg * WB, 16 * wg + 8 + g, tq);
                    const uint4* xs = reinterpret_cast<const uint4*>(xst + stg * XB) + lane;
#pragma unroll
                    for (int m = 0; m < 8; ++m) {
                        uint32_t pa[4], pb[4];
                        LA.pairs(m, pa);
                        LB.pairs(m, pb);
                        const uint4 xv = xs[m * 32];
                        mma16816(A, pa[0], pb[0], pa[1], pb[1], xv.x, xv.y);
                        if constexpr (Cf::kAccSets == 2)
                            mma16816(A2, pa[2], pb[2], pa[3], pb[3], xv.z, xv.w);
                        else
                            mma16816(A, pa[2], pb[2], pa[3], pb[3], xv.z, xv.w);
                    }
                }
                __syncwarp();
                if (lane == 0) ptx::mbar_arrive(&empty[stg]);
            };
            int c = cs;
            for (; c < (ce < Kc ? ce : Kc); ++c) unit(c, acc, acc2);
            if constexpr (PAIR)
                for (; c < ce; ++c) unit(c, accu, accu2);
            if constexpr (Cf::kAccSets == 2) {
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[e] += acc2[e], accu[e] += accu2[e];
            }
            auto put = [&](float* cb, const float(&A)[4]) {
                *reinterpret_cast<float2*>(cb + r0 * RS + 2 * tq) = make_float2(A[0], A[1]);
                *reinterpret_cast<float2*>(cb + (r0 + 8) * RS + 2 * tq) = make_float2(A[2], A[3]);
            };
            auto add = [&](const float* cb, float(&A)[4]) {
                const float2 a = __ldcg(reinterpret_cast<const float2*>(cb + r0 * RS + 2 * tq));
                const float2 b = __ldcg(reinterpret_cast<const float2*>(cb + (r0 + 8) * RS + 2 * tq));
                A[0] += a.x;
                A[1] += a.y;
                A[2] += b.x;
                A[3] += b.y;
            };
            bool store = true;
            if (cs != 0 || ce != kun) {
                const int b0 = worker_of(t * kun), b1 = worker_of(t * kun + kun - 1);
                unsigned* cn = p.cnt + b0;
                if (q != b0) {
                    store = false;
                    float* mine = part_of(q);
                    put(mine, acc);
                    if constexpr (PAIR) put(mine + PB / 4, accu);
                    named_sync(1 + gi, kThreads);
                    if (wg == 0 && lane == 0) {
                        __threadfence();  // the group's partial (ordered by the barrier) before the count
                        const unsigned hooks = *reinterpret_cast<const volatile unsigned*>(&p.status->hooks);
                        if (!(hooks & kHookStreamKSkipCount)) atomicAdd(cn, 1u);
                    }
                } else {
                    if (wg == 0 && lane == 0) {
                        const unsigned need = (unsigned)(b1 - b0);
                        const long long w0 = clock64(), lim = ptx::wait_limit(p.status);
                        int ok = 1;
                        for (;;) {
                            unsigned v;
                            asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(v) : "l"(cn) : "memory");
                            if (v >= need) break;
                            if (*ctl.abort || clock64() - w0 > lim) {
                                if (!*ctl.abort) ptx::raise_timeout(ctl, 53);
                                ok = 0;
                                break;
                            }
                            __nanosleep(64);
                        }
                        s_last[gi] = ok;
                    }
                    named_sync(1 + gi, kThreads);
                    store = s_last[gi];
                    if (store)
                        for (int b = b0 + 1; b <= b1; ++b) {
                            const float* pb = part_of(b);
                            add(pb, acc);
                            if constexpr (PAIR) add(pb + PB / 4, accu);
                        }
                }
            }
            if (!store) continue;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int tok = 2 * tq + (e & 1);
                const int64_t row = (int64_t)tl.tile * TILE_ROWS + r0 + 8 * (e >> 1);
                if (tok < tl.rows && row < p.N) {
                    float v = acc[e];
                    if constexpr (PAIR) v = v / (1.0f + expf(-v)) * accu[e];
                    store_y(p.y, p.y_dtype, ((int64_t)tl.row0 + tok) * p.N + row, v);
                }
            }
        }
    }

    __syncthreads();
    if (s_abort) {
        // Let the copies still in flight land (bounded) before the CTA's shared
        // memory goes away: only the last S tile-chunks issued can be pending.
        asm volatile("cp.async.wait_all;" ::: "memory");
        if (producer && lane == 0) {
            for (int u = w_issued > S ? w_issued - S : 0; u < w_issued; ++u) {
                const long long t0 = clock64();
                while (!ptx::mbar_try_wait(&full[u % S], (uint32_t)(u / S) & 1u) && clock64() - t0 < ptx::kWaitCycles) {
                }
            }
        }
    }
}

template <int TYPE, bool PAIR>
int set_attr() {
    cudaError_t e = cudaFuncSetAttribute(ragged_mma_kernel<TYPE, PAIR>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         (int)Cfg<TYPE, PAIR>::smem);
    return e == cudaSuccess ? NXQ_OK : cuda_fail(e, "cudaFuncSetAttribute (ragged_mma)");
}

template <int TYPE, bool PAIR>
int launch(const Params& p, unsigned grid, cudaStream_t st) {
    const cudaError_t e = launch_overlapped(ragged_mma_kernel<TYPE, PAIR>, grid, Cfg<TYPE, PAIR>::kAll, Cfg<TYPE, PAIR>::smem, st, p);
    note_launches(1);
    return e == cudaSuccess ? NXQ_OK : cuda_fail(e, "ragged_mma launch");
}

template <int TYPE>
int launch_type(const Params& p, bool pair, unsigned grid, cudaStream_t st) {
    return pair ? launch<TYPE, true>(p, grid, st) : launch<TYPE, false>(p, grid, st);
}

}  // namespace

int ragged_mma_init() {
    int rc;
#define NXQ_ATTR(T) \
    if ((rc = set_attr<T, false>()) || (rc = set_attr<T, true>())) return rc;
    NXQ_ATTR(T_Q4_K)
    NXQ_ATTR(T_Q4_0)
    NXQ_ATTR(T_Q8_0)
    NXQ_ATTR(T_Q3_K)
    NXQ_ATTR(T_I4G128)
    NXQ_ATTR(T_Q6_K)
    NXQ_ATTR(T_Q5_K)
    NXQ_ATTR(T_Q4_1)
    NXQ_ATTR(T_Q2_K)
    NXQ_ATTR(T_I4G32)
    NXQ_ATTR(T_I4G64)
    NXQ_ATTR(T_I4G256)
#undef NXQ_ATTR
    return NXQ_OK;
}

// Slots of a row block, or 0 to decline: more than 6 slots per expert that can
// have any, on average.  Measured (64 experts, routed with a bias, Q4_K
// 4096x2048, 2 / 4 / 6 / 8 slots on average): 67 / 80 / 94 / 112 us here, 91 to 94 us
// with the tcgen05 kernel; Q4_0 14336x4096 gate and up, 8 experts, 4 / 8 slots:
// 120 / 175 against 155 to 161; Q3_K, 4 / 8 slots: 53 / 66 against 62.  Other types
// at 4096x2048, 64 experts, 2 / 4 / 6 / 8 slots, here and there: Q8_0 86 / 112 / 132 /
// 157 and 101 / 123 / 130 / 130; Q6_K 72 / 90 / 102 / 123 and 90 / 104 / 105 / 106; Q5_K
// 77 / 95 / 116 / 134 and 83 / 101 / 102 / 102.  One limit for all costs 14 % at worst
// (Q5_K at 6 slots).
int ragged_mma_blk(const RaggedCall& c) {
    const TiledShape& s = c.w->shape;
    if (!mma_supported(s, 1)) return 0;
    const int64_t E = c.w->count < c.R ? c.w->count : c.R;
    if (c.R > 6 * E) return 0;
    // The kernel numbers units in 32 bits.
    const int64_t units = ragged_max_blocks(c.w->count, c.R, kMT) * s.tiles * s.chunks * 2;
    return units < (int64_t)1 << 31 ? kMT : 0;
}

int ragged_mma_workers() { return kGroups * context_sm_count(); }

size_t ragged_mma_partials() { return (size_t)ragged_mma_workers() * 2 * kMT * TILE_ROWS * sizeof(float); }

int ragged_mma(const RaggedCall& c, const __half* xh, int64_t X, const int32_t* rows, const RaggedPlan* plan, float* part,
               unsigned* cnt) {
    const TiledShape& s = c.w->shape;
    const Params p{xh, X, rows, c.y, c.y_dtype, s.N, s.K, (int)s.chunks,
                   (int)s.tiles, plan, part, cnt, context_status()};
    const unsigned grid = (unsigned)context_sm_count();
    switch (s.type) {
        case T_Q4_K: return launch_type<T_Q4_K>(p, c.up != nullptr, grid, c.st);
        case T_Q4_0: return launch_type<T_Q4_0>(p, c.up != nullptr, grid, c.st);
        case T_Q8_0:
        case T_NXF_I8: return launch_type<T_Q8_0>(p, c.up != nullptr, grid, c.st);
        case T_Q3_K: return launch_type<T_Q3_K>(p, c.up != nullptr, grid, c.st);
        case T_I4G128: return launch_type<T_I4G128>(p, c.up != nullptr, grid, c.st);
        case T_Q6_K: return launch_type<T_Q6_K>(p, c.up != nullptr, grid, c.st);
        case T_Q5_K: return launch_type<T_Q5_K>(p, c.up != nullptr, grid, c.st);
        case T_Q4_1: return launch_type<T_Q4_1>(p, c.up != nullptr, grid, c.st);
        case T_Q2_K: return launch_type<T_Q2_K>(p, c.up != nullptr, grid, c.st);
        case T_I4G32: return launch_type<T_I4G32>(p, c.up != nullptr, grid, c.st);
        case T_I4G64: return launch_type<T_I4G64>(p, c.up != nullptr, grid, c.st);
        case T_I4G256: return launch_type<T_I4G256>(p, c.up != nullptr, grid, c.st);
        default: return NXQ_ERR_UNSUPPORTED;
    }
}

}  // namespace nxq
