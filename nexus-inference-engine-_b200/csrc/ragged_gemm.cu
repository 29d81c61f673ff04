// Tensor-core ragged products on tcgen05 / TMEM: y[s] = x[s] W_e^T for the
// slots of every expert, and the SwiGLU form with a gate and an up product.
//
// A persistent grid of one CTA per SM walks the plan's work tiles (ragged.h): 128
// weight rows x one row block of an expert.  The roles are those of the dense
// prefill GEMM (qmm_gemm.cu), per 64-element k-step:
//   warp 26      producer: the packed tile-chunks (256 k) by 1-D bulk copies
//   warp 0       producer: the activations of the row block by TMA, as boxes of
//                64 k x 64 slots (128-byte swizzle, no multicast), only as many
//                as the block has slots for
//   warps 2-17   four dequant warpgroups: thread r decodes row r's 32-element
//                group to f16 and writes it to TMEM, the MMA's A operand
//   warp 1       one lane issues tcgen05.mma kind::f16 M=128, K=16 with N = the
//                block's slots rounded up to 16 (a short block costs less)
//   warps 18-25  epilogue: tcgen05.ld of the accumulator, conversion, store of
//                the block's slots only
// Plain form: row blocks of up to 256 slots, one 256-column fp32 accumulator.
// SwiGLU form (PAIR): row blocks of up to 128 slots and two 128-column
// accumulators; every k-step feeds the same activations to a gate and an up
// MMA (warpgroups 0, 1 decode the gate, 2, 3 the up weight), and the
// epilogue stores silu(gate) * up, so the two products never reach memory.
//
// A k-step's activations and its A operand share one ring stage, released by
// one commit.  There are as many stages as k-steps in a chunk, so every stage
// index is a constant.  The issuing loop runs warp-wide with only the MMA and
// the commit in the elected lane: with the loop in one lane and two rings
// it took 1060 cycles a k-step whatever the block's size (four MMAs
// at ~92 cycles of issue each, measured), twice the 512 of a 256-slot MMA.
//
// An MMA column depends on its own slot's activations only, so what the boxes
// hold behind a block's slots (the next expert's rows, or zeros) reaches no
// stored value.  Every wait is bounded (sm100_ptx.cuh).  Numerics as the dense
// kernels: weights rounded once to f16, f16 activations, fp32 accumulation.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "dq_f16.cuh"
#include "qmm_gemm.h"
#include "ragged.h"
#include "sm100_ptx.cuh"

namespace nxq {

namespace {

constexpr int kDeqGroups = 4;
constexpr int kEpiWarps = 8;
constexpr int kWarpProducer = 0, kWarpMma = 1, kWarpDeq0 = 2, kWarpEpi0 = 2 + 4 * kDeqGroups;
constexpr int kWarpWProducer = kWarpEpi0 + kEpiWarps;
constexpr int kThreads = 32 * (kWarpWProducer + 1);
constexpr int kKS = 64;  // reduction elements per k-step (one swizzle atom)
constexpr int kStepsPerChunk = CHUNK_K / kKS;
constexpr int kStages = kStepsPerChunk;  // ring: activations (shared memory) and A operand (TMEM)
constexpr int kBarBytes = 512;
constexpr uint32_t kColD = 256;     // accumulators: columns 256..511
constexpr uint32_t kTmemCols = 512;
constexpr int kBoxRows = 64;
constexpr int kBoxBytes = kBoxRows * kKS * 2;

template <int TYPE, bool PAIR>
struct Cfg {
    static constexpr int WB = dq::Group<TYPE>::kStage;
    static constexpr int NT = PAIR ? 128 : 256;  // slots per work tile
    static constexpr int XB = NT * kKS * 2;
    static constexpr int kBudget = 227 * 1024 - 1024 - kBarBytes;
    static constexpr int kMats = PAIR ? 2 : 1;
    static constexpr int kACols = 32 * kMats;    // TMEM columns of a stage's A operand
    static constexpr int kWMax = 4 * kMats;
    static constexpr int fit = (kBudget - kStages * XB) / WB;
    static constexpr int kW = fit > kWMax ? kWMax : fit;
    static_assert(kW >= 2, "tile-chunk ring too shallow");
    static_assert(kStages * kACols <= (int)kColD, "A stages overlap the accumulator");
    static constexpr size_t smem = 1024 + (size_t)kStages * XB + (size_t)kW * WB + kBarBytes;
};

struct Params {
    const uint8_t* const* w;
    const uint8_t* const* up;
    TiledShape s;
    void* y;
    int y_dtype;
    const RaggedPlan* plan;
    DeviceStatus* status;
};

template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// y[m0 + j][n] = v[j] for j < cnt (element offset `off` = m0 * N + n).
template <typename T>
__device__ __forceinline__ void store_col(void* y, int64_t off, int64_t N, int cnt, const uint32_t (&v)[32]) {
    T* q = reinterpret_cast<T*>(y) + off;
#pragma unroll
    for (int j = 0; j < 32; ++j, q += N)
        if (j < cnt) *q = from_f32<T>(__uint_as_float(v[j]));
}

__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, const ptx::WaitCtl& c, unsigned where) {
    int ok = 0;
    if ((threadIdx.x & 31) == 0) ok = ptx::mbar_wait(bar, parity, c, where) ? 1 : 0;
    return __shfl_sync(0xFFFFFFFFu, ok, 0) != 0;
}

template <int TYPE, int S>
__device__ __forceinline__ void dq_step(const uint8_t* stage, int r, int h, uint32_t taddr) {
    uint32_t o[16];
    if (h == 0)
        dq::Group<TYPE>::template decode<2 * S>(stage, r, o);
    else
        dq::Group<TYPE>::template decode<2 * S + 1>(stage, r, o);
    ptx::tmem_st16(taddr, o);
}

template <int TYPE, bool PAIR>
__global__ void __launch_bounds__(kThreads, 1) ragged_gemm_kernel(const Params p, const __grid_constant__ CUtensorMap xmap) {
    using C = Cfg<TYPE, PAIR>;
    constexpr int WB = C::WB, XB = C::XB, NT = C::NT, kWStages = C::kW, kMats = C::kMats, kACols = C::kACols;
    static_assert((3 * kStages + 2 * kWStages + 3) * 8 + 8 <= kBarBytes, "barrier area too small");

    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = smem_raw + ((1024 - (ptx::smem_addr(smem_raw) & 1023)) & 1023);
    uint8_t* xs = smem;
    uint8_t* ws = smem + kStages * XB;
    uint64_t* x_full = reinterpret_cast<uint64_t*>(ws + kWStages * WB);  // activations landed
    uint64_t* a_full = x_full + kStages;                                 // A operand written
    uint64_t* empty = a_full + kStages;                                  // the MMA is done with both
    uint64_t* w_full = empty + kStages;
    uint64_t* w_empty = w_full + kWStages;
    uint64_t* d_full = w_empty + kWStages;
    uint64_t* d_empty = d_full + 1;
    uint64_t* drain = d_empty + 1;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

    const int tiles = (int)p.s.tiles;
    const int64_t total = (int64_t)p.plan->blocks * tiles;
    if (blockIdx.x >= total) return;  // the whole CTA, before any barrier or TMEM

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const ptx::WaitCtl ctl{abort_flag, p.status};
    if (threadIdx.x == 0) {
        for (int i = 0; i < kStages; ++i) {
            ptx::mbar_init(&x_full[i], 1);
            ptx::mbar_init(&a_full[i], 8 * kMats);  // the warps that write the A operand
            ptx::mbar_init(&empty[i], 1);
        }
        for (int i = 0; i < kWStages; ++i) {
            ptx::mbar_init(&w_full[i], 1);
            ptx::mbar_init(&w_empty[i], 4 * kDeqGroups / kMats);  // the warps that decode a tile-chunk
        }
        ptx::mbar_init(d_full, 1);
        ptx::mbar_init(d_empty, kEpiWarps);
        ptx::mbar_init(drain, 1);
        *abort_flag = 0;
        ptx::fence_mbar_init();
    }
    if (warp == kWarpProducer) {
        ptx::tmem_alloc(tmem_slot, kTmemCols);
        ptx::tmem_relinquish();
    }
    ptx::tc_fence_before();
    __syncthreads();
    ptx::tc_fence_after();
    const uint32_t tmem = *tmem_slot;

    const int chunks = (int)p.s.chunks;
    const int64_t G = gridDim.x;

    if (warp == kWarpWProducer) {
        if (lane == 0) {
            uint32_t qw = 0;
            bool ok = true;
            RaggedWalk<true> walk;
            walk.start(p.plan, NT, tiles, blockIdx.x);
            for (int64_t g = blockIdx.x; g < total && ok; g += G) {
                const RaggedTile t = walk.at(g);
                const uint8_t* src[kMats];
                src[0] = p.w[t.e] + p.s.chunk_offset(t.tile, 0);
                if constexpr (PAIR) src[1] = p.up[t.e] + p.s.chunk_offset(t.tile, 0);
                for (int c = 0; c < chunks * kMats && ok; ++c, ++qw) {
                    const int sw = qw % kWStages;
                    if (qw >= kWStages && !(ok = ptx::mbar_wait(&w_empty[sw], ((qw / kWStages) & 1) ^ 1u, ctl, 41))) break;
                    ptx::mbar_arrive_expect_tx(&w_full[sw], WB);
                    ptx::bulk_g2s(ws + sw * WB, src[c % kMats] + (int64_t)(c / kMats) * WB, WB, &w_full[sw]);
                }
            }
            // Do not leave with copies in flight (bounded, ignoring the abort flag).
            for (uint32_t k = qw >= kWStages ? qw - kWStages : 0; k < qw; ++k) {
                const long long t0 = clock64();
                while (!ptx::mbar_try_wait(&w_full[k % kWStages], (k / kWStages) & 1) && clock64() - t0 < ptx::kWaitCycles) {
                }
            }
        }
    } else if (warp == kWarpProducer) {
        if (lane == 0) ptx::prefetch_tmap(&xmap);
        uint32_t cc = 0;  // chunks so far: its parity is the stages' phase
        bool ok = true;
        RaggedWalk<true> walk;
        walk.start(p.plan, NT, tiles, blockIdx.x);
        uint32_t issued = 0;  // k-steps requested
        for (int64_t g = blockIdx.x; g < total && ok; g += G) {
            const RaggedTile t = walk.at(g);
            const int boxes = (t.rows + kBoxRows - 1) / kBoxRows;
            for (int c = 0; c < chunks && ok; ++c) {
#pragma unroll
                for (int st = 0; st < kStages; ++st) {
                    ok = ok && ptx::mbar_wait(&empty[st], (cc & 1) ^ 1u, ctl, 42);
                    ok = __all_sync(0xFFFFFFFFu, ok);
                    if (!ok) continue;
                    if (lane == 0) ptx::mbar_arrive_expect_tx(&x_full[st], boxes * kBoxBytes);
                    __syncwarp();
                    if (lane < boxes)
                        ptx::tma_load_2d(xs + st * XB + lane * kBoxBytes, &xmap, c * CHUNK_K + st * kKS,
                                         t.row0 + lane * kBoxRows, &x_full[st]);
                    ++issued;
                }
                if (ok) ++cc;
            }
        }
        // Do not leave with copies in flight (bounded, ignoring the abort flag).
        for (uint32_t k = issued >= kStages ? issued - kStages : 0; k < issued; ++k) {
            const long long t0 = clock64();
            while (!ptx::mbar_try_wait(&x_full[k % kStages], (k / kStages) & 1) && clock64() - t0 < ptx::kWaitCycles) {
            }
        }
    } else if (warp == kWarpMma) {
        uint32_t cc = 0, nt = 0;
        bool ok = true;
        RaggedWalk<true> walk;
        walk.start(p.plan, NT, tiles, blockIdx.x);
        const uint64_t desc0 = ptx::desc_sw128_kmajor(ptx::smem_addr(xs));
        for (int64_t g = blockIdx.x; g < total && ok; g += G, ++nt) {
            const RaggedTile t = walk.at(g);
            const uint32_t idesc = ptx::idesc_f16_f32(128, (t.rows + 15) & ~15);
            ok = nt == 0 || ptx::mbar_wait(d_empty, (nt - 1) & 1, ctl, 43);
            ok = __all_sync(0xFFFFFFFFu, ok);
            ptx::tc_fence_after();
            for (int c = 0; c < chunks && ok; ++c, ++cc) {
#pragma unroll
                for (int st = 0; st < kStages; ++st) {
                    ok = ok && ptx::mbar_wait(&x_full[st], cc & 1, ctl, 44) && ptx::mbar_wait(&a_full[st], cc & 1, ctl, 45);
                    ok = __all_sync(0xFFFFFFFFu, ok);
                    if (!ok) continue;
                    ptx::tc_fence_after();
                    if (ptx::elect_one()) {
#pragma unroll
                        for (int mat = 0; mat < kMats; ++mat)
                            ptx::mma_ts_f16_k64(tmem + kColD + mat * NT, tmem + st * kACols + mat * 32,
                                                desc0 + ((st * XB) >> 4), idesc, (c | st) ? 1u : 0u);
                        ptx::mma_commit(&empty[st]);
                        if (st == kStages - 1 && c == chunks - 1) ptx::mma_commit(d_full);
                    }
                    __syncwarp();
                }
            }
        }
        if (ptx::elect_one()) ptx::mma_commit(drain);
        __syncwarp();
        const long long t0 = clock64();
        while (!ptx::mbar_try_wait(drain, 0) && clock64() - t0 < ptx::kWaitCycles) {
        }
    } else if (warp < kWarpEpi0) {
        // Warpgroup wg decodes k group wg % 2 of a k-step: plain, of the k-steps
        // of parity wg / 2; PAIR, of every k-step of matrix wg / 2.
        const int wg = (warp - kWarpDeq0) >> 2, quad = warp & 3, r = quad * 32 + lane;
        const int h = wg & 1, par = wg >> 1;
        uint32_t qw = PAIR ? par : 0, cc = 0;
        bool ok = true;
        for (int64_t g = blockIdx.x; g < total && ok; g += G) {
            for (int c = 0; c < chunks && ok; ++c, ++cc, qw += kMats) {
                const int sw = qw % kWStages;
                if (!(ok = warp_wait(&w_full[sw], (qw / kWStages) & 1, ctl, 46))) break;
                const uint8_t* stage = ws + sw * WB;
#pragma unroll
                for (int st = 0; st < kStages; ++st) {
                    if (!PAIR && (st & 1) != par) continue;
                    ok = ok && warp_wait(&empty[st], (cc & 1) ^ 1u, ctl, 47);
                    if (!ok) continue;
                    ptx::tc_fence_after();
                    const uint32_t taddr =
                        tmem + ((uint32_t)(quad * 32) << 16) + st * kACols + (PAIR ? 32 * par : 0) + 16 * h;
                    if (st == 0) dq_step<TYPE, 0>(stage, r, h, taddr);
                    if (st == 1) dq_step<TYPE, 1>(stage, r, h, taddr);
                    if (st == 2) dq_step<TYPE, 2>(stage, r, h, taddr);
                    if (st == 3) dq_step<TYPE, 3>(stage, r, h, taddr);
                    ptx::tmem_wait_st();
                    ptx::tc_fence_before();
                    __syncwarp();
                    if (lane == 0) ptx::mbar_arrive(&a_full[st]);
                }
                __syncwarp();
                if (ok && lane == 0) ptx::mbar_arrive(&w_empty[sw]);
            }
        }
    } else {
        // Epilogue: warp (quad, sub) reads TMEM lanes 32 quad .. (its lane
        // quadrant) = weight row n, and the slots of half `sub` of the tile.
        const int ew = warp - kWarpEpi0, quad = warp & 3, r = quad * 32 + lane, sub = ew >> 2;
        const int64_t N = p.s.N;
        uint32_t nt = 0;
        RaggedWalk<true> walk;
        walk.start(p.plan, NT, tiles, blockIdx.x);
        for (int64_t g = blockIdx.x; g < total; g += G, ++nt) {
            const RaggedTile t = walk.at(g);
            if (!warp_wait(d_full, nt & 1, ctl, 48)) break;
            ptx::tc_fence_after();
            const int64_t n = (int64_t)t.tile * TILE_ROWS + r;
#pragma unroll 1
            for (int cb = 0; cb < NT / 64; ++cb) {
                const int c0 = sub * (NT / 2) + 32 * cb;  // slot in the tile
                const int cnt = t.rows - c0;
                if (cnt <= 0) break;
                uint32_t v[32];
                const uint32_t ta = tmem + ((uint32_t)(quad * 32) << 16) + kColD + c0;
                ptx::tmem_ld16(ta, *reinterpret_cast<uint32_t(*)[16]>(&v[0]));
                ptx::tmem_ld16(ta + 16, *reinterpret_cast<uint32_t(*)[16]>(&v[16]));
                if constexpr (PAIR) {
#pragma unroll
                    for (int hf = 0; hf < 2; ++hf) {
                        uint32_t u[16];
                        ptx::tmem_ld16(ta + NT + 16 * hf, u);
                        ptx::tmem_wait_ld();
#pragma unroll
                        for (int j = 0; j < 16; ++j) {
                            const float a = __uint_as_float(v[16 * hf + j]);
                            v[16 * hf + j] = __float_as_uint(a / (1.0f + expf(-a)) * __uint_as_float(u[j]));
                        }
                    }
                } else {
                    ptx::tmem_wait_ld();
                }
                if (n < N) {
                    const int64_t off = ((int64_t)t.row0 + c0) * N + n;
                    if (p.y_dtype == NXQ_BF16)
                        store_col<__nv_bfloat16>(p.y, off, N, cnt, v);
                    else if (p.y_dtype == NXQ_F16)
                        store_col<__half>(p.y, off, N, cnt, v);
                    else
                        store_col<float>(p.y, off, N, cnt, v);
                }
            }
            ptx::tc_fence_before();
            __syncwarp();
            if (lane == 0) ptx::mbar_arrive(d_empty);
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
                                         (int)Cfg<TYPE, false>::smem);
    if (e == cudaSuccess)
        e = cudaFuncSetAttribute(ragged_gemm_kernel<TYPE, true>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                 (int)Cfg<TYPE, true>::smem);
    return e == cudaSuccess ? NXQ_OK : cuda_fail(e, "cudaFuncSetAttribute (ragged_gemm)");
}

template <int TYPE>
int launch(const Params& p, const CUtensorMap& tmap, unsigned grid, cudaStream_t st) {
    if (p.up)
        ragged_gemm_kernel<TYPE, true><<<grid, kThreads, Cfg<TYPE, true>::smem, st>>>(p, tmap);
    else
        ragged_gemm_kernel<TYPE, false><<<grid, kThreads, Cfg<TYPE, false>::smem, st>>>(p, tmap);
    note_launches(1);
    const cudaError_t e = cudaGetLastError();
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

int ragged_gemm_blk(bool pair) { return pair ? 128 : 256; }

int ragged_gemm(const RaggedCall& c, const void* xh, int64_t X, const RaggedPlan* plan) {
    const TiledShape& s = c.w->shape;
    Params p{c.w->dev, c.up ? c.up->dev : nullptr, s, c.y, c.y_dtype, plan, context_status()};
    CUtensorMap tmap;
    if (int rc = gemm_activation_map(&tmap, xh, X, s.K, kBoxRows)) return rc;
    const int64_t work = ragged_max_blocks(c.w->count, c.R, ragged_gemm_blk(c.up != nullptr)) * s.tiles;
    const unsigned grid = (unsigned)(work < context_sm_count() ? work : context_sm_count());
    switch (s.type) {
        case T_Q4_K: return launch<T_Q4_K>(p, tmap, grid, c.st);
        case T_Q4_0: return launch<T_Q4_0>(p, tmap, grid, c.st);
        case T_Q8_0:
        case T_NXF_I8: return launch<T_Q8_0>(p, tmap, grid, c.st);
        case T_Q3_K: return launch<T_Q3_K>(p, tmap, grid, c.st);
        case T_I4G128: return launch<T_I4G128>(p, tmap, grid, c.st);
        case T_Q6_K: return launch<T_Q6_K>(p, tmap, grid, c.st);
        case T_Q5_K: return launch<T_Q5_K>(p, tmap, grid, c.st);
        case T_Q4_1: return launch<T_Q4_1>(p, tmap, grid, c.st);
        case T_Q2_K: return launch<T_Q2_K>(p, tmap, grid, c.st);
        case T_I4G32: return launch<T_I4G32>(p, tmap, grid, c.st);
        case T_I4G64: return launch<T_I4G64>(p, tmap, grid, c.st);
        case T_I4G256: return launch<T_I4G256>(p, tmap, grid, c.st);
        default: return NXQ_ERR_UNSUPPORTED;
    }
}

}  // namespace nxq
