// Products grouped by expert with ragged sizes: y[s] = x[rows[s]] W_e^T for the
// slots s of expert e, with the sizes known on the device only.
//
// A call is a plan kernel, which turns the offsets into a list of the experts
// that have rows (ragged.h) and where needed brings the activations into slot
// order as f16, and a product kernel that walks the plan: warp-level tensor
// cores for few slots per expert (ragged_mma.cu), tcgen05 beyond
// (ragged_gemm.cu), or the exact kernel here, with fp32 decode (formats.cuh,
// decode8) and fp32 products on the CUDA cores, for the block types without a
// tensor-core decoder.
#include "ragged.h"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <mutex>
#include <new>
#include <unordered_set>

namespace nxq {

namespace {

std::mutex g_tables_mu;
std::unordered_set<ExpertTable*> g_tables;

int check_experts(nxq_experts_t h, const ExpertTable** out) {
    ExpertTable* t = reinterpret_cast<ExpertTable*>(h);
    if (!t) return fail(NXQ_ERR_ARG, "null expert table");
    std::lock_guard<std::mutex> lk(g_tables_mu);
    if (!g_tables.count(t)) return fail(NXQ_ERR_ARG, "expert table is not live (released or foreign)");
    *out = t;
    return NXQ_OK;
}

// One CTA of at least E threads, thread = expert: writes the experts that have rows.  An expert's
// range is taken only if both its ends lie in [0, R] and it starts at or behind
// every such offset before it, so the ranges taken never overlap and hold at most
// R slots whatever the offsets are; anything else is reported and left out.  An
// offset outside [0, R] so costs the two experts it bounds, and no other.
__device__ __forceinline__ void make_plan(const int32_t* offsets, int E, int64_t R, int blk, RaggedPlan* plan,
                                          const uint8_t* const* w, const uint8_t* const* up, DeviceStatus* status) {
    __shared__ int warp_n[32], warp_b[32], warp_m[32];
    const int e = threadIdx.x, warp = e >> 5, lane = e & 31;
    const int o0 = e < E ? offsets[e] : 0, o1 = e < E ? offsets[e + 1] : 0;
    const uint8_t* const we = e < E ? w[e] : nullptr;
    const uint8_t* const ue = e < E && up ? up[e] : nullptr;
    int before = o0 <= R ? o0 : 0;  // the largest offset within [0, R] (or 0) up to and including o0
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xFFFFFFFFu, before, o);
        if (lane >= o && v > before) before = v;
    }
    if (lane == 31) warp_m[warp] = before;
    __syncthreads();
    for (int w = 0; w < warp; ++w) before = warp_m[w] > before ? warp_m[w] : before;
    int a = 0, n = 0;
    if (e < E) {
        if (o0 < 0 || o0 > R || o0 < before || o1 < o0 || o1 > R)
            raise_index(status, kIndexOffset);
        else
            a = o0, n = o1 - o0;
    }
    const int has = n > 0, nb = row_blocks(n, blk);
    const unsigned act = __ballot_sync(0xFFFFFFFFu, has);
    int bs = nb;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xFFFFFFFFu, bs, o);
        if (lane >= o) bs += v;
    }
    if (lane == 31) {
        warp_n[warp] = __popc(act);
        warp_b[warp] = bs;
    }
    __syncthreads();
    int n0 = 0, b0 = 0;
    for (int w = 0; w < warp; ++w) {
        n0 += warp_n[w];
        b0 += warp_b[w];
    }
    if (has) plan->it[n0 + __popc(act & ((1u << lane) - 1u))] = RaggedEntry{e, a, n, b0 + bs - nb, we, ue};
    if (e == (int)blockDim.x - 1) {
        plan->entries = n0 + __popc(act);
        plan->blocks = b0 + bs;
    }
}

__device__ __forceinline__ float load_x(const void* x, int dt, int64_t i) {
    if (dt == NXQ_F16) return __half2float(static_cast<const __half*>(x)[i]);
    if (dt == NXQ_BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(x)[i]);
    return static_cast<const float*>(x)[i];
}
__device__ __forceinline__ void store_y(void* y, int dt, int64_t i, float v) {
    if (dt == NXQ_F16)
        static_cast<__half*>(y)[i] = __float2half_rn(v);
    else if (dt == NXQ_BF16)
        static_cast<__nv_bfloat16*>(y)[i] = __float2bfloat16_rn(v);
    else
        static_cast<float*>(y)[i] = v;
}

constexpr int kSimtBlk = 8;  // rows per work tile

struct SimtParams {
    TiledShape s;
    const void* x;
    int x_dtype;
    int64_t X;
    const int32_t* rows;
    void* y;
    int y_dtype;
    const RaggedPlan* plan;
    DeviceStatus* status;
};

// Thread r owns weight row r of the tile for up to kSimtBlk slots.
template <bool PAIR>
__global__ void __launch_bounds__(TILE_ROWS) ragged_simt_kernel(const SimtParams p) {
    __shared__ float xs[kSimtBlk][CHUNK_K];
    __shared__ int64_t src[kSimtBlk];
    const int r = threadIdx.x;
    const int tiles = (int)p.s.tiles;
    const int64_t total = (int64_t)p.plan->blocks * tiles;
    if (blockIdx.x >= total) return;
    RaggedWalk<false> walk;
    walk.start(p.plan, kSimtBlk, tiles, blockIdx.x);
    for (int64_t g = blockIdx.x; g < total; g += gridDim.x) {
        const RaggedTile t = walk.at(g);
        __syncthreads();
        if (r < kSimtBlk) {
            int64_t row = -1;
            if (r < t.rows) {
                row = p.rows ? p.rows[t.row0 + r] : t.row0 + r;
                if (row < 0 || row >= p.X) {
                    raise_index(p.status, kIndexRow);
                    row = -1;
                }
            }
            src[r] = row;
        }
        float acc[kSimtBlk], accu[PAIR ? kSimtBlk : 1];
#pragma unroll
        for (int m = 0; m < kSimtBlk; ++m) {
            acc[m] = 0.0f;
            if constexpr (PAIR) accu[m] = 0.0f;
        }
        for (int64_t c = 0; c < p.s.chunks; ++c) {
            const int64_t k0 = c * CHUNK_K;
            __syncthreads();
            for (int i = r; i < kSimtBlk * CHUNK_K; i += TILE_ROWS) {
                const int m = i / CHUNK_K, kk = i % CHUNK_K;
                xs[m][kk] = src[m] >= 0 && k0 + kk < p.s.K ? load_x(p.x, p.x_dtype, src[m] * p.s.K + k0 + kk) : 0.0f;
            }
            __syncthreads();
            const int kmax = (int)(p.s.K - k0 < CHUNK_K ? p.s.K - k0 : CHUNK_K);
            auto add = [&](const uint8_t* w, float* a) {
                const uint8_t* chunk = w + p.s.chunk_offset(t.tile, c);
                for (int e0 = 0; e0 < kmax; e0 += 8) {
                    float v[8];
                    decode8(p.s.type, chunk, r, e0, v);
#pragma unroll
                    for (int m = 0; m < kSimtBlk; ++m)
#pragma unroll
                        for (int i = 0; i < 8; ++i) a[m] = fmaf(v[i], xs[m][e0 + i], a[m]);
                }
            };
            add(t.w, acc);
            if constexpr (PAIR) add(t.up, accu);
        }
        const int64_t n = (int64_t)t.tile * TILE_ROWS + r;
        if (n >= p.s.N) continue;
#pragma unroll
        for (int m = 0; m < kSimtBlk; ++m)
            if (m < t.rows) {
                float v = acc[m];
                if constexpr (PAIR) v = v / (1.0f + expf(-v)) * accu[m];
                store_y(p.y, p.y_dtype, (int64_t)(t.row0 + m) * p.s.N + n, v);
            }
    }
}

// What a product kernel needs first, in one launch.  CTA 0 makes the plan and
// zeroes the counters; the others (none if xh is null) bring the activations of
// every slot an expert has into slot order as f16, xh[s] = f16(x[rows ? rows[s]
// : s]), a group of kRowThreads threads per slot and 8 or 1 elements per thread
// (VEC).  fp32 and bf16 values beyond the f16 range and row indices outside
// [0, X) (zeros) are reported.
struct PrepParams {
    const int32_t* offsets;
    int E;
    int64_t R;
    int blk;
    RaggedPlan* plan;
    const uint8_t* const* w;
    const uint8_t* const* up;
    unsigned* cnt;
    int n_cnt;
    const void* x;
    int x_dtype;
    int64_t X, K;
    const int32_t* rows;
    __half* xh;
    DeviceStatus* status;
};
constexpr int kRowThreads = 256;

template <int VEC>
__global__ void __launch_bounds__(kMaxExperts) ragged_prep_kernel(const PrepParams p) {
    overlap_begin();  // the product kernel may set itself up meanwhile
    if (blockIdx.x == 0) {
        for (int i = threadIdx.x; i < p.n_cnt; i += blockDim.x) p.cnt[i] = 0u;
        make_plan(p.offsets, p.E, p.R, p.blk, p.plan, p.w, p.up, p.status);
        return;
    }
    // Up to the largest offset within [0, R], which is the last one unless an
    // expert that the plan leaves out comes last.  (A thread per expert.)
    __shared__ int top[32];
    const int o1 = (int)threadIdx.x < p.E ? p.offsets[threadIdx.x + 1] : 0;
    int most = __reduce_max_sync(0xFFFFFFFFu, o1 <= p.R ? o1 : 0);
    if (threadIdx.x % 32 == 0) top[threadIdx.x / 32] = most;
    __syncthreads();
    most = __reduce_max_sync(0xFFFFFFFFu, threadIdx.x % 32 < blockDim.x / 32 ? top[threadIdx.x % 32] : 0);
    const int o0 = p.offsets[0];
    const int64_t lo = o0 > 0 && o0 <= p.R ? o0 : 0, hi = most;  // (a first offset out of range bounds nothing)
    const int group = threadIdx.x / kRowThreads, lane = threadIdx.x % kRowThreads, groups = blockDim.x / kRowThreads;
    bool over = false;
    for (int64_t s = lo + (int64_t)(blockIdx.x - 1) * groups + group; s < hi; s += (int64_t)(gridDim.x - 1) * groups) {
        int64_t row = p.rows ? p.rows[s] : s;
        if (row < 0 || row >= p.X) {
            if (lane == 0) raise_index(p.status, kIndexRow);
            row = -1;
        }
        for (int64_t k = (int64_t)lane * VEC; k < p.K; k += kRowThreads * VEC) {
            const int64_t i = row * p.K + k;
            __half* out = p.xh + s * p.K + k;
            if constexpr (VEC == 1) {
                const float v = row < 0 ? 0.0f : load_x(p.x, p.x_dtype, i);
                over |= f16_overflows(v);
                *out = __float2half_rn(v);
            } else {
                uint4 h = make_uint4(0u, 0u, 0u, 0u);
                if (row >= 0 && p.x_dtype == NXQ_F16) {
                    h = *reinterpret_cast<const uint4*>(static_cast<const __half*>(p.x) + i);
                } else if (row >= 0) {
                    float v[8];
                    if (p.x_dtype == NXQ_F32) {
                        const float4* q = reinterpret_cast<const float4*>(static_cast<const float*>(p.x) + i);
                        const float4 a = q[0], b = q[1];
                        v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
                    } else {
                        const uint4 q = *reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(p.x) + i);
                        const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            v[2 * j] = __uint_as_float(w[j] << 16);
                            v[2 * j + 1] = __uint_as_float(w[j] & 0xFFFF0000u);
                        }
                    }
                    uint32_t o[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        over |= f16_overflows(v[2 * j]) || f16_overflows(v[2 * j + 1]);
                        const __half2 q = __floats2half2_rn(v[2 * j], v[2 * j + 1]);
                        o[j] = *reinterpret_cast<const uint32_t*>(&q);
                    }
                    h = make_uint4(o[0], o[1], o[2], o[3]);
                }
                *reinterpret_cast<uint4*>(out) = h;
            }
        }
    }
    if (over) raise_range(p.status, 1u);
}

cudaError_t launch_prep(const RaggedCall& c, int blk, RaggedPlan* plan, unsigned* cnt, int n_cnt, __half* xh) {
    const PrepParams p{c.offsets, c.w->count, c.R, blk, plan, c.w->dev, c.up ? c.up->dev : nullptr, cnt, n_cnt, c.x, c.x_dtype, c.X, c.w->shape.K, c.rows, xh,
                       context_status()};
    // A thread per expert, in whole warps; whole groups of kRowThreads if rows move.
    const int unit = xh ? kRowThreads : 32;
    const unsigned threads = (unsigned)((c.w->count + unit - 1) / unit * unit);
    const int64_t groups = threads / kRowThreads;
    const int64_t most = (int64_t)context_sm_count() * 8 / (groups ? groups : 1), want = groups ? (c.R + groups - 1) / groups : 0;
    const unsigned grid = 1 + (unsigned)(!xh ? 0 : want < most ? want : most);
    const bool vec = ((uintptr_t)c.x % 16) == 0;  // K is a multiple of 32
    note_launches(1);
    return launch_overlapped(vec ? ragged_prep_kernel<8> : ragged_prep_kernel<1>, grid, threads, 0, c.st, p);
}

int run_simt(const RaggedCall& c, const RaggedPlan* plan) {
    SimtParams p{c.w->shape, c.x, c.x_dtype, c.X, c.rows, c.y, c.y_dtype, plan,
                 context_status()};
    const int64_t work = ragged_max_blocks(c.w->count, c.R, kSimtBlk) * c.w->shape.tiles;
    const int64_t cap = (int64_t)context_sm_count() * 16;
    const unsigned grid = (unsigned)(work < cap ? work : cap);
    if (c.up)
        ragged_simt_kernel<true><<<grid, TILE_ROWS, 0, c.st>>>(p);
    else
        ragged_simt_kernel<false><<<grid, TILE_ROWS, 0, c.st>>>(p);
    note_launches(1);
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? NXQ_OK : cuda_fail(e, "ragged product launch");
}

// Plan, activations and product of a call, in one stream-ordered workspace.
int dispatch(const RaggedCall& c) {
    const int mma = ragged_mma_blk(c);  // few slots per expert
    const bool gemm = !mma && ragged_gemm_supported(c.w->shape);
    const int blk = mma ? mma : gemm ? ragged_gemm_blk() : kSimtBlk;
    // f16 activations are read where they are: by row index (mma), or in slot
    // order (gemm: TMA boxes).
    const bool as_is = (!mma && !gemm) || (c.x_dtype == NXQ_F16 && ((uintptr_t)c.x % 16) == 0 && (mma || !c.rows));
    const int workers = ragged_mma_workers();
    auto up = [](size_t n) { return (n + 255) & ~(size_t)255; };
    const size_t plan_size = up(plan_bytes(c.w->count < c.R ? c.w->count : c.R));
    const size_t cnt_size = mma ? up(workers * sizeof(unsigned)) : 0, part_size = mma ? up(ragged_mma_partials()) : 0;
    const size_t x_size = as_is ? 0 : (size_t)c.R * c.w->shape.K * sizeof(__half);
    uint8_t* ws = nullptr;
    cudaError_t e = cudaMallocAsync((void**)&ws, plan_size + cnt_size + part_size + x_size, c.st);
    if (e != cudaSuccess) return cuda_fail(e, "cudaMallocAsync (ragged workspace)");
    RaggedPlan* plan = reinterpret_cast<RaggedPlan*>(ws);
    unsigned* cnt = reinterpret_cast<unsigned*>(ws + plan_size);
    float* part = reinterpret_cast<float*>(ws + plan_size + cnt_size);
    __half* xh = as_is ? nullptr : reinterpret_cast<__half*>(ws + plan_size + cnt_size + part_size);
    int rc = NXQ_OK;
    if ((e = launch_prep(c, blk, plan, cnt, mma ? workers : 0, xh)) != cudaSuccess)
        rc = cuda_fail(e, "ragged plan launch");
    else if (mma)
        rc = ragged_mma(c, as_is ? static_cast<const __half*>(c.x) : xh, as_is ? c.X : c.R, as_is ? c.rows : nullptr,
                        plan, part, cnt);
    else if (gemm)
        rc = ragged_gemm(c, as_is ? c.x : xh, as_is ? c.X : c.R, plan);
    else
        rc = run_simt(c, plan);
    cudaFreeAsync(ws, c.st);
    return rc;
}

int run(nxq_experts_t he, nxq_experts_t hu, bool pair, const void* x_dev, int x_dtype, int64_t X, const int32_t* rows_dev,
        void* y_dev, int y_dtype, int64_t R, const int32_t* offsets_dev, void* stream) {
    RaggedCall c{};
    int rc = check_experts(he, &c.w);
    if (rc || (pair && (rc = check_experts(hu, &c.up)))) return rc;
    if (pair && (c.w->count != c.up->count || c.w->shape.type != c.up->shape.type || c.w->shape.N != c.up->shape.N ||
                 c.w->shape.K != c.up->shape.K))
        return fail(NXQ_ERR_SHAPE, "ragged swiglu: gate (%d x %s [%lld][%lld]) and up (%d x %s [%lld][%lld]) differ",
                    c.w->count, type_name(c.w->shape.type), (long long)c.w->shape.N, (long long)c.w->shape.K,
                    c.up->count, type_name(c.up->shape.type), (long long)c.up->shape.N, (long long)c.up->shape.K);
    if (R < 0 || R > 0x7FFFFFFF || X < 0) return fail(NXQ_ERR_ARG, "ragged: R=%lld X=%lld", (long long)R, (long long)X);
    if (!dtype_valid(x_dtype) || !dtype_valid(y_dtype)) return fail(NXQ_ERR_ARG, "bad dtype");
    if (R == 0) return NXQ_OK;
    if (!x_dev || !y_dev || !offsets_dev) return fail(NXQ_ERR_ARG, "ragged: null activation, output or offsets");
    if (!aligned_as(x_dev, x_dtype) || !aligned_as(y_dev, y_dtype) || !aligned_4(offsets_dev) || !aligned_4(rows_dev))
        return fail(NXQ_ERR_ARG, "ragged: an array is not aligned to its type");
    if (!rows_dev && X < R)
        return fail(NXQ_ERR_SHAPE, "ragged: %lld activation rows for %lld slots (and no row indices)", (long long)X, (long long)R);
    if ((rc = context_ready())) return rc;
    c.x = x_dev;
    c.x_dtype = x_dtype;
    c.X = X;
    c.rows = rows_dev;
    c.y = y_dev;
    c.y_dtype = y_dtype;
    c.R = R;
    c.offsets = offsets_dev;
    c.st = (cudaStream_t)stream;
    return dispatch(c);
}

}  // namespace

void experts_shutdown() {
    std::lock_guard<std::mutex> lk(g_tables_mu);
    for (ExpertTable* t : g_tables) {
        cudaFree(t->dev);
        delete t;
    }
    g_tables.clear();
}

}  // namespace nxq

using namespace nxq;

extern "C" {

NXQ_API int nxq_experts_create(const nxq_weight_t* hs, int count, nxq_experts_t* out) {
    if (!hs || !out) return fail(NXQ_ERR_ARG, "null argument");
    if (count < 1 || count > kMaxExperts) return fail(NXQ_ERR_ARG, "%d experts (1 to %d)", count, kMaxExperts);
    // The references come first: another thread may release a weight until it has one.
    const uint8_t* dev[kMaxExperts];
    TiledShape shape{};
    int held = 0;
    auto give_back = [&](int status) {
        for (int i = 0; i < held; ++i) weight_table_ref(hs[i], -1);
        return status;
    };
    for (int i = 0; i < count; ++i) {
        Weight* w = nullptr;
        if (int rc = weight_table_ref(hs[i], 1, &w)) return give_back(rc);
        ++held;
        if (i == 0) shape = w->shape;
        if (w->shape.type != shape.type || w->shape.N != shape.N || w->shape.K != shape.K)
            return give_back(fail(NXQ_ERR_SHAPE, "expert %d is %s [%lld][%lld], expert 0 %s [%lld][%lld]", i,
                                  type_name(w->shape.type), (long long)w->shape.N, (long long)w->shape.K,
                                  type_name(shape.type), (long long)shape.N, (long long)shape.K));
        dev[i] = w->dev;
    }
    if (int rc = context_ready()) return give_back(rc);
    ExpertTable* t = new (std::nothrow) ExpertTable();
    if (!t) return give_back(fail(NXQ_ERR_NOMEM, "host allocation failed"));
    t->count = count;
    t->shape = shape;
    const size_t bytes = (size_t)count * sizeof(dev[0]);
    // The copy is waited for: streams that do not synchronize with the default one read the table.
    cudaError_t e = cudaMalloc((void**)&t->dev, bytes);
    if (e == cudaSuccess && (e = cudaMemcpy(t->dev, dev, bytes, cudaMemcpyHostToDevice)) == cudaSuccess)
        e = cudaStreamSynchronize(cudaStreamLegacy);
    int rc = e == cudaSuccess ? NXQ_OK : cuda_fail(e, "expert table");
    if (rc == NXQ_OK) {
        try {
            t->refs.assign(hs, hs + count);
            std::lock_guard<std::mutex> lk(g_tables_mu);
            g_tables.insert(t);
        } catch (const std::bad_alloc&) {
            rc = fail(NXQ_ERR_NOMEM, "host allocation failed");
        }
    }
    if (rc != NXQ_OK) {
        if (t->dev) cudaFree(t->dev);
        delete t;
        return give_back(rc);
    }
    *out = reinterpret_cast<nxq_experts_t>(t);
    return NXQ_OK;
}

NXQ_API int nxq_experts_release(nxq_experts_t h) {
    const ExpertTable* t = nullptr;
    int rc = check_experts(h, &t);
    if (rc || (rc = context_ready())) return rc;
    {
        std::lock_guard<std::mutex> lk(g_tables_mu);
        if (!g_tables.erase(const_cast<ExpertTable*>(t))) return fail(NXQ_ERR_ARG, "expert table is not live");
    }
    // Work queued on any stream may still read the table.
    cudaDeviceSynchronize();
    for (nxq_weight_t w : t->refs) weight_table_ref(w, -1);
    cudaFree(t->dev);
    delete t;
    return NXQ_OK;
}

NXQ_API int nxq_experts_info(nxq_experts_t h, int* count, int* type, int64_t* N, int64_t* K) {
    const ExpertTable* t = nullptr;
    if (int rc = check_experts(h, &t)) return rc;
    if (count) *count = t->count;
    if (type) *type = t->shape.type;
    if (N) *N = t->shape.N;
    if (K) *K = t->shape.K;
    return NXQ_OK;
}

NXQ_API int nxq_qmatmul_ragged(nxq_experts_t e, const void* x_dev, int x_dtype, int64_t X, const int32_t* rows_dev,
                               void* y_dev, int y_dtype, int64_t R, const int32_t* offsets_dev, void* stream) {
    return run(e, nullptr, false, x_dev, x_dtype, X, rows_dev, y_dev, y_dtype, R, offsets_dev, stream);
}

NXQ_API int nxq_qmatmul_ragged_swiglu(nxq_experts_t gate, nxq_experts_t up, const void* x_dev, int x_dtype, int64_t X,
                                      const int32_t* rows_dev, void* h_dev, int h_dtype, int64_t R,
                                      const int32_t* offsets_dev, void* stream) {
    return run(gate, up, true, x_dev, x_dtype, X, rows_dev, h_dev, h_dtype, R, offsets_dev, stream);
}

}  // extern "C"
