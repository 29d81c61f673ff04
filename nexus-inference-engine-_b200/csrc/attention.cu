// nxq_paged_attention: dispatch, and the kernel that joins partial results.
#include "attn_plan.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cmath>

namespace nxq {

namespace {

using namespace attn;

constexpr int kFewRows = 32;
constexpr int kJoinThreads = 128, kJoinWarps = kJoinThreads / 32;

// Joins the pieces of items cut between runs.  CTA (c, g) takes the item that begins in run
// c and ends behind it, if there is one, and of that rows kRowsPer g ...: a warp per row,
// first the largest maximum and the sum of weights over the pieces, then the sum of their
// outputs, in order of the runs whatever order they were written in.
constexpr int kRowsPer = 4 * kJoinWarps;

template <int ROWS, int KEYS>
__global__ void __launch_bounds__(kJoinThreads) attn_join_kernel(const __grid_constant__ AttnParams p, const int runs) {
    __shared__ PlanSmem plan;
    // The lengths are complete before the kernel that writes the pieces begins (it waits for
    // them before it lets this one start); the pieces when it has ended.
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    plan_total<ROWS, KEYS, kJoinThreads>(p, plan);
    const long long total = plan.total, r = blockIdx.x;
    const long long here = run_start(total, r, runs), end = run_start(total, r + 1, runs);
    long long first = 0, last = 0;
    bool cut = here < end && end < total;
    if (cut) {
        plan_locate<ROWS, KEYS, kJoinThreads>(p, plan, end);
        cut = plan.off > 0 && end - plan.off >= here;
    }
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (!cut) return;
    bool bad;
    const Seq q = launch_seq(p, plan.s, &bad);
    const Item it = make_item<ROWS, KEYS>(p, q, plan.item);
    first = end - plan.off;
    last = first + it.units;
    // Piece i: with a unit or more in every run, run r + i; else the run that unit first + i is.
    auto run_of = [&](long long x) { return ((x + 1) * runs - 1) / total; };
    const int pieces = (int)(total >= runs ? run_of(last - 1) - r + 1 : it.units);
    const size_t floats = part_floats(ROWS, p.D);
    auto part_of = [&](int i) {
        const long long run = total >= runs ? r + i : run_of(first + i);
        return p.part + (2 * run + (i == 0 ? 1 : 0)) * floats;
    };
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    for (int k = 0; k < kRowsPer / kJoinWarps; ++k) {
        const int row = (int)blockIdx.y * kRowsPer + k * kJoinWarps + warp;
        if (row >= it.rows) continue;
        float top = -INFINITY;
        for (int i = lane; i < pieces; i += 32) top = fmaxf(top, part_of(i)[(size_t)ROWS * p.D + row]);
        for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
        float sum = 0.0f;
        float acc[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) acc[e] = 0.0f;
#pragma unroll 4
        for (int i = 0; i < pieces; ++i) {
            const float* part = part_of(i);
            const float m = part[(size_t)ROWS * p.D + row], l = part[(size_t)ROWS * p.D + ROWS + row];
            const float f = m > -INFINITY ? exp2f(m - top) : 1.0f;  // (1: zeros, or NaN)
            sum = fmaf(l, f, sum);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int d = 4 * lane + 128 * h;
                if (d < p.D) {
                    const float4 v = *reinterpret_cast<const float4*>(part + (size_t)row * p.D + d);
                    acc[4 * h] = fmaf(v.x, f, acc[4 * h]);
                    acc[4 * h + 1] = fmaf(v.y, f, acc[4 * h + 1]);
                    acc[4 * h + 2] = fmaf(v.z, f, acc[4 * h + 2]);
                    acc[4 * h + 3] = fmaf(v.w, f, acc[4 * h + 3]);
                }
            }
        }
        const int64_t flat = (int64_t)plan.item * ROWS + row, t = flat / p.G;
        const int head = plan.head * p.G + (int)(flat - t * p.G);
        const int64_t at = (q.q0 + t) * p.o_token + head * p.o_head;
        const float f = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int d = 4 * lane + 128 * h + e;
                if (d >= p.D) continue;
                const float v = acc[4 * h + e] * f;
                if (p.y_dtype == NXQ_F32)
                    static_cast<float*>(p.out)[at + d] = v;
                else if (p.y_dtype == NXQ_BF16)
                    static_cast<__nv_bfloat16*>(p.out)[at + d] = __float2bfloat16_rn(v);
                else
                    static_cast<__half*>(p.out)[at + d] = __float2half_rn(v);
            }
        if (p.lse && lane == 0)
            p.lse[(q.q0 + t) * ((int64_t)p.Hk * p.G) + head] = sum == 0.0f ? -INFINITY : (top + log2f(sum)) * 0.6931471805599453f;
    }
}

template <int ROWS, int KEYS>
cudaError_t join(const AttnParams& p, unsigned runs, cudaStream_t st) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(runs, (ROWS + kRowsPer - 1) / kRowsPer);
    cfg.blockDim = dim3(kJoinThreads);
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    note_launches(1);
    return cudaLaunchKernelEx(&cfg, attn_join_kernel<ROWS, KEYS>, p, (int)runs);
}

int attend(const nxq_kv_cache* cache, const nxq_kv_batch* batch, const nxq_heads* q, int64_t T, float scale, int64_t window,
           int64_t sinks, int64_t max_new, const nxq_heads* out, int y_dtype, float* lse, cudaStream_t st) {
    AttnParams p{};
    p.b = make_batch(cache, batch, T);
    p.q = q->dev;
    p.k = cache->k_dev;
    p.v = cache->v_dev;
    p.out = out->dev;
    p.lse = lse;
    p.q_token = q->token_stride, p.q_head = q->head_stride;
    p.o_token = out->token_stride, p.o_head = out->head_stride;
    p.page_stride = cache->page_stride, p.head_stride = cache->head_stride, p.slot_stride = cache->slot_stride;
    p.Hk = cache->heads, p.G = q->heads / cache->heads, p.D = cache->head_dim;
    p.y_dtype = y_dtype;
    p.q_vec = (uintptr_t)q->dev % 16 == 0 && q->token_stride % 8 == 0 && q->head_stride % 8 == 0;
    p.o_vec = (uintptr_t)out->dev % 16 == 0 && out->token_stride % 8 == 0 && out->head_stride % 8 == 0;
    p.page_shift = -1;
    for (int i = 0; i < 31; ++i)
        if (cache->page_size == 1 << i) p.page_shift = i;
    p.c = scale * 1.4426950408889634f;
    // No position reaches kMaxTokens, so a window of that size hides nothing.
    p.window = window < kMaxTokens ? (int)window : 0;
    p.sinks = (int)(sinks < kMaxTokens ? sinks : kMaxTokens);
    p.max_new = (int)(max_new && max_new < T ? max_new : T);
    p.status = context_status();
    p.rows_lo = 0;
    p.rows_hi = INT64_MAX;
    p.first = 1;
    // Sequences of up to kFewRows rows per key head go to the kernel that streams the cache, those
    // with more to the tcgen05 kernel, each by a launch that leaves the others out; only
    // one launch where the host can tell (a sequence alone has T rows in all but odd cases, and
    // the tcgen05 kernel takes any number).
    const int64_t most = (int64_t)p.max_new * p.G;
    const bool tc = most > kFewRows && attn_tc_supported(cache);
    const bool few = !tc || p.b.S > 1;
    const int rows = attn_mma_rows(p.D, tc ? kFewRows : most);
    const unsigned runs = attn_mma_grid(p.D);
    size_t floats = few ? 2 * runs * part_floats(rows, p.D) : 0;
    if (tc && 2 * attn_tc_grid() * part_floats(attn_tc_rows(), p.D) > floats)
        floats = 2 * attn_tc_grid() * part_floats(attn_tc_rows(), p.D);
    cudaError_t e = cudaMallocAsync((void**)&p.part, floats * sizeof(float), st);
    if (e != cudaSuccess) return cuda_fail(e, "cudaMallocAsync (attention workspace)");
    int rc = NXQ_OK;
    if (few) {
        if (tc) p.rows_hi = kFewRows;
        rc = attn_mma(p, cache->dtype, rows, st);
        p.rows_lo = tc ? kFewRows : 0;
        p.rows_hi = INT64_MAX;
        p.first = 0;
    }
    if (tc && rc == NXQ_OK) rc = attn_tc(p, cache, st);
    cudaFreeAsync(p.part, st);
    return rc;
}

}  // namespace

cudaError_t launch_attn_join(const AttnParams& p, int rows, int keys, unsigned runs, cudaStream_t st) {
    if (rows == 16 && keys == 64) return join<16, 64>(p, runs, st);
    if (rows == 32 && keys == 64) return join<32, 64>(p, runs, st);
    if (rows == 256 && keys == 128) return join<256, 128>(p, runs, st);
    return cudaErrorInvalidValue;
}

}  // namespace nxq

using namespace nxq;

extern "C" {

NXQ_API int nxq_paged_attention(const nxq_kv_cache* cache, const nxq_kv_batch* batch, const nxq_heads* q, int64_t T,
                                float scale, int64_t window, int64_t sinks, int64_t max_new, const nxq_heads* out,
                                int y_dtype, float* lse_dev, void* stream) {
    int rc;
    if ((rc = check_cache(cache)) || (rc = check_batch(batch, T))) return rc;
    if (!dtype_valid(y_dtype)) return fail(NXQ_ERR_ARG, "bad dtype");
    if (!(scale > 0.0f) || !std::isfinite(scale)) return fail(NXQ_ERR_ARG, "a scale of %g (finite, above zero)", scale);
    if (window < 0 || sinks < 0 || max_new < 0)
        return fail(NXQ_ERR_ARG, "window %lld, sinks %lld, max_new %lld", (long long)window, (long long)sinks, (long long)max_new);
    if (T == 0) return NXQ_OK;
    if ((rc = check_heads("queries", q, cache->dtype)) || (rc = check_heads("output", out, y_dtype))) return rc;
    if (q->heads % cache->heads || q->heads != out->heads)
        return fail(NXQ_ERR_SHAPE, "%d query heads and %d output heads for %d key heads", q->heads, out->heads, cache->heads);
    if (T * (q->heads / cache->heads) > (int64_t)1 << 34)
        return fail(NXQ_ERR_SHAPE, "%lld rows of %d query heads per key head", (long long)T, q->heads / cache->heads);
    if (!aligned_4(lse_dev)) return fail(NXQ_ERR_ARG, "lse is not aligned to its type");
    if ((rc = context_ready())) return rc;
    return attend(cache, batch, q, T, scale, window, sinks, max_new, out, y_dtype, lse_dev, (cudaStream_t)stream);
}

}  // extern "C"
