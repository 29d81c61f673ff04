// nxq_paged_attention: dispatch, and the kernel that joins partial results.
#include "attn_plan.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cmath>

namespace nxq {

namespace {

using namespace attn;

// Rows of a sequence and key head up to which the kernel that streams the cache is the
// quicker one: 24 sequences of 6 new tokens over 3000, 5 query heads per key head (30
// rows), take 75 us there and 98 on tcgen05, of 8 new tokens (40 rows) 126 and 98; 32 of
// one over 4000 with 32 heads over one 30.6 and 31.5.
constexpr int kFewRows = 32;
constexpr int kJoinThreads = 128, kJoinWarps = kJoinThreads / 32;

// Joins the pieces of items cut between runs.  CTA (c, g) takes the item that begins in run
// c and ends behind it, if there is one, and of that the rows PER g kJoinWarps ...: a warp per
// row, first the largest maximum over the pieces, then the sums of weights and outputs, in
// order of the runs whatever order they were written in.  Nothing but latency counts:
// a row of 128 elements is one load of a warp per piece, eight of them in flight, and a
// CTA has few rows (one item of 16 rows in 37 pieces: 88 us with 16 rows per CTA,
// 4.0 with 4).
template <int ROWS, int PER, bool BF16, int Y>
__global__ void __launch_bounds__(kJoinThreads) attn_join_kernel(const __grid_constant__ AttnParams p, const int runs) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int r = blockIdx.x;
    const int4* const note = reinterpret_cast<const int4*>(static_cast<const Cut*>(p.work) + r);
    const int4 n0 = note[0], n1 = note[1];
    const Cut cut{n0.x, n0.y, n0.z, n0.w, n1.x, n1.y, {0, 0}};
    if (cut.pieces == 0) return;
    const size_t floats = part_floats(ROWS, p.D);
    const float* const slots = reinterpret_cast<const float*>(static_cast<const uint8_t*>(p.work) + cuts_bytes(runs));
    // Piece 0 is in run r's slot 1, piece i in run r + i's slot 0.
    auto part_of = [&](int i) { return slots + (2 * (size_t)(r + i) + (i == 0 ? 1 : 0)) * floats; };
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    bool over = false;
#pragma unroll 1
    for (int k = 0; k < PER; ++k) {
        const int row = ((int)blockIdx.y * PER + k) * kJoinWarps + warp;
        if (row >= cut.rows) break;
        // Outputs of piece i, eight of them asked for at a time, the first before the maxima are known.
        auto outputs = [&](int i, float4 (&v)[2]) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                v[h] = make_float4(0, 0, 0, 0);
                if (i < cut.pieces && 4 * lane + 128 * h < p.D)
                    v[h] = *reinterpret_cast<const float4*>(part_of(i) + (size_t)row * p.D + 4 * lane + 128 * h);
            }
        };
        float4 v[8][2];
#pragma unroll
        for (int i = 0; i < 8; ++i) outputs(i, v[i]);
        // Lane i has the factor of piece i0 + i; more than 32 pieces are looked at again.
        float top = -INFINITY, mine = -INFINITY, sum = 0.0f;
        auto statistics = [&](int i, float& m, float& l) {
            m = -INFINITY, l = 0.0f;
            if (i < cut.pieces) m = part_of(i)[(size_t)ROWS * p.D + row], l = part_of(i)[(size_t)ROWS * p.D + ROWS + row];
        };
        float l0;
        statistics(lane, mine, l0);
        top = mine;
        for (int i = lane + 32; i < cut.pieces; i += 32) {
            float m, l;
            statistics(i, m, l);
            top = fmaxf(top, m);
        }
        for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
        float acc[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) acc[e] = 0.0f;
        for (int i0 = 0; i0 < cut.pieces; i0 += 32) {
            if (i0) statistics(i0 + lane, mine, l0);
            const float factor = mine > -INFINITY ? exp2f(mine - top) : 1.0f;  // (1: zeros, or NaN)
            float part = l0 * factor;
            for (int o = 16; o; o >>= 1) part += __shfl_xor_sync(0xFFFFFFFFu, part, o);
            sum += part;
            const int n = cut.pieces - i0 < 32 ? cut.pieces - i0 : 32;
            for (int j0 = 0; j0 < n; j0 += 8) {
                if (i0 + j0)
#pragma unroll
                    for (int j = 0; j < 8; ++j) outputs(i0 + j0 + j, v[j]);
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float f = __shfl_sync(0xFFFFFFFFu, factor, (j0 + j) & 31);
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        acc[4 * h] = fmaf(v[j][h].x, f, acc[4 * h]);
                        acc[4 * h + 1] = fmaf(v[j][h].y, f, acc[4 * h + 1]);
                        acc[4 * h + 2] = fmaf(v[j][h].z, f, acc[4 * h + 2]);
                        acc[4 * h + 3] = fmaf(v[j][h].w, f, acc[4 * h + 3]);
                    }
                }
            }
        }
        const int g = cut.r0 + row, t = (int)((unsigned)g / (unsigned)p.G), head = cut.head * p.G + (g - t * p.G);
        const int64_t token = (int64_t)cut.q0 + cut.t0 + t, at = token * p.o_token + head * p.o_head;
        const float f = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int d = 4 * lane + 128 * h + e;
                if (d >= p.D) continue;
                const float v = acc[4 * h + e] * f;
                if constexpr (Y == NXQ_F32)
                    static_cast<float*>(p.out)[at + d] = v;
                else if constexpr (Y == NXQ_BF16)
                    static_cast<__nv_bfloat16*>(p.out)[at + d] = __float2bfloat16_rn(v);
                else
                    static_cast<__half*>(p.out)[at + d] = __float2half_rn(for_f16<BF16>(v, over));
            }
        if (p.lse && lane == 0)
            p.lse[token * ((int64_t)p.Hk * p.G) + head] = sum == 0.0f ? -INFINITY : (top + log2f(sum)) * 0.6931471805599453f;
    }
    if (Y == NXQ_F16 && BF16 && over) raise_range(p.status, kRangeAttn);
}

template <int ROWS, int PER>
cudaError_t join(const AttnParams& p, unsigned runs, cudaStream_t st) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(runs, ROWS / (PER * kJoinWarps));
    cfg.blockDim = dim3(kJoinThreads);
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    note_launches(1);
    // (Only f16 outputs depend on the cache's type.)
    auto* kernel = p.y_dtype == NXQ_F32    ? attn_join_kernel<ROWS, PER, false, NXQ_F32>
                   : p.y_dtype == NXQ_BF16 ? attn_join_kernel<ROWS, PER, false, NXQ_BF16>
                   : p.bf16                ? attn_join_kernel<ROWS, PER, true, NXQ_F16>
                                           : attn_join_kernel<ROWS, PER, false, NXQ_F16>;
    return cudaLaunchKernelEx(&cfg, kernel, p, (int)runs);
}

size_t work_bytes(unsigned runs, int rows, int D) { return cuts_bytes(runs) + 2 * runs * part_floats(rows, D) * sizeof(float); }

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
    p.bf16 = cache->dtype == NXQ_BF16;
    p.q_vec = (uintptr_t)q->dev % 16 == 0 && q->token_stride % 8 == 0 && q->head_stride % 8 == 0;
    const uintptr_t o_bits = (uintptr_t)out->dev |
                             (uintptr_t)(out->token_stride | out->head_stride) * (y_dtype == NXQ_F32 ? 4 : 2);
    p.o_vec = o_bits % 32 == 0 ? 2 : o_bits % 16 == 0 ? 1 : 0;
    p.page_shift = -1;
    for (int i = 0; i < 31; ++i)
        if (cache->page_size == 1 << i) p.page_shift = i;
    p.page_align = cache->page_size & -cache->page_size;
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
    // with more to the tcgen05 kernel, each by a launch that leaves the others out.  Where the
    // average is above kFewRows the tcgen05 kernel takes them all.  What that gives depends on
    // the histories, which the host does not know (32 heads over 8 of 128; all on tcgen05, then
    // both): 64 single tokens over 1000 beside a chunk of 512 105 and 123 us, 32 over 4000 beside
    // 2048 232 and 235, but 32 over 4000 beside 512 171 and 160, 64 over 4000 beside 600 304 and 259;
    // on the other side of the rule, 64 over 4000 beside 128 297 and 235, 128 over 2000 beside 256
    // 299 and 246.
    const int64_t most = (int64_t)p.max_new * p.G;
    const bool tc = most > kFewRows && attn_tc_supported(cache);
    const bool few = !tc || T * p.G <= (int64_t)kFewRows * p.b.S;
    const int rows = attn_mma_rows(p.D, tc ? kFewRows : most);
    const unsigned runs = attn_mma_grid(p.D);
    size_t bytes = few ? work_bytes(runs, rows, p.D) : 0;
    if (tc) {
        const size_t b = work_bytes(attn_tc_grid(), attn_tc_rows(), p.D) + attn_tc_grid() * (size_t)attn_tc_rows() * p.D * sizeof(float);
        if (b > bytes) bytes = b;
    }
    cudaError_t e = cudaMallocAsync(&p.work, bytes, st);
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
    cudaFreeAsync(p.work, st);
    return rc;
}

}  // namespace

cudaError_t launch_attn_join(const AttnParams& p, int rows, unsigned runs, cudaStream_t st) {
    if (rows == 16) return join<16, 1>(p, runs, st);
    if (rows == 32) return join<32, 1>(p, runs, st);
    if (rows == 256) return join<256, 2>(p, runs, st);
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
    if (!(scale > 0.0f) || !std::isfinite(scale * 1.4426950408889634f)) return fail(NXQ_ERR_ARG, "a scale of %g (finite, above zero)", scale);
    if (window < 0 || sinks < 0 || max_new < 0)
        return fail(NXQ_ERR_ARG, "window %lld, sinks %lld, max_new %lld", (long long)window, (long long)sinks, (long long)max_new);
    if (T == 0) return NXQ_OK;
    if ((rc = check_heads("queries", q, cache->dtype)) || (rc = check_heads("output", out, y_dtype))) return rc;
    if (q->heads % cache->heads || q->heads != out->heads)
        return fail(NXQ_ERR_SHAPE, "%d query heads and %d output heads for %d key heads", q->heads, out->heads, cache->heads);
    if (q->dev == out->dev && (y_dtype != cache->dtype || (T > 1 && q->token_stride != out->token_stride) ||
                               (q->heads > 1 && q->head_stride != out->head_stride)))
        return fail(NXQ_ERR_ARG, "in place with another type or other strides");
    if (T * (q->heads / cache->heads) > 0x7FFFFFFF)
        return fail(NXQ_ERR_SHAPE, "%lld rows of %d query heads per key head", (long long)T, q->heads / cache->heads);
    if (!aligned_4(lse_dev)) return fail(NXQ_ERR_ARG, "lse is not aligned to its type");
    if ((rc = context_ready())) return rc;
    return attend(cache, batch, q, T, scale, window, sinks, max_new, out, y_dtype, lse_dev, (cudaStream_t)stream);
}

}  // extern "C"
