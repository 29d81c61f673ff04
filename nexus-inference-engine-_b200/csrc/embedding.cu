// Token embedding from a registered table: y[t] = scale * decode(W[ids[t]]).
//
// The table stays in its packed form; a row is decoded with the exact fp32
// decoder (formats.cuh, decode8), so a looked-up value is bit for bit the one
// nxq_dequant gives, times `scale` in fp32, rounded once to the output type.
//
// One thread decodes 8 consecutive elements (one decode8 call: the block's
// scale fields and one to three code words) and stores them with one access of
// 32 or 16 bytes; a warp so covers one chunk of a row.  A resident grid walks all
// (token, 8 elements) items with the next item's id in flight: bound by the
// output it writes.  (One CTA per 1024 elements instead, 32768 of them for 8192
// rows of 4096, was bound by starting CTAs: 45 us.)
#include "nxq_internal.h"

#include <cuda_bf16.h>

namespace nxq {

namespace {

constexpr int kEmbThreads = 256;

__device__ __forceinline__ uint32_t pack_half(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}

// Items are (token, 8 elements), K / 8 to a token.
template <int TYPE>
__global__ void __launch_bounds__(kEmbThreads) embedding_kernel(const uint8_t* __restrict__ tiled, TiledShape s,
                                                                const void* __restrict__ ids, int ids_type, int64_t T,
                                                                float scale, void* __restrict__ y, int y_dtype, int wide,
                                                                DeviceStatus* status) {
    overlap_begin();
    const int64_t per = s.K / 8, total = T * per, step = (int64_t)gridDim.x * kEmbThreads;
    const int64_t dt = step / per, dk = step - dt * per;  // one step in tokens and items
    auto id_of = [&](int64_t t) {
        return ids_type == NXQ_I64 ? static_cast<const int64_t*>(ids)[t] : (int64_t)static_cast<const int32_t*>(ids)[t];
    };
    int64_t i = (int64_t)blockIdx.x * kEmbThreads + threadIdx.x;
    int64_t t = i / per, j = i - t * per;
    int64_t next_id = i < total ? id_of(t) : 0;
    for (; i < total; i += step) {
        const int64_t id = next_id, k = j * 8, o = t * s.K + k;
        t += dt;
        j += dk;
        if (j >= per) {
            j -= per;
            ++t;
        }
        if (i + step < total) next_id = id_of(t);
        float v[8];
        if (id >= 0 && id < s.N) {
            decode8(TYPE, tiled + s.chunk_offset(id / TILE_ROWS, k / CHUNK_K), (int)(id % TILE_ROWS), (int)(k % CHUNK_K), v);
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = __fmul_rn(v[i], scale);
        } else {
            if (k == 0) raise_index(status, kIndexToken);
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = 0.0f;
        }
        if (y_dtype == NXQ_F32) {
            float4* p = reinterpret_cast<float4*>(static_cast<float*>(y) + o);
            if (wide) {
                store_f32x8(static_cast<float*>(y) + o, v);
            } else {
                p[0] = make_float4(v[0], v[1], v[2], v[3]);
                p[1] = make_float4(v[4], v[5], v[6], v[7]);
            }
        } else if (y_dtype == NXQ_F16) {
            *reinterpret_cast<uint4*>(static_cast<__half*>(y) + o) =
                make_uint4(pack_half(v[0], v[1]), pack_half(v[2], v[3]), pack_half(v[4], v[5]), pack_half(v[6], v[7]));
        } else {
            *reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(y) + o) =
                make_uint4(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]), pack_bf16(v[4], v[5]), pack_bf16(v[6], v[7]));
        }
    }
}

}  // namespace

cudaError_t launch_embedding(const uint8_t* tiled, const TiledShape& s, const void* ids, int ids_type, int64_t T,
                             float scale, void* y, int y_dtype, cudaStream_t st) {
    const int64_t want = (T * (s.K / 8) + kEmbThreads - 1) / kEmbThreads, most = (int64_t)context_sm_count() * 8;
    const unsigned grid = (unsigned)(want < most ? want : most);
    const int wide = (uintptr_t)y % 32 == 0;  // rows are multiples of 64 bytes
    cudaError_t e = cudaErrorInvalidValue;
    switch (s.type) {
#define NXQ_EMB_CASE(TY)                                                                                            \
    case TY:                                                                                                        \
        e = launch_overlapped(embedding_kernel<TY>, grid, kEmbThreads, 0, st, tiled, s, ids, ids_type, T, scale, y, \
                              y_dtype, wide, context_status());                                                     \
        break;
        NXQ_EMB_CASE(T_Q4_0)
        NXQ_EMB_CASE(T_Q4_1)
        NXQ_EMB_CASE(T_Q8_0)
        NXQ_EMB_CASE(T_Q2_K)
        NXQ_EMB_CASE(T_Q3_K)
        NXQ_EMB_CASE(T_Q4_K)
        NXQ_EMB_CASE(T_Q5_K)
        NXQ_EMB_CASE(T_Q6_K)
        NXQ_EMB_CASE(T_I4G32)
        NXQ_EMB_CASE(T_I4G64)
        NXQ_EMB_CASE(T_I4G128)
        NXQ_EMB_CASE(T_I4G256)
        NXQ_EMB_CASE(T_NXF_I8)
        NXQ_EMB_CASE(T_NXF_F16)
        NXQ_EMB_CASE(T_NXF_F32)
#undef NXQ_EMB_CASE
        default: return e;
    }
    note_launches(1);
    return e;
}

}  // namespace nxq
