// Token embedding from a registered table: y[t] = scale * decode(W[ids[t]]).
//
// The table stays in its packed form; a row is decoded with the exact fp32
// decoder (formats.cuh, decode8), so a looked-up value is bit for bit the one
// nxq_dequant gives, times `scale` in fp32, rounded once to the output type.
//
// One thread decodes 8 consecutive elements (one decode8 call, up to three
// block fields and at most 32 code bytes) and stores them with 16-byte
// stores; a CTA takes a run of one token's row, so its index is one broadcast load.
#include "nxq_internal.h"

#include <cuda_bf16.h>

namespace nxq {

namespace {

constexpr int kEmbThreads = 128;

__device__ __forceinline__ uint32_t pack_half(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}

// grid = T * segs CTAs (walked with a stride), segs = CTAs per row.
template <int TYPE>
__global__ void __launch_bounds__(kEmbThreads) embedding_kernel(const uint8_t* __restrict__ tiled, TiledShape s,
                                                                const void* __restrict__ ids, int ids_type, int64_t T,
                                                                int segs, float scale, void* __restrict__ y, int y_dtype,
                                                                DeviceStatus* status) {
    for (int64_t b = blockIdx.x; b < T * segs; b += gridDim.x) {
        const int64_t t = b / segs;
        const int64_t k = ((b - t * segs) * kEmbThreads + threadIdx.x) * 8;
        if (k >= s.K) continue;
        const int64_t id = ids_type == NXQ_I64 ? static_cast<const int64_t*>(ids)[t]
                                               : (int64_t)static_cast<const int32_t*>(ids)[t];
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
        const int64_t o = t * s.K + k;
        if (y_dtype == NXQ_F32) {
            float4* p = reinterpret_cast<float4*>(static_cast<float*>(y) + o);
            p[0] = make_float4(v[0], v[1], v[2], v[3]);
            p[1] = make_float4(v[4], v[5], v[6], v[7]);
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
    const int segs = (int)((s.K / 8 + kEmbThreads - 1) / kEmbThreads);
    int64_t grid = T * segs;
    if (grid > (1 << 30)) grid = 1 << 30;
    switch (s.type) {
#define NXQ_EMB_CASE(TY)                                                                                              \
    case TY:                                                                                                          \
        embedding_kernel<TY><<<(unsigned)grid, kEmbThreads, 0, st>>>(tiled, s, ids, ids_type, T, segs, scale, y,      \
                                                                     y_dtype, context_status());                      \
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
        default: return cudaErrorInvalidValue;
    }
    note_launches(1);
    return cudaGetLastError();
}

}  // namespace nxq
