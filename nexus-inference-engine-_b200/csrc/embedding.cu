// Token embedding from a registered table: y[t] = scale * decode(W[ids[t]]).
//
// The table stays in its packed form; a row is decoded by the exact fp32
// arithmetic of formats.cuh (decode8), so a looked-up value is the one
// nxq_dequant gives bit for bit (NaN payloads aside), times `scale` in fp32,
// rounded once to the output type.
//
// One thread decodes 16 consecutive elements, which share one scale in every
// format, from whole code words (decode16), and stores them in accesses of 32
// or 16 bytes.  (Two decode8 calls instead, with their byte-wise addressing,
// took 430 instructions and 39 us for 8192 rows of 4096; now 30.5 us for 153 MB.
// Q2_K, Q3_K and the NXF chunk types still take decode8.)
// A resident grid walks all (token, 16 elements) items; the id of the item after
// next and the record of the next are on their way to the L2 cache meanwhile,
// since a row's records lie 256 elements x 128 rows apart and each is a short
// read of its own.
#include "nxq_internal.h"

#include <cuda_bf16.h>

namespace nxq {

namespace {

constexpr int kEmbThreads = 256, kEmbElems = 16;

__device__ __forceinline__ uint32_t pack_half(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}

__device__ __forceinline__ float half_at(uint32_t bits) { return __half2float(__ushort_as_half((unsigned short)bits)); }

// Elements e0 .. e0 + 15 (e0 a multiple of 16) of row r of a tile-chunk, in
// decode8's operations and order.
template <int TYPE>
__device__ __forceinline__ void decode16(const uint8_t* chunk, int r, int e0, float (&v)[kEmbElems]) {
    const int g = e0 >> 5, half = (e0 >> 4) & 1;  // 32-element group, and which 16 of it
    // Code i of a word of eight in the 4-bit order (q4_code_pos).
    auto nib = [](uint32_t w, int i) { return (int)((w >> (4 * (i >> 1) + 16 * (i & 1))) & 15u); };
    if constexpr (TYPE == T_Q4_K || TYPE == T_Q5_K) {
        const uint8_t* rec = chunk + r * (TYPE == T_Q4_K ? 144 : 176);
        const uint4 hd = *reinterpret_cast<const uint4*>(rec);
        const uint2 q = *reinterpret_cast<const uint2*>(rec + 16 + 16 * g + 8 * half);
        uint32_t h = 0u;
        if constexpr (TYPE == T_Q5_K) h = *reinterpret_cast<const uint32_t*>(rec + 144 + 4 * g) >> (2 * half);
        const uint32_t sb = (g < 4 ? hd.y : hd.z) >> (8 * (g & 3)), eb = hd.w >> (8 * (g & 3));
        const uint32_t sc = sb & 63u, mn = ((sb >> 6) & 3u) | ((g < 4 ? eb & 15u : (eb >> 4) & 15u) << 2);
        const float ds = __fmul_rn(half_at(hd.x), (float)sc), dm = __fmul_rn(half_at(hd.x >> 16), (float)mn);
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            int c = nib(i < 8 ? q.x : q.y, i & 7);
            if constexpr (TYPE == T_Q5_K)  // bit (4 + 4k + 16s) mod 32, + 1 for the second word
                c |= (int)((h >> (((4 + 4 * ((i & 7) >> 1) + 16 * (i & 1)) & 31) + (i >> 3))) & 1u) << 4;
            v[i] = __fsub_rn(__fmul_rn(ds, (float)c), dm);
        }
    } else if constexpr (TYPE == T_Q4_0 || TYPE == T_Q4_1 || is_i4g(TYPE)) {
        constexpr int kRec = TYPE == T_Q4_0 ? 144 : TYPE == T_Q4_1 ? 160 : i4g_hdr(TYPE) + CHUNK_K / 2;
        constexpr int kHdr = TYPE == T_Q4_0 ? 16 : TYPE == T_Q4_1 ? 32 : i4g_hdr(TYPE);
        const uint8_t* rec = chunk + r * kRec;
        const uint2 q = *reinterpret_cast<const uint2*>(rec + kHdr + 16 * g + 8 * half);
        float a, b = 0.0f;
        if constexpr (TYPE == T_Q4_0) {
            a = half_at(rd16(rec + 2 * g));
        } else if constexpr (TYPE == T_Q4_1) {
            const uint32_t dm = *reinterpret_cast<const uint32_t*>(rec + 4 * g);
            a = half_at(dm), b = half_at(dm >> 16);
        } else {
            const float2 sz = *reinterpret_cast<const float2*>(rec + 8 * (e0 / i4g_gs(TYPE)));
            a = sz.x, b = sz.y;
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const int c = nib(i < 8 ? q.x : q.y, i & 7);
            v[i] = TYPE == T_Q4_0   ? __fmul_rn((float)(c - 8), a)
                   : TYPE == T_Q4_1 ? __fadd_rn(__fmul_rn((float)c, a), b)
                                    : __fmul_rn(__fsub_rn((float)c, b), a);
        }
    } else if constexpr (TYPE == T_Q8_0) {
        const uint8_t* rec = chunk + r * 272;
        const uint4 q = *reinterpret_cast<const uint4*>(rec + 16 + e0);
        const float d = half_at(rd16(rec + 2 * g));
        const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
        for (int i = 0; i < 16; ++i) v[i] = __fmul_rn((float)(int8_t)(w[i >> 2] >> (8 * (i & 3))), d);
    } else if constexpr (TYPE == T_Q6_K) {
        const uint8_t* rec = chunk + r * 192 + 24 * g;
        const uint2 l = *reinterpret_cast<const uint2*>(rec + 8 * half);
        const uint32_t h = *reinterpret_cast<const uint32_t*>(rec + 16 + 4 * half);
        const float d = half_at(rd16(chunk + TILE_ROWS * 208 + r * 2));
        const float ds = __fmul_rn(d, (float)*(const int8_t*)(chunk + TILE_ROWS * 192 + r * 16 + (e0 >> 4)));
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const int c = nib(i < 8 ? l.x : l.y, i & 7) |
                          (int)((h >> (((4 + 4 * ((i & 7) >> 1) + 16 * (i & 1)) & 31) + 2 * (i >> 3))) & 3u) << 4;
            v[i] = __fmul_rn(ds, __fsub_rn((float)c, 32.0f));
        }
    } else {
        decode8(TYPE, chunk, r, e0, v);
        decode8(TYPE, chunk, r, e0 + 8, v + 8);
    }
}

// Items are (token, kEmbElems elements); every block holds a multiple of 32 elements.
template <int TYPE>
__global__ void __launch_bounds__(kEmbThreads) embedding_kernel(const uint8_t* __restrict__ tiled, TiledShape s,
                                                                const void* ids, int ids_type, int64_t T,
                                                                float scale, void* y, int y_dtype, int wide,
                                                                DeviceStatus* status) {
    overlap_begin();
    constexpr int kPerChunk = CHUNK_K / kEmbElems;
    const uint32_t per = (uint32_t)(s.K / kEmbElems);  // items of a token
    const int64_t total = T * per, step = (int64_t)gridDim.x * kEmbThreads;
    const int64_t dt = step / per;
    const uint32_t dj = (uint32_t)(step - dt * per);  // one step in tokens and items
    const uint64_t tile_bytes = (uint64_t)s.chunks * (uint64_t)s.tile_chunk_bytes;
    const uint32_t chunk_bytes = (uint32_t)s.tile_chunk_bytes;
    auto advance = [&](int64_t& t, uint32_t& j) {
        t += dt;
        j += dj;
        if (j >= per) {
            j -= per;
            ++t;
        }
    };
    auto id_of = [&](int64_t t) {
        return ids_type == NXQ_I64 ? static_cast<const int64_t*>(ids)[t] : (int64_t)static_cast<const int32_t*>(ids)[t];
    };
    // The tile-chunk of item j of row id (null: no such row).
    auto chunk_of = [&](int64_t id, uint32_t j) -> const uint8_t* {
        if ((uint64_t)id >= (uint64_t)s.N) return nullptr;
        return tiled + ((uint64_t)id / TILE_ROWS) * tile_bytes + (uint64_t)(j / kPerChunk) * chunk_bytes;
    };
    const int64_t i0 = (int64_t)blockIdx.x * kEmbThreads + threadIdx.x;
    if (i0 >= total) return;
    int64_t t = i0 / per, t1;
    uint32_t j = (uint32_t)(i0 - t * per), j1;
    t1 = t, j1 = j;  // the next item
    advance(t1, j1);
    int64_t id = id_of(t), id1 = i0 + step < total ? id_of(t1) : -1;
    const uint8_t* chunk = chunk_of(id, j);
    for (int64_t i = i0; i < total; i += step) {
        int64_t t2 = t1;
        uint32_t j2 = j1;
        advance(t2, j2);
        const int64_t id2 = i + 2 * step < total ? id_of(t2) : -1;
        const uint8_t* const chunk1 = i + step < total ? chunk_of(id1, j1) : nullptr;
        if (chunk1)
            asm volatile("prefetch.global.L2 [%0];" ::"l"(chunk1 + ((uint32_t)id1 % TILE_ROWS) * s.g.crb +
                                                          (j1 % kPerChunk) * s.g.crb / kPerChunk));
        const int64_t o = t * s.K + (int64_t)j * kEmbElems;
        float v[kEmbElems];
        if (chunk) {
            const int row = (int)((uint32_t)id % TILE_ROWS), e0 = (int)(j % kPerChunk) * kEmbElems;
            decode16<TYPE>(chunk, row, e0, v);
#pragma unroll
            for (int m = 0; m < kEmbElems; ++m) v[m] = __fmul_rn(v[m], scale);
        } else {
            if (j == 0) raise_index(status, kIndexToken);
#pragma unroll
            for (int m = 0; m < kEmbElems; ++m) v[m] = 0.0f;
        }
        if (y_dtype == NXQ_F32) {
            float* p = static_cast<float*>(y) + o;
            if (wide) {
                store_f32x8(p, v);
                store_f32x8(p + 8, v + 8);
            } else {
#pragma unroll
                for (int m = 0; m < kEmbElems; m += 4)
                    *reinterpret_cast<float4*>(p + m) = make_float4(v[m], v[m + 1], v[m + 2], v[m + 3]);
            }
        } else {
            uint4* p = reinterpret_cast<uint4*>(static_cast<uint16_t*>(y) + o);
            uint32_t q[kEmbElems / 2];
#pragma unroll
            for (int m = 0; m < kEmbElems / 2; ++m)
                q[m] = y_dtype == NXQ_F16 ? pack_half(v[2 * m], v[2 * m + 1]) : pack_bf16(v[2 * m], v[2 * m + 1]);
            p[0] = make_uint4(q[0], q[1], q[2], q[3]);
            p[1] = make_uint4(q[4], q[5], q[6], q[7]);
        }
        t = t1, j = j1, id = id1, chunk = chunk1;
        t1 = t2, j1 = j2, id1 = id2;
    }
}

}  // namespace

cudaError_t launch_embedding(const uint8_t* tiled, const TiledShape& s, const void* ids, int ids_type, int64_t T,
                             float scale, void* y, int y_dtype, cudaStream_t st) {
    const int64_t want = (T * (s.K / kEmbElems) + kEmbThreads - 1) / kEmbThreads, most = (int64_t)context_sm_count() * 8;
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
