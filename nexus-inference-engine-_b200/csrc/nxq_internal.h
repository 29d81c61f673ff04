// Internal declarations shared by the C-ABI layer and the kernel files.
#pragma once
#include <cuda_runtime.h>

#include <cstdarg>
#include <cstddef>
#include <cstdint>

#include "../../include/nxq.h"
#include "formats.cuh"

namespace nxq {

// A registered, HBM-resident weight (the nxq_weight_t handle).
struct Weight {
    uint32_t magic;       // kWeightMagic while live; guards stale handles
    int device;
    TiledShape shape;
    uint8_t* dev = nullptr;   // tiled copy (shape.total_bytes() + kTailPad)
    size_t dev_bytes = 0;
    size_t packed_bytes = 0;  // N * K/QK * block_bytes (the algorithmic bytes)
    int tables = 0;           // live expert tables that refer to it
};
constexpr uint32_t kWeightMagic = 0x4E58514Bu;  // "NXQK"
constexpr size_t kTailPad = 256;                 // slack after the last tile-chunk

// Records `msg` as the calling thread's last error and returns `status`.
int fail(int status, const char* fmt, ...);
// Maps a CUDA error to NXQ_ERR_CUDA with the call site in the message.
int cuda_fail(cudaError_t e, const char* what);

#define NXQ_CUDA(call)                                          \
    do {                                                        \
        cudaError_t e_ = (call);                                \
        if (e_ != cudaSuccess) return ::nxq::cuda_fail(e_, #call); \
    } while (0)

// Device-side error word of the context: 0 = ok, else the first error a
// kernel raised (kStatusTimeout: a bounded wait ran out; kStatusRange: a
// finite activation was too large for f16; kStatusIndex: an index in device
// memory lay outside its range).  `where` says which wait or
// conversion.  Read by the host after a synchronize (nxq_stream_sync,
// nxq_qmatmul_host).
// The same device allocation also holds the settings kernels read on their
// slow paths: the limit of a bounded wait on another CTA's progress (in SM
// clock cycles; nxq_set_wait_limit) and test hooks (nxq_test_hook).  Drain
// waits (letting a CTA's own copies land before it exits) always use the
// fixed kDrainWaitCycles.
// host_flag is a word of mapped pinned host memory that a kernel raising an
// error also sets, so a host call learns of an error without a device read.
struct DeviceStatus {
    unsigned int code;
    unsigned int where;
    long long wait_cycles;
    unsigned int hooks;  // kHook* bits
    unsigned int pad;
    unsigned int* host_flag;
};
constexpr unsigned kStatusTimeout = 1u;
constexpr unsigned kStatusRange = 2u;
constexpr unsigned kStatusIndex = 3u;
constexpr long long kDefaultWaitCycles = 4000000000LL;  // ~2 s at 2 GHz
constexpr long long kDrainWaitCycles = 4000000000LL;
// Test hook: CTAs of a stream-K launch that publish a partial sum for a tile
// another CTA finishes do not count themselves in, so that CTA's bounded wait
// for the counts runs out (a lost arrival, made on purpose and bounded).
constexpr unsigned kHookStreamKSkipCount = 1u;

// True when a finite v rounds to an infinite f16 (|v| >= 65520): the
// tensor-core kernels compute in f16, so such an activation would turn a
// finite result into inf or NaN.
__device__ __forceinline__ bool f16_overflows(float v) {
    const float a = fabsf(v);
    return a >= 65520.0f && a <= 3.402823466e38f;
}
// Sets the host-visible error flag (mapped pinned memory, written over the bus).
__device__ __forceinline__ void raise_host_flag(DeviceStatus* st) {
    unsigned int* f = st->host_flag;
    if (f) {
        *reinterpret_cast<volatile unsigned int*>(f) = 1u;
        __threadfence_system();
    }
}
// Records a range error (first error wins; `where` names the conversion).
constexpr unsigned kRangeAttn = 5u;
__device__ __forceinline__ void raise_range(DeviceStatus* st, unsigned where) {
    if (st && atomicCAS(&st->code, 0u, kStatusRange) == 0u) {
        st->where = where;
        raise_host_flag(st);
    }
}

// Records an index error (first error wins; `where`: kIndex*).
constexpr unsigned kIndexToken = 1u, kIndexOffset = 2u, kIndexRow = 3u, kIndexSlot = 4u, kIndexSeq = 5u, kIndexPage = 6u,
                   kIndexPosition = 7u;
__device__ __forceinline__ void raise_index(DeviceStatus* st, unsigned where) {
    if (st && atomicCAS(&st->code, 0u, kStatusIndex) == 0u) {
        st->where = where;
        raise_host_flag(st);
    }
}

// The context's device status word and SM count (nxq_api.cu).
DeviceStatus* context_status();
// NXQ_OK once nxq_init has run, with the context's device made current on the
// calling thread; else the status (and message) the C ABI returns.
int context_ready();
int context_sm_count();

// NXQ_OK and the weight behind a live handle, else the status the C ABI returns.
int check_weight(nxq_weight_t h, Weight** out);
// Adds `delta` references of expert tables to the weight behind a live handle and
// gives the weight: with a reference held, nxq_weight_release refuses it.
int weight_table_ref(nxq_weight_t h, int delta, Weight** out = nullptr);
// Releases every expert table (nxq_shutdown; the weights go after it).
void experts_shutdown();

#ifdef __CUDACC__
// Launch with programmatic stream serialization: the kernel may start while the
// one before it on the stream drains, and must run griddepcontrol.wait before
// it touches memory.  What that one may still be writing is not read-only for
// the life of this kernel: no __ldg on it and no const __restrict__ pointer to it
// (which allow loads by the non-coherent path, ahead of the wait).  Registered
// weights are complete before any call can name them and may have both.
template <typename... Params, typename... Args>
cudaError_t launch_overlapped(void (*kernel)(Params...), unsigned grid, unsigned block, size_t smem, cudaStream_t st,
                              const Args&... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(block);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, static_cast<Params>(args)...);
}
// First thing in such a kernel: lets the next one start, then waits for the one before.
__device__ __forceinline__ void overlap_begin() {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
}
// 32 consecutive bytes (32-byte aligned) in one access.
__device__ __forceinline__ void store_f32x8(float* p, const float* v) {
    asm volatile("st.global.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "f"(v[0]), "f"(v[1]), "f"(v[2]),
                 "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7])
                 : "memory");
}
__device__ __forceinline__ void load_f32x8(const float* p, float (&v)[8]) {
    asm volatile("ld.global.v8.f32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7])
                 : "l"(p)
                 : "memory");
}
#endif

inline bool dtype_valid(int d) { return d == NXQ_F32 || d == NXQ_F16 || d == NXQ_BF16; }
// Whether a device pointer (or null) lies on a multiple of its type's size: kernels
// access elements whole, and an access across that boundary is a fault.
inline bool aligned_as(const void* p, int dtype) { return (uintptr_t)p % (dtype == NXQ_F32 ? 4 : 2) == 0; }
inline bool aligned_4(const void* p) { return (uintptr_t)p % 4 == 0; }

// Process-wide count of kernels launched by the library (nxq_launch_count).
void note_launches(unsigned n);

// ---- kernel launchers (return cudaError_t of the launch) -------------------
cudaError_t launch_repack(const uint8_t* src, uint8_t* dst, const TiledShape& s,
                          int64_t row0, int64_t rows, int64_t blk0, int64_t src_row_blocks,
                          cudaStream_t st);
cudaError_t launch_dequant(const uint8_t* tiled, const TiledShape& s, float* y, cudaStream_t st);
// y[t] = scale * decode(row ids[t]) (embedding.cu).
cudaError_t launch_embedding(const uint8_t* tiled, const TiledShape& s, const void* ids, int ids_type, int64_t T,
                             float scale, void* y, int y_dtype, cudaStream_t st);

// CUDA-core fused dequant-GEMV/GEMM with exact fp32 decode; any M (chunked by 32).
// `partials` must hold splits * M * N floats when splits > 1.
cudaError_t launch_qmm_simt(const uint8_t* tiled, const TiledShape& s, const void* x, int x_dtype,
                            void* y, int y_dtype, int64_t M, float* partials, int splits,
                            cudaStream_t st);
int simt_pick_splits(const TiledShape& s, int64_t M, int sm_count);
// The CUDA-core kernel with its split-K partials in a fixed device array
// (no allocation); M * N must not exceed kNoAllocScratchFloats.
constexpr int64_t kNoAllocScratchFloats = 2 * 1024 * 1024;  // 8 MiB of fp32
int launch_qmm_simt_noalloc(const uint8_t* tiled, const TiledShape& s, const void* x, int x_dtype, void* y,
                            int y_dtype, int64_t M, int sm_count, cudaStream_t st);
int simt_rows_per_pass(int64_t M);
const char* type_name(int type);

}  // namespace nxq
