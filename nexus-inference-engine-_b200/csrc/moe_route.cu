// Top-k routing of a mixture of experts, and the weighted sum of its outputs
// (nxq_moe_route, nxq_moe_combine).  The reference routes on the host, token
// by token (MoERouter::route, moe_router.h:47); here the choices, their
// weights and their order by expert stay on the device.
//
// Routing has three steps.  (1) One warp per token: lane l holds the logits of
// experts l, l + 32, ... as order-preserving integer keys and knows its largest;
// k rounds of warp reductions (the largest key, then the lowest index that has it,
// so ties go to the lowest; 16-bit logits hold both in one word and need one)
// pick the choices; a lane keeps its two largest and looks again only when both
// are gone.  The block counts its choices
// of every expert.  (2) An exclusive scan of the counts over blocks, 32 experts
// per CTA.  (3) Every block ranks its own choices: a warp walks a contiguous run of
// choices in order, equal experts among 32 lanes ranked by their lane (match),
// so slots are ordered by (expert, token) and do not depend on timing - the
// counts are integers and no atomic decides a place.  Up to kSmallT tokens one
// CTA does all three.
#include "nxq_internal.h"
#include "sm100_ptx.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace nxq {

namespace {

constexpr int kMaxE = 1024, kMaxK = 32;
constexpr int kRankWarps = 8;        // contiguous runs a block's choices are ranked in
constexpr int kThreads = 32 * kRankWarps;
constexpr int kSmallThreads = 1024;
constexpr int kChooseThreads = 512;
// One CTA up to here: 2.6 us for 1 token, 6.2 for 32, 14.9 for 128 (256 experts, k = 8,
// in a graph), where the three kernels take 14.7.
constexpr int kSmallT = 128;
constexpr int kMaxBlocks = 256;      // of tokens
constexpr float kInf = __builtin_huge_valf();

struct RouteParams {
    const void* logits;
    int dtype;
    int64_t T;
    int E, k, normalize;
    int tb;  // tokens per block
    int blocks;
    int32_t* ids;
    float* weights;
    int32_t* offsets;
    int32_t* rows;
    int32_t* slots;
    int32_t* before;  // [blocks][E]: choices of the expert in the block, then in the blocks before it
    int32_t* total;   // [E]
};

// Larger value, larger key; -0 and +0 equal; 0 for -inf and NaN (never taken).
__device__ __forceinline__ uint32_t key_of(float v) {
    if (!(v > -kInf)) return 0u;
    const uint32_t u = __float_as_uint(v + 0.0f);
    return (u >> 31) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t key) {
    return __uint_as_float((key >> 31) ? (key & 0x7FFFFFFFu) : ~key);
}
// exp(v - m), with the limit for m = +inf.
__device__ __forceinline__ float share_of(float v, float m) { return m == kInf ? (v == kInf ? 1.0f : 0.0f) : expf(v - m); }

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
    return v;
}

// The V logits of type T that a lane holds, as keys of which the warp takes the
// largest again and again.  A 16-bit logit's key and its index fit into one word, so
// one reduction finds a choice; fp32 ones keep the two apart.  (bf16 logits
// that were widened and chosen like fp32 ones: 95 instead of 54 us for 2000
// tokens, 32 of 1024; 27 instead of 25 us for 16384 tokens, 8 of 256.)
template <typename T, int V>
struct Lanes {
    uint32_t key[V];          // 0: never taken
    uint32_t top, top2;       // the two largest behind the last choice,
    int at, at2, known;       // their experts, and how many of the two are left
    __device__ __forceinline__ void set(int i, int, float v) { key[i] = key_of(v); }
    // Looks for the two largest behind (last, last_at).
    __device__ __forceinline__ void look(uint32_t last, int last_at, int lane) {
        top = top2 = 0u;
        at = at2 = 0;
        known = 2;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const int e = lane + 32 * i;
            const uint32_t k = key[i] < last || (key[i] == last && e > last_at) ? key[i] : 0u;
            if (k > top) {
                top2 = top;
                at2 = at;
                top = k;
                at = e;
            } else if (k > top2) {
                top2 = k;
                at2 = e;
            }
        }
    }
    __device__ __forceinline__ void start(int lane) { look(0xFFFFFFFFu, -1, lane); }
    __device__ __forceinline__ uint32_t best() const { return __reduce_max_sync(0xFFFFFFFFu, top); }
    // The expert of the warp's best, which its lane gives up.
    __device__ __forceinline__ int take(uint32_t b, int lane) {
        const int e = (int)__reduce_min_sync(0xFFFFFFFFu, top == b ? (unsigned)at : 0x7FFFFFFFu);
        if (top == b && at == e) {
            if (--known) {
                top = top2;
                at = at2;
            } else {
                look(b, e, lane);
            }
        }
        return e;
    }
    __device__ __forceinline__ static float value(uint32_t b) { return value_of(b); }
    __device__ __forceinline__ float value_at(int i) const { return value_of(key[i]); }
};

template <int V>
struct Lanes16 {
    uint32_t key[V];  // ordered 16 bits of the logit, then 1023 - expert; 0: never taken
    uint32_t top, top2;
    int known;
    __device__ __forceinline__ void look(uint32_t last) {
        top = top2 = 0u;
        known = 2;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const uint32_t k = key[i] < last ? key[i] : 0u;
            top2 = max(top2, min(top, k));
            top = max(top, k);
        }
    }
    __device__ __forceinline__ void start(int) { look(0xFFFFFFFFu); }
    __device__ __forceinline__ uint32_t best() const { return __reduce_max_sync(0xFFFFFFFFu, top); }
    __device__ __forceinline__ int take(uint32_t b, int) {
        if (top == b) {
            if (--known)
                top = top2;
            else
                look(b);
        }
        return (int)(kMaxE - 1 - (b & 0xFFFFu));
    }
    // -0 counts as +0; -inf and NaN are never taken.
    __device__ __forceinline__ void set16(int i, int e, uint32_t u, uint32_t inf) {
        const uint32_t mag = u & 0x7FFFu;
        if (mag == 0u) u = 0u;
        const uint32_t ord = (u & 0x8000u) ? 0xFFFFu - u : u + 0x8000u;
        key[i] = mag > inf || u == (0x8000u | inf) ? 0u : (ord << 16) | (uint32_t)(kMaxE - 1 - e);
    }
    __device__ __forceinline__ static uint32_t bits(uint32_t b) {
        const uint32_t ord = b >> 16;
        return (ord & 0x8000u) ? ord - 0x8000u : 0xFFFFu - ord;
    }
};
template <int V>
struct Lanes<__half, V> : Lanes16<V> {
    __device__ __forceinline__ void set(int i, int e, __half v) { this->set16(i, e, __half_as_ushort(v), 0x7C00u); }
    __device__ __forceinline__ static float value(uint32_t b) {
        return __half2float(__ushort_as_half((unsigned short)Lanes16<V>::bits(b)));
    }
    __device__ __forceinline__ float value_at(int i) const { return value(this->key[i]); }
};
template <int V>
struct Lanes<__nv_bfloat16, V> : Lanes16<V> {
    __device__ __forceinline__ void set(int i, int e, __nv_bfloat16 v) { this->set16(i, e, __bfloat16_as_ushort(v), 0x7F80u); }
    __device__ __forceinline__ static float value(uint32_t b) { return __uint_as_float(Lanes16<V>::bits(b) << 16); }
    __device__ __forceinline__ float value_at(int i) const { return value(this->key[i]); }
};

template <typename T, int V>
__device__ __forceinline__ void read_logits(const RouteParams& p, int64_t t, int lane, T (&logit)[V]) {
    const T* row = static_cast<const T*>(p.logits) + t * p.E;
#pragma unroll
    for (int i = 0; i < V; ++i) logit[i] = lane + 32 * i < p.E ? row[lane + 32 * i] : T(-kInf);
}

// The choices of token t by one warp; lane j < k returns choice j (-1: none).
// logit: its logits as read_logits left them; they are replaced by token next's
// (none if < 0), whose loads so overlap the choosing.
template <typename T, int V>
__device__ __forceinline__ int choose(const RouteParams& p, int64_t t, int64_t next, int lane, T (&logit)[V]) {
    Lanes<T, V> l;
#pragma unroll
    for (int i = 0; i < V; ++i) l.set(i, lane + 32 * i, logit[i]);
    if (next >= 0) read_logits<T, V>(p, next, lane, logit);
    l.start(lane);
    uint32_t best = l.best();
    const float m = best ? l.value(best) : 0.0f;
    float all = 0.0f;  // sum over every expert
    if (!p.normalize && best) {
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (l.key[i]) all += share_of(l.value_at(i), m);
        all = warp_sum(all);
    }
    int my_id = -1;
    uint32_t my_key = 0u;
    for (int j = 0; j < p.k && best; ++j) {
        const int e = l.take(best, lane);
        if (lane == j) {
            my_id = e;
            my_key = best;
        }
        best = l.best();
    }
    const float my_p = my_id >= 0 ? share_of(l.value(my_key), m) : 0.0f;
    const float z = p.normalize ? warp_sum(my_p) : all;
    if (lane < p.k) {
        p.ids[t * p.k + lane] = my_id;
        p.weights[t * p.k + lane] = my_id >= 0 ? my_p / z : 0.0f;
    }
    return my_id;
}

// Ranks the choices of tokens [t0, t1): warp w < kRankWarps takes the w-th run
// of them.  base[e] is the first slot of the block's choices of expert e; start
// ([kRankWarps][E], shared) is scratch.
__device__ __forceinline__ void rank_choices(const RouteParams& p, int64_t t0, int64_t t1, int32_t* start,
                                             const int32_t* base, int threads) {
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int64_t c0 = t0 * p.k, n = (t1 - t0) * p.k;
    const int64_t per = ((n + kRankWarps - 1) / kRankWarps + 31) & ~(int64_t)31;
    const int64_t a = c0 + (warp * per < n ? warp * per : n), z = c0 + ((warp + 1) * per < n ? (warp + 1) * per : n);
    for (int i = tid; i < kRankWarps * p.E; i += threads) start[i] = 0;
    __syncthreads();
    if (warp < kRankWarps)
        for (int64_t c = a + lane; c < z; c += 32) {
            const int e = p.ids[c];
            if (e >= 0) atomicAdd(&start[warp * p.E + e], 1);
        }
    __syncthreads();
    for (int e = tid; e < p.E; e += threads) {
        int at = base[e];
#pragma unroll
        for (int w = 0; w < kRankWarps; ++w) {
            const int cnt = start[w * p.E + e];
            start[w * p.E + e] = at;
            at += cnt;
        }
    }
    __syncthreads();
    if (warp >= kRankWarps) return;
    for (int64_t c = a; c < z; c += 32) {
        const bool in = c + lane < z;
        const int e = in ? p.ids[c + lane] : -1;
        const unsigned same = __match_any_sync(0xFFFFFFFFu, e);
        const int rank = __popc(same & ((1u << lane) - 1u));
        int slot = -1;
        if (e >= 0) slot = start[warp * p.E + e] + rank;
        __syncwarp();
        if (e >= 0 && rank == 0) start[warp * p.E + e] += __popc(same);
        __syncwarp();
        if (in) {
            p.slots[c + lane] = slot;
            if (slot >= 0) p.rows[slot] = (int32_t)((c + lane) / p.k);
        }
    }
}

// Exclusive scan of cnt[0 .. E) (shared) into out[0 .. E) (shared) by warp 0;
// returns nothing, out[E] = total.
__device__ __forceinline__ void scan_experts(const int32_t* cnt, int32_t* out, int E) {
    if (threadIdx.x < 32) {
        const int lane = threadIdx.x, per = (E + 31) / 32, b = lane * per;
        int s = 0;
        for (int i = 0; i < per; ++i)
            if (b + i < E) s += cnt[b + i];
        int at = s;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xFFFFFFFFu, at, o);
            if (lane >= o) at += v;
        }
        if (lane == 31) out[E] = at;
        at -= s;
        for (int i = 0; i < per; ++i)
            if (b + i < E) {
                const int c = cnt[b + i];
                out[b + i] = at;
                at += c;
            }
    }
    __syncthreads();
}

template <typename T, int V>
__global__ void __launch_bounds__(kSmallThreads) route_small_kernel(const RouteParams p) {
    extern __shared__ int32_t sm[];
    int32_t* hist = sm;                // [E]
    int32_t* base = hist + p.E;        // [E + 1]
    int32_t* start = base + p.E + 1;   // [kRankWarps][E]
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, threads = blockDim.x;
    for (int e = tid; e < p.E; e += threads) hist[e] = 0;
    overlap_begin();
    __syncthreads();
    int id = -1;
    T logit[V];
    if (warp < p.T) read_logits<T, V>(p, warp, lane, logit);
    for (int64_t t = warp; t < p.T; t += threads / 32) {
        id = choose<T, V>(p, t, t + threads / 32 < p.T ? t + threads / 32 : -1, lane, logit);
        if (id >= 0) atomicAdd(&hist[id], 1);
    }
    __syncthreads();
    scan_experts(hist, base, p.E);
    for (int e = tid; e <= p.E; e += threads) p.offsets[e] = base[e];
    for (int64_t s = base[p.E] + tid; s < p.T * p.k; s += threads) p.rows[s] = -1;
    if (p.T == 1) {  // one choice of an expert at most: its slot is the expert's first
        if (warp == 0 && lane < p.k) {
            const int slot = id >= 0 ? base[id] : -1;
            p.slots[lane] = slot;
            if (slot >= 0) p.rows[slot] = 0;
        }
        return;
    }
    rank_choices(p, 0, p.T, start, base, threads);
}

template <typename T, int V>
__global__ void __launch_bounds__(kChooseThreads) route_choose_kernel(const RouteParams p) {
    extern __shared__ int32_t cnt[];  // [E]
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    for (int e = tid; e < p.E; e += kChooseThreads) cnt[e] = 0;
    overlap_begin();
    __syncthreads();
    const int64_t t0 = (int64_t)blockIdx.x * p.tb, t1 = t0 + p.tb < p.T ? t0 + p.tb : p.T;
    constexpr int kStep = kChooseThreads / 32;
    T logit[V];
    if (t0 + warp < t1) read_logits<T, V>(p, t0 + warp, lane, logit);
    for (int64_t t = t0 + warp; t < t1; t += kStep) {
        const int id = choose<T, V>(p, t, t + kStep < t1 ? t + kStep : -1, lane, logit);
        if (id >= 0) atomicAdd(&cnt[id], 1);
    }
    __syncthreads();
    for (int e = tid; e < p.E; e += kChooseThreads) p.before[(int64_t)blockIdx.x * p.E + e] = cnt[e];
}

// 32 experts per CTA, lane = expert; the 32 warps scan a run of blocks each.
__global__ void __launch_bounds__(1024) route_scan_kernel(const RouteParams p) {
    __shared__ int32_t part[32][33];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int e = blockIdx.x * 32 + lane;
    overlap_begin();
    constexpr int kPer = kMaxBlocks / 32;  // blocks of a warp, at most
    const int per = (p.blocks + 31) / 32, b0 = warp * per;
    int c[kPer], s = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        c[i] = i < per && b0 + i < p.blocks && e < p.E ? p.before[(int64_t)(b0 + i) * p.E + e] : 0;
        s += c[i];
    }
    part[warp][lane] = s;
    __syncthreads();
    int at = 0, all = 0;
#pragma unroll
    for (int w = 0; w < 32; ++w) {
        const int v = part[w][lane];
        if (w < warp) at += v;
        all += v;
    }
    if (e >= p.E) return;
    if (warp == 0) p.total[e] = all;
#pragma unroll
    for (int i = 0; i < kPer; ++i)
        if (i < per && b0 + i < p.blocks) {
            p.before[(int64_t)(b0 + i) * p.E + e] = at;
            at += c[i];
        }
}

__global__ void __launch_bounds__(kThreads) route_rank_kernel(const RouteParams p) {
    extern __shared__ int32_t sm[];
    int32_t* cnt = sm;
    int32_t* base = cnt + p.E;        // [E + 1]
    int32_t* start = base + p.E + 1;  // [kRankWarps][E]
    const int tid = threadIdx.x;
    overlap_begin();
    for (int e = tid; e < p.E; e += kThreads) cnt[e] = p.total[e];
    __syncthreads();
    scan_experts(cnt, base, p.E);
    const int64_t n = p.T * p.k;
    if (blockIdx.x == 0)
        for (int e = tid; e <= p.E; e += kThreads) p.offsets[e] = base[e];
    for (int64_t s = base[p.E] + (int64_t)blockIdx.x * kThreads + tid; s < n; s += (int64_t)gridDim.x * kThreads) p.rows[s] = -1;
    __syncthreads();
    for (int e = tid; e < p.E; e += kThreads) base[e] += p.before[(int64_t)blockIdx.x * p.E + e];
    __syncthreads();
    const int64_t t0 = (int64_t)blockIdx.x * p.tb, t1 = t0 + p.tb < p.T ? t0 + p.tb : p.T;
    rank_choices(p, t0, t1, start, base, kThreads);
}

template <typename T, int V>
cudaError_t launch_choose(const RouteParams& p, bool small, size_t smem, cudaStream_t st) {
    note_launches(1);
    if (small) {
        const unsigned warps = p.T < 4 ? 4 : p.T < 32 ? (unsigned)p.T : 32;
        return launch_overlapped(route_small_kernel<T, V>, 1, 32 * warps, smem, st, p);
    }
    return launch_overlapped(route_choose_kernel<T, V>, (unsigned)p.blocks, kChooseThreads, p.E * sizeof(int32_t), st, p);
}

template <typename T>
cudaError_t launch_choose(const RouteParams& p, bool small, size_t smem, cudaStream_t st) {
    const int v = (p.E + 31) / 32;
    return v <= 1    ? launch_choose<T, 1>(p, small, smem, st)
           : v <= 2  ? launch_choose<T, 2>(p, small, smem, st)
           : v <= 4  ? launch_choose<T, 4>(p, small, smem, st)
           : v <= 8  ? launch_choose<T, 8>(p, small, smem, st)
           : v <= 16 ? launch_choose<T, 16>(p, small, smem, st)
                     : launch_choose<T, 32>(p, small, smem, st);
}

cudaError_t launch_choose(const RouteParams& p, bool small, size_t smem, cudaStream_t st) {
    return p.dtype == NXQ_F32   ? launch_choose<float>(p, small, smem, st)
           : p.dtype == NXQ_F16 ? launch_choose<__half>(p, small, smem, st)
                                : launch_choose<__nv_bfloat16>(p, small, smem, st);
}

// ---- combine -------------------------------------------------------------------

// One warp sums 32 VEC columns of one token: lane j holds slot and weight j, the
// rows of up to kBatch experts are loaded before the first is used, and the
// next item's slots meanwhile.  Bound by reading T k rows of h, so what counts
// is loads in flight; nothing synchronizes the warps.  (With slots and weights
// staged once per CTA and two barriers an item: 225 us for 8192 tokens x 8 rows
// of 4096 bf16.)
constexpr int kCombThreads = 256;
constexpr int kBatch = 8;

// VEC (8, 2 or 1) consecutive values of h as loaded.
template <int VEC, bool F32>
struct Raw {
    static constexpr int kWords = F32 ? VEC : (VEC + 1) / 2;
    uint32_t w[kWords];
    __device__ __forceinline__ void load(const void* p, int64_t i) {
        if constexpr (VEC == 8) {
            const uint4* a = F32 ? reinterpret_cast<const uint4*>(static_cast<const float*>(p) + i)
                                 : reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p) + i);
#pragma unroll
            for (int j = 0; j < kWords / 4; ++j) {
                const uint4 q = __ldcs(a + j);
                w[4 * j] = q.x, w[4 * j + 1] = q.y, w[4 * j + 2] = q.z, w[4 * j + 3] = q.w;
            }
        } else if constexpr (F32 && VEC == 2) {
            const uint2 q = __ldcs(reinterpret_cast<const uint2*>(static_cast<const float*>(p) + i));
            w[0] = q.x, w[1] = q.y;
        } else if constexpr (F32 || VEC == 2) {
            w[0] = __ldcs(F32 ? static_cast<const uint32_t*>(p) + i
                              : reinterpret_cast<const uint32_t*>(static_cast<const uint16_t*>(p) + i));
        } else {
            w[0] = __ldcs(static_cast<const uint16_t*>(p) + i);
        }
    }
    __device__ __forceinline__ void widen(int dt, float (&v)[VEC]) const {
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            if constexpr (F32) {
                v[j] = __uint_as_float(w[j]);
            } else {
                const uint32_t u = w[j / 2];
                if (dt == NXQ_F16)
                    v[j] = __half2float(__ushort_as_half((unsigned short)(j & 1 ? u >> 16 : u & 0xFFFFu)));
                else
                    v[j] = __uint_as_float(j & 1 ? u & 0xFFFF0000u : u << 16);
            }
        }
    }
};

__device__ __forceinline__ void store_as(void* p, int dt, int64_t i, float v) {
    if (dt == NXQ_F32)
        static_cast<float*>(p)[i] = v;
    else if (dt == NXQ_F16)
        static_cast<__half*>(p)[i] = __float2half_rn(v);
    else
        static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
}

// Eight consecutive outputs (fp32: 32-byte, else 16-byte aligned).
__device__ __forceinline__ void store8(void* y, int dt, int64_t o, const float (&v)[8]) {
    if (dt == NXQ_F32) {
        store_f32x8(static_cast<float*>(y) + o, v);
        return;
    }
    uint32_t q[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (dt == NXQ_F16) {
            const __half2 p = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
            q[i] = *reinterpret_cast<const uint32_t*>(&p);
        } else {
            const __nv_bfloat162 p = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
            q[i] = *reinterpret_cast<const uint32_t*>(&p);
        }
    }
    *reinterpret_cast<uint4*>(static_cast<uint16_t*>(y) + o) = make_uint4(q[0], q[1], q[2], q[3]);
}

// Items are (token, 32 VEC columns), segs to a token.  VEC = 8 needs N % 8 == 0,
// h and y 16-byte and an fp32 residual or output 32-byte aligned; VEC = 2 an
// even N and h aligned to two values.  F32: h's type.
template <int VEC, bool F32>
__global__ void __launch_bounds__(kCombThreads) combine_kernel(const void* h, int h_dtype, int64_t R, int64_t N,
                                                               const int32_t* slots,
                                                               const float* weights, int64_t T, int k,
                                                               const float* res, void* y, int y_dtype, int64_t segs,
                                                               DeviceStatus* status) {
    overlap_begin();
    const int lane = threadIdx.x & 31;
    const int64_t items = T * segs, step = (int64_t)gridDim.x * (kCombThreads / 32);
    const int64_t dt = step / segs, dseg = step - dt * segs;  // one step in tokens and segments
    const int64_t it0 = (int64_t)blockIdx.x * (kCombThreads / 32) + (threadIdx.x >> 5);
    int64_t t = it0 / segs, seg = it0 - t * segs;
    int next_s = -1;
    float next_w = 0.0f;
    auto fetch = [&](int64_t tok) {
        if (tok < T && lane < k) {
            next_s = slots[tok * k + lane];
            next_w = weights[tok * k + lane];
        }
    };
    fetch(t);
    for (int64_t it = it0; it < items; it += step) {
        const int64_t n = (seg * 32 + lane) * VEC, o = t * N + n;
        int my_s = next_s;
        const float my_w = next_w;
        if (my_s >= R) {
            raise_index(status, kIndexSlot);
            my_s = -1;
        }
        t += dt;
        seg += dseg;
        if (seg >= segs) {
            seg -= segs;
            ++t;
        }
        float acc[VEC], rv[VEC];
#pragma unroll
        for (int i = 0; i < VEC; ++i) acc[i] = rv[i] = 0.0f;
        if (res && n < N) {
            if constexpr (VEC == 8) {
                load_f32x8(res + o, rv);
            } else {
#pragma unroll
                for (int i = 0; i < VEC; ++i) rv[i] = res[o + i];
            }
        }
        for (int j0 = 0; j0 < k; j0 += kBatch) {
            Raw<VEC, F32> r[kBatch];
#pragma unroll
            for (int j = 0; j < kBatch; ++j) {
                const int s = __shfl_sync(0xFFFFFFFFu, my_s, (j0 + j) & 31);
                if (j0 + j < k && s >= 0 && n < N) r[j].load(h, (int64_t)s * N + n);
            }
            if (j0 + kBatch >= k) fetch(t);
#pragma unroll
            for (int j = 0; j < kBatch; ++j) {
                const int s = __shfl_sync(0xFFFFFFFFu, my_s, (j0 + j) & 31);
                const float w = __shfl_sync(0xFFFFFFFFu, my_w, (j0 + j) & 31);
                if (j0 + j < k && s >= 0) {
                    float v[VEC];
                    r[j].widen(h_dtype, v);
#pragma unroll
                    for (int i = 0; i < VEC; ++i) acc[i] = fmaf(w, v[i], acc[i]);
                }
            }
        }
        if (n >= N) continue;
#pragma unroll
        for (int i = 0; i < VEC; ++i) acc[i] += rv[i];
        if constexpr (VEC == 8) {
            store8(y, y_dtype, o, acc);
        } else {
#pragma unroll
            for (int i = 0; i < VEC; ++i) store_as(y, y_dtype, o + i, acc[i]);
        }
    }
}

// ---- combine of many tokens ------------------------------------------------------
// One persistent CTA per SM: a producer warp brings the k rows of a token (or
// of `seg` columns of it) into a ring of shared memory by one bulk copy each,
// lane j row j, and 16 warps sum them with a thread per 8 columns; the residual
// is loaded while the rows are awaited.  Rows of several KB in flight per copy
// and no registers to hold them.
constexpr int kBulkWarps = 16, kBulkThreads = 32 * (kBulkWarps + 1);
constexpr int kBulkStages = 3;
constexpr int kBulkStage = 72 * 1024;  // bytes of a stage

// A CTA needs 0.9 us and 0.06 us a row for a token however short the rows are,
// where combine_kernel's time goes by the bytes.  So: from 4 tokens per SM, and
// from 6 KB + 2.25 KB a row of h per token.  Measured, combine_kernel / this one
// in us, fp32 residual and output:
//   4000 tokens, bf16:  k = 2, N = 2048 (8 KB): 39 / 29;    k = 8, N = 1024 (16 KB): 27 / 36
//     k = 8, N = 1536 (24 KB): 38 / 38;  N = 2048 (32 KB): 49 / 40;  N = 4096: 90 / 61
//     k = 16, N = 1024 (32 KB): 42 / 53;  N = 1536 (48 KB): 61 / 56
//     k = 32, N = 512 (32 KB): 38 / 88;  N = 1024 (64 KB): 71 / 88
//   8192 tokens, bf16, k = 8:  N = 64: 10.5 / 66;  N = 1024: 50 / 70;  N = 2048: 92 / 79;  N = 4096: 176 / 121
//   600 tokens, bf16, k = 8:  N = 512: 3.1 / 7.5;  N = 2048: 9.3 / 8.7;  N = 4096: 15.7 / 12.6
inline bool combine_by_bulk(int64_t T, int k, int64_t row_bytes, int sms) {
    return T >= 4 * (int64_t)sms && row_bytes >= 2304 + 6144 / k;
}

template <bool F32>
__global__ void __launch_bounds__(kBulkThreads, 1) combine_bulk_kernel(const void* h, int h_dtype, int64_t R,
                                                                       int64_t N, const int32_t* slots,
                                                                       const float* weights, int64_t T, int k,
                                                                       const float* res, void* y, int y_dtype, int64_t segs,
                                                                       int seg, DeviceStatus* status) {
    constexpr int kSize = F32 ? 4 : 2;
    extern __shared__ __align__(128) uint8_t ring[];
    __shared__ uint64_t full[kBulkStages], empty[kBulkStages];
    __shared__ int s_slot[kBulkStages][kMaxK];  // -1: skipped
    __shared__ float s_w[kBulkStages][kMaxK];
    __shared__ int s_abort;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int i = 0; i < kBulkStages; ++i) {
            ptx::mbar_init(&full[i], 1);
            ptx::mbar_init(&empty[i], kBulkWarps);
        }
        s_abort = 0;
        ptx::fence_mbar_init();
    }
    __syncthreads();
    const ptx::WaitCtl ctl{&s_abort, status};
    overlap_begin();
    const int64_t items = T * segs;
    if (warp == kBulkWarps) {
        // h was written through the generic proxy; the copies read it through the async one.
        asm volatile("fence.proxy.async;" ::: "memory");
        uint32_t u = 0;
        for (int64_t it = blockIdx.x; it < items; it += gridDim.x, ++u) {
            const int st = u % kBulkStages;
            const int64_t t = it / segs, n0 = (it - t * segs) * seg;
            const uint32_t bytes = (uint32_t)(N - n0 < seg ? N - n0 : seg) * kSize;
            int s = -1;
            float w = 0.0f;
            if (lane < k) {
                s = slots[t * k + lane];
                w = weights[t * k + lane];
                if (s >= R) {
                    raise_index(status, kIndexSlot);
                    s = -1;
                }
            }
            int ok = 1;
            if (u >= kBulkStages) ok = ptx::mbar_wait(&empty[st], (u / kBulkStages - 1) & 1u, ctl, 61) ? 1 : 0;
            if (!__all_sync(0xFFFFFFFFu, ok)) break;
            if (lane < k) {
                s_slot[st][lane] = s;
                s_w[st][lane] = w;
            }
            const unsigned rows = __ballot_sync(0xFFFFFFFFu, s >= 0);
            __syncwarp();
            if (lane == 0) ptx::mbar_arrive_expect_tx(&full[st], __popc(rows) * bytes);
            __syncwarp();
            if (s >= 0)
                ptx::bulk_g2s(ring + (size_t)st * kBulkStage + (size_t)lane * seg * kSize,
                              static_cast<const uint8_t*>(h) + ((int64_t)s * N + n0) * kSize, bytes, &full[st]);
        }
        // Do not leave with copies in flight (bounded, ignoring the abort flag).
        for (uint32_t i = u >= kBulkStages ? u - kBulkStages : 0; i < u; ++i) {
            const long long t0 = clock64();
            while (!ptx::mbar_try_wait(&full[i % kBulkStages], (i / kBulkStages) & 1u) && clock64() - t0 < ptx::kWaitCycles) {
            }
        }
        return;
    }
    uint32_t u = 0;
    for (int64_t it = blockIdx.x; it < items; it += gridDim.x, ++u) {
        const int st = u % kBulkStages;
        const int64_t t = it / segs, n0 = (it - t * segs) * seg;
        const int cols = (int)(N - n0 < seg ? N - n0 : seg);
        bool landed = false;
        for (int c = threadIdx.x * 8; c < cols || !landed; c += kBulkWarps * 32 * 8) {
            const int64_t o = t * N + n0 + c;
            float acc[8], rv[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) acc[i] = rv[i] = 0.0f;
            if (res && c < cols) load_f32x8(res + o, rv);
            if (!landed) {
                if (!ptx::mbar_wait(&full[st], (u / kBulkStages) & 1u, ctl, 62)) return;
                landed = true;
            }
            if (c >= cols) break;
            const uint8_t* base = ring + (size_t)st * kBulkStage + (size_t)c * kSize;
            for (int j = 0; j < k; ++j) {
                if (s_slot[st][j] < 0) continue;
                const float w = s_w[st][j];
                Raw<8, F32> r;
                const uint4* q = reinterpret_cast<const uint4*>(base + (size_t)j * seg * kSize);
#pragma unroll
                for (int i = 0; i < (F32 ? 2 : 1); ++i) {
                    const uint4 x = q[i];
                    r.w[4 * i] = x.x, r.w[4 * i + 1] = x.y, r.w[4 * i + 2] = x.z, r.w[4 * i + 3] = x.w;
                }
                float v[8];
                r.widen(h_dtype, v);
#pragma unroll
                for (int i = 0; i < 8; ++i) acc[i] = fmaf(w, v[i], acc[i]);
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) acc[i] += rv[i];
            store8(y, y_dtype, o, acc);
        }
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(&empty[st]);
    }
}

}  // namespace

}  // namespace nxq

using namespace nxq;

extern "C" {

NXQ_API int nxq_moe_route(const void* logits_dev, int dtype, int64_t T, int E, int k, int normalize, int32_t* ids_dev,
                          float* weights_dev, int32_t* offsets_dev, int32_t* rows_dev, int32_t* slots_dev,
                          void* stream) {
    if (E < 1 || E > kMaxE) return fail(NXQ_ERR_ARG, "route: E=%d (1 to %d experts)", E, kMaxE);
    if (k < 1 || k > kMaxK || k > E) return fail(NXQ_ERR_ARG, "route: k=%d of %d experts (at most %d)", k, E, kMaxK);
    if (T < 0 || T > (int64_t)0x7FFFFFFF / k) return fail(NXQ_ERR_ARG, "route: T=%lld, k=%d", (long long)T, k);
    if (!dtype_valid(dtype)) return fail(NXQ_ERR_ARG, "bad dtype");
    if (!offsets_dev) return fail(NXQ_ERR_ARG, "route: null offsets");
    if (T > 0 && (!logits_dev || !ids_dev || !weights_dev || !rows_dev || !slots_dev))
        return fail(NXQ_ERR_ARG, "route: null array");
    if (!aligned_as(logits_dev, dtype) || !aligned_4(ids_dev) || !aligned_4(weights_dev) || !aligned_4(offsets_dev) ||
        !aligned_4(rows_dev) || !aligned_4(slots_dev))
        return fail(NXQ_ERR_ARG, "route: an array is not aligned to its type");
    if (int rc = context_ready()) return rc;
    cudaStream_t st = (cudaStream_t)stream;
    if (T == 0) {
        NXQ_CUDA(cudaMemsetAsync(offsets_dev, 0, (size_t)(E + 1) * sizeof(int32_t), st));
        return NXQ_OK;
    }
    RouteParams p{logits_dev, dtype, T, E, k, normalize, 0, 0, ids_dev, weights_dev, offsets_dev, rows_dev, slots_dev, nullptr, nullptr};
    const size_t smem = (size_t)(2 * E + 1 + kRankWarps * E) * sizeof(int32_t);
    if (T <= kSmallT) {
        cudaError_t e = launch_choose(p, true, smem, st);
        return e == cudaSuccess ? NXQ_OK : cuda_fail(e, "route launch");
    }
    p.tb = (int)((T + kMaxBlocks - 1) / kMaxBlocks);
    if (p.tb < 64) p.tb = 64;
    p.blocks = (int)((T + p.tb - 1) / p.tb);
    cudaError_t e = cudaMallocAsync((void**)&p.before, ((size_t)p.blocks + 1) * E * sizeof(int32_t), st);
    if (e != cudaSuccess) return cuda_fail(e, "cudaMallocAsync (route workspace)");
    p.total = p.before + (size_t)p.blocks * E;
    e = launch_choose(p, false, smem, st);
    if (e == cudaSuccess) e = launch_overlapped(route_scan_kernel, (unsigned)((E + 31) / 32), 1024, 0, st, p);
    if (e == cudaSuccess) e = launch_overlapped(route_rank_kernel, (unsigned)p.blocks, kThreads, smem, st, p);
    note_launches(2);
    cudaFreeAsync(p.before, st);
    return e == cudaSuccess ? NXQ_OK : cuda_fail(e, "route launch");
}

NXQ_API int nxq_moe_combine(const void* h_dev, int h_dtype, int64_t R, int64_t N, const int32_t* slots_dev,
                            const float* weights_dev, int64_t T, int k, const float* res_dev, void* y_dev,
                            int y_dtype, void* stream) {
    if (T < 0 || N < 0 || R < 0 || R > 0x7FFFFFFF || k < 1 || k > kMaxK)
        return fail(NXQ_ERR_ARG, "combine: T=%lld N=%lld R=%lld k=%d", (long long)T, (long long)N, (long long)R, k);
    if (!dtype_valid(h_dtype) || !dtype_valid(y_dtype)) return fail(NXQ_ERR_ARG, "bad dtype");
    if (T == 0 || N == 0) return NXQ_OK;
    if (!slots_dev || !weights_dev || !y_dev || (R > 0 && !h_dev)) return fail(NXQ_ERR_ARG, "combine: null array");
    if (!aligned_as(h_dev, h_dtype) || !aligned_as(y_dev, y_dtype) || !aligned_4(slots_dev) || !aligned_4(weights_dev) ||
        !aligned_4(res_dev))
        return fail(NXQ_ERR_ARG, "combine: an array is not aligned to its type");
    if ((const void*)y_dev == (const void*)res_dev && y_dtype != NXQ_F32)
        return fail(NXQ_ERR_ARG, "combine: y may be the residual only as fp32");
    if (int rc = context_ready()) return rc;
    const bool vec = N % 8 == 0 && (uintptr_t)h_dev % 16 == 0 && (uintptr_t)res_dev % 32 == 0 &&
                     (uintptr_t)y_dev % (y_dtype == NXQ_F32 ? 32 : 16) == 0;
    const bool f32 = h_dtype == NXQ_F32;
    if (vec && combine_by_bulk(T, k, N * (f32 ? 4 : 2), context_sm_count()) && T <= ((int64_t)1 << 62) / N) {
        int64_t seg = kBulkStage / (k * (f32 ? 4 : 2)) / 64 * 64;  // columns of a stage
        int64_t segs = (N + seg - 1) / seg;
        seg = ((N + segs - 1) / segs + 63) / 64 * 64;
        segs = (N + seg - 1) / seg;
        auto* kernel = f32 ? combine_bulk_kernel<true> : combine_bulk_kernel<false>;
        cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kBulkStages * kBulkStage);
        if (e == cudaSuccess)
            e = launch_overlapped(kernel, (unsigned)context_sm_count(), kBulkThreads, kBulkStages * kBulkStage,
                                  (cudaStream_t)stream, h_dev, h_dtype, R, N, slots_dev, weights_dev, T, k, res_dev, y_dev,
                                  y_dtype, segs, (int)seg, context_status());
        note_launches(1);
        return e == cudaSuccess ? NXQ_OK : cuda_fail(e, "combine launch");
    }
    const bool pairs = N % 2 == 0 && (uintptr_t)h_dev % (f32 ? 8 : 4) == 0;
    const int64_t per = 32 * (vec ? 8 : pairs ? 2 : 1), segs = (N + per - 1) / per;
    if (T > ((int64_t)1 << 62) / segs) return fail(NXQ_ERR_ARG, "combine: T=%lld N=%lld", (long long)T, (long long)N);
    const int64_t want = (T * segs + kCombThreads / 32 - 1) / (kCombThreads / 32), most = (int64_t)context_sm_count() * 8;
    auto* kernel = vec ? (f32 ? combine_kernel<8, true> : combine_kernel<8, false>)
                   : pairs ? (f32 ? combine_kernel<2, true> : combine_kernel<2, false>)
                           : (f32 ? combine_kernel<1, true> : combine_kernel<1, false>);
    const cudaError_t e = launch_overlapped(kernel, (unsigned)(want < most ? want : most), kCombThreads, 0,
                                            (cudaStream_t)stream, h_dev, h_dtype, R, N, slots_dev, weights_dev, T, k,
                                            res_dev, y_dev, y_dtype, segs, context_status());
    note_launches(1);
    return e == cudaSuccess ? NXQ_OK : cuda_fail(e, "combine launch");
}

}  // extern "C"
