// Norm and position rotation of heads, plain (nxq_rope) and on the way into a
// paged cache (nxq_kv_append).
//
// Pair i of a head at position p is turned by the angle p f_i.  f_i is held as turns
// per position in units of 2^-64, so p f_i modulo a turn is one 64-bit product, exact
// at any position; its upper 32 bits, as a signed fraction of a half turn and rounded to
// fp32, go to sincospif (off by at most 2^-25 of a half turn, 9e-8 radians; the product p f_i in
// fp32 would be off by 0.06 radians at position 10^6).
//
// A CTA takes one to eight tokens: it finds their positions (append: their sequence, by a
// 32-ary search of the offsets, and their page), computes each token's dims / 2 sines and
// cosines once into shared memory, and then walks the (token, head) pairs of queries,
// keys and values: 16 elements per lane, as two 8-element vectors that hold whole
// pairs in either layout, the fewest lanes (a power of two) that cover a head, so the
// norm's sum is a few shuffles; the next pair's loads are in flight meanwhile, and
// the first's before the positions are known.  Heads, strides or rotated parts that 8-element
// vectors do not fit take one warp per head and one pair per lane.
//
// Bound by memory: T (heads in and out) and nothing else of size.  8192 tokens of 40 heads of
// 128 (168 MB): 38.0 us, 4.4 TB/s, 0.69 of the copy rate; 16800 tokens of 64 + 8 + 8 into the
// cache: 144 us, 4.8 TB/s, 0.74 (scattered heads in flight per lane, not instructions: issue slots are
// 0.70 used).  One token is a launch: 3.5 us.  Sizes that vectors do not fit load 2 bytes at a
// time with nothing ahead: 8192 tokens of 40 heads of 96 (126 MB) with 24 elements turned 175 us,
// with all 96 turned, by vectors, 36.
#include "attention.h"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cmath>
#include <mutex>
#include <new>
#include <unordered_set>

namespace nxq {

namespace {

constexpr int kRopeThreads = 256, kMaxHeadDim = 512, kMaxTokensPerCta = kRopeThreads / 32;

struct HeadRows {
    void* dev;
    int heads;
    int64_t token, head;  // strides in elements
};

struct RopeParams {
    int64_t T;
    int D, dims, layout, lanes;  // lanes of a head
    float scale, eps;
    const uint64_t* turns;
    HeadRows in[3], out[3];  // queries, keys, values (heads 0: none); out[1], out[2] of an append are the cache
    const float* norm[3];
    int norm_vec;  // norms are 16-byte aligned
    int x_dtype, y_dtype, c_dtype;
    const void* positions;  // nxq_rope
    int positions_type;
    // nxq_kv_append
    Batch b;
    int64_t page_stride, slot_stride;
    DeviceStatus* status;
};

__device__ __forceinline__ float load1(const void* x, int dt, int64_t i) {
    if (dt == NXQ_F16) return __half2float(static_cast<const __half*>(x)[i]);
    if (dt == NXQ_BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(x)[i]);
    return static_cast<const float*>(x)[i];
}
__device__ __forceinline__ bool store1(void* y, int dt, int64_t i, float v) {
    if (dt == NXQ_F16) {
        static_cast<__half*>(y)[i] = __float2half_rn(v);
        return f16_overflows(v);
    }
    if (dt == NXQ_BF16)
        static_cast<__nv_bfloat16*>(y)[i] = __float2bfloat16_rn(v);
    else
        static_cast<float*>(y)[i] = v;
    return false;
}

// 8 consecutive elements (16-byte aligned).
__device__ __forceinline__ bool store8(void* y, int dt, int64_t i, const float (&v)[8]) {
    if (dt == NXQ_F32) {
        float4* q = reinterpret_cast<float4*>(static_cast<float*>(y) + i);
        q[0] = make_float4(v[0], v[1], v[2], v[3]);
        q[1] = make_float4(v[4], v[5], v[6], v[7]);
        return false;
    }
    uint32_t w[4];
    bool over = false;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        if (dt == NXQ_F16) {
            const __half2 h = __floats2half2_rn(v[2 * j], v[2 * j + 1]);
            w[j] = *reinterpret_cast<const uint32_t*>(&h);
            over |= f16_overflows(v[2 * j]) || f16_overflows(v[2 * j + 1]);
        } else {
            const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * j], v[2 * j + 1]);
            w[j] = *reinterpret_cast<const uint32_t*>(&h);
        }
    }
    *reinterpret_cast<uint4*>(static_cast<uint16_t*>(y) + i) = make_uint4(w[0], w[1], w[2], w[3]);
    return over;
}

// (x, y) turned by the angle of k = (cos, sin): the same bits wherever it is compiled.
__device__ __forceinline__ void turn(float& x, float& y, float2 k) {
    const float a = x, b = y;
    x = fmaf(a, k.x, -__fmul_rn(b, k.y));
    y = fmaf(a, k.y, __fmul_rn(b, k.x));
}

// The last sequence whose first row is <= t (-1: none), by a converged warp; right
// wherever the offsets ascend.
__device__ __forceinline__ int find_seq(const int32_t* off, int S, int64_t t) {
    const int lane = threadIdx.x & 31;
    int lo = 0, n = S;
    while (true) {
        const int step = (n + 31) / 32, i = lane * step;
        const unsigned m = __ballot_sync(0xFFFFFFFFu, i < n && off[lo + i] <= t);
        if (!m) return lo - 1;  // only in the first round
        const int at = (31 - __clz(m)) * step;
        lo += at;
        n = n - at < step ? n - at : step;
        if (step == 1) return lo;
    }
}

// A token of the CTA: its position, and where it goes in the cache (element offset
// of its slot in head 0; -1: it is left out).
struct Token {
    int64_t pos, slot;
};

// The two 8-element vectors of a lane, as they lie in memory.
template <bool X32>
struct Raw {
    uint4 a[X32 ? 2 : 1], b[X32 ? 2 : 1];
};
template <bool X32>
__device__ __forceinline__ void fetch8(const void* x, int64_t i, uint4 (&v)[X32 ? 2 : 1]) {
    if constexpr (X32) {
        const uint4* q = reinterpret_cast<const uint4*>(static_cast<const float*>(x) + i);
        v[0] = q[0], v[1] = q[1];
    } else {
        v[0] = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(x) + i);
    }
}
template <bool X32>
__device__ __forceinline__ void widen8(const uint4 (&q)[X32 ? 2 : 1], int dt, float (&v)[8]) {
    if constexpr (X32) {
        const uint32_t w[8] = {q[0].x, q[0].y, q[0].z, q[0].w, q[1].x, q[1].y, q[1].z, q[1].w};
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = __uint_as_float(w[j]);
    } else {
        const uint32_t w[4] = {q[0].x, q[0].y, q[0].z, q[0].w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (dt == NXQ_F16) {
                const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[j]));
                v[2 * j] = f.x, v[2 * j + 1] = f.y;
            } else {
                v[2 * j] = __uint_as_float(w[j] << 16), v[2 * j + 1] = __uint_as_float(w[j] & 0xFFFF0000u);
            }
        }
    }
}

template <int VEC, bool APPEND, bool X32>
__global__ void __launch_bounds__(kRopeThreads) rope_kernel(const __grid_constant__ RopeParams p, const int tokens,
                                                            const int splits) {
    extern __shared__ float2 sc[];  // [tokens][dims / 2] (cos, sin) * scale
    __shared__ Token tok[kMaxTokensPerCta];
    overlap_begin();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int cta = blockIdx.x / splits, split = blockIdx.x - cta * splits;  // `splits` CTAs share their tokens' heads
    const int64_t t0 = (int64_t)cta * tokens;
    const int nt = (int)(p.T - t0 < tokens ? p.T - t0 : tokens);

    // The (token, head) pairs of this thread's group of lanes, and their place in memory.
    const int heads = p.in[0].heads + p.in[1].heads + p.in[2].heads;
    const int L = VEC == 8 ? p.lanes : 32, group = threadIdx.x / L, u = threadIdx.x % L, groups = kRopeThreads / L * splits;
    const unsigned mates = L == 32 ? 0xFFFFFFFFu : ((1u << L) - 1u) << (lane & ~(L - 1));  // lanes of the same head
    struct Pair {
        int part, head;
        int64_t x;   // offset of the head in the part's input
        int a, b;    // offsets of the lane's two vectors
        bool turned;
    };
    auto pair_at = [&](int t, int h) {
        Pair q{0, h, 0, 0, 0, false};
        while (q.head >= p.in[q.part].heads) q.head -= p.in[q.part++].heads;
        q.x = (t0 + t) * p.in[q.part].token + q.head * p.in[q.part].head;
        const int dims = q.part == 2 ? 0 : p.dims;  // values stay
        q.turned = u < dims / 16;
        if (q.turned && p.layout == NXQ_ROPE_HALF)
            q.a = 8 * u, q.b = dims / 2 + 8 * u;
        else
            q.a = 16 * u, q.b = q.a + 8;
        return q;
    };
    auto fetch = [&](const Pair& q, Raw<X32>& r) {
        if (q.a < p.D) fetch8<X32>(p.in[q.part].dev, q.x + q.a, r.a);
        if (q.b < p.D) fetch8<X32>(p.in[q.part].dev, q.x + q.b, r.b);
    };
    auto advance = [&](int& t, int& h) {
        for (h += groups; h >= heads; h -= heads) ++t;
    };
    // The first pair's loads go out before its position is known.
    const int first = split * (kRopeThreads / L) + group;
    int t = first / heads, h = first % heads;
    Raw<X32> raw{};
    Pair q{};
    if (t < nt) {
        q = pair_at(t, h);
        if constexpr (VEC == 8) fetch(q, raw);
    }
    if (APPEND) {
        if (warp < nt) {
            const int64_t row = t0 + warp;
            const int s = find_seq(p.b.q_off, p.b.S, row);
            Token k{0, -1};
            if (s >= 0 && lane == 0) {
                bool bad;
                const Seq q = read_seq(p.b, s, p.T, &bad);
                if (bad) {
                    raise_index(p.status, kIndexSeq);
                } else if (row < (int64_t)q.q0 + q.n) {
                    k.pos = (int64_t)q.len - q.n + (row - q.q0);
                    if (k.pos < 0) {
                        raise_index(p.status, kIndexPosition);
                    } else {
                        const int page = p.b.table[s * p.b.table_stride + k.pos / p.b.page];
                        if (page < 0 || page >= p.b.pages)
                            raise_index(p.status, kIndexPage);
                        else
                            k.slot = page * p.page_stride + k.pos % p.b.page * p.slot_stride;
                    }
                }
            }
            if (lane == 0) tok[warp] = k;
        }
        // Offsets that descend leave no row to meet them: one CTA looks at all.
        if (blockIdx.x == gridDim.x - 1)
            for (int s = threadIdx.x; s < p.b.S; s += kRopeThreads) {
                bool bad;
                read_seq(p.b, s, p.T, &bad);
                if (bad) raise_index(p.status, kIndexSeq);
            }
    } else if ((int)threadIdx.x < nt) {
        const int64_t row = t0 + threadIdx.x;
        tok[threadIdx.x] = Token{!p.turns                      ? 0
                                 : p.positions_type == NXQ_I64 ? static_cast<const int64_t*>(p.positions)[row]
                                                               : static_cast<const int32_t*>(p.positions)[row],
                                 0};
    }
    __syncthreads();
    const int pairs = p.dims / 2;
    for (int i = threadIdx.x; i < nt * pairs; i += kRopeThreads) {
        const int k = i / pairs, j = i - k * pairs;
        const uint64_t angle = (uint64_t)tok[k].pos * p.turns[j];
        float s, c;
        sincospif((float)(int32_t)(angle >> 32) * 0x1p-31f, &s, &c);
        // (Vectors: pair 8 u + j at [j][u], where the lanes of a head read it without conflicts.)
        sc[VEC == 8 ? k * pairs + (j & 7) * (pairs >> 3) + (j >> 3) : i] = make_float2(c * p.scale, s * p.scale);
    }
    __syncthreads();

    const float inv_d = 1.0f / (float)p.D;
    bool over = false;
    while (t < nt) {
        int t1 = t, h1 = h;
        advance(t1, h1);
        Raw<X32> next{};
        Pair q1{};
        if (t1 < nt) {
            q1 = pair_at(t1, h1);
            if constexpr (VEC == 8) fetch(q1, next);
        }
        const bool skip = APPEND && tok[t].slot < 0;
        const HeadRows& out = p.out[q.part];
        const bool cached = APPEND && q.part > 0;
        const int64_t yi = (cached ? tok[t].slot : (t0 + t) * out.token) + q.head * out.head;
        const int ydt = cached ? p.c_dtype : p.y_dtype;
        const float* norm = p.norm[q.part];
        const int dims = q.part == 2 ? 0 : p.dims;
        const float2* cs = sc + t * pairs;
        if constexpr (VEC == 8) {
            const bool has_a = q.a < p.D, has_b = q.b < p.D;
            float va[8], vb[8];
            widen8<X32>(raw.a, p.x_dtype, va);
            widen8<X32>(raw.b, p.x_dtype, vb);
            if (norm) {
                float sum = 0.0f;
                if (has_a)
#pragma unroll
                    for (int j = 0; j < 8; ++j) sum = fmaf(va[j], va[j], sum);
                if (has_b)
#pragma unroll
                    for (int j = 0; j < 8; ++j) sum = fmaf(vb[j], vb[j], sum);
                for (int o = L / 2; o; o >>= 1) sum += __shfl_xor_sync(mates, sum, o);
                const float r = 1.0f / sqrtf(fmaf(sum, inv_d, p.eps));
                auto scale = [&](float (&v)[8], int at) {
                    if (p.norm_vec) {
                        const float4 x = *reinterpret_cast<const float4*>(norm + at), y = *reinterpret_cast<const float4*>(norm + at + 4);
                        const float w[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
#pragma unroll
                        for (int j = 0; j < 8; ++j) v[j] = v[j] * r * w[j];
                    } else {
#pragma unroll
                        for (int j = 0; j < 8; ++j) v[j] = v[j] * r * norm[at + j];
                    }
                };
                if (has_a) scale(va, q.a);
                if (has_b) scale(vb, q.b);
            }
            if (q.turned) {
                if (p.layout == NXQ_ROPE_HALF) {
#pragma unroll
                    for (int j = 0; j < 8; ++j) turn(va[j], vb[j], cs[j * (pairs >> 3) + u]);
                } else {
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        turn(va[2 * j], va[2 * j + 1], cs[j * (pairs >> 3) + u]);
                        turn(vb[2 * j], vb[2 * j + 1], cs[(4 + j) * (pairs >> 3) + u]);
                    }
                }
            }
            if (has_a && !skip) over |= store8(out.dev, ydt, yi + q.a, va);
            if (has_b && !skip) over |= store8(out.dev, ydt, yi + q.b, vb);
            raw = next;
        } else if (!skip) {  // (a whole warp)
            const HeadRows& in = p.in[q.part];
            float r = 1.0f;
            if (norm) {
                float sum = 0.0f;
                for (int d = u; d < p.D; d += 32) {
                    const float x = load1(in.dev, p.x_dtype, q.x + d);
                    sum = fmaf(x, x, sum);
                }
                for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
                r = 1.0f / sqrtf(fmaf(sum, inv_d, p.eps));
            }
            auto at = [&](int d) {
                const float x = load1(in.dev, p.x_dtype, q.x + d);
                return norm ? x * r * norm[d] : x;
            };
            for (int i = u; i < dims / 2; i += 32) {
                const int a = p.layout == NXQ_ROPE_HALF ? i : 2 * i, b = p.layout == NXQ_ROPE_HALF ? i + dims / 2 : a + 1;
                float x = at(a), y = at(b);
                turn(x, y, cs[i]);
                over |= store1(out.dev, ydt, yi + a, x);
                over |= store1(out.dev, ydt, yi + b, y);
            }
            for (int d = dims + u; d < p.D; d += 32) over |= store1(out.dev, ydt, yi + d, at(d));
        }
        t = t1, h = h1, q = q1;
    }
    if (over) raise_range(p.status, 4u);
}

// Whether rows of heads can be read and written as vectors of 8 elements.
bool vec_rows(const HeadRows& h, int dtype) {
    return (uintptr_t)h.dev % 16 == 0 && h.token % 8 == 0 && h.head % 8 == 0 && dtype_valid(dtype);
}

cudaError_t launch_rope(RopeParams& p, bool append, cudaStream_t st) {
    bool vec = p.D % 8 == 0 && p.dims % 16 == 0;
    for (int i = 0; i < 3; ++i) {
        if (!p.in[i].heads) continue;
        vec = vec && vec_rows(p.in[i], p.x_dtype);
        if (!append || i == 0) vec = vec && vec_rows(p.out[i], p.y_dtype);  // (a cache always can)
    }
    int lanes = 1;
    while (lanes * 16 < p.D) lanes *= 2;
    p.lanes = lanes;
    p.status = context_status();
    // Few tokens: a CTA for each.  Many: several share one, with fewer barriers per byte.  (40
    // heads of 128, bf16, in us with 1, 4, 8 tokens a CTA: 592 tokens 4.4, 5.5, 9.2; 1200 9.0,
    // 9.1, 13.1; 2400 14.9, 12.1, 16.5; 4736 29.2, 20.2, 19.4; 16384 99.6, 68.4, 69.0.)
    const int64_t sms = context_sm_count();
    const int tokens = p.T <= 4 * sms ? 1 : p.T <= 32 * sms ? 4 : kMaxTokensPerCta;
    p.norm_vec = (uintptr_t)p.norm[0] % 16 == 0 && (uintptr_t)p.norm[1] % 16 == 0;
    const size_t smem = (size_t)tokens * (p.dims / 2) * sizeof(float2);
    // Fewer tokens than SMs: several CTAs for each, so that no thread has a second head to wait for
    // (the same heads in us with one and several: 1 token 2.87, 2.36; 148 3.15, 2.84; 300 4.1, 4.8).
    const int heads = p.in[0].heads + p.in[1].heads + p.in[2].heads, per = kRopeThreads / (vec ? lanes : 32);
    const int splits = p.T <= sms ? (heads + per - 1) / per : 1;
    const unsigned grid = (unsigned)((p.T + tokens - 1) / tokens * splits);
    note_launches(1);
    const bool wide = p.x_dtype == NXQ_F32;
    auto* kernel = !vec    ? (append ? rope_kernel<1, true, false> : rope_kernel<1, false, false>)
                   : wide  ? (append ? rope_kernel<8, true, true> : rope_kernel<8, false, true>)
                           : (append ? rope_kernel<8, true, false> : rope_kernel<8, false, false>);
    return launch_overlapped(kernel, grid, kRopeThreads, smem, st, p, tokens, splits);
}

std::mutex g_ropes_mu;
std::unordered_set<Rope*> g_ropes;

HeadRows rows_of(const nxq_heads* h) { return h ? HeadRows{h->dev, h->heads, h->token_stride, h->head_stride} : HeadRows{}; }

// Rotation and its handle's part of the parameters.
int take_rope(nxq_rope_t h, int D, RopeParams* p) {
    if (!h) return NXQ_OK;
    const Rope* r = nullptr;
    if (int rc = check_rope(h, &r)) return rc;
    if (r->dims > D) return fail(NXQ_ERR_SHAPE, "a rotation of %d elements for heads of %d", r->dims, D);
    p->dims = r->dims;
    p->layout = r->layout;
    p->scale = r->scale;
    p->turns = r->turns;
    return NXQ_OK;
}

// In place means that a head's output lies where the head lay; other threads may not have read what
// lies anywhere else.
int same_heads(const char* what, const nxq_heads* in, const nxq_heads* out, int64_t T, int x_dtype, int y_dtype) {
    if (in->heads != out->heads) return fail(NXQ_ERR_SHAPE, "%s: %d heads in, %d out", what, in->heads, out->heads);
    if (in->dev == out->dev && (x_dtype != y_dtype || (T > 1 && in->token_stride != out->token_stride) ||
                                (in->heads > 1 && in->head_stride != out->head_stride)))
        return fail(NXQ_ERR_ARG, "%s: in place with another type or other strides", what);
    return NXQ_OK;
}

}  // namespace

int check_rope(nxq_rope_t h, const Rope** out) {
    Rope* r = reinterpret_cast<Rope*>(h);
    if (!r) return fail(NXQ_ERR_ARG, "null rotation");
    std::lock_guard<std::mutex> lk(g_ropes_mu);
    if (!g_ropes.count(r)) return fail(NXQ_ERR_ARG, "rotation is not live (released or foreign)");
    *out = r;
    return NXQ_OK;
}

void ropes_shutdown() {
    std::lock_guard<std::mutex> lk(g_ropes_mu);
    for (Rope* r : g_ropes) {
        cudaFree(r->turns);
        delete r;
    }
    g_ropes.clear();
}

int check_heads(const char* what, const nxq_heads* h, int dtype) {
    if (!h || !h->dev) return fail(NXQ_ERR_ARG, "%s: null heads", what);
    if (h->heads < 1 || h->heads > 65536) return fail(NXQ_ERR_ARG, "%s: %d heads", what, h->heads);
    if (h->token_stride < 0 || h->head_stride < 0) return fail(NXQ_ERR_ARG, "%s: negative stride", what);
    if (!aligned_as(h->dev, dtype)) return fail(NXQ_ERR_ARG, "%s: not aligned to its type", what);
    return NXQ_OK;
}

int check_cache(const nxq_kv_cache* c) {
    if (!c || !c->k_dev || !c->v_dev) return fail(NXQ_ERR_ARG, "null cache");
    if (c->dtype != NXQ_F16 && c->dtype != NXQ_BF16) return fail(NXQ_ERR_ARG, "a cache of type %d (f16 or bf16)", c->dtype);
    if (c->pages < 1 || c->pages > 0x7FFFFFFF || c->page_size < 1 || c->heads < 1 || c->heads > 65536)
        return fail(NXQ_ERR_ARG, "a cache of %lld pages of %d slots, %d heads", (long long)c->pages, c->page_size, c->heads);
    if (c->head_dim < 8 || c->head_dim > 256 || c->head_dim % 8)
        return fail(NXQ_ERR_SHAPE, "a cache with heads of %d elements (a multiple of 8 up to 256)", c->head_dim);
    const int64_t s[3] = {c->page_stride, c->head_stride, c->slot_stride};
    for (int64_t v : s)
        if (v <= 0 || v % 8) return fail(NXQ_ERR_ARG, "a cache stride of %lld (positive multiples of 8)", (long long)v);
    if ((uintptr_t)c->k_dev % 16 || (uintptr_t)c->v_dev % 16) return fail(NXQ_ERR_ARG, "the cache is not aligned to 16 bytes");
    return NXQ_OK;
}

int check_batch(const nxq_kv_batch* b, int64_t T) {
    if (!b) return fail(NXQ_ERR_ARG, "null batch");
    if (b->sequences < 1 || b->sequences > 65536) return fail(NXQ_ERR_ARG, "%d sequences (1 to 65536)", b->sequences);
    if (T < 0 || T > kMaxTokens) return fail(NXQ_ERR_ARG, "%lld rows of new tokens (at most 2^30)", (long long)T);
    if (b->table_pages < 0 || b->table_pages > 0x7FFFFFFF || b->table_stride < 0)
        return fail(NXQ_ERR_ARG, "a block table of %lld pages per sequence, stride %lld", (long long)b->table_pages,
                    (long long)b->table_stride);
    if (!b->q_offsets_dev || !b->kv_lens_dev || (!b->block_table_dev && b->table_pages))
        return fail(NXQ_ERR_ARG, "batch: null offsets, lengths or block table");
    if (!aligned_4(b->q_offsets_dev) || !aligned_4(b->kv_lens_dev) || !aligned_4(b->block_table_dev))
        return fail(NXQ_ERR_ARG, "batch: an array is not aligned to its type");
    return NXQ_OK;
}

Batch make_batch(const nxq_kv_cache* c, const nxq_kv_batch* b, int64_t T) {
    const int64_t capacity = b->table_pages * c->page_size;
    return Batch{b->q_offsets_dev, b->kv_lens_dev, b->block_table_dev, b->table_stride,
                 capacity < kMaxTokens ? capacity : kMaxTokens, T, b->sequences, c->page_size, c->pages};
}

}  // namespace nxq

using namespace nxq;

extern "C" {

NXQ_API int nxq_rope_frequencies(int dims, double base, int scaling, double factor, double trained, double low,
                                 double high, double* inv_freq, float* scale) {
    if (!inv_freq) return fail(NXQ_ERR_ARG, "null frequencies");
    if (dims < 2 || dims > kMaxHeadDim || dims % 2) return fail(NXQ_ERR_ARG, "a rotation of %d elements (even, 2 to 512)", dims);
    if (scaling < NXQ_ROPE_PLAIN || scaling > NXQ_ROPE_BLEND) return fail(NXQ_ERR_ARG, "bad scaling %d", scaling);
    if (!(base > 1.0) || !std::isfinite(base)) return fail(NXQ_ERR_ARG, "a base of %g", base);
    const bool ramp = scaling == NXQ_ROPE_YARN || scaling == NXQ_ROPE_BLEND;
    if (scaling != NXQ_ROPE_PLAIN && (!(factor >= 1.0) || !std::isfinite(factor))) return fail(NXQ_ERR_ARG, "a factor of %g", factor);
    if (ramp) {
        if (low == 0.0 && high == 0.0) low = 1.0, high = scaling == NXQ_ROPE_YARN ? 32.0 : 4.0;
        if (!(trained >= 1.0) || !(low > 0.0) || !(high > low) || !std::isfinite(trained) || !std::isfinite(high))
            return fail(NXQ_ERR_ARG, "a ramp from %g to %g turns in %g positions", low, high, trained);
    }
    if (scaling == NXQ_ROPE_NTK) {
        if (dims == 2) return fail(NXQ_ERR_ARG, "one pair has no other base");
        base *= std::pow(factor, (double)dims / (dims - 2));
    }
    constexpr double kTurn = 6.283185307179586476925;
    // YaRN: the (fractional) index of the pair that makes `turns` turns in `trained` positions.
    auto index = [&](double turns) { return dims * std::log(trained / (turns * kTurn)) / (2.0 * std::log(base)); };
    for (int i = 0; i < dims / 2; ++i) {
        const double f = std::pow(base, -2.0 * i / dims);
        double keep = 1.0;  // share of the unscaled frequency
        if (scaling == NXQ_ROPE_LINEAR) keep = 0.0;
        if (scaling == NXQ_ROPE_YARN) {
            const double a = std::fmax(std::floor(index(high)), 0.0), b = std::fmin(std::ceil(index(low)), dims - 1.0);
            keep = 1.0 - std::fmin(std::fmax((i - a) / std::fmax(b - a, 0.001), 0.0), 1.0);
        }
        if (scaling == NXQ_ROPE_BLEND) keep = std::fmin(std::fmax((trained * f / kTurn - low) / (high - low), 0.0), 1.0);
        inv_freq[i] = scaling == NXQ_ROPE_PLAIN || scaling == NXQ_ROPE_NTK ? f : (1.0 - keep) * f / factor + keep * f;
    }
    if (scale) *scale = scaling == NXQ_ROPE_YARN ? (float)(0.1 * std::log(factor) + 1.0) : 1.0f;
    return NXQ_OK;
}

NXQ_API int nxq_rope_create(const double* inv_freq, int dims, int layout, float scale, nxq_rope_t* out) {
    if (!inv_freq || !out) return fail(NXQ_ERR_ARG, "null argument");
    if (dims < 2 || dims > kMaxHeadDim || dims % 2) return fail(NXQ_ERR_ARG, "a rotation of %d elements (even, 2 to 512)", dims);
    if (layout != NXQ_ROPE_HALF && layout != NXQ_ROPE_INTERLEAVED) return fail(NXQ_ERR_ARG, "bad layout %d", layout);
    if (!std::isfinite(scale)) return fail(NXQ_ERR_ARG, "a scale that is not finite");
    uint64_t turns[kMaxHeadDim / 2];
    for (int i = 0; i < dims / 2; ++i) {
        if (!std::isfinite(inv_freq[i])) return fail(NXQ_ERR_ARG, "frequency %d is not finite", i);
        // Extended precision: 64 bits of the fraction, as the fixed point holds.
        long double t = (long double)inv_freq[i] / 6.283185307179586476925286766559005768L;
        t -= floorl(t);
        const long double units = roundl(ldexpl(t, 64));
        turns[i] = units >= 0x1p64L ? 0 : (uint64_t)units;
    }
    if (int rc = context_ready()) return rc;
    Rope* r = new (std::nothrow) Rope();
    if (!r) return fail(NXQ_ERR_NOMEM, "host allocation failed");
    r->dims = dims;
    r->layout = layout;
    r->scale = scale;
    const size_t bytes = (size_t)(dims / 2) * sizeof(uint64_t);
    // The copy is waited for: streams that do not synchronize with the default one read it.
    cudaError_t e = cudaMalloc((void**)&r->turns, bytes);
    if (e == cudaSuccess && (e = cudaMemcpy(r->turns, turns, bytes, cudaMemcpyHostToDevice)) == cudaSuccess)
        e = cudaStreamSynchronize(cudaStreamLegacy);
    int rc = e == cudaSuccess ? NXQ_OK : cuda_fail(e, "rotation table");
    if (rc == NXQ_OK) {
        try {
            std::lock_guard<std::mutex> lk(g_ropes_mu);
            g_ropes.insert(r);
        } catch (const std::bad_alloc&) {
            rc = fail(NXQ_ERR_NOMEM, "host allocation failed");
        }
    }
    if (rc != NXQ_OK) {
        if (r->turns) cudaFree(r->turns);
        delete r;
        return rc;
    }
    *out = reinterpret_cast<nxq_rope_t>(r);
    return NXQ_OK;
}

NXQ_API int nxq_rope_release(nxq_rope_t h) {
    const Rope* r = nullptr;
    int rc = check_rope(h, &r);
    if (rc || (rc = context_ready())) return rc;
    {
        std::lock_guard<std::mutex> lk(g_ropes_mu);
        if (!g_ropes.erase(const_cast<Rope*>(r))) return fail(NXQ_ERR_ARG, "rotation is not live");
    }
    // Work queued on any stream may still read the table.
    cudaDeviceSynchronize();
    cudaFree(r->turns);
    delete r;
    return NXQ_OK;
}

NXQ_API int nxq_rope(nxq_rope_t rope, const void* positions_dev, int positions_type, int64_t T, int head_dim,
                     const nxq_heads* q, const float* q_norm, const nxq_heads* k, const float* k_norm, float eps,
                     int x_dtype, const nxq_heads* q_out, const nxq_heads* k_out, int y_dtype, void* stream) {
    if (!dtype_valid(x_dtype) || !dtype_valid(y_dtype)) return fail(NXQ_ERR_ARG, "bad dtype");
    if (T < 0 || T > 0x7FFFFFFF) return fail(NXQ_ERR_ARG, "%lld tokens", (long long)T);
    if (head_dim < 1 || head_dim > kMaxHeadDim) return fail(NXQ_ERR_ARG, "heads of %d elements (1 to 512)", head_dim);
    if (!!k != !!k_out) return fail(NXQ_ERR_ARG, "keys without outputs, or outputs without keys");
    if (positions_type != NXQ_I32 && positions_type != NXQ_I64) return fail(NXQ_ERR_ARG, "bad position type");
    if (T == 0) return NXQ_OK;
    int rc;
    if ((rc = check_heads("queries", q, x_dtype)) || (rc = check_heads("query outputs", q_out, y_dtype)) ||
        (rc = same_heads("queries", q, q_out, T, x_dtype, y_dtype)))
        return rc;
    if (k && ((rc = check_heads("keys", k, x_dtype)) || (rc = check_heads("key outputs", k_out, y_dtype)) ||
              (rc = same_heads("keys", k, k_out, T, x_dtype, y_dtype))))
        return rc;
    if (!aligned_4(q_norm) || !aligned_4(k_norm)) return fail(NXQ_ERR_ARG, "a norm is not aligned to its type");
    RopeParams p{};
    if (rope) {
        if (!positions_dev) return fail(NXQ_ERR_ARG, "null positions");
        if ((uintptr_t)positions_dev % (positions_type == NXQ_I64 ? 8 : 4)) return fail(NXQ_ERR_ARG, "positions are not aligned to their type");
        if ((rc = take_rope(rope, head_dim, &p))) return rc;
    }
    if ((rc = context_ready())) return rc;
    p.T = T;
    p.D = head_dim;
    p.eps = eps;
    p.in[0] = rows_of(q);
    p.in[1] = rows_of(k);
    p.out[0] = rows_of(q_out);
    p.out[1] = rows_of(k_out);
    p.norm[0] = q_norm;
    p.norm[1] = k_norm;
    p.x_dtype = x_dtype;
    p.y_dtype = y_dtype;
    p.positions = positions_dev;
    p.positions_type = positions_type;
    const cudaError_t e = launch_rope(p, false, (cudaStream_t)stream);
    return e == cudaSuccess ? NXQ_OK : cuda_fail(e, "rotation launch");
}

NXQ_API int nxq_kv_append(const nxq_kv_cache* cache, const nxq_kv_batch* batch, int64_t T, const nxq_heads* k,
                          const nxq_heads* v, const float* k_norm, nxq_rope_t rope, const nxq_heads* q,
                          const float* q_norm, float eps, int x_dtype, const nxq_heads* q_out, int y_dtype,
                          void* stream) {
    int rc;
    if (!dtype_valid(x_dtype) || !dtype_valid(y_dtype)) return fail(NXQ_ERR_ARG, "bad dtype");
    if ((rc = check_cache(cache)) || (rc = check_batch(batch, T))) return rc;
    if (!!q != !!q_out) return fail(NXQ_ERR_ARG, "queries without outputs, or outputs without queries");
    if (T == 0) return NXQ_OK;
    if ((rc = check_heads("keys", k, x_dtype)) || (rc = check_heads("values", v, x_dtype))) return rc;
    if (k->heads != cache->heads || v->heads != cache->heads)
        return fail(NXQ_ERR_SHAPE, "%d key and %d value heads for a cache of %d", k->heads, v->heads, cache->heads);
    if (q && ((rc = check_heads("queries", q, x_dtype)) || (rc = check_heads("query outputs", q_out, y_dtype)) ||
              (rc = same_heads("queries", q, q_out, T, x_dtype, y_dtype))))
        return rc;
    if (!aligned_4(q_norm) || !aligned_4(k_norm)) return fail(NXQ_ERR_ARG, "a norm is not aligned to its type");
    RopeParams p{};
    if ((rc = take_rope(rope, cache->head_dim, &p))) return rc;
    if ((rc = context_ready())) return rc;
    p.T = T;
    p.D = cache->head_dim;
    p.eps = eps;
    p.in[0] = rows_of(q);
    p.in[1] = rows_of(k);
    p.in[2] = rows_of(v);
    p.out[0] = rows_of(q_out);
    p.out[1] = HeadRows{cache->k_dev, cache->heads, 0, cache->head_stride};
    p.out[2] = HeadRows{cache->v_dev, cache->heads, 0, cache->head_stride};
    p.norm[0] = q_norm;
    p.norm[1] = k_norm;
    p.x_dtype = x_dtype;
    p.y_dtype = y_dtype;
    p.c_dtype = cache->dtype;
    p.b = make_batch(cache, batch, T);
    p.page_stride = cache->page_stride;
    p.slot_stride = cache->slot_stride;
    const cudaError_t e = launch_rope(p, true, (cudaStream_t)stream);
    return e == cudaSuccess ? NXQ_OK : cuda_fail(e, "append launch");
}

}  // extern "C"
