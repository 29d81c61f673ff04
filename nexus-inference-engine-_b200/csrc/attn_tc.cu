// Attention over the paged cache for many rows per sequence and key head (chunks and
// whole prompts), on tcgen05 / TMEM.
//
// A persistent grid of one CTA per SM, each with an equal share of the call's units
// (attn_plan.cuh): an item is 256 rows of one (sequence, key head) as two tiles of 128, a
// unit one block of 128 keys with its values, which both tiles share.  Roles:
//   warp 0      producer: keys and values by TMA, one box per page (or part of one) and 64
//               elements, straight from the scattered pages into 128-byte-swizzled
//               blocks [64 elements][128 keys]; five of them in a ring
//   warp 1      issues tcgen05.mma: S_t = Q_t K^T (fp32 in TMEM), O_t += P_t V with P_t
//               from TMEM and V as it lies (its head elements contiguous)
//   warps 2, 3  bring an item's queries into shared memory, and look through the values of
//               units that not all rows see for any that is infinite or NaN (they take
//               part in handing every block back: a wait by phase parity must see every phase)
//   warps 4-7   softmax of tile 0, 8-11 of tile 1: a thread per row, so a row's maximum
//               and sum need no shuffles; reads S_t, writes P_t over it, corrects O_t
//               when the maximum in use is raised, and stores the outputs
// While one tile's weights are computed, the other's products run: S_t of a unit is
// issued right after O_t of the one before.  tcgen05.mma of one thread run in order, so
// S_t being there tells that O_t is up to date, and the next S_t may be issued over a
// P_t that is still to be read.
//
// Bound by the exponentials and the products alike: a unit is 4 x 512 cycles of MMA (D =
// 128) and 2 x 128 x 128 exponentials, 16 a cycle, 2048 cycles.
//
// Weights are relative to a maximum that is raised only when a score passes it by
// 2^8 (so O_t is seldom read back), f16 ones times 2^7; rounding and SPLIT as in
// attn_mma.cu.  Every wait is bounded (sm100_ptx.cuh).
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "attn_plan.cuh"
#include "qmm_gemm.h"
#include "sm100_ptx.cuh"

namespace nxq {

namespace {

using namespace attn;

constexpr int kThreads = 384, kTile = 128, kRows = 2 * kTile, kKeys = 128;
constexpr int kWarpProducer = 0, kWarpMma = 1, kWarpHelper0 = 2, kHelpers = 64, kWarpSoft0 = 4;
constexpr int kSlots = 5;
constexpr uint32_t kTmemCols = 512;
constexpr int kColS = 0, kColO = 2 * kKeys;  // S_t at kColS + 128 t, O_t at kColO + 128 t
constexpr float kSlack = 8.0f;
constexpr int kChunkBytes = kKeys * 128;  // 64 elements of 128 keys (or rows)

template <int DP>
struct Shape {
    static constexpr int kChunks = DP / 64;
    static constexpr int kBlock = kChunks * kChunkBytes;  // 128 keys, values, or rows of queries
    static constexpr int kSmem = 1024 + 2 * kBlock + kSlots * kBlock + 512;
    static_assert(sizeof(PlanSmem) <= kSlots * kBlock, "the plan is made where the ring will be");
    static_assert(kSmem <= 227 * 1024, "");
};

__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint64_t pair(float a, float b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float2 unpair(uint64_t v) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
    return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
template <bool BF16>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
    if constexpr (BF16) {
        const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&v);
    } else {
        const __half2 v = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&v);
    }
}
template <bool BF16>
__device__ __forceinline__ float value_of(uint32_t bits) {
    if constexpr (BF16) return __uint_as_float(bits << 16);
    return __half2float(__ushort_as_half((unsigned short)bits));
}
template <bool BF16>
__device__ __forceinline__ bool not_finite(uint32_t bits) {
    constexpr uint32_t m = BF16 ? 0x7F80u : 0x7C00u;
    return (bits & m) == m;
}

// A and B of the same 16-bit type, fp32 accumulation; b_mn: B's N elements are contiguous.
__host__ __device__ constexpr uint32_t idesc16(bool bf16, int n, bool b_mn) {
    return (1u << 4) | ((bf16 ? 1u : 0u) << 7) | ((bf16 ? 1u : 0u) << 10) | ((b_mn ? 1u : 0u) << 16) |
           ((uint32_t)(n >> 3) << 17) | ((uint32_t)(kTile >> 4) << 24);
}

// Position in the ring of key and value blocks, and the parity of its current use.
struct Ring {
    int i = 0;
    uint32_t ph = 0;
    __device__ __forceinline__ void next() {
        if (++i == kSlots) {
            i = 0;
            ph ^= 1u;
        }
    }
};

// Whether there are keys in a unit that a row of the item does not see (a box brings a
// page's slots whether any row sees them or not).
__device__ __forceinline__ bool mixed(const AttnParams& p, const Item& it, int j0) { return !all_see(p, it, j0, kKeys); }

template <bool BF16, bool SPLIT, int DP>
__global__ void __launch_bounds__(kThreads, 1)
    attn_tc_kernel(const __grid_constant__ AttnParams p, const __grid_constant__ CUtensorMap kmap,
                   const __grid_constant__ CUtensorMap vmap, const int box) {
    using Sh = Shape<DP>;
    using W = Walk<kRows, kKeys>;
    constexpr float kShift = BF16 ? 0.0f : 7.0f;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* const smem = smem_raw + ((1024 - (ptx::smem_addr(smem_raw) & 1023)) & 1023);
    uint8_t* const qs = smem;
    uint8_t* const ring = qs + 2 * Sh::kBlock;
    uint64_t* const bars = reinterpret_cast<uint64_t*>(ring + kSlots * Sh::kBlock);
    uint64_t* const kv_full = bars;
    uint64_t* const kv_empty = kv_full + kSlots;
    uint64_t* const looked = kv_empty + kSlots;  // [slot] the helpers have looked through its values
    uint64_t* const q_full = looked + kSlots;
    uint64_t* const q_empty = q_full + 1;
    uint64_t* const s_full = q_empty + 1;  // [tile]
    uint64_t* const p_full = s_full + 2;
    uint64_t* const o_full = p_full + 2;
    uint64_t* const meet = o_full + 2;  // the softmax warps: of tile 0 alone, of both
    uint64_t* const drain = meet + 2;
    uint32_t* const tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
    volatile int* const abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    volatile int* const found = abort_flag + 1;     // [slot] its values are not all finite
    volatile int* const started = found + kSlots;   // [tile] O_t was set before its first product

    PlanSmem& plan = *reinterpret_cast<PlanSmem*>(ring);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const ptx::WaitCtl ctl{abort_flag, p.status};
    if (threadIdx.x == 0) {
        for (int i = 0; i < kSlots; ++i) {
            ptx::mbar_init(&kv_full[i], 1);
            ptx::mbar_init(&kv_empty[i], 1 + kHelpers / 32);  // the products, and both helpers
            ptx::mbar_init(&looked[i], kHelpers / 32);
            found[i] = 0;
        }
        ptx::mbar_init(q_full, kHelpers / 32);
        ptx::mbar_init(q_empty, 1);
        for (int t = 0; t < 2; ++t) {
            ptx::mbar_init(&s_full[t], 1);
            ptx::mbar_init(&p_full[t], 4);
            ptx::mbar_init(&o_full[t], 1);
            ptx::mbar_init(&meet[t], t ? 8 : 4);
            started[t] = 0;
        }
        ptx::mbar_init(drain, 1);
        *abort_flag = 0;
        ptx::fence_mbar_init();
    }
    __syncwarp();
    if (warp == kWarpProducer) {
        ptx::tmem_alloc(tmem_slot, kTmemCols);
        ptx::tmem_relinquish();
    }
    ptx::tc_fence_before();
    __syncthreads();
    ptx::tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    // The join kernel may start its set-up when all before this kernel is complete.
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

    plan_total<kRows, kKeys, kThreads>(p, plan);
    const long long total = plan.total, first = run_start(total, blockIdx.x, gridDim.x);
    const long long units = run_start(total, blockIdx.x + 1, gridDim.x) - first;
    W w;
    bool go = units > 0;
    if (go) {
        plan_locate<kRows, kKeys, kThreads>(p, plan, first);
        w.start(p, plan, units);
    }
    __syncthreads();  // the plan has been read: its memory is the ring's

    if (warp == kWarpProducer) {
        if (lane == 0) {
            ptx::prefetch_tmap(&kmap);
            ptx::prefetch_tmap(&vmap);
        }
        // The plan, and the cache, were written through the generic proxy; TMA works through the async one.
        asm volatile("fence.proxy.async;" ::: "memory");
        Ring r;
        uint32_t issued = 0;
        bool ok = true;
        const int boxes = kKeys / box, b = lane % boxes, chunk = lane / boxes;
        const bool mine = chunk < Sh::kChunks;
        while (go && ok) {
            const int32_t* const table = p.b.table + w.s * p.b.table_stride;
            for (int u = 0; u < w.count && ok; ++u) {
                const int j = w.key0(u) + b * box;
                // Boxes without a key that a row sees read nothing: a page of -1 gives zeros.
                const bool want = mine && j <= w.it.p_hi &&
                                  (p.window <= 0 || j + box - 1 > w.it.p_lo - p.window || j < p.sinks);
                int page = -1, slot = 0;
                if (want) {
                    const int n = p.page_shift >= 0 ? j >> p.page_shift : j / p.b.page;
                    slot = j - n * p.b.page;
                    page = table[n];
                    if (page < 0 || page >= p.b.pages) {
                        raise_index(p.status, kIndexPage);
                        page = -1;
                    }
                }
#pragma unroll
                for (int kv = 0; kv < 2; ++kv) {
                    ok = ok && ptx::warp_mbar_wait(&kv_empty[r.i], r.ph ^ 1u, ctl, 61);
                    if (!ok) continue;
                    if (lane == 0) ptx::mbar_arrive_expect_tx(&kv_full[r.i], Sh::kBlock);
                    __syncwarp();
                    if (mine)
                        ptx::tma_load_4d(ring + r.i * Sh::kBlock + chunk * kChunkBytes + b * box * 128, kv ? &vmap : &kmap,
                                         64 * chunk, slot, w.head, page, &kv_full[r.i]);
                    r.next();
                    ++issued;
                }
            }
            go = w.next(p);
        }
        // Do not leave with copies in flight (bounded, ignoring the abort flag).
        for (uint32_t k = issued >= kSlots ? issued - kSlots : 0; k < issued; ++k) {
            const long long t0 = clock64();
            while (!ptx::mbar_try_wait(&kv_full[k % kSlots], (k / kSlots) & 1) && clock64() - t0 < ptx::kWaitCycles) {
            }
        }
    } else if (warp == kWarpMma) {
        const uint64_t qd = ptx::desc_sw128_kmajor(ptx::smem_addr(qs)), kd = ptx::desc_sw128_kmajor(ptx::smem_addr(ring));
        const uint64_t vd = ptx::desc_sw128_mnmajor(ptx::smem_addr(ring), kChunkBytes);
        constexpr uint32_t kIdS = idesc16(BF16, kKeys, false), kIdO = idesc16(BF16, DP, true);
        // S_t = Q_t K^T, from the block in slot i.
        const bool lead = ptx::elect_one();  // one lane issues, and commits what it issued
        auto scores = [&](int t, int i) {
            if (!lead) return;
            const uint64_t a = qd + ((uint32_t)(t * Sh::kBlock) >> 4), b = kd + ((uint32_t)(i * Sh::kBlock) >> 4);
#pragma unroll
            for (int c = 0; c < Sh::kChunks; ++c)
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    ptx::mma_ss_f16(tmem + kColS + kKeys * t, a + c * (kChunkBytes >> 4) + 2 * k, b + c * (kChunkBytes >> 4) + 2 * k,
                                    kIdS, c || k ? 1u : 0u);
        };
        // O_t (+)= P_t V, from the block in slot i.
        auto outputs = [&](int t, int i, uint32_t accumulate) {
            if (!lead) return;
            const uint64_t b = vd + ((uint32_t)(i * Sh::kBlock) >> 4);
#pragma unroll
            for (int h = 0; h < (SPLIT ? 2 : 1); ++h)
#pragma unroll
                for (int k = 0; k < kKeys / 16; ++k)
                    ptx::mma_ts_f16(tmem + kColO + 128 * t, tmem + kColS + kKeys * t + 64 * h + 8 * k, b + k * (2048 >> 4), kIdO,
                                    h || k ? 1u : accumulate);
        };
        auto commit = [&](uint64_t* bar) {
            if (lead) ptx::mma_commit(bar);
            __syncwarp();
        };
        Ring kr, vr;   // the next block of keys, and of values
        vr.next();
        uint32_t q_ph = 0, p_ph[2] = {0, 0};
        bool ok = true;
        auto two = [](const W& x) { return x.it.rows > kTile; };
        auto queries = [&]() {  // of the next piece
            ok = ok && ptx::warp_mbar_wait(q_full, q_ph, ctl, 62);
            q_ph ^= 1u;
        };
        int tiles = 0;
        if (go) {
            queries();
            ok = ok && ptx::warp_mbar_wait(&kv_full[kr.i], kr.ph, ctl, 63);
            ptx::tc_fence_after();
            tiles = two(w) ? 2 : 1;
            if (ok)
                for (int t = 0; t < tiles; ++t) {
                    scores(t, kr.i);
                    __syncwarp();
                    commit(&s_full[t]);
                }
            if (ok) {
                commit(&kv_empty[kr.i]);
                if (w.count == 1) commit(q_empty);
            }
            kr.next();
            kr.next();
        }
        while (go && ok) {
            for (int u = 0; u < w.count && ok; ++u) {
                const bool last = u + 1 == w.count;
                W after = w;
                const bool more = !last || after.next(p);
                const int next_tiles = !more ? 0 : last ? (two(after) ? 2 : 1) : tiles;
                if (!(ok = ptx::warp_mbar_wait(&kv_full[vr.i], vr.ph, ctl, 64))) break;
                bool keys = false;  // the next unit's keys (and queries) are there
                for (int t = 0; t < 2 && ok; ++t) {
                    if (t < tiles) {
                        if (!(ok = ptx::warp_mbar_wait(&p_full[t], p_ph[t], ctl, 65))) break;
                        p_ph[t] ^= 1u;
                        ptx::tc_fence_after();
                        outputs(t, vr.i, u > 0 || started[t] ? 1u : 0u);
                        __syncwarp();
                        if (last) commit(&o_full[t]);
                    }
                    if (t == tiles - 1) commit(&kv_empty[vr.i]);
                    if (t < next_tiles) {
                        if (!keys) {
                            if (last) queries();
                            ok = ok && ptx::warp_mbar_wait(&kv_full[kr.i], kr.ph, ctl, 66);
                            if (!ok) break;
                            ptx::tc_fence_after();
                            keys = true;
                        }
                        scores(t, kr.i);
                        __syncwarp();
                        commit(&s_full[t]);
                        if (t == next_tiles - 1) {
                            commit(&kv_empty[kr.i]);
                            if ((last ? after.count : w.count - u - 1) == 1) commit(q_empty);
                        }
                    }
                }
                if (more) {
                    kr.next();
                    kr.next();
                }
                vr.next();
                vr.next();
                if (last) {
                    go = more;
                    w = after;
                    tiles = next_tiles;
                    break;
                }
            }
        }
        commit(drain);
        const long long t0 = clock64();
        while (!ptx::mbar_try_wait(drain, 0) && clock64() - t0 < ptx::kWaitCycles) {
        }
    } else if (warp < kWarpSoft0) {
        // Helpers: warp h brings tile h's queries.
        const int tile = warp - kWarpHelper0, tid = threadIdx.x - 32 * kWarpHelper0;
        bool ok = true;
        uint32_t q_ph = 0;
        bool first_piece = true;
        Ring r;
        while (go && ok) {
            if (!first_piece) {
                ok = ptx::warp_mbar_wait(q_empty, q_ph, ctl, 67);
                q_ph ^= 1u;
                if (!ok) break;
            }
            first_piece = false;
            const int64_t row0 = (int64_t)w.item * kRows + tile * kTile;
            const int rows = w.it.rows - tile * kTile;
            if (rows > 0) {
                int64_t at[4];  // of rows lane, lane + 32, ...: their offset in q, -1 behind the last
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int64_t f = row0 + 32 * i + lane, t = f / p.G;
                    at[i] = 32 * i + lane < rows ? (w.q.q0 + t) * p.q_token + ((int64_t)w.head * p.G + (f - t * p.G)) * p.q_head : -1;
                }
                uint8_t* const dst = qs + tile * Sh::kBlock;
                const uint32_t dst32 = ptx::smem_addr(dst);
                constexpr int kPer = DP / 8;  // 16-byte pieces of a row
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll 4
                    for (int e = lane; e < 32 * kPer; e += 32) {
                        const int r0 = e / kPer, c = e % kPer;
                        const int64_t a = __shfl_sync(0xFFFFFFFFu, at[i], r0);
                        const int row = 32 * i + r0;
                        const uint32_t o = (c >> 3) * kChunkBytes + row * 128 + (((c & 7) ^ (row & 7)) << 4);
                        const bool read = a >= 0 && c * 8 < p.D;
                        const uint16_t* src = static_cast<const uint16_t*>(p.q) + (read ? a + c * 8 : 0);
                        if (p.q_vec) {
                            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst32 + o), "l"(src), "r"(read ? 16 : 0)
                                         : "memory");
                        } else {
                            uint32_t h[4] = {0u, 0u, 0u, 0u};
                            if (read)
#pragma unroll
                                for (int k = 0; k < 4; ++k) h[k] = (uint32_t)src[2 * k] | (uint32_t)src[2 * k + 1] << 16;
                            *reinterpret_cast<uint4*>(dst + o) = make_uint4(h[0], h[1], h[2], h[3]);
                        }
                    }
                asm volatile("cp.async.wait_all;" ::: "memory");
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            }
            __syncwarp();
            if (lane == 0) ptx::mbar_arrive(q_full);
            for (int u = 0; u < w.count && ok; ++u) {
                const bool look = mixed(p, w.it, w.key0(u));
                for (int kv = 0; kv < 2 && ok; ++kv, r.next()) {
                    if (!(ok = ptx::warp_mbar_wait(&kv_full[r.i], r.ph, ctl, 68))) break;
                    if (kv && look) {
                        bool bad = false;
#pragma unroll 4
                        for (int i = tid; i < Sh::kBlock / 16; i += kHelpers) {
                            const uint4 v = *reinterpret_cast<const uint4*>(ring + r.i * Sh::kBlock + 16 * i);
                            const uint32_t x[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                            for (int k = 0; k < 4; ++k) bad |= not_finite<BF16>(x[k] & 0xFFFFu) || not_finite<BF16>(x[k] >> 16);
                        }
                        bad = __any_sync(0xFFFFFFFFu, bad);
                        if (lane == 0) {
                            if (bad) found[r.i] = 1;
                            ptx::mbar_arrive(&looked[r.i]);
                        }
                    }
                    __syncwarp();
                    if (lane == 0) ptx::mbar_arrive(&kv_empty[r.i]);
                }
            }
            go = w.next(p);
        }
    } else {
        // Softmax of tile t: a thread per row.
        const int t = (warp - kWarpSoft0) >> 2, quad = warp & 3, row = quad * 32 + lane;
        const uint32_t lanes = (uint32_t)(quad * 32) << 16;
        const uint32_t ts = tmem + lanes + kColS + kKeys * t, to = tmem + lanes + kColO + 128 * t;
        uint32_t s_ph = 0, o_ph = 0, meet_ph[2] = {0, 0}, looked_ph = 0;  // looked_ph: a bit per slot
        Ring r;
        r.next();  // values
        bool ok = true;
        while (go && ok) {
            const int tiles = w.it.rows > kTile ? 2 : 1;
            if (t >= tiles) {  // (the ring moves on, and so do the units looked through)
                for (int u = 0; u < w.count; ++u, r.next(), r.next())
                    if (mixed(p, w.it, w.key0(u))) looked_ph ^= 1u << r.i;
                go = w.next(p);
                continue;
            }
            const int64_t flat = (int64_t)w.item * kRows + t * kTile + row, tok = flat / p.G;
            const int head = w.head * p.G + (int)(flat - tok * p.G);
            const bool mine = t * kTile + row < w.it.rows;
            const int pos = mine ? w.q.len - w.q.n + (int)tok : -1;
            float m = -INFINITY, l = 0.0f;
            for (int u = 0; u < w.count; ++u, r.next(), r.next()) {
                const int j0 = w.key0(u);
                if (!(ok = ptx::warp_mbar_wait(&s_full[t], s_ph, ctl, 69))) break;
                s_ph ^= 1u;
                ptx::tc_fence_after();
                uint32_t s[4][32];
#pragma unroll
                for (int i = 0; i < 4; ++i) ptx::tmem_ld32(ts + 32 * i, s[i]);
                ptx::tmem_wait_ld();
                const bool hidden = mixed(p, w.it, j0);
                if (hidden) {
                    const int hi = pos - j0, lo = p.window > 0 ? pos - p.window - j0 : -1, sk = p.sinks - j0;
#pragma unroll
                    for (int i = 0; i < 4; ++i)
#pragma unroll
                        for (int k = 0; k < 32; ++k) {
                            const int j = 32 * i + k;
                            if (j > hi || (j <= lo && j >= sk)) s[i][k] = 0xFF800000u;
                        }
                }
                float top[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    top[i] = __uint_as_float(s[i][0]);
#pragma unroll
                    for (int k = 1; k < 32; k += 1) top[i] = fmaxf(top[i], __uint_as_float(s[i][k]));
                }
                const float now = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])) * p.c;
                const bool raise = now > m + kSlack || (m == -INFINITY && now > -INFINITY);
                if (__any_sync(0xFFFFFFFFu, raise)) {
                    const float to_m = fmaxf(m, now), f = m == -INFINITY ? 0.0f : exp2_fast(m - to_m);
                    m = to_m;
                    l *= f;
                    if (u > 0) {
#pragma unroll 1
                        for (int d = 0; d < DP; d += 16) {
                            uint32_t o[16];
                            ptx::tmem_ld16(to + d, o);
                            ptx::tmem_wait_ld();
#pragma unroll
                            for (int k = 0; k < 16; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * f);
                            ptx::tmem_st16(to + d, o);
                        }
                        ptx::tmem_wait_st();
                    }
                }
                const float base = m == -INFINITY ? 0.0f : m - kShift;
                // A value that not all rows see may be infinite or NaN, and a weight of zero must
                // not meet it: such elements are added to the rows that see them here, and are zeros
                // to the product.
                if (hidden) {
                    if (!(ok = ptx::warp_mbar_wait(&looked[r.i], (looked_ph >> r.i) & 1u, ctl, 70))) break;
                    looked_ph ^= 1u << r.i;
                    if (found[r.i]) {
                        uint8_t* const vs = ring + r.i * Sh::kBlock;
                        auto value = [&](int k, int d) {
                            return reinterpret_cast<uint16_t*>(vs + (d >> 6) * kChunkBytes + k * 128 +
                                                               ((((d >> 3) & 7) ^ (k & 7)) << 4)) + (d & 7);
                        };
                        if (u == 0) {
#pragma unroll 1
                            for (int d = 0; d < DP; ++d) ptx::tmem_st1(to + d, 0u);
                            ptx::tmem_wait_st();
                            if (row == 0) started[t] = 1;
                        }
#pragma unroll 1
                        for (int k = 0; k < kKeys; ++k)
#pragma unroll 1
                            for (int d = 0; d < DP; ++d) {
                                const uint32_t bits = *value(k, d);
                                if (!not_finite<BF16>(bits)) continue;  // (the same in all lanes)
                                float x = __uint_as_float(ptx::tmem_ld1(ts + k)), o = __uint_as_float(ptx::tmem_ld1(to + d));
                                ptx::tmem_wait_ld();
                                if (sees(p, pos, j0 + k)) o += exp2_fast(fmaf(x, p.c, -base)) * value_of<BF16>(bits);
                                ptx::tmem_st1(to + d, __float_as_uint(o));
                                ptx::tmem_wait_st();
                            }
                        // Everybody has read them; then everybody has cleared them.
                        for (int step = 0; step < 2 && ok; ++step) {
                            __syncwarp();
                            if (lane == 0) ptx::mbar_arrive(&meet[tiles - 1]);
                            ok = ptx::warp_mbar_wait(&meet[tiles - 1], meet_ph[tiles - 1], ctl, 71);
                            meet_ph[tiles - 1] ^= 1u;
                            if (step == 0 && ok) {
                                for (int i = threadIdx.x - 32 * kWarpSoft0; i < Sh::kBlock / 2; i += tiles * kTile) {
                                    uint16_t* e = reinterpret_cast<uint16_t*>(vs) + i;
                                    if (not_finite<BF16>(*e)) *e = 0;
                                }
                                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                            }
                        }
                        if (!ok) break;
                        if (warp == kWarpSoft0 && lane == 0) found[r.i] = 0;
                    }
                }
                const uint64_t c2 = pair(p.c, p.c), b2 = pair(-base, -base);
                uint64_t sum[4] = {0ull, 0ull, 0ull, 0ull};
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    uint32_t hi[16], lo[SPLIT ? 16 : 1];
#pragma unroll
                    for (int k = 0; k < 16; ++k) {
                        float2 x = unpair(fma2(pair(__uint_as_float(s[i][2 * k]), __uint_as_float(s[i][2 * k + 1])), c2, b2));
                        x.x = exp2_fast(x.x);
                        x.y = exp2_fast(x.y);
                        sum[k & 3] = add2(sum[k & 3], pair(x.x, x.y));
                        hi[k] = pack2<BF16>(x.x, x.y);
                        if constexpr (SPLIT)
                            lo[k] = pack2<BF16>(x.x - value_of<BF16>(hi[k] & 0xFFFFu), x.y - value_of<BF16>(hi[k] >> 16));
                    }
                    ptx::tmem_st16(ts + 16 * i, hi);
                    if constexpr (SPLIT) ptx::tmem_st16(ts + 64 + 16 * i, lo);
                }
                ptx::tmem_wait_st();
                ptx::tc_fence_before();
                __syncwarp();
                if (lane == 0) ptx::mbar_arrive(&p_full[t]);
                const float2 a = unpair(add2(add2(sum[0], sum[1]), add2(sum[2], sum[3])));
                l += a.x + a.y;
            }
            if (!ok) break;
            if (!(ok = ptx::warp_mbar_wait(&o_full[t], o_ph, ctl, 72))) break;
            o_ph ^= 1u;
            ptx::tc_fence_after();
            if (row == 0) started[t] = 0;
            const bool whole = w.whole();
            float* const part = whole ? nullptr : p.part + (2ll * blockIdx.x + w.slot()) * part_floats(kRows, p.D);
            const float f = !whole ? 1.0f : l == 0.0f ? 0.0f : 1.0f / l;
            const int64_t token = w.q.q0 + tok, at = token * p.o_token + head * p.o_head;
#pragma unroll 1
            for (int d = 0; d < DP && d < p.D; d += 16) {
                uint32_t o[16];
                ptx::tmem_ld16(to + d, o);
                ptx::tmem_wait_ld();
                if (!mine) continue;
                float v[16];
#pragma unroll
                for (int k = 0; k < 16; ++k) v[k] = __uint_as_float(o[k]) * f;
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int e = d + 8 * h;
                    if (e >= p.D) continue;
                    const float* x = v + 8 * h;
                    if (!whole || p.y_dtype == NXQ_F32) {
                        float* q = whole ? static_cast<float*>(p.out) + at + e : part + (int64_t)(t * kTile + row) * p.D + e;
                        if (!whole || p.o_vec) {
                            *reinterpret_cast<float4*>(q) = make_float4(x[0], x[1], x[2], x[3]);
                            *reinterpret_cast<float4*>(q + 4) = make_float4(x[4], x[5], x[6], x[7]);
                        } else {
#pragma unroll
                            for (int k = 0; k < 8; ++k) q[k] = x[k];
                        }
                    } else {
                        uint32_t y[4];
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            y[k] = p.y_dtype == NXQ_BF16 ? pack2<true>(x[2 * k], x[2 * k + 1]) : pack2<false>(x[2 * k], x[2 * k + 1]);
                        uint16_t* q = static_cast<uint16_t*>(p.out) + at + e;
                        if (p.o_vec) {
                            *reinterpret_cast<uint4*>(q) = make_uint4(y[0], y[1], y[2], y[3]);
                        } else {
#pragma unroll
                            for (int k = 0; k < 8; ++k) q[k] = (uint16_t)(y[k >> 1] >> (16 * (k & 1)));
                        }
                    }
                }
            }
            if (mine && !whole) {
                part[(int64_t)kRows * p.D + t * kTile + row] = m == -INFINITY ? m : m - kShift;
                part[(int64_t)kRows * p.D + kRows + t * kTile + row] = l;
            }
            if (mine && whole && p.lse)
                p.lse[token * ((int64_t)p.Hk * p.G) + head] =
                    l == 0.0f ? -INFINITY : (m - kShift + log2f(l)) * 0.6931471805599453f;
            ptx::tc_fence_before();
            go = w.next(p);
        }
    }

    ptx::tc_fence_before();
    __syncthreads();
    if (warp == kWarpProducer) {
        ptx::tc_fence_after();
        ptx::tmem_dealloc(tmem, kTmemCols);
    }
}

template <int DP>
auto* kernel_of(bool bf16, bool split) {
    return bf16 ? (split ? attn_tc_kernel<true, true, DP> : attn_tc_kernel<true, false, DP>)
                : (split ? attn_tc_kernel<false, true, DP> : attn_tc_kernel<false, false, DP>);
}

template <int DP>
int set_attr() {
    for (int i = 0; i < 4; ++i) {
        const cudaError_t e = cudaFuncSetAttribute(kernel_of<DP>(i & 1, i & 2), cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                   Shape<DP>::kSmem);
        if (e != cudaSuccess) return cuda_fail(e, "cudaFuncSetAttribute (attn_tc)");
    }
    return NXQ_OK;
}

// Rows of a box: the largest power of two that divides a page and a unit.
int box_rows(int page) {
    int b = 1;
    while (b < kKeys && page % (2 * b) == 0) b *= 2;
    return b;
}

int cache_map(CUtensorMap* map, const nxq_kv_cache* c, const void* base, int box) {
    const uint64_t dims[4] = {(uint64_t)c->head_dim, (uint64_t)c->page_size, (uint64_t)c->heads, (uint64_t)c->pages};
    const uint64_t strides[3] = {2 * (uint64_t)c->slot_stride, 2 * (uint64_t)c->head_stride, 2 * (uint64_t)c->page_stride};
    const uint32_t boxes[4] = {64, (uint32_t)box, 1, 1};
    if (const int e = tensor_map_16(map, c->dtype == NXQ_BF16, base, 4, dims, strides, boxes))
        return fail(NXQ_ERR_CUDA, "cuTensorMapEncodeTiled failed (%d)", e);
    return NXQ_OK;
}

}  // namespace

int attn_tc_init() {
    int rc;
    if ((rc = set_attr<64>()) || (rc = set_attr<128>())) return rc;
    return NXQ_OK;
}

// Pages of whole groups of 8 slots (a box then starts at a swizzle atom), heads of 64 to 128
// elements, strides that a tensor map takes.
bool attn_tc_supported(const nxq_kv_cache* c) {
    const int64_t far = (int64_t)1 << 38;
    return tensor_maps() && c->page_size % 8 == 0 && c->head_dim >= 64 && c->head_dim <= 128 && c->page_stride < far &&
           c->head_stride < far && c->slot_stride < far;
}

int attn_tc_rows() { return kRows; }
unsigned attn_tc_grid() { return (unsigned)context_sm_count(); }

int attn_tc(const AttnParams& p, const nxq_kv_cache* cache, cudaStream_t st) {
    const int box = box_rows(cache->page_size);
    CUtensorMap k, v;
    int rc;
    if ((rc = cache_map(&k, cache, cache->k_dev, box)) || (rc = cache_map(&v, cache, cache->v_dev, box))) return rc;
    const bool bf = cache->dtype == NXQ_BF16, split = p.y_dtype == NXQ_F32;
    note_launches(1);
    const cudaError_t e =
        p.D <= 64 ? launch_overlapped(kernel_of<64>(bf, split), attn_tc_grid(), kThreads, Shape<64>::kSmem, st, p, k, v, box)
                  : launch_overlapped(kernel_of<128>(bf, split), attn_tc_grid(), kThreads, Shape<128>::kSmem, st, p, k, v, box);
    if (e != cudaSuccess) return cuda_fail(e, "attention launch (tcgen05)");
    const cudaError_t j = launch_attn_join(p, kRows, kKeys, attn_tc_grid(), st);
    return j == cudaSuccess ? NXQ_OK : cuda_fail(j, "attention join launch");
}

}  // namespace nxq
