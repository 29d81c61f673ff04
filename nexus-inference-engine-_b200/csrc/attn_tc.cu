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
//               from TMEM and V as it lies (its head elements contiguous): the products of 64 keys
//               as soon as their weights are there, then the other 64's and the next scores
//   warp 2      brings an item's queries into shared memory, and looks through the values of
//               units that not all rows see for any that is infinite or NaN, and clears those that
//               no row sees (it takes part in handing every block back: a wait by phase parity
//               must see every phase)
//   warps 4-7   softmax of tile 0, 8-11 of tile 1: a thread per row, so a row's maximum
//               and sum need no shuffles; reads S_t, writes P_t over it, corrects O_t
//               when the maximum in use is raised, and stores the outputs
// (Warp 3 only fills the group of four.)  S_t of a unit is issued behind O_t of the unit before
// - tcgen05.mma of one thread run in order, so it may go over a P_t still to be read - and across
// items as well.  One tile's softmax runs beside the other's products.
//
// What bounds it (one prompt of 8192 tokens, 32 heads over 8, D = 128: 602 us, 913 TFLOP/s, 0.55 of
// the measured GEMM rate; 330 us at that rate): a tile's chain of scores, softmax, products.  128
// keys take both tiles 2057 cycles of tcgen05.mma (scores are bound by the reads of both operands
// from shared memory, 64 cycles for 16 elements) and 2048 of the exponential unit (16 a
// cycle), but some 3900 go by: softmax 2200, a tile's wait for its products 1000 to 1400, the
// rest barriers.  Loops must stay short: code of seldom ways inside them costs every turn
// its fetch (masks inside the score loops: 740 us; in a pass of their own: 624).  Tried,
// and no faster beyond the spread between runs: blocks of 64 keys with two score buffers
// (48 cycles of MMA for 32 of arithmetic), an issuing warp for each tile, tiles that take turns at
// the exponentials, a register split by setmaxnreg (spills), an eighth to a half of the exponentials as
// a polynomial of degree 4 on the FMA units, a shorter loop over the outputs.
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
constexpr int kWarpProducer = 0, kWarpMma = 1, kWarpHelper = 2, kWarpSoft0 = 4;
constexpr int kSlots = 5, kAhead = 1;
constexpr uint32_t kTmemCols = 512;
constexpr int kColO = 2 * kKeys;  // S_t at kKeys t, O_t at kColO + 128 t
constexpr float kSlack = 8.0f;
// tcgen05 sums toward zero: every accumulation loses up to 2^-23 of the sum, on average some 2^-26
// (2500 of them, 20000 keys with SPLIT: 2.4e-5).  So every kFlush units O_t moves to fp32 sums in
// the workspace, and begins anew.
constexpr int flush_units(bool split) { return split ? 8 : 64; }
constexpr int kChunkBytes = kKeys * 128, kQChunkBytes = kTile * 128;  // 64 elements of a block's keys, of a tile's rows

template <int DP>
struct Shape {
    static constexpr int kChunks = DP / 64;
    static constexpr int kBlock = kChunks * kChunkBytes;    // keys, or values, of a unit
    static constexpr int kQTile = kChunks * kQChunkBytes;  // queries of a tile
    static constexpr int kSmem = 1024 + 2 * kQTile + kSlots * kBlock + 512 + kRows * 4;
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
// The lowest n bits.
__device__ __forceinline__ uint32_t below(int n) { return n >= 32 ? ~0u : n <= 0 ? 0u : (1u << n) - 1u; }
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

// The larger of a and |b| in both halves; NaN if either is.
template <bool BF16>
__device__ __forceinline__ uint32_t max_abs2(uint32_t a, uint32_t b) {
    uint32_t r;
    b &= 0x7FFF7FFFu;
    if constexpr (BF16)
        asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    else
        asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}

// A and B of the same 16-bit type, fp32 accumulation; b_mn: B's N elements are contiguous.
__host__ __device__ constexpr uint32_t idesc16(bool bf16, int n, bool b_mn) {
    return (1u << 4) | ((bf16 ? 1u : 0u) << 7) | ((bf16 ? 1u : 0u) << 10) | ((b_mn ? 1u : 0u) << 16) |
           ((uint32_t)(n >> 3) << 17) | ((uint32_t)(kTile >> 4) << 24);
}

// The blocks of a run's units: keys of unit 0, then values of unit g and keys of unit g + 1
// (while there are), g = 0, 1, ...  Position in the ring, and the parity of its current use.
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

// Y: the outputs' type (SPLIT: fp32).
template <bool BF16, int Y, int DP>
__global__ void __launch_bounds__(kThreads, 1)
    attn_tc_kernel(const __grid_constant__ AttnParams p, const __grid_constant__ CUtensorMap kmap,
                   const __grid_constant__ CUtensorMap vmap, const __grid_constant__ CUtensorMap qmap, const int box,
                   const int q_boxes) {
    constexpr bool SPLIT = Y == NXQ_F32;
    using Sh = Shape<DP>;
    using W = Walk<kRows, kKeys>;
    constexpr float kShift = BF16 ? 0.0f : 7.0f;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* const smem = smem_raw + ((1024 - (ptx::smem_addr(smem_raw) & 1023)) & 1023);
    uint8_t* const qs = smem;
    uint8_t* const ring = qs + 2 * Sh::kQTile;
    uint64_t* const bars = reinterpret_cast<uint64_t*>(ring + kSlots * Sh::kBlock);
    uint64_t* const kv_full = bars;
    uint64_t* const kv_empty = kv_full + kSlots;
    uint64_t* const looked = kv_empty + kSlots;  // [slot] the helpers have looked through its values
    uint64_t* const q_full = looked + kSlots;
    uint64_t* const q_empty = q_full + 1;
    uint64_t* const s_full = q_empty + 1;  // [tile]
    uint64_t* const p_full = s_full + 2;   // [tile]
    uint64_t* const p_half = p_full + 2;   // [tile] the weights of the second 64 keys, which come first
    uint64_t* const o_full = p_half + 2;   // [tile] the item's products are in O_t
    uint64_t* const meet = o_full + 2;     // the softmax warps: of tile 0 alone, of both
    uint64_t* const drain = meet + 2;
    uint32_t* const tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
    volatile int* const abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    volatile int* const found = abort_flag + 1;     // [slot] its values are not all finite
    volatile int* const anew = found + kSlots;      // [tile] the unit's product begins O_t anew
    static_assert((3 * kSlots + 2 + 8 + 2 + 1) * 8 + (2 + kSlots + 2) * 4 <= 512, "barrier area too small");

    float* const moved_m = reinterpret_cast<float*>(reinterpret_cast<uint8_t*>(bars) + 512);  // [kRows]
    PlanSmem& plan = *reinterpret_cast<PlanSmem*>(ring);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const ptx::WaitCtl ctl{abort_flag, p.status};
    if (threadIdx.x == 0) {
        for (int i = 0; i < kSlots; ++i) {
            ptx::mbar_init(&kv_full[i], 1);
            ptx::mbar_init(&kv_empty[i], 2);  // the products, and the helper
            ptx::mbar_init(&looked[i], 1);
            found[i] = 0;
        }
        ptx::mbar_init(q_full, 1);
        ptx::mbar_init(q_empty, 1);
        for (int t = 0; t < 2; ++t) {
            ptx::mbar_init(&s_full[t], 1);
            ptx::mbar_init(&p_full[t], 4);
            ptx::mbar_init(&p_half[t], 4);
            ptx::mbar_init(&o_full[t], 1);
            ptx::mbar_init(&meet[t], t ? 8 : 4);
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
    const Runs runs(plan.total, gridDim.x);
    const int units = (int)runs.units(blockIdx.x);  // (a run of 2^31 units would take an hour)
    W w;
    bool go = units > 0;
    if (go) {
        plan_locate<kRows, kKeys, kThreads>(p, plan, runs.start(blockIdx.x));
        w.start(p, plan, units);
    }
    Cut* const note = static_cast<Cut*>(p.work) + blockIdx.x;
    float* const slots = reinterpret_cast<float*>(static_cast<uint8_t*>(p.work) + cuts_bytes(gridDim.x));
    __syncthreads();  // the plan has been read: its memory is the ring's

    if (warp == kWarpProducer) {
        if (lane == 0) {
            ptx::prefetch_tmap(&kmap);
            ptx::prefetch_tmap(&vmap);
            note->pieces = 0;
        }
        // The plan, and the cache, were written through the generic proxy; TMA works through the async one.
        asm volatile("fence.proxy.async;" ::: "memory");
        Ring r;
        uint32_t issued = 0;
        bool ok = true;
        const int boxes = kKeys / box, b = lane % boxes, chunk = lane / boxes;
        const bool mine = chunk < Sh::kChunks;
        // Where a unit's box of this lane lies.  The page entries of keys are asked for a unit
        // ahead (a load of some 700 cycles, twice a unit, was what the ring waited for), and values
        // take the places of their keys two units before.
        struct Place {
            int page, slot, head;
        };
        Place places[kAhead + 1];  // of the keys copied last, the oldest first; then the next ones'
        bool asked = false;        // a page is wanted for the last of them
        int u = 0;                 // of w, whose unit is looked up next
        auto look_up = [&]() {
            const int j = w.key0(u) + b * box;
            // Boxes without a key that a row sees read nothing: a page of -1 gives zeros.
            Place& x = places[kAhead];
            x = Place{-1, 0, w.head};
            asked = mine && j <= w.it.p_hi && (p.window <= 0 || j + box - 1 > w.it.p_lo - p.window || j < p.sinks);
            if (asked) {
                const int n = p.page_shift >= 0 ? j >> p.page_shift : (int)((unsigned)j / (unsigned)p.b.page);
                x.slot = j - n * p.b.page;
                x.page = p.b.table[w.s * p.b.table_stride + n];
            }
            if (u == 0 && lane == 0) w.cut(runs, blockIdx.x, note);
            if (++u == w.count) {
                u = 0;
                w.next(p);
            }
        };
        auto copy = [&](const Place& x, const CUtensorMap* map) {
            if (!(ok = ptx::warp_mbar_wait(&kv_empty[r.i], r.ph ^ 1u, ctl, 61))) return;
            if (lane == 0) ptx::mbar_arrive_expect_tx(&kv_full[r.i], Sh::kBlock);
            __syncwarp();
            if (mine)
                ptx::tma_load_4d(ring + r.i * Sh::kBlock + chunk * kChunkBytes + b * box * 128, map, 64 * chunk, x.slot, x.head, x.page,
                                 &kv_full[r.i]);
            r.next();
            ++issued;
        };
        if (go) {
            look_up();
            for (int g = -kAhead; g < units && ok; ++g) {
                if (g >= 0) copy(places[0], &vmap);
#pragma unroll
                for (int i = 0; i < kAhead; ++i) places[i] = places[i + 1];
                if (ok && g + kAhead < units) {
                    Place& x = places[kAhead - 1];
                    if (asked && (x.page < 0 || x.page >= p.b.pages)) {
                        raise_index(p.status, kIndexPage);
                        x.page = -1;
                    }
                    if (g + kAhead + 1 < units) look_up();
                    copy(x, &kmap);
                }
            }
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
        const bool lead = ptx::elect_one();  // one lane issues, and commits what it issued
        // S_t = Q_t K^T, the keys in slot i.
        auto scores = [&](int t, int i) {
            const uint64_t a = qd + ((uint32_t)(t * Sh::kQTile) >> 4), b = kd + ((uint32_t)(i * Sh::kBlock) >> 4);
#pragma unroll
            for (int c = 0; c < Sh::kChunks; ++c)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    ptx::mma_ss_f16(tmem + kKeys * t, a + c * (kQChunkBytes >> 4) + 2 * e, b + c * (kChunkBytes >> 4) + 2 * e, kIdS,
                                    c || e ? 1u : 0u);
            ptx::mma_commit(&s_full[t]);
        };
        // O_t (+)= P_t V, the values in slot i.
        auto outputs = [&](int t, int i, int half, bool last) {
            const uint64_t b = vd + ((uint32_t)(i * Sh::kBlock) >> 4);
            const uint32_t accumulate = anew[t] ? 0u : 1u;
#pragma unroll
            for (int h = 0; h < (SPLIT ? 2 : 1); ++h)
#pragma unroll
                for (int e = kKeys / 32 * half; e < kKeys / 32 * (half + 1); ++e)
                    ptx::mma_ts_f16(tmem + kColO + 128 * t, tmem + kKeys * t + 32 * (e >> 1) + 16 * h + 8 * (e & 1), b + e * (2048 >> 4), kIdO,
                                    h || e != kKeys / 32 ? 1u : accumulate);
            if (last && !half) ptx::mma_commit(&o_full[t]);
        };
        Ring r;
        uint32_t q_ph = 0, p_ph0 = 0, p_ph1 = 0;
        bool ok = true;
        if (go) {
            int left = w.count;  // units of the piece from unit g on
            bool two = w.it.rows > kTile;
            // Step g: outputs of unit g and scores of unit g + 1, tile 0's and then tile 1's: a wait for all
            // that a tile's need (different lanes for each barrier) and one go of the issuing lane.
            for (int g = -1; g < units; ++g) {
                const bool has_o = g >= 0, has_s = g + 1 < units, last = has_o && left == 1, had = two && has_o;
                const bool s_fresh = has_s && (last || !has_o);
                if (last && has_s) {
                    w.next(p);
                    left = w.count + 1;
                    two = w.it.rows > kTile;
                }
                const bool s_last = has_s && left == (has_o ? 2 : 1);
                const Ring v = r;
                if (has_o) r.next();
                const Ring k = r;
                if (has_s) r.next();
                uint64_t* bar = has_o ? &kv_full[v.i] : &kv_full[k.i];
                uint32_t ph = has_o ? v.ph : k.ph;
                const int part = lane & 3;
                if (part == 1 && has_o) bar = &p_half[0], ph = p_ph0;
                if (part == 2 && !has_o && s_fresh) bar = q_full, ph = q_ph;
                if (!(ok = ptx::warp_mbar_wait(bar, ph, ctl, 64))) break;
                ptx::tc_fence_after();
                if (has_o) {
                    if (lead) outputs(0, v.i, 1, last);
                    __syncwarp();
                    bar = part == 1 && has_s ? &kv_full[k.i] : part == 2 && s_fresh ? q_full : &p_full[0];
                    ph = part == 1 && has_s ? k.ph : part == 2 && s_fresh ? q_ph : p_ph0;
                    if (!(ok = ptx::warp_mbar_wait(bar, ph, ctl, 64))) break;
                    ptx::tc_fence_after();
                }
                if (lead) {
                    if (has_o) outputs(0, v.i, 0, last);
                    if (has_s) scores(0, k.i);
                }
                __syncwarp();
                if (had) {
                    if (!(ok = ptx::warp_mbar_wait(&p_half[1], p_ph1, ctl, 65))) break;
                    ptx::tc_fence_after();
                    if (lead) outputs(1, v.i, 1, last);
                    __syncwarp();
                    if (!(ok = ptx::warp_mbar_wait(&p_full[1], p_ph1, ctl, 65))) break;
                    ptx::tc_fence_after();
                }
                if (lead) {
                    if (had) outputs(1, v.i, 0, last);
                    if (has_o) ptx::mma_commit(&kv_empty[v.i]);
                    if (has_s && two) scores(1, k.i);
                    if (has_s) ptx::mma_commit(&kv_empty[k.i]);
                    if (s_last) ptx::mma_commit(q_empty);
                }
                __syncwarp();
                p_ph0 ^= has_o;
                p_ph1 ^= had;
                q_ph ^= s_fresh;
                left -= has_o;
            }
        }
        if (lead) ptx::mma_commit(drain);
        __syncwarp();
        const long long t0 = clock64();
        while (!ptx::mbar_try_wait(drain, 0) && clock64() - t0 < ptx::kWaitCycles) {
        }
    } else if (warp == kWarpHelper) {
        bool ok = true;
        if (lane == 0 && q_boxes) ptx::prefetch_tmap(&qmap);
        asm volatile("fence.proxy.async;" ::: "memory");  // (queries, as the cache above)
        uint32_t q_ph = 0, q_loads = 0;
        bool first_piece = true;
        auto queries = [&](const W& x) {
            if (!first_piece) {
                ok = ptx::warp_mbar_wait(q_empty, q_ph, ctl, 67);
                q_ph ^= 1u;
                if (!ok) return;
            }
            first_piece = false;
            const int tiles = x.it.rows > kTile ? 2 : 1;
            if (q_boxes) {
                // Whole tokens in every tile: a box of their group's heads for each 64 elements.  (Rows
                // behind the item's are other rows of q, or zeros, and are not stored.)
                if (lane == 0) ptx::mbar_arrive_expect_tx(q_full, tiles * Sh::kQTile);
                __syncwarp();
                if (lane < tiles * Sh::kChunks) {
                    const int tile = lane / Sh::kChunks, c = lane % Sh::kChunks;
                    ptx::tma_load_3d(qs + tile * Sh::kQTile + c * kQChunkBytes, &qmap, 64 * c, x.head * p.G,
                                     x.q.q0 + x.it.t0 + tile * (kTile / p.G), q_full);
                }
                __syncwarp();
                ++q_loads;
                return;
            }
            // A lane has one 16-byte piece of rows kStep apart.
            constexpr int kPer = DP / 8, kStep = 32 / kPer;
            const int piece = lane % kPer, first = lane / kPer;
            const int f = x.it.r0 + first, t = (int)((unsigned)f / (unsigned)p.G);
            int g = f - t * p.G;
            const uint16_t* src = static_cast<const uint16_t*>(p.q) + ((int64_t)x.q.q0 + x.it.t0 + t) * p.q_token +
                                  ((int64_t)x.head * p.G + g) * p.q_head + piece * 8;
            const int64_t to_token = p.q_token - p.G * p.q_head;
            uint8_t* const dst = qs + (piece >> 3) * kQChunkBytes + first * 128;
            const bool in_head = piece * 8 < p.D;
#pragma unroll 8
            for (int row = first, i = 0; i < tiles * kTile; row += kStep, i += kStep) {
                uint8_t* const to = dst + (i / kTile) * (Sh::kQTile - kQChunkBytes) + i * 128 + (((piece & 7) ^ (row & 7)) << 4);
                const bool read = row < x.it.rows && in_head;
                if (p.q_vec) {
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(ptx::smem_addr(to)), "l"(read ? src : p.q),
                                 "r"(read ? 16 : 0)
                                 : "memory");
                } else {
                    uint32_t h[4] = {0u, 0u, 0u, 0u};
                    if (read)
#pragma unroll
                        for (int k = 0; k < 4; ++k) h[k] = (uint32_t)src[2 * k] | (uint32_t)src[2 * k + 1] << 16;
                    *reinterpret_cast<uint4*>(to) = make_uint4(h[0], h[1], h[2], h[3]);
                }
                src += kStep * p.q_head;
                for (g += kStep; g >= p.G; g -= p.G) src += to_token;
            }
            asm volatile("cp.async.wait_all;" ::: "memory");
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) ptx::mbar_arrive(q_full);
        };
        if (go) {
            Ring r;
            W wk = w, wv = w;
            int uk = 0, uv = 0;
            for (int g = -kAhead; g < units && ok; ++g) {
                if (g >= 0) {
                    const int j0 = wv.key0(uv);
                    const Item it = wv.it;
                    if (++uv == wv.count) {
                        uv = 0;
                        wv.next(p);
                    }
                    if (!(ok = ptx::warp_mbar_wait(&kv_full[r.i], r.ph, ctl, 68))) break;
                    if (mixed(p, it, j0)) {
                        // Keys `behind` .. end - 1 and those before `before`, but for sinks, are seen by some rows only: the
                        // largest magnitude of their values, NaN above all.  Keys from `end` on and before `gone` are
                        // seen by none: what lies there (the rest of a page; tokens that left the window) is zeros to
                        // the product if it is not finite.
                        const bool windowed = p.window > 0;
                        const int behind = it.p_lo + 1 - j0, end = it.p_hi + 1 - j0, sinks = windowed ? p.sinks - j0 : 0;
                        const int gone = windowed ? it.p_lo - p.window + 1 - j0 : 0, before = windowed ? it.p_hi - p.window + 1 - j0 : 0;
                        uint8_t* const block = ring + r.i * Sh::kBlock;
                        uint32_t big = 0;
                        bool cleared = false;
                        auto look = [&](int from, int to) {
                            from = from > 0 ? from : 0, to = to < kKeys ? to : kKeys;
                            if (from >= to) return;  // (8 * from would pass 31 bits with 2^30 sinks)
#pragma unroll 1
                            for (int i = 8 * from + lane; i < 8 * to; i += 32)
#pragma unroll
                                for (int c = 0; c < Sh::kChunks; ++c) {
                                    const uint4 v = *reinterpret_cast<const uint4*>(block + c * kChunkBytes + 16 * i);
                                    big = max_abs2<BF16>(max_abs2<BF16>(max_abs2<BF16>(max_abs2<BF16>(big, v.x), v.y), v.z), v.w);
                                }
                        };
                        look(gone > sinks ? gone : sinks, before);
                        look(behind, end);
                        // (Boxes without a key that a row sees are zeros already.)
                        const int upto = (sinks + box - 1) & -box, whole = gone & -box;
#pragma unroll 1
                        for (int part = windowed ? 0 : 2; part < 3; ++part) {
                            int from = part == 0 ? sinks : part == 1 ? (whole > sinks ? whole : sinks) : end;
                            int to = part == 0 ? (upto < gone ? upto : gone) : part == 1 ? gone : (end + box - 1) & -box;
                            from = from > 0 ? from : 0, to = to < kKeys ? to : kKeys;
                            if (from >= to) continue;
#pragma unroll 1
                            for (int i = 8 * from + lane; i < 8 * to; i += 32)
#pragma unroll
                                for (int c = 0; c < Sh::kChunks; ++c) {
                                    uint4* const at = reinterpret_cast<uint4*>(block + c * kChunkBytes + 16 * i);
                                    const uint4 v = *at;
                                    const uint32_t top = max_abs2<BF16>(max_abs2<BF16>(max_abs2<BF16>(v.x & 0x7FFF7FFFu, v.y), v.z), v.w);
                                    if (not_finite<BF16>(top & 0xFFFFu) || not_finite<BF16>(top >> 16)) {
                                        *at = make_uint4(0u, 0u, 0u, 0u);
                                        cleared = true;
                                    }
                                }
                        }
                        if (cleared) asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                        const bool bad = __any_sync(0xFFFFFFFFu, not_finite<BF16>(big & 0xFFFFu) || not_finite<BF16>(big >> 16));
                        if (lane == 0) {
                            if (bad) found[r.i] = 1;
                            ptx::mbar_arrive(&looked[r.i]);
                        }
                    }
                    __syncwarp();
                    if (lane == 0) ptx::mbar_arrive(&kv_empty[r.i]);
                    r.next();
                }
                if (g + kAhead < units) {
                    if (uk == 0) {
                        queries(wk);
                        if (!ok) break;
                    }
                    if (++uk == wk.count) {
                        uk = 0;
                        wk.next(p);
                    }
                    if (!(ok = ptx::warp_mbar_wait(&kv_full[r.i], r.ph, ctl, 68))) break;
                    if (lane == 0) ptx::mbar_arrive(&kv_empty[r.i]);
                    __syncwarp();
                    r.next();
                }
            }
        }
        // Do not leave with copies in flight (as the producer).
        if (q_loads) {
            const long long t0 = clock64();
            while (!ptx::mbar_try_wait(q_full, (q_loads - 1) & 1) && clock64() - t0 < ptx::kWaitCycles) {
            }
        }
    } else if (warp >= kWarpSoft0) {
        // Softmax of tile t: a thread per row.
        const int t = (warp - kWarpSoft0) >> 2, quad = warp & 3, row = quad * 32 + lane;
        const uint32_t lanes = (uint32_t)(quad * 32) << 16;
        const uint32_t ts = tmem + lanes + kKeys * t, to = tmem + lanes + kColO + 128 * t;
        uint32_t s_ph = 0, o_ph = 0;
        uint32_t meet_ph[2] = {0, 0}, looked_ph = 0;  // looked_ph: a bit per slot
        int left = units;        // of the run, from the piece's unit on
        Ring r;                  // the unit's values
        for (int i = 0; i < (units < kAhead ? units : kAhead); ++i) r.next();
        auto step = [&]() {
            r.next();
            if (left > kAhead) r.next();
            --left;
        };
        bool ok = true;
        while (go && ok) {
            const int tiles = w.it.rows > kTile ? 2 : 1;
            if (t >= tiles) {  // (the ring moves on, and so do the units looked through)
                for (int u = 0; u < w.count; ++u, step())
                    if (mixed(p, w.it, w.key0(u))) looked_ph ^= 1u << r.i;
                go = w.next(p);
                continue;
            }
            const int flat = w.it.r0 + t * kTile + row, tok = (int)((unsigned)flat / (unsigned)p.G);
            const int head = w.head * p.G + (flat - tok * p.G);
            const bool mine = t * kTile + row < w.it.rows;
            const int pos = mine ? w.it.p_lo + tok : w.it.p_hi;  // (what rows behind the item's see is nobody's)
            // The maximum in use.  A warp's rows are raised together, and rows behind the item's must have no
            // say in that (theirs are scores of whatever lies there): nothing is above +inf.
            float m = mine ? -INFINITY : INFINITY, l = 0.0f;
            // What has left O_t, relative to the maximum that was in use then.
            constexpr int kFlush = flush_units(SPLIT);
            float& m_moved = moved_m[t * kTile + row];
            auto moved_to = [&]() {
                return reinterpret_cast<float*>(static_cast<uint8_t*>(p.work) + cuts_bytes(gridDim.x)) +
                       2 * (size_t)gridDim.x * part_floats(kRows, p.D) + ((size_t)blockIdx.x * kRows + t * kTile + row) * p.D;
            };
            auto factor_moved = [&]() { return m_moved == -INFINITY ? 1.0f : exp2_fast(m_moved - m); };  // (1: zeros, or NaN)
            auto move = [&](bool first) {
                const float f = first ? 0.0f : factor_moved();
                float* const moved = moved_to();
#pragma unroll 1
                for (int d = 0; d < DP && d < p.D; d += 8) {
                    uint32_t o[8];
                    ptx::tmem_ld8(to + d, o);
                    ptx::tmem_wait_ld();
                    if (mine) {
                        float v[8], x[8];
#pragma unroll
                        for (int k = 0; k < 8; ++k) v[k] = __uint_as_float(o[k]);
                        if (!first) {
                            load_f32x8(moved + d, x);
#pragma unroll
                            for (int k = 0; k < 8; ++k) v[k] = fmaf(x[k], f, v[k]);
                        }
                        store_f32x8(moved + d, v);
                    }
                    __syncwarp();
                }
                m_moved = m;
            };
            // Raises the maximum in use of rows whose new one is too far above, and corrects what
            // has been summed in unit u - 1 and before.
            auto raise_to = [&](float now, int u) {
                if (!__any_sync(0xFFFFFFFFu, now > m + kSlack || (m == -INFINITY && now > -INFINITY))) return;
                const float to_m = fmaxf(m, now), f = m == -INFINITY ? 0.0f : exp2_fast(m - to_m);
                m = to_m;
                l *= f;
                if (u == 0) return;
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
            };
            for (int u = 0; u < w.count; ++u, step()) {
                const int j0 = w.key0(u);
                // (With S_t of a unit O_t has the unit before.)
                if (!(ok = ptx::warp_mbar_wait(&s_full[t], s_ph, ctl, 69))) break;
                s_ph ^= 1u;
                ptx::tc_fence_after();
                bool fresh = u % kFlush == 0;
                if (fresh && u > 0) move(u == kFlush);
                const bool hidden = mixed(p, w.it, j0);
                if (hidden) {
                    if (!(ok = ptx::warp_mbar_wait(&looked[r.i], (looked_ph >> r.i) & 1u, ctl, 70))) break;
                    looked_ph ^= 1u << r.i;
                    // A value that not all rows see may be infinite or NaN, and a weight of zero must
                    // not meet it: such elements are added to the rows that see them here, and are
                    // zeros to the product.
                    if (found[r.i]) {
                        float now = -INFINITY;
#pragma unroll 1
                        for (int k = 0; k < kKeys; ++k) {
                            const float x = __uint_as_float(ptx::tmem_ld1(ts + k));
                            ptx::tmem_wait_ld();
                            if (sees(p, pos, j0 + k)) now = fmaxf(now, x * p.c);
                            __syncwarp();
                        }
                        raise_to(now, u);
                        const float base = m == -INFINITY ? 0.0f : m - kShift;
                        uint8_t* const vs = ring + r.i * Sh::kBlock;
                        if (fresh) {
#pragma unroll 1
                            for (int d = 0; d < DP; ++d) ptx::tmem_st1(to + d, 0u);
                            ptx::tmem_wait_st();
                            fresh = false;
                        }
                        // (A lane looks at 8 elements; the pieces found are gone through by all.)
                        constexpr int kPer = DP / 8;
                        auto piece_at = [&](int i) {
                            return vs + (i % kPer >> 3) * kChunkBytes + i / kPer * 128 + (((i % kPer & 7) ^ (i / kPer & 7)) << 4);
                        };
#pragma unroll 1
                        for (int i = lane; i < kKeys * kPer; i += 32) {
                            const uint4 v = *reinterpret_cast<const uint4*>(piece_at(i));
                            const uint32_t top = max_abs2<BF16>(max_abs2<BF16>(max_abs2<BF16>(v.x & 0x7FFF7FFFu, v.y), v.z), v.w);
                            uint32_t hits = __ballot_sync(0xFFFFFFFFu, not_finite<BF16>(top & 0xFFFFu) || not_finite<BF16>(top >> 16));
#pragma unroll 1
                            for (; hits; hits &= hits - 1) {
                                const int j = i - lane + __ffs(hits) - 1, k = j / kPer;
#pragma unroll 1
                                for (int e = 0; e < 8; ++e) {
                                    const uint32_t bits = reinterpret_cast<const uint16_t*>(piece_at(j))[e];
                                    if (!not_finite<BF16>(bits)) continue;  // (the same in all lanes)
                                    const int d = j % kPer * 8 + e;
                                    float x = __uint_as_float(ptx::tmem_ld1(ts + k)), o = __uint_as_float(ptx::tmem_ld1(to + d));
                                    ptx::tmem_wait_ld();
                                    if (sees(p, pos, j0 + k)) o += exp2_fast(fmaf(x, p.c, -base)) * value_of<BF16>(bits);
                                    __syncwarp();
                                    ptx::tmem_st1(to + d, __float_as_uint(o));
                                    ptx::tmem_wait_st();
                                }
                            }
                        }
                        // Everybody has read them; then everybody has cleared them.
                        for (int both = 0; both < 2 && ok; ++both) {
                            __syncwarp();
                            if (lane == 0) ptx::mbar_arrive(&meet[tiles - 1]);
                            ok = ptx::warp_mbar_wait(&meet[tiles - 1], meet_ph[tiles - 1], ctl, 71);
                            meet_ph[tiles - 1] ^= 1u;
                            if (both == 0 && ok) {
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
                // Scores that a row does not see become -inf in place, 32 keys at a time against the positions of
                // the warp's rows (most are seen by all or by none), before and apart from the loops below: with the
                // masks inside them, as long as they are, every unit took 500 cycles more.
                if (hidden) {
                    const int hi = pos - j0, lo = p.window > 0 ? pos - p.window - j0 : -1, sk = p.sinks - j0;
                    const int hi_min = __reduce_min_sync(0xFFFFFFFFu, hi), hi_max = __reduce_max_sync(0xFFFFFFFFu, hi);
                    const int lo_min = __reduce_min_sync(0xFFFFFFFFu, lo), lo_max = __reduce_max_sync(0xFFFFFFFFu, lo);
#pragma unroll 1
                    for (int j = 0; j < kKeys; j += 16) {
                        if (j + 15 <= hi_min && (j > lo_max || j + 15 < sk)) continue;
                        const uint32_t seen = below(hi - j + 1) & (~below(lo - j + 1) | below(sk - j));
                        uint32_t x[16];
                        if (j <= hi_max && (j + 15 > lo_min || j < sk)) {
                            ptx::tmem_ld16(ts + j, x);
                            ptx::tmem_wait_ld();
                        }
#pragma unroll
                        for (int k = 0; k < 16; ++k)
                            if (!(seen >> k & 1)) x[k] = 0xFF800000u;
                        ptx::tmem_st16(ts + j, x);
                    }
                    ptx::tmem_wait_st();
                }
                // 64 keys at a time: the first for the maximum, the other for the maximum and the weights, the
                // first again for the weights, which go over the first half of each 32 scores' columns (what
                // their rounding leaves, SPLIT, over the other).  Loops of two rather than 128 of
                // everything: those neither fit the registers nor a scheduler's instruction cache.
                uint32_t s[2][32];
                auto read = [&](int half) {
                    ptx::tmem_ld32(ts + 64 * half, s[0]);
                    ptx::tmem_ld32(ts + 64 * half + 32, s[1]);
                    ptx::tmem_wait_ld();
                };
                float now = -INFINITY;
#pragma unroll 1
                for (int half = 0; half < 2; ++half) {
                    read(half);
                    float top[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const uint32_t* x = s[i >> 1] + 16 * (i & 1);
                        top[i] = fmaxf(__uint_as_float(x[0]), __uint_as_float(x[1]));
#pragma unroll
                        for (int k = 2; k < 16; k += 2) top[i] = fmaxf(fmaxf(top[i], __uint_as_float(x[k])), __uint_as_float(x[k + 1]));
                    }
                    now = fmaxf(now, fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])));
                }
                raise_to(now * p.c, u);
                const float base = m == -INFINITY ? 0.0f : m - kShift;
                const uint64_t c2 = pair(p.c, p.c), b2 = pair(-base, -base);
                if (row == 0) anew[t] = fresh;
                __syncwarp();
                uint64_t sum[4] = {0ull, 0ull, 0ull, 0ull};
#pragma unroll 1
                for (int half = 1; half >= 0; --half) {
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        uint32_t y[16], z[SPLIT ? 16 : 1];
#pragma unroll
                        for (int k = 0; k < 16; ++k) {
                            float2 x = unpair(fma2(pair(__uint_as_float(s[i][2 * k]), __uint_as_float(s[i][2 * k + 1])), c2, b2));
                            x.x = exp2_fast(x.x);
                            x.y = exp2_fast(x.y);
                            sum[k & 3] = add2(sum[k & 3], pair(x.x, x.y));
                            y[k] = pack2<BF16>(x.x, x.y);
                            if constexpr (SPLIT)
                                z[k] = pack2<BF16>(x.x - value_of<BF16>(y[k] & 0xFFFFu), x.y - value_of<BF16>(y[k] >> 16));
                        }
                        ptx::tmem_st16(ts + 64 * half + 32 * i, y);
                        if constexpr (SPLIT) ptx::tmem_st16(ts + 64 * half + 32 * i + 16, z);
                    }
                    ptx::tmem_wait_st();
                    ptx::tc_fence_before();
                    __syncwarp();
                    if (lane == 0) ptx::mbar_arrive(half ? &p_half[t] : &p_full[t]);
                    __syncwarp();
                    if (half) read(0);
                }
                const float2 a = unpair(add2(add2(sum[0], sum[1]), add2(sum[2], sum[3])));
                l += a.x + a.y;
            }
            if (!ok) break;
            const bool whole = w.whole();
            float* const part = whole ? nullptr : slots + (2ll * blockIdx.x + w.slot()) * part_floats(kRows, p.D);
            const float f = !whole ? 1.0f : l == 0.0f ? 0.0f : 1.0f / l;
            const int64_t token = (int64_t)w.q.q0 + w.it.t0 + tok, at = token * p.o_token + head * p.o_head;
            const bool wide = p.o_vec > 1;
            const bool has_moved = w.count > kFlush;
            go = w.next(p);  // (while the last products run)
            if (!(ok = ptx::warp_mbar_wait(&o_full[t], o_ph, ctl, 73))) break;
            o_ph ^= 1u;
            ptx::tc_fence_after();
            const float f_moved = has_moved ? factor_moved() : 0.0f;
            float* const moved = moved_to();
            bool over = false;
#pragma unroll 1
            for (int d = 0; d < DP && d < p.D; d += 32) {
                uint32_t o[32];
                ptx::tmem_ld32(to + d, o);
                ptx::tmem_wait_ld();
                if (mine) {
                    float v[32];
#pragma unroll
                    for (int k = 0; k < 32; ++k) v[k] = __uint_as_float(o[k]);
                    if (has_moved)
#pragma unroll
                        for (int h = 0; h < 4; ++h) {
                            if (d + 8 * h >= p.D) break;
                            float x[8];
                            load_f32x8(moved + d + 8 * h, x);
#pragma unroll
                            for (int k = 0; k < 8; ++k) v[8 * h + k] = fmaf(x[k], f_moved, v[8 * h + k]);
                        }
#pragma unroll
                    for (int k = 0; k < 32; ++k) v[k] *= f;
                    if (!whole || Y == NXQ_F32) {
                        float* const q = whole ? static_cast<float*>(p.out) + at + d : part + (int64_t)(t * kTile + row) * p.D + d;
#pragma unroll
                        for (int h = 0; h < 4; ++h) {
                            if (d + 8 * h >= p.D) break;
                            if (!whole || wide) {
                                store_f32x8(q + 8 * h, v + 8 * h);
                            } else {
#pragma unroll
                                for (int k = 0; k < 8; ++k) q[8 * h + k] = v[8 * h + k];
                            }
                        }
                    } else if constexpr (Y != NXQ_F32) {
                        if constexpr (Y == NXQ_F16)
#pragma unroll
                            for (int k = 0; k < 32; ++k) v[k] = for_f16<BF16>(v[k], over);
                        uint16_t* const q = static_cast<uint16_t*>(p.out) + at + d;
                        uint32_t y[16];
#pragma unroll
                        for (int k = 0; k < 16; ++k) y[k] = pack2<Y == NXQ_BF16>(v[2 * k], v[2 * k + 1]);
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            if (d + 16 * h >= p.D) break;
                            if (wide && d + 16 * h + 16 <= p.D) {
                                store_f32x8(reinterpret_cast<float*>(q + 16 * h), reinterpret_cast<const float*>(y + 8 * h));
                            } else {
#pragma unroll
                                for (int e = 0; e < 2; ++e) {
                                    if (d + 16 * h + 8 * e >= p.D) break;
                                    const uint32_t* z = y + 8 * h + 4 * e;
                                    uint16_t* const to_y = q + 16 * h + 8 * e;
                                    if (p.o_vec) {
                                        *reinterpret_cast<uint4*>(to_y) = make_uint4(z[0], z[1], z[2], z[3]);
                                    } else {
#pragma unroll
                                        for (int k = 0; k < 8; ++k) to_y[k] = (uint16_t)(z[k >> 1] >> (16 * (k & 1)));
                                    }
                                }
                            }
                        }
                    }
                }
                __syncwarp();
            }
            if (Y == NXQ_F16 && BF16 && over) raise_range(p.status, kRangeAttn);
            if (mine && !whole) {
                part[(int64_t)kRows * p.D + t * kTile + row] = m == -INFINITY ? m : m - kShift;
                part[(int64_t)kRows * p.D + kRows + t * kTile + row] = l;
            }
            if (mine && whole && p.lse)
                p.lse[token * ((int64_t)p.Hk * p.G) + head] =
                    l == 0.0f ? -INFINITY : (m - kShift + log2f(l)) * 0.6931471805599453f;
            __syncwarp();
            ptx::tc_fence_before();
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
auto* kernel_of(bool bf16, int y) {
    return y == NXQ_F32   ? (bf16 ? attn_tc_kernel<true, NXQ_F32, DP> : attn_tc_kernel<false, NXQ_F32, DP>)
           : y == NXQ_F16 ? (bf16 ? attn_tc_kernel<true, NXQ_F16, DP> : attn_tc_kernel<false, NXQ_F16, DP>)
                          : (bf16 ? attn_tc_kernel<true, NXQ_BF16, DP> : attn_tc_kernel<false, NXQ_BF16, DP>);
}

template <int DP>
int set_attr() {
    for (const int y : {NXQ_F32, NXQ_F16, NXQ_BF16})
        for (const bool bf16 : {false, true}) {
            const cudaError_t e = cudaFuncSetAttribute(kernel_of<DP>(bf16, y), cudaFuncAttributeMaxDynamicSharedMemorySize,
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

// Queries [tokens][heads][D] in boxes of a group's heads and as many tokens as a tile has.
int query_map(CUtensorMap* map, const AttnParams& p, bool bf16) {
    const uint64_t dims[3] = {(uint64_t)p.D, (uint64_t)p.Hk * p.G, (uint64_t)p.b.T};
    const uint64_t strides[2] = {2 * (uint64_t)p.q_head, 2 * (uint64_t)p.q_token};
    const uint32_t boxes[3] = {64, (uint32_t)p.G, (uint32_t)(kTile / p.G)};
    if (const int e = tensor_map_16(map, bf16, p.q, 3, dims, strides, boxes))
        return fail(NXQ_ERR_CUDA, "cuTensorMapEncodeTiled failed (%d)", e);
    return NXQ_OK;
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
    const bool bf = cache->dtype == NXQ_BF16;
    CUtensorMap k, v, q{};
    int rc;
    if ((rc = cache_map(&k, cache, cache->k_dev, box)) || (rc = cache_map(&v, cache, cache->v_dev, box))) return rc;
    // Queries by TMA where tiles hold whole tokens and rows are such that a tensor map takes them; by
    // 16-byte copies of one warp otherwise (4096 tokens, 8 key heads of 128: 4 query heads for each
    // 207 us, 8 364; 3 280, 5 412, 7 547).
    const int64_t far = (int64_t)1 << 38;
    const int q_boxes = kTile % p.G == 0 && p.q_vec && p.q_head > 0 && p.q_token > 0 && p.q_head < far && p.q_token < far;
    if (q_boxes && (rc = query_map(&q, p, bf))) return rc;
    note_launches(1);
    const cudaError_t e = p.D <= 64 ? launch_overlapped(kernel_of<64>(bf, p.y_dtype), attn_tc_grid(), kThreads, Shape<64>::kSmem, st,
                                                        p, k, v, q, box, q_boxes)
                                    : launch_overlapped(kernel_of<128>(bf, p.y_dtype), attn_tc_grid(), kThreads, Shape<128>::kSmem,
                                                        st, p, k, v, q, box, q_boxes);
    if (e != cudaSuccess) return cuda_fail(e, "attention launch (tcgen05)");
    const cudaError_t j = launch_attn_join(p, kRows, attn_tc_grid(), st);
    return j == cudaSuccess ? NXQ_OK : cuda_fail(j, "attention join launch");
}

}  // namespace nxq
