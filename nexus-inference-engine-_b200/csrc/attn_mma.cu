// Attention over the paged cache for few rows per sequence and key head: single
// new tokens, drafted ones (and every shape that the tcgen05 kernel does not take).
//
// Bound by memory: a key and its value are read once per key head and meet up to 16
// MT rows.  So the kernel is built around loads: two CTAs per SM, each with an equal
// share of the call's units of 64 keys (128 for short heads; attn_plan.cuh), each of its
// four warps streaming its own quarter of a unit through a ring of its own by cp.async
// (16 bytes a lane, pages looked up a unit ahead), with no barrier between units.  Rows of
// a key that no query of the item sees are filled with zeros instead of read.
//
// A warp multiplies on mma.sync.m16n8k16: scores of 16 MT rows x 16 keys, then weights
// times values, with the maximum, the sum of weights and the output of its own keys
// in registers (fp32).  At 64 keys per unit that is 128 instructions per 32 KB, 256
// of the 1390 cycles in which an SM gets 32 KB.  An item ends with the four warps'
// states joined in shared memory.
//
// 64 sequences of 200 to 8000 keys, 32 heads over 8 (bf16, 1.2 GB): 199 us, 6.1 TB/s, 0.94 of the
// copy rate; one of 131072 keys, 128 heads over 8: 101 us with its join, 83 at that rate.  Two
// tiles of rows (MT = 2; 24 sequences of 2 to 6 new tokens, 5 heads per key head) take 78 us where the
// cache's bytes take 41: a unit's chain of products, maximum, exponentials and products with two
// warps on a scheduler, whose issue slots are 0.29 used; more warps would have too few registers (255).
//
// Weights are relative to a maximum that is raised only when a score passes it by
// 2^8, so most units need no rescaling; an f16 cache's weights get a factor 2^7 on top,
// which keeps small ones out of f16's subnormals (2^15 at most).  They are rounded to the
// cache's type for the product with the values, which takes both operands in one type: bf16
// outputs are off by 0.0023 of their size (their own rounding alone 0.0017), f16 by 0.00029 (0.00021).
// Where the output is fp32 (SPLIT) what the rounding leaves goes through a second product, so that
// they keep twice its digits (203 us instead of 199, two tiles of rows 86 instead of 78).
#include "attn_plan.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace nxq {

namespace {

using namespace attn;

constexpr int kThreads = 128, kWarps = 4;
constexpr float kSlack = 8.0f;

__device__ __forceinline__ uint32_t smem_of(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }
// 16 bytes global -> shared, or 16 zeros.
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool read) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(read ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void ldsm4(uint32_t a, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(a)
                 : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t a, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(a)
                 : "memory");
}
template <bool BF16>
__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (BF16)
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
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
// Whether a 16-bit value is infinite or NaN.
template <bool BF16>
__device__ __forceinline__ bool not_finite(uint32_t bits) {
    constexpr uint32_t m = BF16 ? 0x7F80u : 0x7C00u;
    return (bits & m) == m;
}

template <int DP, int MT>
struct Shape {
    static constexpr int kSlice = DP == 64 ? 32 : 16;  // keys of a unit per warp: 4 KB or more of each
    static constexpr int kKeys = kWarps * kSlice;
    static constexpr int kStatic = 512;  // shared memory besides (Walks)
    static constexpr int kStages = DP <= 128 && MT == 1 ? 3 : 2;
    static constexpr int kRows = 16 * MT;
    static constexpr int kSliceBytes = kSlice * DP * 2;                 // a warp's keys (or values) of a unit
    static constexpr int kRing = kWarps * kStages * 2 * kSliceBytes;
    static constexpr bool kQInRegs = MT == 1 && DP <= 128;
    static constexpr int kQBytes = kRows * DP * 2;
    static constexpr int kJoin = 2 * 16 * DP * 4 + kWarps * kRows * 8;  // two warps' outputs of 16 rows, all statistics
    // The plan, the queries (if they go on to registers) and the join share one region.
    static constexpr int kShared0 = kJoin > (int)sizeof(PlanSmem) ? kJoin : (int)sizeof(PlanSmem);
    static constexpr int kShared = kShared0 > kQBytes ? kShared0 : kQBytes;
    static constexpr int kSmem = kRing + kShared + (kQInRegs ? 0 : kQBytes);
    static constexpr int kCtas = 2 * (kSmem + 1024 + kStatic) <= 228 * 1024 ? 2 : 1;
};

// Swizzled offset of 16-byte chunk c of row r in a block of rows of DP 16-bit elements.
template <int DP>
__device__ __forceinline__ uint32_t chunk_at(int r, int c) {
    return (uint32_t)(r * DP * 2 + ((c ^ (r & 7)) << 4));
}

// MULTI: sequences may have several new tokens, so rows of an item may differ in what they see.
// FRESH: a unit's products are summed from zero and added to the outputs here.  The tensor
// cores sum toward zero: 131072 keys in one accumulator fall short by 1.5e-4 (with SPLIT
// 1.8e-4), by nothing that shows with fresh sums.  It costs nothing where there are registers for it (single tokens, 1.2 GB: 199 us
// either way), which two tiles of rows over heads of 128 lack: 88 us against 78 (24
// sequences of 2 to 6 new tokens), so those do it only in long sums (sums_fresh).
// Y: the outputs' type (SPLIT: fp32).
template <bool BF16, int Y, bool MULTI, bool FRESH, int DP, int MT>
__global__ void __launch_bounds__(kThreads, Shape<DP, MT>::kCtas) attn_mma_kernel(const __grid_constant__ AttnParams p) {
    using Sh = Shape<DP, MT>;
    constexpr bool SPLIT = Y == NXQ_F32;
    constexpr int kRows = Sh::kRows, kStages = Sh::kStages, kSlice = Sh::kSlice, kKeys = Sh::kKeys;
    constexpr int kChunks = DP / 8, kSteps = DP / 16, kTiles = DP / 8, kNT = kSlice / 8;
    constexpr float kShift = BF16 ? 0.0f : 7.0f;
    using W = Walk<kRows, kKeys>;
    extern __shared__ __align__(128) uint8_t smem[];
    uint8_t* const shared = smem + Sh::kRing;
    PlanSmem& plan = *reinterpret_cast<PlanSmem*>(shared);
    float* const join = reinterpret_cast<float*>(shared);
    float* const join_ml = join + 2 * 16 * DP;  // [warp][kRows] maximum, then sum
    uint8_t* const qs = Sh::kQInRegs ? shared : shared + Sh::kShared;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    // The join kernel may start when all before this kernel is complete.
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    Cut* const note = static_cast<Cut*>(p.work) + blockIdx.x;
    float* const slots = reinterpret_cast<float*>(static_cast<uint8_t*>(p.work) + cuts_bytes(gridDim.x));
    if (threadIdx.x == 0) note->pieces = 0;
    plan_total<kRows, kKeys, kThreads>(p, plan);
    const long long total = plan.total, units = Runs(total, gridDim.x).units(blockIdx.x);
    if (units == 0) return;
    plan_locate<kRows, kKeys, kThreads>(p, plan, Runs(total, gridDim.x).start(blockIdx.x));

    // The piece being computed, and the one being loaded, each warp's for itself and in shared
    // memory: registers are short.
    __shared__ W aheads[kWarps];
    __shared__ long long all_units;
    static_assert(sizeof(aheads) + sizeof(all_units) <= Sh::kStatic, "");
    W w;
    w.start(p, plan, units);
    W& ahead = aheads[warp];
    if (lane == 0) ahead = w;
    if (threadIdx.x == 0) all_units = total;
    __syncthreads();  // the plan has been read: its memory is the join's
    int au = 0;       // unit of `ahead` whose pages are looked up next
    bool more = true;

    // The unit after the one being copied: the page entry and slot of its keys, and which
    // of them are wanted.  Where pages hold whole slices a warp's keys share one entry, its
    // first key's slot and a range (rows below `upto`, but not gap0 .. gap1 - 1); else
    // lane i has key i's (lanes from kSlice on repeat).
    const bool paged = p.page_align >= kSlice;
    int entry = 0, slot = 0, entry_head = 0, upto = 0, gap0 = 0, gap1 = 0;
    bool want = false;
    auto look_up = [&]() {
        want = false;
        if (!more) return;
        int j = ahead.key0(au) + warp * kSlice;
        entry_head = ahead.head;
        if (paged) {
            upto = ahead.it.p_hi + 1 - j;
            want = upto > 0;
            upto = upto < kSlice ? upto : kSlice;
            gap0 = gap1 = 0;
            if (p.window > 0) {
                gap0 = p.sinks > j ? p.sinks - j : 0;
                gap1 = ahead.it.p_lo - p.window + 1 - j;
                want = want && !(gap0 == 0 && gap1 >= upto);
            }
        } else {
            j += lane & (kSlice - 1);
            want = any_sees(p, ahead.it, j);
        }
        if (want) {
            const int page = p.page_shift >= 0 ? j >> p.page_shift : (int)((unsigned)j / (unsigned)p.b.page);
            slot = j - page * p.b.page;
            entry = p.b.table[ahead.s * p.b.table_stride + page];
        }
        if (++au == ahead.count) {
            au = 0;
            __syncwarp();  // (all have read it)
            if (lane == 0) more = ahead.next(p);
            more = __shfl_sync(0xFFFFFFFFu, more, 0);
            __syncwarp();
        }
    };
    const uint32_t ring = smem_of(smem) + warp * kStages * 2 * Sh::kSliceBytes;
    // A lane copies 16-byte pieces of rows kStep apart.
    constexpr int kPieces = kSlice * kChunks / 32, kStep = kChunks >= 32 ? 1 : 32 / kChunks;
    const int lane_row = lane / kChunks, lane_chunk = lane % kChunks;
    const bool in_head = lane_chunk * 8 < p.D;
    auto copy_unit = [&](int stage) {
        int64_t at = -1;
        if (want) {
            if (entry < 0 || entry >= p.b.pages)
                raise_index(p.status, kIndexPage);
            else
                at = entry * p.page_stride + slot * p.slot_stride + entry_head * p.head_stride;
        }
        const uint32_t dst = ring + stage * 2 * Sh::kSliceBytes + lane_row * DP * 2;
        auto piece = [&](int i, const uint16_t* k, const uint16_t* v, bool read) {
            const uint32_t d = dst + i * kStep * DP * 2 + ((lane_chunk ^ lane_row ^ ((i * kStep) & 7)) << 4);
            copy16(d, k, read);
            copy16(d + Sh::kSliceBytes, v, read);
        };
        static_assert(kChunks <= 32, "a lane has one place in its rows");
        if (paged) {
            const bool some = at >= 0 && in_head;
            const int64_t o = some ? at + lane_row * p.slot_stride + lane_chunk * 8 : 0, step = some ? kStep * p.slot_stride : 0;
            const uint16_t* k = static_cast<const uint16_t*>(p.k) + o;
            const uint16_t* v = static_cast<const uint16_t*>(p.v) + o;
            if (upto == kSlice && gap1 <= gap0) {
#pragma unroll
                for (int i = 0; i < kPieces; ++i, k += step, v += step) piece(i, k, v, some);
            } else {
#pragma unroll
                for (int i = 0; i < kPieces; ++i) {
                    const int r = lane_row + i * kStep;
                    const bool read = some && r < upto && (r < gap0 || r >= gap1);
                    piece(i, read ? k + i * step : static_cast<const uint16_t*>(p.k),
                          read ? v + i * step : static_cast<const uint16_t*>(p.v), read);
                }
            }
        } else {
#pragma unroll
            for (int i = 0; i < kPieces; ++i) {
                const int64_t row = __shfl_sync(0xFFFFFFFFu, at, lane_row + i * kStep);
                const bool read = row >= 0 && in_head;
                const int64_t o = read ? row + lane_chunk * 8 : 0;
                piece(i, static_cast<const uint16_t*>(p.k) + o, static_cast<const uint16_t*>(p.v) + o, read);
            }
        }
    };
    look_up();
    for (int i = 0; i < kStages - 1; ++i) {
        copy_unit(i);
        copies_commit();
        look_up();
    }

    int stage = 0;
    bool go = true;
    while (go) {
        // Queries of the piece: rows of DP, zeros behind D and behind the item's rows.
        auto token_of = [&](int r) { return (int)((unsigned)(w.it.r0 + r) / (unsigned)p.G); };  // from the item's first on
        auto query_at = [&](int r) {  // row r's place in q
            const int t = token_of(r), g = w.it.r0 + r - t * p.G;
            return ((int64_t)w.q.q0 + w.it.t0 + t) * p.q_token + ((int64_t)w.head * p.G + g) * p.q_head;
        };
        for (int e = threadIdx.x; e < kRows * kChunks; e += kThreads) {
            const int r = e / kChunks, c = e % kChunks;
            uint4 v = make_uint4(0u, 0u, 0u, 0u);
            if (r < w.it.rows && c * 8 < p.D) {
                const uint16_t* src = static_cast<const uint16_t*>(p.q) + query_at(r) + c * 8;
                if (p.q_vec) {
                    v = *reinterpret_cast<const uint4*>(src);
                } else {
                    uint32_t h[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) h[i] = (uint32_t)src[2 * i] | (uint32_t)src[2 * i + 1] << 16;
                    v = make_uint4(h[0], h[1], h[2], h[3]);
                }
            }
            *reinterpret_cast<uint4*>(qs + chunk_at<DP>(r, c)) = v;
        }
        __syncthreads();
        const uint32_t qa = smem_of(qs);
        // A fragment of 16 rows x 16 elements: lanes 0-15 rows, low 8 elements; 16-31 the same rows, high 8.
        auto query = [&](int mt, int ks, uint32_t (&a)[4]) {
            ldsm4(qa + chunk_at<DP>(16 * mt + (lane & 15), 2 * ks + (lane >> 4)), a);
        };
        uint32_t qf[Sh::kQInRegs ? kSteps : 1][4];
        if constexpr (Sh::kQInRegs) {
#pragma unroll
            for (int ks = 0; ks < kSteps; ++ks) query(0, ks, qf[ks]);
        }
        int pos[MT][2];  // positions of this lane's rows (-1: none)
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int r = 16 * mt + 8 * h + (lane >> 2);
                pos[mt][h] = r < w.it.rows ? w.it.p_lo + token_of(r) : -1;
            }
        float o[MT][kTiles][4], m[MT][2], l[MT][2];  // m: maximum in use, in units of c q k
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
            for (int t = 0; t < kTiles; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i) o[mt][t][i] = 0.0f;
            m[mt][0] = m[mt][1] = -INFINITY;
            l[mt][0] = l[mt][1] = 0.0f;
        }

        for (int u = 0; u < w.count; ++u) {
            copies_wait<kStages - 2>();
            __syncwarp();  // the unit is there, and the one before has been read by all lanes: its stage takes the unit kStages - 1 ahead
            copy_unit(stage == 0 ? kStages - 1 : stage - 1);
            copies_commit();
            look_up();
            const uint32_t ks0 = ring + stage * 2 * Sh::kSliceBytes, vs0 = ks0 + Sh::kSliceBytes;
            const int j0 = w.key0(u) + warp * kSlice;
            float s[MT][kNT][4];
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                for (int nt = 0; nt < kNT; ++nt)
#pragma unroll
                    for (int i = 0; i < 4; ++i) s[mt][nt][i] = 0.0f;
#pragma unroll
            for (int ks = 0; ks < kSteps; ++ks) {
                uint32_t b[kNT / 2][4];  // of 16 keys: 0-7 low, high elements; 8-15 low, high
#pragma unroll
                for (int n = 0; n < kNT / 2; ++n)
                    ldsm4(ks0 + chunk_at<DP>(16 * n + (lane & 7) + ((lane >> 4) << 3), 2 * ks + ((lane >> 3) & 1)), b[n]);
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) {
                    uint32_t a[4];
                    if constexpr (Sh::kQInRegs) {
#pragma unroll
                        for (int i = 0; i < 4; ++i) a[i] = qf[ks][i];
                    } else {
                        query(mt, ks, a);
                    }
#pragma unroll
                    for (int n = 0; n < kNT / 2; ++n) {
                        mma<BF16>(s[mt][2 * n], a, b[n][0], b[n][1]);
                        mma<BF16>(s[mt][2 * n + 1], a, b[n][2], b[n][3]);
                    }
                }
            }
            const bool masked = !all_see(p, w.it, j0, kSlice);
            if (masked)
#pragma unroll
                for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                    for (int nt = 0; nt < kNT; ++nt)
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            if (!sees(p, pos[mt][i >> 1], j0 + 8 * nt + 2 * (lane & 3) + (i & 1))) s[mt][nt][i] = -INFINITY;
            // Maxima of the rows; lanes of a quad share a row.
            bool raise = false;
            float top[MT][2];
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    float v = fmaxf(s[mt][0][2 * h], s[mt][0][2 * h + 1]);
#pragma unroll
                    for (int nt = 1; nt < kNT; ++nt) v = fmaxf(v, fmaxf(s[mt][nt][2 * h], s[mt][nt][2 * h + 1]));
                    v = fmaxf(v, __shfl_xor_sync(0xFFFFFFFFu, v, 1));
                    v = fmaxf(v, __shfl_xor_sync(0xFFFFFFFFu, v, 2)) * p.c;
                    top[mt][h] = v;
                    raise |= v > m[mt][h] + kSlack || (m[mt][h] == -INFINITY && v > -INFINITY);
                }
            if (__any_sync(0xFFFFFFFFu, raise)) {
#pragma unroll
                for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const float now = fmaxf(m[mt][h], top[mt][h]);
                        // (From -inf: nothing has been added yet.)
                        const float f = m[mt][h] == -INFINITY ? 0.0f : exp2_fast(m[mt][h] - now);
                        m[mt][h] = now;
                        l[mt][h] *= f;
#pragma unroll
                        for (int t = 0; t < kTiles; ++t) {
                            o[mt][t][2 * h] *= f;
                            o[mt][t][2 * h + 1] *= f;
                        }
                    }
            }
            uint32_t pa[MT][kNT / 2][4], pb[SPLIT ? MT : 1][kNT / 2][4];
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const float base = m[mt][h] == -INFINITY ? 0.0f : m[mt][h] - kShift;
#pragma unroll
                    for (int nt = 0; nt < kNT; ++nt) {
                        float& x = s[mt][nt][2 * h];
                        float& y = s[mt][nt][2 * h + 1];
                        x = exp2_fast(fmaf(x, p.c, -base));
                        y = exp2_fast(fmaf(y, p.c, -base));
                        l[mt][h] += x + y;
                        const uint32_t two = pack2<BF16>(x, y);
                        pa[mt][nt >> 1][2 * (nt & 1) + h] = two;
                        if constexpr (SPLIT)
                            pb[mt][nt >> 1][2 * (nt & 1) + h] = pack2<BF16>(x - value_of<BF16>(two & 0xFFFFu), y - value_of<BF16>(two >> 16));
                    }
                }
            }
            // A value that not all rows see may be infinite or NaN, and its weight of zero
            // must not meet it: such elements are added to the rows that see them one by
            // one, and are zeros to the product below.
            if (MULTI && masked && w.it.p_lo != w.it.p_hi) {
                bool bad = false;
#pragma unroll
                for (int i = 0; i < kPieces; ++i) {
                    uint32_t v[4];
                    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3])
                                 : "r"(vs0 + (i * 32 + lane) * 16)
                                 : "memory");
#pragma unroll
                    for (int k = 0; k < 4; ++k) bad |= not_finite<BF16>(v[k] & 0xFFFFu) || not_finite<BF16>(v[k] >> 16);
                }
                if (__any_sync(0xFFFFFFFFu, bad)) {
                    uint8_t* const vs = smem + (vs0 - smem_of(smem));
#pragma unroll 1
                    for (int k = 0; k < kSlice; ++k) {
                        float wt[MT][2];
                        bool see[MT][2];
#pragma unroll
                        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                            for (int h = 0; h < 2; ++h) {
                                // Key k's weight is in lane (k % 8) / 2 of the quad, element k % 2 of tile k / 8.
                                float e = 0.0f;
#pragma unroll
                                for (int nt = 0; nt < kNT; ++nt)
                                    if (k >> 3 == nt) e = (k & 1) ? s[mt][nt][2 * h + 1] : s[mt][nt][2 * h];
                                wt[mt][h] = __shfl_sync(0xFFFFFFFFu, e, (lane & ~3) | ((k & 7) >> 1));
                                see[mt][h] = sees(p, pos[mt][h], j0 + k);
                            }
#pragma unroll
                        for (int t = 0; t < kTiles; ++t) {
                            const uint32_t two = *reinterpret_cast<const uint32_t*>(vs + chunk_at<DP>(k, t) + 4 * (lane & 3));
#pragma unroll
                            for (int e = 0; e < 2; ++e) {
                                const uint32_t bits = e ? two >> 16 : two & 0xFFFFu;
                                if (not_finite<BF16>(bits)) {
#pragma unroll
                                    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                                        for (int h = 0; h < 2; ++h)
                                            if (see[mt][h]) o[mt][t][2 * h + e] += wt[mt][h] * value_of<BF16>(bits);
                                }
                            }
                        }
                    }
                    __syncwarp();
                    for (int i = lane; i < kSlice * DP; i += 32) {
                        uint16_t* e = reinterpret_cast<uint16_t*>(vs) + i;
                        if (not_finite<BF16>(*e)) *e = 0;
                    }
                    __syncwarp();
                }
            }
#pragma unroll
            for (int t = 0; t < kTiles; t += 2) {
                uint32_t b[kNT / 2][4];  // tile t: keys 0-7, 8-15; tile t + 1: the same
#pragma unroll
                for (int n = 0; n < kNT / 2; ++n) ldsm4t(vs0 + chunk_at<DP>(16 * n + (lane & 15), t + (lane >> 4)), b[n]);
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) {
                    float d[2][4] = {};
#pragma unroll
                    for (int n = 0; n < kNT / 2; ++n)
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            float(&sum)[4] = FRESH ? d[i] : o[mt][t + i];
                            mma<BF16>(sum, pa[mt][n], b[n][2 * i], b[n][2 * i + 1]);
                            if constexpr (SPLIT) mma<BF16>(sum, pb[mt][n], b[n][2 * i], b[n][2 * i + 1]);
                        }
                    if constexpr (FRESH)
#pragma unroll
                        for (int i = 0; i < 8; ++i) o[mt][t + (i >> 2)][i & 3] += d[i >> 2][i & 3];
                }
            }
            if (++stage == kStages) stage = 0;
        }

        // Join the warps: everybody's factor against the largest maximum, then outputs
        // of warps 2, 3 onto 0, 1, and of 1 onto 0, 16 rows at a time.
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                l[mt][h] += __shfl_xor_sync(0xFFFFFFFFu, l[mt][h], 1);
                l[mt][h] += __shfl_xor_sync(0xFFFFFFFFu, l[mt][h], 2);
            }
        __syncthreads();  // (queries are read from here on no more)
        if ((lane & 3) == 0)
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int r = 16 * mt + 8 * h + (lane >> 2);
                    join_ml[warp * kRows + r] = m[mt][h];
                    join_ml[(kWarps + warp) * kRows + r] = l[mt][h];
                }
        __syncthreads();
        float big[MT][2], sum[MT][2];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int r = 16 * mt + 8 * h + (lane >> 2);
                float x = -INFINITY, y = 0.0f;
                for (int k = 0; k < kWarps; ++k) x = fmaxf(x, join_ml[k * kRows + r]);
                for (int k = 0; k < kWarps; ++k) {  // (without a maximum the sum is 0, or NaN)
                    const float mk = join_ml[k * kRows + r], lk = join_ml[(kWarps + k) * kRows + r];
                    y += mk > -INFINITY ? lk * exp2_fast(mk - x) : lk;
                }
                big[mt][h] = x;
                sum[mt][h] = y;
                const float f = m[mt][h] == -INFINITY ? 1.0f : exp2_fast(m[mt][h] - x);  // (1: zeros, or NaN)
#pragma unroll
                for (int t = 0; t < kTiles; ++t) {
                    o[mt][t][2 * h] *= f;
                    o[mt][t][2 * h + 1] *= f;
                }
            }
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
            for (int step = 2; step; step >>= 1) {
                if (mt || step == 1) __syncthreads();
                if (warp >= step && warp < 2 * step) {
                    float4* d = reinterpret_cast<float4*>(join + (warp - step) * 16 * DP) + lane;
#pragma unroll
                    for (int t = 0; t < kTiles; ++t) d[t * 32] = make_float4(o[mt][t][0], o[mt][t][1], o[mt][t][2], o[mt][t][3]);
                }
                __syncthreads();
                if (warp < step) {
                    const float4* d = reinterpret_cast<const float4*>(join + warp * 16 * DP) + lane;
#pragma unroll
                    for (int t = 0; t < kTiles; ++t) {
                        const float4 x = d[t * 32];
                        o[mt][t][0] += x.x, o[mt][t][1] += x.y, o[mt][t][2] += x.z, o[mt][t][3] += x.w;
                    }
                }
            }
        }
        if (warp == 0) {
            const bool whole = w.whole();
            bool over = false;
            if (lane == 0) w.cut(Runs(all_units, gridDim.x), blockIdx.x, note);
            float* const part = whole ? nullptr : slots + (2ll * blockIdx.x + w.slot()) * part_floats(kRows, p.D);
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int r = 16 * mt + 8 * h + (lane >> 2);
                    if (r >= w.it.rows) continue;
                    const int t = token_of(r), head = w.head * p.G + (w.it.r0 + r - t * p.G);
                    const int64_t row = (int64_t)w.q.q0 + w.it.t0 + t;
                    if (whole) {
                        const float f = sum[mt][h] == 0.0f ? 0.0f : 1.0f / sum[mt][h];
                        const int64_t at = row * p.o_token + head * p.o_head;
#pragma unroll
                        for (int tt = 0; tt < kTiles; ++tt) {
                            const int d = 8 * tt + 2 * (lane & 3);
                            if (d >= p.D) break;
                            float x = o[mt][tt][2 * h] * f, y = o[mt][tt][2 * h + 1] * f;
                            if constexpr (Y == NXQ_F32) {
                                float* e = static_cast<float*>(p.out) + at + d;
                                e[0] = x, e[1] = y;
                            } else {
                                if constexpr (Y == NXQ_F16) x = for_f16<BF16>(x, over), y = for_f16<BF16>(y, over);
                                const uint32_t two = pack2<Y == NXQ_BF16>(x, y);
                                uint16_t* e = static_cast<uint16_t*>(p.out) + at + d;
                                if (p.o_vec) {
                                    *reinterpret_cast<uint32_t*>(e) = two;
                                } else {
                                    e[0] = (uint16_t)two, e[1] = (uint16_t)(two >> 16);
                                }
                            }
                        }
                        if (p.lse && (lane & 3) == 0)
                            p.lse[row * ((int64_t)p.Hk * p.G) + head] =
                                sum[mt][h] == 0.0f ? -INFINITY : (big[mt][h] - kShift + log2f(sum[mt][h])) * 0.6931471805599453f;
                    } else {
#pragma unroll
                        for (int tt = 0; tt < kTiles; ++tt) {
                            const int d = 8 * tt + 2 * (lane & 3);
                            if (d >= p.D) break;
                            *reinterpret_cast<float2*>(part + (int64_t)r * p.D + d) = make_float2(o[mt][tt][2 * h], o[mt][tt][2 * h + 1]);
                        }
                        if ((lane & 3) == 0) {
                            part[(int64_t)kRows * p.D + r] = big[mt][h] - kShift;
                            part[(int64_t)kRows * p.D + kRows + r] = sum[mt][h];
                        }
                    }
                }
            if (Y == NXQ_F16 && BF16 && over) raise_range(p.status, kRangeAttn);
        }
        __syncthreads();  // the join's memory is the next piece's queries'
        go = w.next(p);
    }
    copies_wait<0>();
}

// Whether a kernel's sums are fresh ones anyway.
template <int DP, int MT, bool SPLIT>
constexpr bool kAlwaysFresh = SPLIT || MT == 1 || DP <= 64;
// Whether they must be where there is a choice: a unit (64 keys) is one sum more toward zero, 7.5e-8 of the
// result each, and together they are to stay below a sixth of half a step of the output's type.  (No
// sequence is longer than its row of the block table.)
bool sums_fresh(const AttnParams& p) { return p.b.capacity / 64 > (p.y_dtype == NXQ_F16 ? 1 << 10 : 1 << 13); }

template <int DP, int MT, bool BF16, int Y>
auto* kernel_of(bool multi, bool fresh) {
    constexpr bool kF = kAlwaysFresh<DP, MT, Y == NXQ_F32>;
    return multi ? (fresh ? attn_mma_kernel<BF16, Y, true, true, DP, MT> : attn_mma_kernel<BF16, Y, true, kF, DP, MT>)
                 : (fresh ? attn_mma_kernel<BF16, Y, false, true, DP, MT> : attn_mma_kernel<BF16, Y, false, kF, DP, MT>);
}
template <int DP, int MT, bool BF16>
auto* kernel_of(int y, bool multi, bool fresh) {
    return y == NXQ_F32   ? kernel_of<DP, MT, BF16, NXQ_F32>(multi, fresh)
           : y == NXQ_F16 ? kernel_of<DP, MT, BF16, NXQ_F16>(multi, fresh)
                          : kernel_of<DP, MT, BF16, NXQ_BF16>(multi, fresh);
}
template <int DP, int MT>
auto* kernel_of(bool bf16, int y, bool multi, bool fresh) {
    return bf16 ? kernel_of<DP, MT, true>(y, multi, fresh) : kernel_of<DP, MT, false>(y, multi, fresh);
}

template <int DP, int MT>
int set_attr() {
    for (const int y : {NXQ_F32, NXQ_F16, NXQ_BF16})
        for (int i = 0; i < 8; ++i) {
            const cudaError_t e = cudaFuncSetAttribute(kernel_of<DP, MT>(i & 1, y, i & 2, i & 4),
                                                       cudaFuncAttributeMaxDynamicSharedMemorySize, Shape<DP, MT>::kSmem);
            if (e != cudaSuccess) return cuda_fail(e, "cudaFuncSetAttribute (attn_mma)");
        }
    return NXQ_OK;
}

template <int DP>
unsigned grid_of() {
    static_assert(DP == 256 || Shape<DP, 1>::kCtas == Shape<DP, 2>::kCtas, "one grid for both");
    return (unsigned)context_sm_count() * Shape<DP, 1>::kCtas;
}

template <int DP, int MT>
cudaError_t launch(const AttnParams& p, bool bf16, cudaStream_t st) {
    return launch_overlapped(kernel_of<DP, MT>(bf16, p.y_dtype, p.max_new > 1, sums_fresh(p)), grid_of<DP>(), kThreads,
                            Shape<DP, MT>::kSmem, st, p);
}

}  // namespace

int attn_mma_init() {
    int rc;
    if ((rc = set_attr<64, 1>()) || (rc = set_attr<64, 2>()) || (rc = set_attr<128, 1>()) || (rc = set_attr<128, 2>()) ||
        (rc = set_attr<256, 1>()))
        return rc;
    return NXQ_OK;
}

// (Heads beyond 128 elements: 32 rows of outputs do not fit the registers.)
int attn_mma_rows(int D, int64_t rows) { return rows <= 16 || D > 128 ? 16 : 32; }

unsigned attn_mma_grid(int D) { return D <= 64 ? grid_of<64>() : D <= 128 ? grid_of<128>() : grid_of<256>(); }

int attn_mma(const AttnParams& p, int dtype, int rows, cudaStream_t st) {
    note_launches(1);
    const bool bf = dtype == NXQ_BF16, two = rows == 32;
    const cudaError_t e = p.D <= 64    ? (two ? launch<64, 2>(p, bf, st) : launch<64, 1>(p, bf, st))
                          : p.D <= 128 ? (two ? launch<128, 2>(p, bf, st) : launch<128, 1>(p, bf, st))
                                       : launch<256, 1>(p, bf, st);
    if (e != cudaSuccess) return cuda_fail(e, "attention launch");
    const cudaError_t j = launch_attn_join(p, rows, attn_mma_grid(p.D), st);
    return j == cudaSuccess ? NXQ_OK : cuda_fail(j, "attention join launch");
}

}  // namespace nxq
