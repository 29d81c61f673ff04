// The work of an attention launch, derived by every CTA from the lengths on the device.
//
// A row is one (new token, query head) pair of a sequence and key head: row r is token
// r / G, query head r % G of the group, so the rows of a group share every key they
// read.  An item is ROWS consecutive rows of one (sequence, key head); a unit is one of its
// blocks of KEYS keys, those with at least one key that a row of the item sees (an
// item that sees none has one unit all the same, which writes its zeros).  Units are numbered
// by sequence, key head, item, key block, and each of the launch's runs gets an equal
// share of consecutive units, whatever the lengths are.  A run that holds an item
// whole writes its output; pieces of an item cut between runs go to the workspace,
// two slots a run (0: a piece that starts inside an item, 1: one that starts an item
// and does not end it), the run in which the item starts leaves a note of it, and the
// join kernel adds the pieces up in order of the runs.
#pragma once
#include "attention.h"

namespace nxq {
namespace attn {

constexpr int kPlanChunk = 256;  // sequences looked at together

__device__ __forceinline__ long long divide(long long n, int d) {
    return (unsigned long long)n >> 32 ? n / d : (long long)((unsigned)n / (unsigned)d);
}

// An item's rows: row r is token t0 + (r0 + r) / G of its sequence's new ones, query head
// (r0 + r) % G.
struct Item {
    int rows;
    int t0, r0;
    int p_lo, p_hi;        // positions of the first and the last row
    int head_blocks;       // units that hold the sinks (blocks 0 ..)
    int skip;              // unit u >= head_blocks is block u + skip
    int units;
};

template <int ROWS, int KEYS>
__device__ __forceinline__ Item make_item(const AttnParams& p, const Seq& q, int j) {
    Item it;
    const int total = q.n * p.G, row0 = j * ROWS;  // below 2^31 (nxq_paged_attention)
    it.rows = total - row0 < ROWS ? total - row0 : ROWS;
    it.t0 = (int)((unsigned)row0 / (unsigned)p.G);
    it.r0 = row0 - it.t0 * p.G;
    it.p_lo = q.len - q.n + it.t0;
    it.p_hi = it.p_lo + (int)((unsigned)(it.r0 + it.rows - 1) / (unsigned)p.G);
    const int end = it.p_hi < 0 ? 0 : it.p_hi / KEYS + 1;  // blocks up to the last visible key
    int lo = 0, heads = 0;
    if (p.window > 0 && it.p_lo >= p.window) {
        const int first = it.p_lo - p.window + 1;
        lo = first / KEYS;
        const int sinks = p.sinks < first ? p.sinks : first;
        heads = (sinks + KEYS - 1) / KEYS;
        if (heads > lo) heads = lo;
    }
    it.head_blocks = heads;
    it.skip = lo - heads;
    const int units = heads + (end - lo);
    it.units = units > 0 ? units : 1;
    return it;
}

// Items of a sequence and key head.
template <int ROWS>
__device__ __forceinline__ int items_of(const AttnParams& p, const Seq& q) {
    return (int)(((unsigned)(q.n * p.G) + ROWS - 1) / ROWS);
}
// Sequence s if it is this launch's, else one without rows.
__device__ __forceinline__ Seq launch_seq(const AttnParams& p, int s, bool* bad) {
    Seq q = read_seq(p.b, s, p.max_new, bad);
    const int64_t rows = (int64_t)q.n * p.G;
    if (rows <= p.rows_lo || rows > p.rows_hi) q.n = 0;
    return q;
}

struct PlanSmem {
    Seq seqs[kPlanChunk];              // of the chunk looked at last
    long long units[kPlanChunk];       // of each of them, per key head
    long long chunks[65536 / kPlanChunk];  // of each chunk
    long long total;                   // of all sequences and key heads
    // A unit's place.
    Seq q;
    int s, head, item, off;
};

// Units of the sequences of one chunk into sm.units, by the whole CTA.  With few
// sequences several threads share one, for their item counts may be large.
template <int ROWS, int KEYS, int THREADS>
__device__ __forceinline__ void plan_chunk(const AttnParams& p, PlanSmem& sm, int chunk, bool report) {
    const int s0 = chunk * kPlanChunk, n = p.b.S - s0 < kPlanChunk ? p.b.S - s0 : kPlanChunk;
    int share = 1;
    while (share < 32 && 2 * share * n <= THREADS) share *= 2;
    for (int i0 = 0; i0 < n; i0 += THREADS / share) {
        const int i = i0 + threadIdx.x / share, part = threadIdx.x % share;
        long long u = 0;
        Seq q{0, 0, 0};
        if (i < n) {
            bool bad;
            q = launch_seq(p, s0 + i, &bad);
            if (bad && report && part == 0) raise_index(p.status, kIndexSeq);
            const int items = items_of<ROWS>(p, q);
            for (int j = part; j < items; j += share) u += make_item<ROWS, KEYS>(p, q, j).units;
        }
        for (int o = share / 2; o; o >>= 1) u += __shfl_xor_sync(0xFFFFFFFFu, u, o);
        if (i < n && part == 0) {
            sm.units[i] = u;
            sm.seqs[i] = q;
        }
    }
    for (int i = n + threadIdx.x; i < kPlanChunk; i += THREADS) sm.units[i] = 0;
}

__device__ __forceinline__ long long warp_sum(long long v) {
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
    return v;
}
// By a converged warp: the first i < n (n a multiple of 32) with a running sum of v(0 .. i) > x, and x
// less the sum before it.  There is one.
template <typename F>
__device__ __forceinline__ int warp_locate(F v, int n, long long& x) {
    const int lane = threadIdx.x & 31;
    for (int i0 = 0; i0 < n; i0 += 32) {
        const long long mine = v(i0 + lane);
        long long sum = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long t = __shfl_up_sync(0xFFFFFFFFu, sum, o);
            if (lane >= o) sum += t;
        }
        const unsigned m = __ballot_sync(0xFFFFFFFFu, sum > x);
        if (m) {
            const int at = __ffs(m) - 1;
            x -= __shfl_sync(0xFFFFFFFFu, sum - mine, at);
            return i0 + at;
        }
        x -= __shfl_sync(0xFFFFFFFFu, sum, 31);
    }
    return n - 1;
}

// First pass: all units (sm.total).  By the whole CTA; ends with a barrier.
template <int ROWS, int KEYS, int THREADS>
__device__ __forceinline__ void plan_total(const AttnParams& p, PlanSmem& sm) {
    const int chunks = (p.b.S + kPlanChunk - 1) / kPlanChunk;
    for (int c = 0; c < chunks; ++c) {
        plan_chunk<ROWS, KEYS, THREADS>(p, sm, c, p.first && blockIdx.x == 0);
        __syncthreads();
        if (threadIdx.x < 32) {
            long long u = 0;
            for (int i = threadIdx.x; i < kPlanChunk; i += 32) u += sm.units[i];
            u = warp_sum(u);
            if (threadIdx.x == 0) {
                sm.chunks[c] = u;
                sm.total = (c ? sm.total : 0) + u * p.Hk;
            }
        }
        __syncthreads();
    }
}

// Unit x < sm.total of the launch: its sequence, key head, item and place in the item
// (sm.s, .head, .item, .off).  After plan_total, by the whole CTA; ends with a barrier.
template <int ROWS, int KEYS, int THREADS>
__device__ __forceinline__ void plan_locate(const AttnParams& p, PlanSmem& sm, long long x) {
    const int chunks = (p.b.S + kPlanChunk - 1) / kPlanChunk;
    int c = 0;
    if (chunks > 1) {  // sm.units holds the last chunk: make the one that x lies in
        long long y = x;
        c = warp_locate([&](int i) { return i < chunks ? sm.chunks[i] * p.Hk : 0ll; }, (chunks + 31) / 32 * 32, y);
        __syncthreads();
        plan_chunk<ROWS, KEYS, THREADS>(p, sm, c, false);
        __syncthreads();
        x = y;
    }
    if (threadIdx.x < 32) {
        const int i = warp_locate([&](int i) { return sm.units[i] * p.Hk; }, kPlanChunk, x);
        const long long per = sm.units[i];
        const int head = (int)(((unsigned long long)x | per) >> 32 ? x / per : (unsigned)x / (unsigned)per);
        x -= head * per;
        const Seq q = sm.seqs[i];
        const int items = items_of<ROWS>(p, q);
        const int j = warp_locate([&](int j) { return j < items ? (long long)make_item<ROWS, KEYS>(p, q, j).units : 0ll; },
                                  (items + 31) / 32 * 32, x);
        if (threadIdx.x == 0) {
            sm.q = q;
            sm.s = c * kPlanChunk + i;
            sm.head = head;
            sm.item = j;
            sm.off = (int)x;
        }
    }
    __syncthreads();
}

// The units of a launch's runs: run r < live has units each, or one more if r < more;
// the other runs (fewer units than runs) have none.
struct Runs {
    long long each;
    int more, live;
    __device__ __forceinline__ Runs(long long total, int grid) {
        live = total < grid ? (int)total : grid;
        each = live ? divide(total, live) : 0;
        more = (int)(total - each * live);
    }
    __device__ __forceinline__ long long start(int r) const { return r < live ? each * r + (r < more ? r : more) : each * live + more; }
    __device__ __forceinline__ long long units(int r) const { return r < live ? each + (r < more) : 0; }
    // Runs that `left` units behind run r, directly after it, reach into.
    __device__ __forceinline__ int behind(int r, int left) const {
        if (each >= left) return 1;
        const unsigned e = (unsigned)each, big = more > r + 1 ? more - r - 1 : 0;  // of them with a unit more
        return (unsigned long long)big * (e + 1) >= (unsigned)left ? (left + e) / (e + 1) : big + (left - big * (e + 1) + e - 1) / e;
    }
};

// What the join kernel has to do for a run: the item that begins in it and ends behind it.
struct Cut {
    int pieces;  // 0: there is none
    int rows, r0, t0;
    int q0, head, pad[2];
};
__host__ __device__ inline size_t cuts_bytes(unsigned runs) { return runs * sizeof(Cut); }

// Walks a run's pieces.  Every lane of a warp holds the same values.
template <int ROWS, int KEYS>
struct Walk {
    Seq q;
    Item it;
    int s, head, item, off;  // the piece: units off .. off + count - 1 of the item
    int count;
    int items;
    long long left;  // units of the run from the piece on

    __device__ __forceinline__ void piece() { count = (int)(it.units - off < left ? it.units - off : left); }
    __device__ __forceinline__ void start(const AttnParams& p, const PlanSmem& sm, long long units) {
        q = sm.q, s = sm.s, head = sm.head, item = sm.item, off = sm.off;
        left = units;
        items = items_of<ROWS>(p, q);
        it = make_item<ROWS, KEYS>(p, q, item);
        piece();
    }
    // The next piece; false at the end of the run.
    __device__ __forceinline__ bool next(const AttnParams& p) {
        left -= count;
        if (left <= 0) return false;
        off = 0;
        if (++item == items) {
            item = 0;
            if (++head == p.Hk) {
                head = 0;
                do {  // (units are left, so a sequence is)
                    if (++s >= p.b.S) return false;
                    bool bad;
                    q = launch_seq(p, s, &bad);
                } while (q.n == 0);
                items = items_of<ROWS>(p, q);
            }
        }
        it = make_item<ROWS, KEYS>(p, q, item);
        piece();
        return true;
    }
    __device__ __forceinline__ bool whole() const { return count == it.units; }
    __device__ __forceinline__ int slot() const { return off ? 0 : 1; }  // of a piece that is not whole
    // The cut of run r, if this piece is its first.
    __device__ __forceinline__ void cut(const Runs& runs, int r, Cut* to) const {
        if (off || whole()) return;
        *to = Cut{1 + runs.behind(r, it.units - count), it.rows, it.r0, it.t0, q.q0, head, {0, 0}};
    }
    // First key of the piece's unit u.
    __device__ __forceinline__ int key0(int u) const {
        u += off;
        return (u < it.head_blocks ? u : u + it.skip) * KEYS;
    }
};

// Whether the query at position pos sees key j.
__device__ __forceinline__ bool sees(const AttnParams& p, int pos, int j) {
    return j <= pos && (p.window <= 0 || j > pos - p.window || j < p.sinks);
}
// Whether keys j0 .. j0 + n - 1 are seen by all rows of the item.
__device__ __forceinline__ bool all_see(const AttnParams& p, const Item& it, int j0, int n) {
    return j0 + n - 1 <= it.p_lo && (p.window <= 0 || j0 > it.p_hi - p.window || j0 + n <= p.sinks);
}
// Whether any row of the item may see key j (its keys and values are read).
__device__ __forceinline__ bool any_sees(const AttnParams& p, const Item& it, int j) {
    return j <= it.p_hi && (p.window <= 0 || j > it.p_lo - p.window || j < p.sinks);
}

// The workspace: Cut [runs], then slots [runs][2] of partial results (then, tcgen05 kernel, fp32
// sums [runs][ROWS][D]).
// A partial result: [ROWS][D] fp32 sums of weights times values, then
// [ROWS] maxima (in units of c q k) and [ROWS] sums of weights, all relative to the maximum.
__host__ __device__ inline size_t part_floats(int rows, int D) { return (size_t)rows * (D + 2); }

// An output on its way to f16.  A finite one beyond that type is the largest value where the cache
// is f16 (the average of f16 values lies among them, but weights rounded to f16 put it up to 2^-11
// of itself outside), and is reported where it is bf16.
template <bool BF16>
__device__ __forceinline__ float for_f16(float x, bool& over) {
    if (!f16_overflows(x)) return x;
    if constexpr (!BF16) return copysignf(65504.0f, x);
    over = true;
    return x;
}

}  // namespace attn
}  // namespace nxq
