// Attention over a paged cache of keys and values: what the position rotation, the
// append and the attention kernels share.
#pragma once
#include "nxq_internal.h"

namespace nxq {

// A registered position rotation (the nxq_rope_t handle).
struct Rope {
    int dims;    // rotated elements of a head
    int layout;  // NXQ_ROPE_HALF / _INTERLEAVED
    float scale;
    // Turns per position of each pair, modulo 1, in units of 2^-64: position * turns
    // modulo 2^64 is the angle of any position, without an error that grows with it.
    uint64_t* turns = nullptr;
};
// NXQ_OK and the rotation behind a live handle, else the status the C ABI returns.
int check_rope(nxq_rope_t h, const Rope** out);
void ropes_shutdown();

// Tokens of a batch and of a sequence's cache at most: positions, and positions less
// a window, are ints.
constexpr int64_t kMaxTokens = 1 << 30;

// The sequences of a step as the kernels see them.
struct Batch {
    const int32_t *q_off, *kv_len, *table;
    int64_t table_stride;
    int64_t capacity;  // positions that a row of the table has pages for, kMaxTokens at most
    int64_t T;
    int S, page;
    int64_t pages;
};

// One sequence's new tokens: rows q0 .. q0 + n - 1, at positions len - n ...  A
// sequence that is left out has n = 0.
struct Seq {
    int q0, n, len;
};
__device__ __forceinline__ Seq read_seq(const Batch& b, int s, int64_t max_new, bool* bad) {
    const int q0 = b.q_off[s], q1 = b.q_off[s + 1], len = b.kv_len[s];
    *bad = q0 < 0 || q1 < q0 || q1 > b.T || len < 0 || len > b.capacity || (int64_t)q1 - q0 > max_new;
    return *bad ? Seq{0, 0, 0} : Seq{q0, q1 - q0, len};
}

// Checks of the C ABI (host).  `elem` is the size of an element.
int check_cache(const nxq_kv_cache* c);
int check_batch(const nxq_kv_batch* b, int64_t T);
int check_heads(const char* what, const nxq_heads* h, int dtype);
Batch make_batch(const nxq_kv_cache* c, const nxq_kv_batch* b, int64_t T);

// A call of the attention kernels.
struct AttnParams {
    Batch b;
    const void *q, *k, *v;
    void* out;
    float* lse;  // or null
    int64_t q_token, q_head, o_token, o_head;          // strides in elements
    int64_t page_stride, head_stride, slot_stride;
    int Hk, G, D;      // key heads, query heads per key head, elements of a head
    int y_dtype;
    int bf16;          // the cache's type
    int q_vec, o_vec;  // rows of q (of the output) are multiples of 16 bytes, at such an address (o_vec 2: of 32)
    int page_shift;    // log2 of the page size, or -1
    int page_align;    // the largest power of two that divides the page size
    float c;           // scale * log2(e): weights are exp2(c q k)
    int window, sinks; // window 0: none
    int max_new;
    int64_t rows_lo, rows_hi;  // sequences of rows_lo < n G <= rows_hi rows are this launch's
    int first;             // reports what is wrong with the batch
    void* work;            // partial results of runs (attn_plan.cuh)
    DeviceStatus* status;
};

// Kernel of few rows per sequence and key head, or of any (attn_mma.cu): a grid of
// attn_mma_grid(p) runs.
int attn_mma_init();
int attn_mma_rows(int D, int64_t rows);           // rows of an item where a sequence has `rows` at most
unsigned attn_mma_grid(int D);
int attn_mma(const AttnParams& p, int dtype, int rows, cudaStream_t st);

// Kernel of many rows (attn_tc.cu), for caches that it can read: a grid of
// attn_tc_grid() runs, items of attn_tc_rows() rows.
int attn_tc_init();
bool attn_tc_supported(const nxq_kv_cache* c);
int attn_tc_rows();
unsigned attn_tc_grid();
int attn_tc(const AttnParams& p, const nxq_kv_cache* cache, cudaStream_t st);

// Joins the partial results of a launch of `runs` runs with items of `rows` rows (attention.cu).
cudaError_t launch_attn_join(const AttnParams& p, int rows, unsigned runs, cudaStream_t st);

}  // namespace nxq
