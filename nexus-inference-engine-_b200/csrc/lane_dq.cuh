// Per-lane f16 decoders of the register-fragment kernels (qmm_mma.cu,
// ragged_mma.cu): the warp-level MMA they feed, and for each block type the
// 64-element slice of a row of a staged tile-chunk that one lane decodes.
#pragma once
#include "dq_f16.cuh"

namespace nxq {
namespace lane {

using dq::h2u;
using dq::u2h;

// C[16 rows][8 tokens] += A[16 rows][16 k] * B[16 k][8 tokens]; f16 in, fp32 accumulate.
__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                         uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
        "{%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t word_of(const uint4& v, int i) {
    return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w;
}

// ---------------------------------------------------------------------------
// Per-format lane decoders.  load() reads the lane's 64-element slice (chunk
// elements 64t .. 64t+63) of row `row` of a staged tile-chunk and its scales;
// pairs(m, p) returns elements 8m .. 8m+7 of the slice as four f16 pairs
// (2i, 2i+1), i = 0..3.
// ---------------------------------------------------------------------------
template <int TYPE>
struct Lane;

// Q4_K / Q5_K header hd = (d, dmin, scales[12]): the f16 scale and offset
// pairs of sub-blocks 2t, 2t+1.  Scale bytes 2t, 2t+1 hold the 6-bit scale
// and the low 2 bits of the min, nibbles of bytes 8 + 2(t&1) + {0,1} the high
// 4 bits of the min.  (scale, min) pairs become exact f16 integers by the
// magic number; one f16 multiply by (d, d) / (-dmin, -dmin) then rounds d*sc
// and -dmin*m once each, as fp32 math followed by one rounding would.
__device__ __forceinline__ void kquant_lane_scales(const uint4& hd, int t, __half2 (&s2)[2], __half2 (&o2)[2]) {
    const uint32_t v = __byte_perm(((t < 2 ? hd.y : hd.z) >> (16 * (t & 1))), 0u, 0x4140u);
    const uint32_t e = __byte_perm(((hd.w >> (16 * (t & 1))) >> (4 * (t >> 1))), 0u, 0x4140u);
    const __half2 magic = u2h(0x64006400u);
    const __half2 sc = __hsub2(u2h((v & 0x003F003Fu) | 0x64006400u), magic);
    const __half2 mn = __hsub2(u2h(((v >> 6) & 0x00030003u) | ((e & 0x000F000Fu) << 2) | 0x64006400u), magic);
    const uint32_t sp = h2u(__hmul2(sc, u2h(__byte_perm(hd.x, 0u, 0x1010u))));
    const uint32_t op = h2u(__hmul2(mn, u2h(__byte_perm(hd.x, 0u, 0x3232u) ^ 0x80008000u)));
    s2[0] = u2h(__byte_perm(sp, 0u, 0x1010u));
    s2[1] = u2h(__byte_perm(sp, 0u, 0x3232u));
    o2[0] = u2h(__byte_perm(op, 0u, 0x1010u));
    o2[1] = u2h(__byte_perm(op, 0u, 0x3232u));
}

// Q4_K (gguf_importer.cpp:838-873): record = block (d, dmin, scales[12], qs[128]);
// the slice is sub-blocks 2t, 2t+1 = code bytes 32t .. 32t+31.
template <>
struct Lane<T_Q4_K> {
    static constexpr int kStage = TILE_ROWS * 144;
    uint4 q0, q1;
    __half2 s2[2], o2[2];
    __device__ __forceinline__ void load(const uint8_t* st, int row, int t) {
        const uint8_t* rec = st + row * 144;
        const uint4 hd = *reinterpret_cast<const uint4*>(rec);
        q0 = *reinterpret_cast<const uint4*>(rec + 16 + 32 * t);
        q1 = *reinterpret_cast<const uint4*>(rec + 32 + 32 * t);
        kquant_lane_scales(hd, t, s2, o2);
    }
    __device__ __forceinline__ void pairs(int m, uint32_t (&p)[4]) const {
        dq::q4_word_pairs(word_of(m < 4 ? q0 : q1, m & 3), s2[m >> 2], o2[m >> 2], p);
    }
};

// Q5_K (gguf_importer.cpp:878-915): record = [d, dmin, scales[12]][L words of
// 8 groups][H words] (formats.cuh, q5_hi_bit); the slice is sub-blocks 2t,
// 2t+1: L words at 16 + 32t, H words at 144 + 8t.
template <>
struct Lane<T_Q5_K> {
    static constexpr int kStage = TILE_ROWS * 176;
    uint4 q0, q1;
    uint2 hh;
    __half2 s2[2], o2[2];
    __device__ __forceinline__ void load(const uint8_t* st, int row, int t) {
        const uint8_t* rec = st + row * 176;
        const uint4 hd = *reinterpret_cast<const uint4*>(rec);
        q0 = *reinterpret_cast<const uint4*>(rec + 16 + 32 * t);
        q1 = *reinterpret_cast<const uint4*>(rec + 32 + 32 * t);
        hh = *reinterpret_cast<const uint2*>(rec + 144 + 8 * t);
        kquant_lane_scales(hd, t, s2, o2);
    }
    __device__ __forceinline__ void pairs(int m, uint32_t (&p)[4]) const {
        const uint32_t l = word_of(m < 4 ? q0 : q1, m & 3), h = m < 4 ? hh.x : hh.y;
        switch (m & 3) {
            case 0: dq::q5_word_pairs<0>(l, h, s2[m >> 2], o2[m >> 2], p); break;
            case 1: dq::q5_word_pairs<1>(l, h, s2[m >> 2], o2[m >> 2], p); break;
            case 2: dq::q5_word_pairs<2>(l, h, s2[m >> 2], o2[m >> 2], p); break;
            default: dq::q5_word_pairs<3>(l, h, s2[m >> 2], o2[m >> 2], p); break;
        }
    }
};

// Q6_K (gguf_importer.cpp:924-954): plane A = 8 x [L0 L1 L2 L3 H0 H1] per row
// (formats.cuh, q6_lo_bit); the slice (elements 64t .. 64t+63) is groups 2t,
// 2t+1 = 48 bytes at r*192 + 48t, with scales 4t .. 4t+3 (16 elements each)
// and d.  Weights fl16((q - 32) * fl16(d * sc)).
template <>
struct Lane<T_Q6_K> {
    static constexpr int kStage = TILE_ROWS * 210;
    uint32_t L[8], H[4];
    __half2 s2[4];
    __device__ __forceinline__ void load(const uint8_t* st, int row, int t) {
        const uint4* rec = reinterpret_cast<const uint4*>(st + row * 192 + 48 * t);
        const uint4 a = rec[0], b = rec[1], c = rec[2];
        L[0] = a.x; L[1] = a.y; L[2] = a.z; L[3] = a.w;
        H[0] = b.x; H[1] = b.y;
        L[4] = b.z; L[5] = b.w; L[6] = c.x; L[7] = c.y;
        H[2] = c.z; H[3] = c.w;
        const uint32_t sc = *reinterpret_cast<const uint32_t*>(st + TILE_ROWS * 192 + row * 16 + 4 * t);
        const float d = __half2float(__ushort_as_half(*reinterpret_cast<const uint16_t*>(st + TILE_ROWS * 208 + row * 2)));
#pragma unroll
        for (int i = 0; i < 4; ++i) s2[i] = __float2half2_rn(d * (float)(int8_t)(sc >> (8 * i)));
    }
    // Elements 8m .. 8m+7 of the slice: group m >> 2, L word m & 3, scale m >> 1.
    __device__ __forceinline__ void pairs(int m, uint32_t (&p)[4]) const {
        const int g = m >> 2, wl = m & 3;
        if (wl & 1)
            dq::q6_word_pairs<2>(L[4 * g + wl], H[2 * g + (wl >> 1)], s2[m >> 1], p);
        else
            dq::q6_word_pairs<0>(L[4 * g + wl], H[2 * g + (wl >> 1)], s2[m >> 1], p);
    }
};

// NXF INT4 groups (quant/gptq.cpp:9-27): record = [(scale, zero) per group of
// the chunk, padded to H bytes][codes x8 of 16 B]; sub-blocks 2t, 2t+1 of the
// slice lie in groups 64t / gs and (64t + 32) / gs.  Weights
// fl16(q * fl16(scale) + fl16(-(zero * scale))).
template <int TYPE>
struct LaneI4G {
    static constexpr int GS = i4g_gs(TYPE), H = i4g_hdr(TYPE), REC = H + CHUNK_K / 2;
    static constexpr int kStage = TILE_ROWS * REC;
    uint4 q0, q1;
    __half2 s2[2], o2[2];
    __device__ __forceinline__ void load(const uint8_t* st, int row, int t) {
        const uint8_t* rec = st + row * REC;
        q0 = *reinterpret_cast<const uint4*>(rec + H + 32 * t);
        q1 = *reinterpret_cast<const uint4*>(rec + H + 16 + 32 * t);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const float2 sz = *reinterpret_cast<const float2*>(rec + 8 * ((64 * t + 32 * h) / GS));
            s2[h] = __float2half2_rn(sz.x);
            o2[h] = __float2half2_rn(-(sz.y * sz.x));
        }
    }
    __device__ __forceinline__ void pairs(int m, uint32_t (&p)[4]) const {
        dq::q4_word_pairs(word_of(m < 4 ? q0 : q1, m & 3), s2[m >> 2], o2[m >> 2], p);
    }
};
template <>
struct Lane<T_I4G32> : LaneI4G<T_I4G32> {};
template <>
struct Lane<T_I4G64> : LaneI4G<T_I4G64> {};
template <>
struct Lane<T_I4G128> : LaneI4G<T_I4G128> {};
template <>
struct Lane<T_I4G256> : LaneI4G<T_I4G256> {};

// Q4_0 (gguf_importer.cpp:679-695): record = [d x8][codes x8 of 16 B]; the
// slice is blocks 2t, 2t+1.
template <>
struct Lane<T_Q4_0> {
    static constexpr int kStage = TILE_ROWS * 144;
    uint4 q0, q1;
    __half2 s2[2], o2[2];
    __device__ __forceinline__ void load(const uint8_t* st, int row, int t) {
        const uint8_t* rec = st + row * 144;
        const uint32_t dw = *reinterpret_cast<const uint32_t*>(rec + 4 * t);
        q0 = *reinterpret_cast<const uint4*>(rec + 16 + 32 * t);
        q1 = *reinterpret_cast<const uint4*>(rec + 32 + 32 * t);
        const __half2 neg8 = u2h(0xC800C800u);
        s2[0] = u2h((dw & 0xFFFFu) | (dw << 16));
        s2[1] = u2h((dw >> 16) | (dw & 0xFFFF0000u));
        o2[0] = __hmul2(s2[0], neg8);  // exact
        o2[1] = __hmul2(s2[1], neg8);
    }
    __device__ __forceinline__ void pairs(int m, uint32_t (&p)[4]) const {
        dq::q4_word_pairs(word_of(m < 4 ? q0 : q1, m & 3), s2[m >> 2], o2[m >> 2], p);
    }
};

// Q4_1 (gguf_importer.cpp:699-717): record = [(d, m) x8][codes x8 of 16 B];
// the slice is blocks 2t, 2t+1; weights fl16(q * d + m).
template <>
struct Lane<T_Q4_1> {
    static constexpr int kStage = TILE_ROWS * 160;
    uint4 q0, q1;
    __half2 s2[2], o2[2];
    __device__ __forceinline__ void load(const uint8_t* st, int row, int t) {
        const uint8_t* rec = st + row * 160;
        const uint2 dm = *reinterpret_cast<const uint2*>(rec + 8 * t);
        q0 = *reinterpret_cast<const uint4*>(rec + 32 + 32 * t);
        q1 = *reinterpret_cast<const uint4*>(rec + 48 + 32 * t);
        s2[0] = u2h((dm.x & 0xFFFFu) | (dm.x << 16));
        o2[0] = u2h((dm.x >> 16) | (dm.x & 0xFFFF0000u));
        s2[1] = u2h((dm.y & 0xFFFFu) | (dm.y << 16));
        o2[1] = u2h((dm.y >> 16) | (dm.y & 0xFFFF0000u));
    }
    __device__ __forceinline__ void pairs(int m, uint32_t (&p)[4]) const {
        dq::q4_word_pairs(word_of(m < 4 ? q0 : q1, m & 3), s2[m >> 2], o2[m >> 2], p);
    }
};

// Q2_K (gguf_importer.cpp:756-786): plane A = [scales[16]][8 x [L0 L1]] per
// row (formats.cuh, q2_tiled_byte), plane B = (dmin, d); the slice (elements
// 64t .. 64t+63) is code words 4t .. 4t+3 with scale bytes 4t .. 4t+3.
template <>
struct Lane<T_Q2_K> {
    static constexpr int kStage = TILE_ROWS * 84;
    uint4 q;
    __half2 s2[4], o2[4];
    __device__ __forceinline__ void load(const uint8_t* st, int row, int t) {
        const uint8_t* rec = st + row * 80;
        q = *reinterpret_cast<const uint4*>(rec + 16 + 16 * t);
        const uint32_t sc = *reinterpret_cast<const uint32_t*>(rec + 4 * t);
        const uint32_t dd = *reinterpret_cast<const uint32_t*>(st + TILE_ROWS * 80 + row * 4);
        const float dmin = __half2float(__ushort_as_half((unsigned short)(dd & 0xFFFFu)));
        const float d = __half2float(__ushort_as_half((unsigned short)(dd >> 16)));
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t b = (sc >> (8 * i)) & 0xFFu;
            s2[i] = __float2half2_rn(d * (float)(b & 15u));
            o2[i] = __float2half2_rn(-(dmin * (float)(b >> 4)));
        }
    }
    // Elements 8m .. 8m+7: code word m >> 1 (low or high byte of each half),
    // scale group m >> 1.
    __device__ __forceinline__ void pairs(int m, uint32_t (&p)[4]) const {
        const uint32_t l = word_of(q, m >> 1);
        dq::q2_half_pairs((m & 1) ? l >> 8 : l, s2[m >> 1], o2[m >> 1], p);
    }
};

// Q8_0 (gguf_importer.cpp:721-733): record = [d x8][codes x8 of 32 B]; the
// slice is blocks 2t, 2t+1 = code bytes 64t .. 64t+63.
template <>
struct Lane<T_Q8_0> {
    static constexpr int kStage = TILE_ROWS * 272;
    uint4 c[4];
    __half2 s2[2];
    __device__ __forceinline__ void load(const uint8_t* st, int row, int t) {
        const uint8_t* rec = st + row * 272;
        const uint32_t dw = *reinterpret_cast<const uint32_t*>(rec + 4 * t);
        const uint4* cv = reinterpret_cast<const uint4*>(rec + 16 + 64 * t);
#pragma unroll
        for (int i = 0; i < 4; ++i) c[i] = cv[i];
        s2[0] = u2h((dw & 0xFFFFu) | (dw << 16));
        s2[1] = u2h((dw >> 16) | (dw & 0xFFFF0000u));
    }
    __device__ __forceinline__ void pairs(int m, uint32_t (&p)[4]) const {
        // Signed byte b -> f16 1152 + b via (b ^ 0x80) in the mantissa of 1024.
        const __half2 bias = u2h(0x64806480u);
        const uint32_t w0 = word_of(c[m >> 1], 2 * (m & 1)), w1 = word_of(c[m >> 1], 2 * (m & 1) + 1);
        const __half2 s = s2[m >> 2];
        p[0] = h2u(__hmul2(__hsub2(u2h(__byte_perm(w0, 0u, 0x4140u) ^ 0x64806480u), bias), s));
        p[1] = h2u(__hmul2(__hsub2(u2h(__byte_perm(w0, 0u, 0x4342u) ^ 0x64806480u), bias), s));
        p[2] = h2u(__hmul2(__hsub2(u2h(__byte_perm(w1, 0u, 0x4140u) ^ 0x64806480u), bias), s));
        p[3] = h2u(__hmul2(__hsub2(u2h(__byte_perm(w1, 0u, 0x4342u) ^ 0x64806480u), bias), s));
    }
};

// Q3_K (gguf_importer.cpp:791-833): plane A = 8 x [L0 L1 H] per row (tiled
// code order, formats.cuh q3_lo_pos), plane B = [scales 12][d] at 128*96 +
// row*14.  The slice's elements are groups 2t, 2t+1 = bytes 24t .. 24t+23 of
// the row's plane-A record, in four 16-element scale groups.
template <>
struct Lane<T_Q3_K> {
    static constexpr int kStage = TILE_ROWS * 110;
    uint32_t L[4], H[2], Hr[2];  // L0, L1 of group 2t, then of 2t+1; their high-bit words
    __half2 s2[4];
    __device__ __forceinline__ void load(const uint8_t* st, int row, int t) {
        const uint8_t* rec = st + row * 96 + 24 * t;
        const uint2 a = *reinterpret_cast<const uint2*>(rec);
        const uint2 b = *reinterpret_cast<const uint2*>(rec + 8);
        const uint2 c = *reinterpret_cast<const uint2*>(rec + 16);
        L[0] = a.x;
        L[1] = a.y;
        H[0] = b.x;
        L[2] = b.y;
        L[3] = c.x;
        H[1] = c.y;
        Hr[0] = __funnelshift_r(H[0], H[0], 8);
        Hr[1] = __funnelshift_r(H[1], H[1], 8);
        const uint16_t* tl = reinterpret_cast<const uint16_t*>(st + TILE_ROWS * 96 + row * 14);
        // Groups G = 4t + gg (gg = 0..3): i8 = G & 7 = 4(t&1) + gg; the low 4
        // bits of the 6-bit scale are nibble (t >> 1) of scale byte i8, the
        // high 2 bits are bits 2(t >> 1) + {0,1} of nibble (gg & 1) of byte
        // 8 + 2(t&1) + (gg >> 1).  (scale - 32) * d as one f16 rounding of the
        // exact product, through exact f16 integers.
        const uint32_t lo4 = ((t & 1) ? (tl[2] | ((uint32_t)tl[3] << 16)) : (tl[0] | ((uint32_t)tl[1] << 16)));
        const uint32_t hi2 = (uint32_t)tl[4 + (t & 1)];  // bytes 8 + 2(t&1), +1
        const uint32_t sh = 4 * (t >> 1), hs = 2 * (t >> 1);
        const __half2 d2 = u2h(__byte_perm((uint32_t)tl[6], 0u, 0x1010u));
        const __half2 bias = u2h(0x64206420u);  // 1056 = magic + 32
#pragma unroll
        for (int pr = 0; pr < 2; ++pr) {  // groups gg = 2pr, 2pr+1
            const uint32_t l = (__byte_perm(lo4, 0u, 0x4040u | ((2 * pr + 1) << 8) | (2 * pr)) >> sh) & 0x000F000Fu;
            const uint32_t hb = (hi2 >> (8 * pr)) & 0xFFu;  // byte for gg = 2pr, 2pr+1: nibbles 0, 1
            const uint32_t h = (((hb >> hs) & 3u) | ((((hb >> 4) >> hs) & 3u) << 16)) << 4;
            const uint32_t sp = h2u(__hmul2(__hsub2(u2h(l | h | 0x64006400u), bias), d2));
            s2[2 * pr] = u2h(__byte_perm(sp, 0u, 0x1010u));
            s2[2 * pr + 1] = u2h(__byte_perm(sp, 0u, 0x3232u));
        }
    }
    // Elements 8m .. 8m+7 of the slice: group m >> 2, L word (m & 3) >> 1,
    // pairs 4((m & 3) & 1) .. +3 of that word.
    __device__ __forceinline__ void pairs(int m, uint32_t (&p)[4]) const {
        const int g = m >> 2, j = (m & 3) >> 1;
        uint32_t l = L[2 * g + j], h = j ? Hr[g] : H[g];
        if (m & 1) {
            l >>= 8;
            h >>= 1;
        }
        const __half2 s = s2[m >> 1];
        p[0] = dq::q3_pair<0>(l, h, s);
        p[1] = dq::q3_pair<1>(l, h, s);
        p[2] = dq::q3_pair<2>(l, h, s);
        p[3] = dq::q3_pair<3>(l, h, s);
    }
};

}  // namespace lane
}  // namespace nxq
