// The 4-bit KV cache: where a row's values sit, and how they are encoded.
//
// One plane holds the k (or the v) rows of one sequence and layer: KH heads of
// R rows (q4_plane_rows(maxT)), 64 bytes of codes a row and head, all heads' codes first, then all
// heads' fp16 scales, [KH][R][128 / G].  A row of a head is the Q4 format of
// the expert store along its 128 dimensions: groups of G values, the scale
// fp16(fp32(absmax / 7)), the code clip(round_half_even(v / scale), -8, 7) + 8.
//
// Heads come before rows, so that what one (sequence, head) reads is one
// contiguous stream.  Within a row the codes sit as the matrix cores take them
// (v_mfma_f32_16x16x32 gives lane l of A or B index l % 16 and 8 of the
// contraction's 32 steps, 8 (l / 16) ..):
//   k  dword 4 c + s of a row holds dimensions 32 s + 8 c .. + 7, lowest nibble
//      first: the 16 bytes c of a row are what lane group c feeds to the 4
//      contraction steps s over the head
//   v  rows in blocks of 4: dword 4 n + r % 4 of a block's 64 holds the
//      dimensions 16 j + n of row r, j = 0 .. 7 from the lowest nibble: 16
//      bytes are 4 rows of the 8 output tiles j at lane n
// A row's codes are whole dwords of its own in both, so rows are written
// independently of each other.
#pragma once

#include "jm_device.h"
#include "jm_kernels.h"

namespace jm {

// The rows of one head in one plane.
template <int NG>
struct Q4Head {
    gptr<uint32_t> codes;       // [R][16] (k), [R / 4][64] (v)
    gptr<uint16_t> scales;      // [R][NG]
    __device__ __forceinline__ Q4Head(unsigned long long plane, int kh, int KH, int R) {
        codes = (gptr<uint32_t>)plane + (size_t)kh * R * 16;
        scales = (gptr<uint16_t>)(plane + (size_t)KH * R * 64) + (size_t)kh * R * NG;
    }
    __device__ __forceinline__ gptr<uint32_t> k_dword(int r, int p) const { return codes + (size_t)r * 16 + p; }
    __device__ __forceinline__ gptr<uint32_t> v_dword(int r, int n) const {
        return codes + (size_t)(r >> 2) * 64 + 4 * n + (r & 3);
    }
    __device__ __forceinline__ gptr<uint16_t> scale(int r, int g) const { return scales + (size_t)r * NG + g; }
};

// The sequence and cache row of the four tokens t0 .. t0 + 3 of a call (not the
// decoder's form) in the wave's four rows of 16 lanes: each lane gets its row's
// token's; false for a token that has none (behind the last sequence, or a row
// outside the cache).
__device__ __forceinline__ bool q4_places(const Q4KvArgs& c, int t0, int& seq, int& pos) {
    const int lane = threadIdx.x & 63, i = lane >> 4, t = t0 + i;
    seq = t;
    int first = t;
    if (c.cu) {
        int n = 0;
        for (int s = 0; s <= c.n_seq; s += 64) {
            const int x = c.cu[min(s + lane, c.n_seq)];
#pragma unroll
            for (int q = 0; q < 4; q++) {
                const int upto = __popcll(__ballot(s + lane <= c.n_seq && x <= t0 + q));
                n += i == q ? upto : 0;
            }
        }
        seq = n - 1;
        if (t >= c.N || seq < 0 || seq >= c.n_seq) return false;
        first = c.cu[seq];
    } else if (t >= c.N || t >= c.n_seq) {
        return false;
    }
    const long long p = (long long)c.start[seq] + (t - first);
    pos = (int)(p < 0 ? -1 : p >= c.maxT ? c.maxT : p);
    return p >= 0 && p < c.maxT;
}

__device__ __forceinline__ unsigned long long q4_plane(const Q4KvArgs& c, int seq, int which) {
    if (c.pos) return c.tab[((size_t)seq * c.L + c.layer) * 2 + which];
    return (unsigned long long)(uintptr_t)(which ? c.v : c.k) + (unsigned long long)seq * c.seq_stride;
}

// A group's scale from the bits of its largest magnitude (a NaN's are the
// largest of all), and its values' codes + 8.  The quotient is the correctly
// rounded fp32 one: the scale's reciprocal rounded, then one Newton step on the
// quotient with the exact remainder.
struct Q4Group {
    uint32_t m;
    _Float16 s16;
    float s, inv;
    __device__ __forceinline__ explicit Q4Group(uint32_t largest) : m(largest) {
        const float top = m > 0x2B8CBCCCu ? __uint_as_float(m) : 1e-12f;       // (the bits of 1e-12f)
        s16 = (_Float16)__fdiv_rn(top, 7.0f);
        s = (float)s16;
        inv = __fdiv_rn(1.0f, s);
    }
    __device__ __forceinline__ uint32_t code(float x) const {
        const float a = __fmul_rn(x, inv);
        const float f = __builtin_fmaf(__builtin_fmaf(-a, s, x), inv, a);
        float n = fminf(fmaxf(rintf(f), -8.0f), 7.0f);
        // a scale of 0 (a group below 7 * 2^-25): +-inf or NaN over 0
        if (s == 0.0f) n = x > 0.0f ? 7.0f : x < 0.0f ? -8.0f : 0.0f;
        // NaN, or an infinite scale: 0, and the scale makes the value non-finite
        if (m >= 0x7F800000u || s == INFINITY) n = 0.0f;
        return (uint32_t)((int)n + 8);
    }
};

// 8 codes a lane and 8 lanes: nibble e of lane m against nibble m of lane e.
__device__ __forceinline__ uint32_t q4_transpose(uint32_t d, int m) {
    constexpr int XOR3 = 0x1B;              // quad_perm(3,2,1,0)
    uint32_t o = (uint32_t)dpp_i<XOR3>(dpp_i<DPP_HALF_MIRROR>((int)d));     // lane ^ 4
    d = __builtin_amdgcn_perm(o, d, m & 4 ? 0x03020706u : 0x05040100u);
    o = (uint32_t)dpp_i<DPP_XOR2>((int)d);
    d = __builtin_amdgcn_perm(o, d, m & 2 ? 0x03070105u : 0x06020400u);
    o = (uint32_t)dpp_i<DPP_XOR1>((int)d);
    const uint32_t keep = m & 1 ? 0xF0F0F0F0u : 0x0F0F0F0Fu;
    return (d & keep) | ((m & 1 ? o >> 4 : o << 4) & ~keep);
}

// One head's 128 values of one row by 16 lanes (a row of the wave), lane 8 g + m
// with the 8 dimensions from 8 q4_chunk() on; k (isk) or v.
__device__ __forceinline__ int q4_chunk() { return 2 * (threadIdx.x & 7) + ((threadIdx.x >> 3) & 1); }
__device__ __forceinline__ int q4_k_at(int chunk) { return 4 * (chunk & 3) + (chunk >> 2); }    // its dword of a k row

template <int NG>
__device__ __forceinline__ void q4_store_chunk(const float (&x)[8], bool isk, int r, const Q4Head<NG>& h) {
    const int o = q4_chunk();
    uint32_t m = 0;
#pragma unroll
    for (int e = 0; e < 8; e++) m = max(m, __float_as_uint(x[e]) & 0x7FFFFFFFu);
    m = max(m, (uint32_t)dpp_i<DPP_XOR1>((int)m));
    if (NG == 2) m = max(m, (uint32_t)dpp_i<DPP_XOR2>((int)m));
    m = max(m, (uint32_t)dpp_i<DPP_ROR8>((int)m));
    const Q4Group q(m);
    uint32_t d = 0;
#pragma unroll
    for (int e = 0; e < 8; e++) d |= q.code(x[e]) << (4 * e);
    if (o % (16 / NG) == 0) *h.scale(r, o / (16 / NG)) = __builtin_bit_cast(uint16_t, q.s16);
    const uint32_t y = q4_transpose(d, threadIdx.x & 7);
    *(isk ? h.k_dword(r, q4_k_at(o)) : h.v_dword(r, threadIdx.x & 15)) = isk ? d : y;
}

template <int NG>
__device__ __forceinline__ void q4_load_chunk(float (&x)[8], bool isk, int r, const Q4Head<NG>& h) {
    const int o = q4_chunk();
    uint32_t d = *(isk ? h.k_dword(r, q4_k_at(o)) : h.v_dword(r, threadIdx.x & 15));
    const float s = fp16_hw(*h.scale(r, o / (16 / NG)));
    const uint32_t y = q4_transpose(d, threadIdx.x & 7);
    d = isk ? d : y;
#pragma unroll
    for (int e = 0; e < 8; e++) x[e] = __fmul_rn((float)((int)((d >> (4 * e)) & 15u) - 8), s);
}

// The same store by 32 lanes (an aligned half of the wave; lane j holds
// dimensions 4 j .. + 3), as the decoder's append has them.
template <int NG>
__device__ __forceinline__ void q4_store_row(const float (&x)[4], bool isk, int r, int j, const Q4Head<NG>& h) {
    uint32_t m = 0;
#pragma unroll
    for (int e = 0; e < 4; e++) m = max(m, __float_as_uint(x[e]) & 0x7FFFFFFFu);
#pragma unroll
    for (int o = 1; o < 32 / NG; o <<= 1) m = max(m, (uint32_t)__shfl_xor((int)m, o, JM_WAVE));
    const Q4Group g(m);
    uint32_t q[4];
#pragma unroll
    for (int e = 0; e < 4; e++) q[e] = g.code(x[e]);
    if (j % (32 / NG) == 0) *h.scale(r, j / (32 / NG)) = __builtin_bit_cast(uint16_t, g.s16);
    if (isk) {
        const uint32_t half = q[0] | (q[1] << 4) | (q[2] << 8) | (q[3] << 12);
        const uint32_t other = (uint32_t)__shfl_xor((int)half, 1, JM_WAVE);
        const int o = j >> 1;               // dimensions 8 o .. + 7
        if ((j & 1) == 0) *h.k_dword(r, 4 * (o & 3) + (o >> 2)) = half | (other << 16);
    } else {
        // nibble j / 4 of dwords 4 (j % 4) + e: gathered over lanes 4, 8 and 16 apart
        uint32_t d[4];
#pragma unroll
        for (int e = 0; e < 4; e++) d[e] = q[e] << (4 * (j >> 2));
        const bool h16 = j & 16, h8 = j & 8;
        uint32_t a0 = h16 ? d[2] : d[0], a1 = h16 ? d[3] : d[1];
        a0 |= (uint32_t)__shfl_xor((int)(h16 ? d[0] : d[2]), 16, JM_WAVE);
        a1 |= (uint32_t)__shfl_xor((int)(h16 ? d[1] : d[3]), 16, JM_WAVE);
        uint32_t b = h8 ? a1 : a0;
        b |= (uint32_t)__shfl_xor((int)(h8 ? a0 : a1), 8, JM_WAVE);
        b |= (uint32_t)__shfl_xor((int)b, 4, JM_WAVE);
        if ((j & 4) == 0) *h.v_dword(r, 4 * (j & 3) + (h16 ? 2 : 0) + (h8 ? 1 : 0)) = b;
    }
}

}  // namespace jm
