// The 4-bit KV cache's operators: rows quantised as they are written, read
// back, and attended over (jm_q4kv.h has the layout).
#include <algorithm>

#include "jm_q4kv.h"

namespace jm {

// 4 consecutive values of a float32 or bf16 tensor.
template <bool BF>
__device__ __forceinline__ void load4(const void* p, size_t i, float (&v)[4]) {
    if (BF) {
        const uint2 u = *(const uint2*)((const uint16_t*)p + i);
        v[0] = bf16_bits_to_f32(u.x & 0xFFFFu);
        v[1] = __uint_as_float(u.x & 0xFFFF0000u);
        v[2] = bf16_bits_to_f32(u.y & 0xFFFFu);
        v[3] = __uint_as_float(u.y & 0xFFFF0000u);
    } else {
        const float4 u = *(const float4*)((const float*)p + i);
        v[0] = u.x; v[1] = u.y; v[2] = u.z; v[3] = u.w;
    }
}

template <bool BF>
__device__ __forceinline__ void store4(void* p, size_t i, const float (&v)[4]) {
    if (BF) *(uint2*)((uint16_t*)p + i) = make_uint2(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]));
    else *(float4*)((float*)p + i) = make_float4(v[0], v[1], v[2], v[3]);
}

// One wave per (token, KV head): lanes 0..31 the k row, 32..63 the v row.
template <int NG, bool BF>
__global__ void __launch_bounds__(256)
k_q4_write(Q4KvArgs c, const void* __restrict__ k, const void* __restrict__ v, long long kts, long long khs,
           long long vts, long long vhs) {
    const int lane = threadIdx.x & 63, j = lane & 31;
    const int item = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int t = item / c.KH, kh = item % c.KH;
    if (t >= c.N) return;
    int seq, r;
    if (!q4_place(c, t, seq, r)) return;
    const bool isk = lane < 32;
    float x[4];
    load4<BF>(isk ? k : v, (size_t)(isk ? t * kts + kh * khs : t * vts + kh * vhs) + 4 * j, x);
    const Q4Head<NG> h(q4_plane(c, seq, isk ? 0 : 1), kh, c.KH, c.R);
    q4_store_row<NG>(x, isk, r, j, h);
}

// The rows back, one wave per (token, KV head): the exact values, bf16 rounded.
template <int NG, bool BF>
__global__ void __launch_bounds__(256)
k_q4_read(Q4KvArgs c, void* __restrict__ k, void* __restrict__ v) {
    const int lane = threadIdx.x & 63, j = lane & 31;
    const int item = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int t = item / c.KH, kh = item % c.KH;
    if (t >= c.N) return;
    int seq, r;
    if (!q4_place(c, t, seq, r)) return;
    const bool isk = lane < 32;
    const Q4Head<NG> h(q4_plane(c, seq, isk ? 0 : 1), kh, c.KH, c.R);
    const float s = fp16_hw(*h.scale(r, j / (32 / NG)));
    float x[4];
    if (isk) {
        const int o = j >> 1;
        const uint32_t w = *h.k_dword(r, 4 * (o & 3) + (o >> 2)) >> (16 * (j & 1));
#pragma unroll
        for (int e = 0; e < 4; e++) x[e] = __fmul_rn((float)((int)((w >> (4 * e)) & 15u) - 8), s);
    } else {
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const uint32_t w = *h.v_dword(r, 4 * (j & 3) + e) >> (4 * (j >> 2));
            x[e] = __fmul_rn((float)((int)(w & 15u) - 8), s);
        }
    }
    store4<BF>(isk ? k : v, (size_t)item * 128 + 4 * j, x);
}

// ---------------------------------------------------------------- attention
//
// A unit is what one block takes of the queries: a KV head and up to 8 query
// rows of one sequence, 8 / qpk consecutive tokens of the head's qpk query
// heads.  The cache rows that its last token sees are cut into S ranges of
// 32-row tiles; wave w of block (head, unit, range) takes every fourth tile of
// the range with a running maximum and sum of its own, the block merges its
// waves and k_q4_merge the ranges.  No cache byte goes through LDS: rows come in
// the order in which the matrix cores take them (jm_q4kv.h).
//
// Operands.  One AND-OR gives two codes as fp16, 1024 + q from nibbles 0 and 4
// of a dword, or 1024 + 16 q from 1 and 5, and one packed subtraction q - 8, or 16
// times that (which the other operand or the end takes back), exactly.  (The
// codes' bits as subnormals, without either, came out of the matrix cores right
// to only 2^-14 of a sum: 7e-5 of the output instead of 5e-7.)
//
//   scores   v_mfma_f32_16x16x32_f16, 16 cache rows as A, the 8 query rows as B
//            in columns n < 8, q brought to [1, 2) by a power of two and rounded
//            to fp16, the rest of it times 2^11 in columns n + 8; one product a
//            32 dimensions, one scale a group.  Lane (g, n) gets column n of rows
//            4 g + i: with the two halves added (one DPP move), the scores of
//            query row n % 8 at 8 rows of the tile.
//   weights  exp2(score - ref), ref common to a column's lanes and chosen so that
//            weight x V scale stays below 2^15: raised only when a lane meets a
//            product above 2^14, to where the largest is 2^6, so that most tiles
//            need no exchange between lanes.  Each lane sums its own weights.
//   P . V    16 dimensions a product (dimension 16 j + m is row m of product j,
//            nibble j of the lane's V dwords) as A, weight x scale in fp16, the
//            rest times 2^11 in columns n + 8, as B, from the lanes that formed
//            them: contraction index 8 g + e is row 16 (e / 4) + 4 g + e % 4.
// q and the weights carry 21 bits so; for bf16 queries (BF) q is exact without
// the second half, and the weights are rounded to fp16 once (2^-11 of each).

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ f16x8 as_f16x8(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    return __builtin_bit_cast(f16x8, make_uint4(a, b, c, d));
}

// The codes less 8 of nibbles 0 and 4 of w, and 16 times those of nibbles 1 and 5.
__device__ __forceinline__ uint32_t q4_even(uint32_t w) {
    const f16x2 h = __builtin_bit_cast(f16x2, (w & 0x000F000Fu) | 0x64006400u) - f16x2{(_Float16)1032.0f, (_Float16)1032.0f};
    return __builtin_bit_cast(uint32_t, h);
}
__device__ __forceinline__ uint32_t q4_odd(uint32_t w) {
    const f16x2 h = __builtin_bit_cast(f16x2, (w & 0x00F000F0u) | 0x64006400u) - f16x2{(_Float16)1152.0f, (_Float16)1152.0f};
    return __builtin_bit_cast(uint32_t, h);
}

__device__ __forceinline__ float pow2f(float x) { return __builtin_amdgcn_exp2f(x); }

// The KV head's query rows of one unit: which sequence, its first token, how
// many tokens, the first token's cache row.
struct Q4Unit {
    int seq, tok, n, pos;
};

// Unit u of the call for tp tokens a unit (without cu and in the decoder's form:
// token u alone); false if there is none.  The same in every lane.
__device__ __forceinline__ bool q4_unit(const Q4KvArgs& c, int u, int tp, Q4Unit& q) {
    if (!c.cu) {
        q.seq = q.tok = u;
        q.n = 1;
        q.pos = c.pos ? c.pos[u] : c.start[u];
        return true;
    }
    const int lane = threadIdx.x & 63;
    int base = 0;
    for (int s0 = 0; s0 < c.n_seq; s0 += 64) {
        const int s = s0 + lane;
        const int t0 = c.cu[min(s, c.n_seq)], t1 = c.cu[min(s + 1, c.n_seq)];
        const int n = s < c.n_seq ? max(t1 - t0, 0) : 0;
        const unsigned units = (unsigned)((n + tp - 1) / tp), upto = wave_inclusive_scan(units);
        const unsigned long long below = __ballot(base + (int)upto <= u);
        const int all = base + (int)__builtin_amdgcn_readlane((int)upto, 63);
        if (u < all) {
            const int l = __popcll(below);                  // the first sequence whose units pass u
            const int k = u - base - (int)__builtin_amdgcn_readlane((int)(upto - units), l);
            q.seq = s0 + l;
            q.tok = __builtin_amdgcn_readlane(t0, l) + k * tp;
            q.n = min(tp, __builtin_amdgcn_readlane(n, l) - k * tp);
            q.n = min(q.n, c.N - q.tok);
            const long long p = (long long)c.start[q.seq] + k * tp;
            q.pos = (int)(p < -c.N ? -c.N : p > c.maxT ? c.maxT : p);
            return q.n > 0 && q.tok >= 0;
        }
        base = all;
    }
    return false;
}

struct Q4AttnArgs {
    const void* q;              // strides qts, qhs
    long long qts, qhs;
    int H, qpk, tp;             // tp tokens a unit
    float scale2;               // score scale times log2(e)
    void* out;                  // [N][H][128]
    int units, S;
    float* part_o;              // [units][KH][S][qpk tp][128]: not divided by the sum
    float* part_ml;             // [units][KH][S][qpk tp][2]: ref, sum
};

constexpr float Q4_LO = 2048.0f;        // what the second halves are times

// The two fp16 halves of a and b: the values rounded towards 0, and the rest
// times 2^11.
__device__ __forceinline__ void split_f16x2(float a, float b, uint32_t& hi, uint32_t& lo) {
    const auto h = __builtin_amdgcn_cvt_pkrtz(a, b);
    const float ra = __builtin_fmaf((float)h[0], -Q4_LO, __fmul_rn(a, Q4_LO));
    const float rb = __builtin_fmaf((float)h[1], -Q4_LO, __fmul_rn(b, Q4_LO));
    hi = __builtin_bit_cast(uint32_t, h);
    lo = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(ra, rb));
}

template <bool BF>
__device__ __forceinline__ void store_out(void* p, size_t i, float4 v) {
    if (BF) *(uint2*)((uint16_t*)p + i) = make_uint2(pack_bf16x2(v.x, v.y), pack_bf16x2(v.z, v.w));
    else *(float4*)((float*)p + i) = v;
}

// One tile of 32 cache rows as a lane gets it: 16 bytes of K codes of rows
// 16 t + l % 16, of V codes of the row blocks 4 t + l / 16, and the scales of
// rows 16 t + 4 (l / 16) .. + 3.
template <int NG>
struct Q4Tile {
    u32x4_t k[2], v[2];
    u32x4_t ks[NG], vs[NG];     // (NG / 2 words of 16 bytes a row group t)
};

template <int NG>
__device__ __forceinline__ void q4_load_tile(Q4Tile<NG>& x, const Q4Head<NG>& k, const Q4Head<NG>& v, int tile, int lane) {
    const int g = lane >> 4, n = lane & 15;
#pragma unroll
    for (int t = 0; t < 2; t++) {
        const size_t r = (size_t)32 * tile + 16 * t;
        x.k[t] = *(gptr<const u32x4_t>)(k.codes + (r + n) * 16 + 4 * g);
        x.v[t] = *(gptr<const u32x4_t>)(v.codes + r * 16 + 64 * g + 4 * n);
#pragma unroll
        for (int i = 0; i < NG / 2; i++) {
            x.ks[t * (NG / 2) + i] = ((gptr<const u32x4_t>)(k.scales + (r + 4 * g) * NG))[i];
            x.vs[t * (NG / 2) + i] = ((gptr<const u32x4_t>)(v.scales + (r + 4 * g) * NG))[i];
        }
    }
}

// scale of row i (0..3) of row group t, group e
template <int NG>
__device__ __forceinline__ float q4_scale(const u32x4_t (&s)[NG], int t, int i, int e) {
    const int h = i * NG + e;                               // fp16 index within the row group
    const uint32_t w = s[t * (NG / 2) + h / 8][(h % 8) / 2];
    return (float)__builtin_bit_cast(f16x2, w)[h % 2];
}

template <int NG, bool BF>
__global__ void __launch_bounds__(256, 2)
k_q4_attn(Q4KvArgs c, Q4AttnArgs a) {
    constexpr int HD = 128, GS = 4 / NG;                    // contraction steps a group
    __shared__ __align__(16) float ow[4][8][HD];
    __shared__ float mls[4][8][2];
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int g = lane >> 4, n = lane & 15, col = n & 7;
    const int kh = blockIdx.x % c.KH, u = blockIdx.x / c.KH % a.units, s = blockIdx.x / c.KH / a.units;
    Q4Unit un;
    if (!q4_unit(c, u, a.tp, un)) return;                   // (block-uniform)
    const int ncol = a.qpk * un.n;
    const int ct = min(col / a.qpk, un.n - 1), head = kh * a.qpk + col % a.qpk;
    const int last = min(un.pos + un.n - 1, c.maxT - 1);    // the last row any token sees
    const int crow = min(un.pos + ct, c.maxT - 1);          // and this column's
    const int NT = (last + 32) / 32;                        // (0 where last < 0)
    const int t_end = (int)((long long)NT * (s + 1) / a.S);
    int t = (int)((long long)NT * s / a.S) + w;

    const Q4Head<NG> kk(q4_plane(c, un.seq, 0), kh, c.KH, c.R), vv(q4_plane(c, un.seq, 1), kh, c.KH, c.R);
    Q4Tile<NG> cur, nxt;
    if (t < t_end) q4_load_tile(cur, kk, vv, t, lane);

    // the query columns: dimensions 32 st + 8 g + e, pairs (e, e + 4)
    const bool lo_col = !BF && n >= 8;
    f16x8 qb[4];
    float lf;
    {
        float x[4][8];
        float top = 0.0f;
        const size_t qi = (size_t)((un.tok + ct) * a.qts + head * a.qhs);
#pragma unroll
        for (int st = 0; st < 4; st++) {
            float y[4];
            load4<BF>(a.q, qi + 32 * st + 8 * g, y);
#pragma unroll
            for (int e = 0; e < 4; e++) x[st][e] = y[e];
            load4<BF>(a.q, qi + 32 * st + 8 * g + 4, y);
#pragma unroll
            for (int e = 0; e < 4; e++) x[st][4 + e] = y[e];
        }
#pragma unroll
        for (int st = 0; st < 4; st++)
#pragma unroll
            for (int e = 0; e < 8; e++) top = fmaxf(top, fabsf(x[st][e]));
        top = fmaxf(top, swz_xor16_f(top));
        top = fmaxf(top, __shfl_xor(top, 32, JM_WAVE));
        // the power of two below the column's largest value
        const uint32_t ex = min(max(__float_as_uint(top) >> 23, 2u), 252u);
        const float f = __uint_as_float((254u - ex) << 23);
        // q's power of two, the scale and the halves' factor
        lf = __fmul_rn(__fmul_rn(__uint_as_float(ex << 23), a.scale2), lo_col ? 1.0f / Q4_LO : 1.0f);
#pragma unroll
        for (int st = 0; st < 4; st++) {
            uint32_t b[4];
#pragma unroll
            for (int e = 0; e < 4; e++) {
                uint32_t hi, lo;
                split_f16x2(__fmul_rn(x[st][e], f), __fmul_rn(x[st][e + 4], f), hi, lo);
                const f16x2 h = __builtin_bit_cast(f16x2, lo_col ? lo : hi);
                // codes of nibbles 1, 3, 5 and 7 come 16 times too large
                b[e] = __builtin_bit_cast(uint32_t, e & 1 ? h * (_Float16)0.0625f : h);
            }
            qb[st] = as_f16x8(b[0], b[1], b[2], b[3]);
        }
    }

    f32x4 O[8];
#pragma unroll
    for (int j = 0; j < 8; j++) O[j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    float ref = -INFINITY, l = 0.0f;

    for (; t < t_end; t += 4) {
        if (t + 4 < t_end) q4_load_tile(nxt, kk, vv, t + 4, lane);
        // ---- scores
        float y[8];
#pragma unroll
        for (int rt = 0; rt < 2; rt++) {
            f32x4 S = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int e = 0; e < NG; e++) {
                f32x4 acc = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int st = e * GS; st < (e + 1) * GS; st++) {
                    const uint32_t d = cur.k[rt][st], d8 = d >> 8;
                    acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(
                        as_f16x8(q4_even(d), q4_odd(d), q4_even(d8), q4_odd(d8)), qb[st], acc, 0, 0, 0);
                }
#pragma unroll
                for (int i = 0; i < 4; i++) S[i] = __builtin_fmaf(q4_scale(cur.ks, rt, i, e), acc[i], S[i]);
            }
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const float v = __fmul_rn(S[i], lf);
                y[4 * rt + i] = BF ? v : __fadd_rn(v, dpp_f<DPP_ROR8>(v));
            }
        }
        float sv[8][NG];
#pragma unroll
        for (int i = 0; i < 8; i++)
#pragma unroll
            for (int e = 0; e < NG; e++) sv[i][e] = q4_scale(cur.vs, i >> 2, i & 3, e);
        if (32 * t + 31 > un.pos) {                         // some column does not see the whole tile
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const bool in = 32 * t + 16 * (i >> 2) + 4 * g + (i & 3) <= crow;
                y[i] = in ? y[i] : -INFINITY;
#pragma unroll
                for (int e = 0; e < NG; e++) sv[i][e] = in ? sv[i][e] : 0.0f;
            }
        }
        // ---- the reference: the largest weight x scale, to the exponent
        float ym = y[0], sm = 0.0f;
#pragma unroll
        for (int i = 1; i < 8; i++) ym = fmaxf(ym, y[i]);
#pragma unroll
        for (int i = 0; i < 8; i++)
#pragma unroll
            for (int e = 0; e < NG; e++) sm = fmaxf(sm, sv[i][e]);
        // (sm < 2^(exponent + 1); 0, which no scale that counts is below, as 2^-24)
        float z = ym + (float)((int)(__float_as_uint(fmaxf(sm, 5.9604645e-8f)) >> 23) - 126);
        if (__any(z > ref + 14.0f)) {
            z = fmaxf(z, swz_xor16_f(z));
            z = fmaxf(z, __shfl_xor(z, 32, JM_WAVE));
            const float nref = fmaxf(ref, z - 6.0f);
            const float f = ref == -INFINITY ? 0.0f : pow2f(ref - nref);
            l *= f;
#pragma unroll
            for (int j = 0; j < 8; j++) O[j] *= f;
            ref = nref;
        }
        const float r0 = ref == -INFINITY ? 0.0f : ref;     // (a column that has seen nothing yet)
        float p[8];
#pragma unroll
        for (int i = 0; i < 8; i++) {
            p[i] = pow2f(__fsub_rn(y[i], r0));
            l = __fadd_rn(l, p[i]);
        }
        f16x8 pb[NG];
#pragma unroll
        for (int e = 0; e < NG; e++) {
            uint32_t b[4];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const float x0 = __fmul_rn(p[2 * i], sv[2 * i][e]), x1 = __fmul_rn(p[2 * i + 1], sv[2 * i + 1][e]);
                if (BF) {
                    b[i] = __builtin_bit_cast(uint32_t, f16x2{(_Float16)x0, (_Float16)x1});
                } else {
                    uint32_t hi, lo;
                    split_f16x2(x0, x1, hi, lo);
                    b[i] = lo_col ? lo : hi;
                }
            }
            pb[e] = as_f16x8(b[0], b[1], b[2], b[3]);
        }
        // ---- P . V: pairs of rows (2 i, 2 i + 1), nibbles 0..3 and 4..7
        uint32_t vl[4], vh[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const uint32_t d0 = cur.v[i >> 1][2 * (i & 1)], d1 = cur.v[i >> 1][2 * (i & 1) + 1];
            vl[i] = __builtin_amdgcn_perm(d1, d0, 0x05040100u);
            vh[i] = __builtin_amdgcn_perm(d1, d0, 0x07060302u);
        }
#pragma unroll
        for (int h = 0; h < 2; h++) {
            uint32_t (&v)[4] = h ? vh : vl;
#pragma unroll
            for (int b8 = 0; b8 < 2; b8++) {
                const int j = 4 * h + 2 * b8, e = 16 * j / (HD / NG);
                O[j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
                    as_f16x8(q4_even(v[0]), q4_even(v[1]), q4_even(v[2]), q4_even(v[3])), pb[e], O[j], 0, 0, 0);
                O[j + 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
                    as_f16x8(q4_odd(v[0]), q4_odd(v[1]), q4_odd(v[2]), q4_odd(v[3])), pb[e], O[j + 1], 0, 0, 0);
#pragma unroll
                for (int i = 0; i < 4; i++) v[i] >>= 8;
            }
        }
        cur = nxt;
    }

    // ---- the wave's outputs: dimension 16 j + 4 g + i of column n
    l += swz_xor16_f(l);
    l += __shfl_xor(l, 32, JM_WAVE);
#pragma unroll
    for (int j = 0; j < 8; j++) {
        float o[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float v = O[j][i] * (j & 1 ? 0.0625f : 1.0f);
            o[i] = BF ? v : __builtin_fmaf(dpp_f<DPP_ROR8>(v), 1.0f / Q4_LO, v);
        }
        if (n < 8) *(float4*)&ow[w][n][16 * j + 4 * g] = make_float4(o[0], o[1], o[2], o[3]);
    }
    if (g == 0 && n < 8) {
        mls[w][n][0] = ref;
        mls[w][n][1] = l;
    }
    __syncthreads();

    // ---- the block's: thread = column tid / 32, dimensions 4 (tid % 32) ..
    const int oc = threadIdx.x >> 5, od = 4 * (threadIdx.x & 31);
    if (oc >= ncol) return;
    const float M = fmaxf(fmaxf(mls[0][oc][0], mls[1][oc][0]), fmaxf(mls[2][oc][0], mls[3][oc][0]));
    float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    float L = 0.0f;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        if (mls[i][oc][0] == -INFINITY) continue;
        const float f = pow2f(mls[i][oc][0] - M);
        const float4 x = *(const float4*)&ow[i][oc][od];
        v.x = __builtin_fmaf(x.x, f, v.x);
        v.y = __builtin_fmaf(x.y, f, v.y);
        v.z = __builtin_fmaf(x.z, f, v.z);
        v.w = __builtin_fmaf(x.w, f, v.w);
        L = __builtin_fmaf(mls[i][oc][1], f, L);
    }
    if (a.S == 1) {
        if (un.pos + oc / a.qpk >= c.maxT) return;
        const float inv = M == -INFINITY ? 0.0f : __fdiv_rn(1.0f, L);       // no row to see: 0
        const size_t oi = ((size_t)(un.tok + oc / a.qpk) * a.H + kh * a.qpk + oc % a.qpk) * HD + od;
        store_out<BF>(a.out, oi, make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv));
        return;
    }
    const size_t pi = (((size_t)u * c.KH + kh) * a.S + s) * (a.qpk * a.tp) + oc;
    if (M != -INFINITY) *(float4*)(a.part_o + pi * HD + od) = v;
    if ((threadIdx.x & 31) == 0) {
        a.part_ml[2 * pi] = M;
        a.part_ml[2 * pi + 1] = L;
    }
}

// The ranges of one (KV head, unit) merged into the output.
template <bool BF>
__global__ void __launch_bounds__(256)
k_q4_merge(Q4KvArgs c, Q4AttnArgs a) {
    constexpr int HD = 128;
    const int kh = blockIdx.x % c.KH, u = blockIdx.x / c.KH;
    Q4Unit un;
    if (!q4_unit(c, u, a.tp, un)) return;
    const int oc = threadIdx.x >> 5, od = 4 * (threadIdx.x & 31), nc = a.qpk * a.tp;
    if (oc >= a.qpk * un.n || un.pos + oc / a.qpk >= c.maxT) return;
    const size_t p0 = ((size_t)u * c.KH + kh) * a.S * nc + oc;
    float M = -INFINITY;
    for (int s = 0; s < a.S; s++) M = fmaxf(M, a.part_ml[2 * (p0 + (size_t)s * nc)]);
    float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    float L = 0.0f;
    for (int s = 0; s < a.S; s++) {
        const size_t pi = p0 + (size_t)s * nc;
        const float m = a.part_ml[2 * pi];
        if (m == -INFINITY) continue;
        const float f = pow2f(m - M);
        const float4 x = *(const float4*)(a.part_o + pi * HD + od);
        v.x = __builtin_fmaf(x.x, f, v.x);
        v.y = __builtin_fmaf(x.y, f, v.y);
        v.z = __builtin_fmaf(x.z, f, v.z);
        v.w = __builtin_fmaf(x.w, f, v.w);
        L = __builtin_fmaf(a.part_ml[2 * pi + 1], f, L);
    }
    const float inv = M == -INFINITY ? 0.0f : __fdiv_rn(1.0f, L);
    const size_t oi = ((size_t)(un.tok + oc / a.qpk) * a.H + kh * a.qpk + oc % a.qpk) * HD + od;
    store_out<BF>(a.out, oi, make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv));
}

#define JM_Q4_CASE(NGV, BFV, KERNEL, GRID, BLK, ...)                                              \
    if (c.group == 128 / NGV && bf == BFV)                                                        \
        hipLaunchKernelGGL((KERNEL<NGV, BFV>), GRID, BLK, 0, st, __VA_ARGS__)
#define JM_Q4_EACH(KERNEL, GRID, BLK, ...)                                                        \
    JM_Q4_CASE(2, false, KERNEL, GRID, BLK, __VA_ARGS__); else JM_Q4_CASE(2, true, KERNEL, GRID, BLK, __VA_ARGS__); \
    else JM_Q4_CASE(4, false, KERNEL, GRID, BLK, __VA_ARGS__); else JM_Q4_CASE(4, true, KERNEL, GRID, BLK, __VA_ARGS__); \
    else return hipErrorInvalidValue

hipError_t launch_q4_write(const Q4KvArgs& c, const void* k, const void* v, bool bf, const long long (&st4)[4],
                           hipStream_t st) {
    if (c.N == 0) return hipSuccess;
    const dim3 grid((unsigned)(((long long)c.N * c.KH + 3) / 4));
    JM_Q4_EACH(k_q4_write, grid, dim3(256), c, k, v, st4[0], st4[1], st4[2], st4[3]);
    return hipGetLastError();
}

hipError_t launch_q4_read(const Q4KvArgs& c, void* k, void* v, bool bf, hipStream_t st) {
    if (c.N == 0) return hipSuccess;
    const dim3 grid((unsigned)(((long long)c.N * c.KH + 3) / 4));
    JM_Q4_EACH(k_q4_read, grid, dim3(256), c, k, v);
    return hipGetLastError();
}

// How the attention of a call is cut: tokens a unit, units, ranges of rows.
Q4AttnPlan q4_attn_plan(const Q4KvArgs& c, int H) {
    Q4AttnPlan p;
    const int qpk = H / c.KH;
    p.tp = c.cu ? 8 / qpk : 1;
    // (every sequence's tokens are rounded up to whole units)
    p.units = (int)std::min<long long>(c.N, (long long)c.N / p.tp + c.n_seq);
    const long long blocks = (long long)p.units * c.KH;
    // enough blocks for 4 a CU, at least 128 rows (a tile a wave) each
    p.S = (int)std::max<long long>(1, std::min<long long>((1024 + blocks - 1) / blocks, (c.maxT + 127) / 128));
    const size_t cols = (size_t)blocks * p.S * qpk * p.tp;
    p.o_floats = p.S > 1 ? cols * 128 : 0;
    p.ml_floats = p.S > 1 ? cols * 2 : 0;
    return p;
}

hipError_t launch_q4_attn(const Q4KvArgs& c, const Q4AttnPlan& p, const void* q, bool bf, long long qts, long long qhs,
                          int H, float scale, void* out, float* part_o, float* part_ml, hipStream_t st) {
    if (c.N == 0) return hipSuccess;
    Q4AttnArgs a{};
    a.q = q; a.qts = qts; a.qhs = qhs; a.H = H; a.qpk = H / c.KH; a.tp = p.tp;
    a.scale2 = scale * 1.4426950408889634f;
    a.out = out; a.units = p.units; a.S = p.S; a.part_o = part_o; a.part_ml = part_ml;
    const dim3 grid((unsigned)c.KH * p.units * p.S);
    JM_Q4_EACH(k_q4_attn, grid, dim3(256), c, a);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || p.S == 1) return e;
    const dim3 mg((unsigned)c.KH * p.units);
    if (bf) hipLaunchKernelGGL(k_q4_merge<true>, mg, dim3(256), 0, st, c, a);
    else hipLaunchKernelGGL(k_q4_merge<false>, mg, dim3(256), 0, st, c, a);
    return hipGetLastError();
}

}  // namespace jm
