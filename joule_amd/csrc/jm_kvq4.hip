// The 4-bit KV cache's operators: rows quantised as they are written, read
// back, and attended over (jm_q4kv.h has the layout).
#include <algorithm>

#include "jm_q4kv.h"

namespace jm {

// Rows in and out: one wave per (KV head, 4 consecutive tokens), 16 lanes a row,
// 8 dimensions a lane, so that a row moves in 16-byte pieces (the v codes change
// hands between 8 lanes in registers).  Bound by memory where there is much: 112016
// tokens of 8 heads read back as bf16 in 40 us, 5.7 TB/s of codes and values.  What
// is read back is stored past the caches, which it would only go through: with
// ordinary stores, into outputs that were not there before, 65 us.  3 prompts of up
// to 1531 bf16 tokens written in 6.7 us; 8 tokens of 4 heads in 3.4 (the launch).
template <int NG, bool BF>
__global__ void __launch_bounds__(256)
k_q4_write(Q4KvArgs c, const void* __restrict__ k, const void* __restrict__ v, long long kts, long long khs,
           long long vts, long long vhs) {
    const int item = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int t0 = 4 * (item / c.KH), kh = item % c.KH, t = t0 + ((threadIdx.x & 63) >> 4);
    int seq, r;
    if (t0 >= c.N || !call_places(c, t0, seq, r)) return;
    float x[8], y[8];
    load8<BF>(k, (size_t)(t * kts + kh * khs) + 8 * q4_chunk(), x);
    load8<BF>(v, (size_t)(t * vts + kh * vhs) + 8 * q4_chunk(), y);
    q4_store_chunk<NG>(x, true, r, Q4Head<NG>(q4_plane(c, seq, 0), kh, c.KH, c.R));
    q4_store_chunk<NG>(y, false, r, Q4Head<NG>(q4_plane(c, seq, 1), kh, c.KH, c.R));
}

// (the exact values, bf16 rounded)
template <int NG, bool BF>
__global__ void __launch_bounds__(256)
k_q4_read(Q4KvArgs c, void* __restrict__ k, void* __restrict__ v) {
    const int item = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int t0 = 4 * (item / c.KH), kh = item % c.KH, t = t0 + ((threadIdx.x & 63) >> 4);
    int seq, r;
    if (t0 >= c.N || !call_places(c, t0, seq, r)) return;
    float x[8], y[8];
    q4_load_chunk<NG>(x, true, r, Q4Head<NG>(q4_plane(c, seq, 0), kh, c.KH, c.R));
    q4_load_chunk<NG>(y, false, r, Q4Head<NG>(q4_plane(c, seq, 1), kh, c.KH, c.R));
    const size_t at = ((size_t)t * c.KH + kh) * 128 + 8 * q4_chunk();
    store8<BF>(k, at, x);
    store8<BF>(v, at, y);
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
//            in columns n < 8, q brought to [2^10, 2^11) by a power of two and
//            rounded to fp16, the rest of it in columns n + 8; one product a
//            32 dimensions, one scale a group.  Lane (g, n) gets column n of rows
//            4 g + i: with the two halves added (one DPP move), the scores of
//            query row n % 8 at 8 rows of the tile.
//   weights  exp2(score - ref), ref common to a column's lanes and chosen so that
//            weight x V scale stays below 2^15: raised only when a lane meets a
//            product above 2^14, to where the largest is 2^6, so that most tiles
//            need no exchange between lanes.  Each row's weight counts with its own
//            scale: a large V without weight must not raise ref, under which the
//            other products would fall out of fp16's range (5 % of the output for a
//            V 10^8 times the others').  Each lane sums its own weights.
//   P . V    16 dimensions a product (dimension 16 j + m is row m of product j,
//            nibble j of the lane's V dwords) as A, weight x scale in fp16, the
//            rest in columns n + 8, as B, from the lanes that formed
//            them: contraction index 8 g + e is row 16 (e / 4) + 4 g + e % 4.
// q and the weights carry 21 bits so; for bf16 queries (BF) q is exact without
// the second half, and the weights are rounded to fp16 once (2^-11 of each, a
// fraction of the output's own rounding; with both halves the 32 long sequences
// below take 108 us instead of 98).
//
// Measured, kernels alone, caches as long as their rows: 1 token behind 777 rows of 4
// KV heads 9.8 us, in one range; with k_q4_merge, 8 tokens behind 2048 rows each 7.7 +
// 2.9 (a tile a wave takes 6.4 us: the launch, the unit's place, q and the tile, the
// waves joined; each further tile 0.6); 6 drafts of 5 tokens behind 3001 rows of 16
// heads (26 MB) 15.4 + 3.1, on 576 blocks of 4 tiles a wave; 32 bf16 tokens behind
// 16003 rows each of 8 heads (441 MB, groups of 32) 93.4 + 4.8 us, 4.7 TB/s: memory.

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef unsigned short u16x2_t __attribute__((ext_vector_type(2)));

__device__ __forceinline__ f16x8 as_f16x8(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    return __builtin_bit_cast(f16x8, make_uint4(a, b, c, d));
}

// The codes less 8 of nibbles 0 and 4 of w, and 16 times those of nibbles 1 and 5.
// The constants come from registers (one of them a vector register), so that
// each mask and exponent is one v_and_or_b32.
struct Q4Bits {
    uint32_t even = 0x000F000Fu, odd = 0x00F000F0u, one = 0x64006400u;
    __device__ __forceinline__ Q4Bits() { __asm__("" : "+s"(even), "+s"(odd), "+v"(one)); }
    __device__ __forceinline__ uint32_t lo(uint32_t w) const {
        const f16x2 h = __builtin_bit_cast(f16x2, (w & even) | one) - f16x2{(_Float16)1032.0f, (_Float16)1032.0f};
        return __builtin_bit_cast(uint32_t, h);
    }
    __device__ __forceinline__ uint32_t hi(uint32_t w) const {
        const f16x2 h = __builtin_bit_cast(f16x2, (w & odd) | one) - f16x2{(_Float16)1152.0f, (_Float16)1152.0f};
        return __builtin_bit_cast(uint32_t, h);
    }
};

__device__ __forceinline__ float pow2f(float x) { return __builtin_amdgcn_exp2f(x); }

// y + log2(the largest of some V scales, given as fp16 bits) + 15, the logarithm read
// off the bits (at most 0.09 below it, and at least -15; an infinity's and a NaN's
// are above every finite one's).
__device__ __forceinline__ float q4_weight_exp(float y, u16x2_t m) { return __builtin_fmaf((float)max(m.x, m.y), 0x1p-10f, y); }

// ... of a row's scales, two a word
template <int NG>
__device__ __forceinline__ float q4_weight_exp(float y, const uint32_t* w) {
    u16x2_t m = __builtin_bit_cast(u16x2_t, w[0]);
#pragma unroll
    for (int e = 1; e < NG / 2; e++) m = __builtin_elementwise_max(m, __builtin_bit_cast(u16x2_t, w[e]));
    return q4_weight_exp(y, m);
}

struct Q4AttnArgs {
    const void* q;              // strides qts, qhs
    long long qts, qhs;
    int H, qpk, lq, tp;         // qpk = 2^lq; tp tokens a unit
    float scale2;               // score scale times log2(e)
    void* out;                  // [N][H][128]
    int units, S;
    float* part_o;              // [units][KH][S][qpk tp][128]: not divided by the sum
    float* part_ml;             // [units][KH][S][qpk tp][2]: ref, sum
};

// Constants from registers, unknown to the compiler: a fused multiply-add with
// an fp16 factor is one v_fma_mix_f32, where it would make a product or a
// difference of it (exactly as good) two instructions.
struct Q4Mix {
    float zero = 0.0f, minus1 = -1.0f;
    __device__ __forceinline__ Q4Mix() { __asm__("" : "+s"(zero), "+s"(minus1)); }
    __device__ __forceinline__ float mul(float a, _Float16 b) const { return __builtin_fmaf(a, (float)b, zero); }
    __device__ __forceinline__ float sub(float a, _Float16 b) const { return __builtin_fmaf((float)b, minus1, a); }
};

// The two fp16 halves of a and b: the values rounded towards 0, and the rest.
__device__ __forceinline__ void split_f16x2(const Q4Mix& mix, float a, float b, uint32_t& hi, uint32_t& lo) {
    const auto h = __builtin_amdgcn_cvt_pkrtz(a, b);
    const float ra = mix.sub(a, (_Float16)h[0]);
    const float rb = mix.sub(b, (_Float16)h[1]);
    hi = __builtin_bit_cast(uint32_t, h);
    lo = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(ra, rb));
}

// Whether a running maximum and sum are those of no row at all (a NaN among the
// scores leaves the maximum, but not the sum).
__device__ __forceinline__ bool q4_dead(float ref, float sum) { return ref == -INFINITY && sum == 0.0f; }

// One tile of 32 cache rows as a lane gets it: 16 bytes of K codes of rows
// 16 t + l % 16, of V codes of the row blocks 4 t + l / 16, and the scales of
// rows 16 t + 4 (l / 16) .. + 3.
template <int NG>
struct Q4Tile {
    u32x4_t k[2], v[2];
    u32x4_t ks[NG], vs[NG];     // (NG / 2 words of 16 bytes a row group t)
};

// Where a lane's share of a tile lies, and of the tiles after it.
template <int NG>
struct Q4TileAt {
    gptr<const u32x4_t> k, v, ks, vs;
    __device__ __forceinline__ Q4TileAt(const Q4Head<NG>& kk, const Q4Head<NG>& vv, int tile, int lane) {
        const int g = lane >> 4, n = lane & 15;
        const size_t r = (size_t)32 * tile;
        k = (gptr<const u32x4_t>)(kk.codes + (r + n) * 16 + 4 * g);
        v = (gptr<const u32x4_t>)(vv.codes + r * 16 + 64 * g + 4 * n);
        ks = (gptr<const u32x4_t>)(kk.scales + (r + 4 * g) * NG);
        vs = (gptr<const u32x4_t>)(vv.scales + (r + 4 * g) * NG);
    }
    __device__ __forceinline__ void skip(int tiles) {
        k += tiles * 128;       // (16 bytes of a row's 64, 32 rows a tile)
        v += tiles * 128;
        ks += tiles * 4 * NG;
        vs += tiles * 4 * NG;
        // (from registers: left to the compiler, the additions come ahead of the loads)
        __asm__("" : "+v"(k), "+v"(v), "+v"(ks), "+v"(vs));
    }
    __device__ __forceinline__ void load(Q4Tile<NG>& x) const {
#pragma unroll
        for (int t = 0; t < 2; t++) {
            // (past the caches: 32 sequences of 16384 rows 4% faster, and no slower
            // where units share rows)
            x.k[t] = __builtin_nontemporal_load(k + 64 * t);
            x.v[t] = __builtin_nontemporal_load(v + 64 * t);
#pragma unroll
            for (int i = 0; i < NG / 2; i++) {
                x.ks[t * (NG / 2) + i] = ks[2 * NG * t + i];
                x.vs[t * (NG / 2) + i] = vs[2 * NG * t + i];
            }
        }
    }
};

// scale of row i (0..3) of row group t, group e
template <int NG>
__device__ __forceinline__ float q4_scale(const u32x4_t (&s)[NG], int t, int i, int e) {
    const int h = i * NG + e;                               // fp16 index within the row group
    const uint32_t w = s[t * (NG / 2) + h / 8][(h % 8) / 2];
    return (float)__builtin_bit_cast(f16x2, w)[h % 2];
}

// The 8 query rows of one unit over tiles t0 .. t_end - 1, a wave taking every W-th;
// all W waves joined, and the output, or (several ranges) the partial outputs of
// unit u and range s from their row row0 on.  ow and mls: LDS for the W waves.
template <int NG, bool BF, int W>
__device__ __forceinline__ void q4_attn_unit(const Q4KvArgs& c, const Q4AttnArgs& a, const CallUnit& un, int kh, int t0,
                                             int t_end, int u, int s, int row0, float (*ow)[8][128], float (*mls)[8][2]) {
    constexpr int HD = 128, GS = 4 / NG;                    // contraction steps a group
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int g = lane >> 4, n = lane & 15, col = n & 7;
    const int ncol = a.qpk * un.n;
    int t = t0 + w;
    const int ct = min(col >> a.lq, un.n - 1), head = kh * a.qpk + (col & (a.qpk - 1));
    const int crow = min(un.pos + ct, c.maxT - 1);          // the last row that this column sees

    const Q4Head<NG> kk(q4_plane(c, un.seq, 0), kh, c.KH, c.R), vv(q4_plane(c, un.seq, 1), kh, c.KH, c.R);
    const Q4Mix mix;
    Q4Tile<NG> cur, nxt;
    Q4TileAt<NG> at(kk, vv, t, lane);
    if (t < t_end) at.load(cur);
    at.skip(W);

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
        // q times a power of two, its largest value in [2^10, 2^11)
        const uint32_t ex = min(max(__float_as_uint(top) >> 23, 12u), 252u);
        const float f = __uint_as_float((264u - ex) << 23);
        lf = __fmul_rn(__uint_as_float((ex - 10u) << 23), a.scale2);
#pragma unroll
        for (int st = 0; st < 4; st++) {
            uint32_t b[4];
#pragma unroll
            for (int e = 0; e < 4; e++) {
                uint32_t hi, lo;
                split_f16x2(mix, __fmul_rn(x[st][e], f), __fmul_rn(x[st][e + 4], f), hi, lo);
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
    const Q4Bits bits;

    for (; t < t_end; t += W) {
        if (t + W < t_end) at.load(nxt);
        at.skip(W);
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
                        as_f16x8(bits.lo(d), bits.hi(d), bits.lo(d8), bits.hi(d8)), qb[st], acc, 0, 0, 0);
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
        uint32_t sv[8][NG / 2];                             // V's scales, two a word
#pragma unroll
        for (int i = 0; i < 8; i++)
#pragma unroll
            for (int e = 0; e < NG / 2; e++) {
                const int at = (i & 3) * (NG / 2) + e;
                sv[i][e] = cur.vs[(i >> 2) * (NG / 2) + at / 4][at % 4];
            }
        if (32 * t + 31 > un.pos) {                         // some column does not see the whole tile
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const bool in = 32 * t + 16 * (i >> 2) + 4 * g + (i & 3) <= crow;
                y[i] = in ? y[i] : -INFINITY;
#pragma unroll
                for (int e = 0; e < NG / 2; e++) sv[i][e] = in ? sv[i][e] : 0u;
            }
        }
        // ---- the reference: the largest weight x scale, to the exponent; row by row
        // only where the largest weight times the largest scale passes it
        float ym = y[0];
        u16x2_t sm = 0;
#pragma unroll
        for (int i = 1; i < 8; i++) ym = fmaxf(ym, y[i]);
#pragma unroll
        for (int i = 0; i < 8; i++)
#pragma unroll
            for (int e = 0; e < NG / 2; e++) sm = __builtin_elementwise_max(sm, __builtin_bit_cast(u16x2_t, sv[i][e]));
        const float pass = ref + 29.0f;                     // (q4_weight_exp's 15 among it)
        if (__any(q4_weight_exp(ym, sm) > pass)) {
            float z = -INFINITY;
#pragma unroll
            for (int i = 0; i < 8; i++) z = fmaxf(z, q4_weight_exp<NG>(y[i], sv[i]));
            if (__any(z > pass)) {
                z = fmaxf(z, swz_xor16_f(z));
                z = fmaxf(z, __shfl_xor(z, 32, JM_WAVE));
                const float nref = fmaxf(ref, z - 21.0f);
                const float f = ref == -INFINITY ? 0.0f : pow2f(ref - nref);
                l *= f;
#pragma unroll
                for (int j = 0; j < 8; j++) O[j] *= f;
                ref = nref;
            }
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
                const float x0 = mix.mul(p[2 * i], __builtin_bit_cast(f16x2, sv[2 * i][e / 2])[e % 2]);
                const float x1 = mix.mul(p[2 * i + 1], __builtin_bit_cast(f16x2, sv[2 * i + 1][e / 2])[e % 2]);
                if (BF) {
                    b[i] = __builtin_bit_cast(uint32_t, f16x2{(_Float16)x0, (_Float16)x1});
                } else {
                    uint32_t hi, lo;
                    split_f16x2(mix, x0, x1, hi, lo);
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
                    as_f16x8(bits.lo(v[0]), bits.lo(v[1]), bits.lo(v[2]), bits.lo(v[3])), pb[e], O[j], 0, 0, 0);
                O[j + 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
                    as_f16x8(bits.hi(v[0]), bits.hi(v[1]), bits.hi(v[2]), bits.hi(v[3])), pb[e], O[j + 1], 0, 0, 0);
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
            o[i] = BF ? v : __fadd_rn(v, dpp_f<DPP_ROR8>(v));
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
    float M = mls[0][oc][0];
#pragma unroll
    for (int i = 1; i < W; i++) M = fmaxf(M, mls[i][oc][0]);
    float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    float L = 0.0f;
#pragma unroll
    for (int i = 0; i < W; i++) {
        if (q4_dead(mls[i][oc][0], mls[i][oc][1])) continue;
        const float f = pow2f(mls[i][oc][0] - M);
        const float4 x = *(const float4*)&ow[i][oc][od];
        v.x = __builtin_fmaf(x.x, f, v.x);
        v.y = __builtin_fmaf(x.y, f, v.y);
        v.z = __builtin_fmaf(x.z, f, v.z);
        v.w = __builtin_fmaf(x.w, f, v.w);
        L = __builtin_fmaf(mls[i][oc][1], f, L);
    }
    if (a.S == 1) {
        if (un.pos + (oc >> a.lq) >= c.maxT) return;
        // a row below 0 sees none: 0.  (A sum of 0 elsewhere is that of scores that are
        // all -infinity, as an infinite query makes them: NaN.)
        const float inv = un.pos + (oc >> a.lq) < 0 ? 0.0f : __fdiv_rn(1.0f, L);
        const size_t oi = ((size_t)(un.tok + (oc >> a.lq)) * a.H + kh * a.qpk + (oc & (a.qpk - 1))) * HD + od;
        store_out<BF>(a.out, oi, make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv));
        return;
    }
    const size_t pi = (((size_t)u * c.KH + kh) * a.S + s) * (a.qpk * a.tp) + row0 + oc;
    if (!q4_dead(M, L)) *(float4*)(a.part_o + pi * HD + od) = v;
    if ((threadIdx.x & 31) == 0) {
        a.part_ml[2 * pi] = M;
        a.part_ml[2 * pi + 1] = L;
    }
}

template <int NG, bool BF>
__global__ void __launch_bounds__(256, 2)
k_q4_attn(Q4KvArgs c, Q4AttnArgs a) {
    __shared__ __align__(16) float ow[4][8][128];
    __shared__ float mls[4][8][2];
    const int kh = blockIdx.x % c.KH, u = blockIdx.x / c.KH % a.units, s = blockIdx.x / c.KH / a.units;
    CallUnit un;
    if (!call_unit(c, u, a.tp, un)) return;                 // (block-uniform)
    const int last = min(un.pos + un.n - 1, c.maxT - 1);    // the last row any token sees
    const int NT = (last + 32) / 32;                        // (0 where last < 0)
    q4_attn_unit<NG, BF, 4>(c, a, un, kh, (int)((long long)NT * s / a.S), (int)((long long)NT * (s + 1) / a.S), u, s, 0, ow, mls);
}

// The ranges of one (KV head, unit) merged into the output, 8 query rows a block.
template <bool BF>
__global__ void __launch_bounds__(256)
k_q4_merge(Q4KvArgs c, Q4AttnArgs a) {
    constexpr int HD = 128;
    const int nc = a.qpk * a.tp, nb = (nc + 7) / 8;
    const int kh = blockIdx.x % c.KH, u = blockIdx.x / c.KH / nb;
    CallUnit un;
    if (c.pos) {
        un.tok = u * a.tp;
        un.n = min(a.tp, c.N - un.tok);
    } else if (!call_unit(c, u, a.tp, un)) {
        return;
    }
    const int oc = 8 * (blockIdx.x / c.KH % nb) + (threadIdx.x >> 5), od = 4 * (threadIdx.x & 31);
    if (oc >= a.qpk * un.n) return;
    const int pos = c.pos ? c.pos[un.tok + (oc >> a.lq)] : un.pos + (oc >> a.lq);
    if (pos >= c.maxT) return;
    const size_t p0 = ((size_t)u * c.KH + kh) * a.S * nc + oc;
    // lane j of the 32 has the factors of ranges j, j + 32, ..; the ranges' outputs
    // are on their way four at a time
    const int j = threadIdx.x & 31, half = threadIdx.x & 32;
    float M = -INFINITY;
    for (int s = j; s < a.S; s += 32) M = fmaxf(M, a.part_ml[2 * (p0 + (size_t)s * nc)]);
    M = seg_max<32>(M);
    float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    float L = 0.0f;
    for (int s0 = 0; s0 < a.S; s0 += 32) {
        float f = -1.0f;                // (a range without a row: it has no output; and past the end)
        if (s0 + j < a.S) {
            const float2 x = *(const float2*)(a.part_ml + 2 * (p0 + (size_t)(s0 + j) * nc));
            if (!q4_dead(x.x, x.y)) {
                f = pow2f(x.x - M);
                L = __builtin_fmaf(x.y, f, L);
            }
        }
        for (int e = s0; e < min(s0 + 32, a.S); e += 4) {
            float4 x[4];
#pragma unroll
            for (int q = 0; q < 4; q++)
                x[q] = *(const float4*)(a.part_o + (p0 + (size_t)min(e + q, a.S - 1) * nc) * HD + od);
#pragma unroll
            for (int q = 0; q < 4; q++) {
                const float y = __shfl(f, half + e - s0 + q, JM_WAVE);
                if (y < 0.0f) continue;         // (0 counts: it may meet a NaN)
                v.x = __builtin_fmaf(x[q].x, y, v.x);
                v.y = __builtin_fmaf(x[q].y, y, v.y);
                v.z = __builtin_fmaf(x[q].z, y, v.z);
                v.w = __builtin_fmaf(x[q].w, y, v.w);
            }
        }
    }
    L = seg_sum<32>(L);
    const float inv = pos < 0 ? 0.0f : __fdiv_rn(1.0f, L);                  // (as in k_q4_attn)
    const size_t oi = ((size_t)(un.tok + (oc >> a.lq)) * a.H + kh * a.qpk + (oc & (a.qpk - 1))) * HD + od;
    store_out<BF>(a.out, oi, make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv));
}

// ------------------------------------------------------- many query tokens
//
// The same for prompts: block (KV head, unit of RG x 32 QB query rows), 8 waves =
// RG row groups x PS position strides; in a step wave (rg, ps) takes the 32 cache
// rows ps of the step's 32 PS for its 32 QB query rows, with an online softmax,
// and the PS waves of a row group merge once at the end.  The step's codes are
// turned into fp16 once for all of them, in LDS, while the step before is
// multiplied (two buffers, one barrier a step; the codes of the step after are on
// their way).
//
//   scores   v_mfma_f32_32x32x16_f16, cache rows as A (lane l: row l % 32, the 8
//            dimensions of the row's code dword 4 c + s with s = kk / 2, c = 2 (kk % 2)
//            + l / 32), query rows as B: lane l holds query row l % 32 at cache
//            rows 8 (v / 4) + 4 (l / 32) + v % 4
//   P . V    V^T as A (lane l: dimension 32 nt + l % 32) from the rows' blocks of 4
//            as the plane has them, the weights as B from the lanes that formed
//            them: contraction index j of half h in step s is row 16 s + 8 (j / 4) +
//            4 h + j % 4
//
// Two forms.  float32 queries: the codes less 8 are exact in LDS, q and the
// weights are two fp16 halves each, every group's scores are scaled on their own
// and the V scale goes into the weights, as in k_q4_attn.  bf16 queries (BF): K and
// V are scaled in LDS and rounded to fp16 (2^-11 of the value, or 2^-15 of the
// largest scale of 16 rows), relative to the 16 rows' largest scale, whose exponent
// goes into the scores and the weights; q is exact, the weights are fp16 once (their
// sum is of the float32 ones: where 16 rows of V are far below the others, fp16 no
// longer holds weights that count).  That is one product where the other form takes
// two, no arithmetic on scales between them, and 64 query rows a wave (QB = 2), which
// halves the LDS reads a product.
//
// Rows of which one is below 2^-8 of the largest of its 16 do not bear that: a later
// token's row would take the bits of an earlier token's.  A block that finds such
// among the scales of its range does the range as k_q4_attn does.  Looking takes some
// 1.3 us (509 tokens 25.7 -> 27.0 us, 2047 behind 4099 rows 224 -> 227); looking while
// staging, or branching behind the loop, spilled the loop's registers.  Where there
// are such rows these take 90 and 1070 us.
//
// Measured at 2047 tokens behind 4099 rows, 32 query heads on 8 (172 GFLOP, 147 us
// at the rate of a large library product): 222 us a call in a run of them, 245 alone
// under a profiler, whose clock is lower.  Vector work bounds it: 49.2 million vector
// instructions beside 5.3 million products, 296 a wave and step beside 32, and the
// two waves of a SIMD, half a step apart, hide most but not all of it (225 us with
// both in step; for the 509 float32 tokens, of which a block has 4 steps at most,
// 20.7 in step and 21.0 apart).

typedef float f32x16 __attribute__((ext_vector_type(16)));

// Byte offsets in a step's LDS: chunk p (16 bytes, one code dword) of cache row r
// of K; chunk (s, h) of dimension d of V^T of 32-row tile t.  Spread over the
// banks for the reads of 16 lanes.
__device__ __forceinline__ int q4t_k(int r, int p) { return r * 256 + 16 * (p ^ (r & 15)); }
__device__ __forceinline__ int q4t_v(int t, int d, int sh) { return t * 8192 + d * 64 + 16 * (sh ^ ((d >> 2) & 3)); }

// 2^e as fp16, twice, for e in [-15, 15]
__device__ __forceinline__ f16x2 q4t_pow2(int e) {
    const _Float16 f = (_Float16)__uint_as_float((uint32_t)(127 + e) << 23);
    return f16x2{f, f};
}

// Two codes times their scales, (q - 8) s 2^-10, in one fused multiply-add: the
// codes' bits are the subnormals q 2^-24 (or 16 times that), and -8 s 2^-10 is
// exact.  s is at most 2 (one scale of each half's row).
struct Q4Scaled {
    f16x2 even, odd, off;
    __device__ __forceinline__ void set(f16x2 s) {
        even = s * (_Float16)16384.0f;
        odd = s * (_Float16)1024.0f;
        off = s * (_Float16)-0.0078125f;
    }
    __device__ __forceinline__ uint32_t lo(uint32_t w) const {
        return __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(__builtin_bit_cast(f16x2, w & 0x000F000Fu), even, off));
    }
    __device__ __forceinline__ uint32_t hi(uint32_t w) const {
        return __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(__builtin_bit_cast(f16x2, w & 0x00F000F0u), odd, off));
    }
};

// the largest over the wave, the same in every lane (DPP: within rows of 16, then
// the row ends onto the rows behind)
template <int CTRL>
__device__ __forceinline__ uint32_t dpp_max_u(uint32_t v) {
    return max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xF, 0xF, false));
}
__device__ __forceinline__ uint32_t wave_max_u(uint32_t v) {
    v = dpp_max_u<0x111>(v);                // row_shr 1, 2, 4, 8
    v = dpp_max_u<0x112>(v);
    v = dpp_max_u<0x114>(v);
    v = dpp_max_u<0x118>(v);
    v = dpp_max_u<0x142>(v);                // row_bcast 15 and 31
    v = dpp_max_u<0x143>(v);
    return (uint32_t)__builtin_amdgcn_readlane((int)v, 63);
}

// Whether of rows r0 .. r1 - 1 (r0 a multiple of 16) one's largest scale is below 2^-8
// of the largest of its 16 (rows of zeros, exact at any exponent, and scales that
// are not finite do not count): this thread's share of the 512 threads'.
template <int NG>
__device__ __forceinline__ bool q4_rows_apart(const Q4Head<NG>& k, const Q4Head<NG>& v, int r0, int r1) {
    constexpr int RPL = 8 / NG;                 // rows a lane: 16 bytes of scales
    bool far = false;
    auto look = [&](u32x4_t x, int r) __attribute__((always_inline)) {
        uint32_t m[RPL], top = 0, least = 0xFFFFFFFFu;
#pragma unroll
        for (int i = 0; i < RPL; i++) {
            u16x2_t h = 0;
#pragma unroll
            for (int e = 0; e < NG / 2; e++) {
                uint32_t y = x[i * (NG / 2) + e] & 0x7FFF7FFFu;
                if ((y & 0x7C00u) == 0x7C00u) y &= 0xFFFF0000u;
                if ((y & 0x7C000000u) == 0x7C000000u) y &= 0xFFFFu;
                h = __builtin_elementwise_max(h, __builtin_bit_cast(u16x2_t, y));
            }
            m[i] = r + i < r1 ? max(h.x, h.y) : 0u;
            top = max(top, m[i]);
            least = min(least, m[i] - 1u);      // (0 last of all)
        }
        top = max(top, (uint32_t)dpp_i<DPP_XOR1>((int)top));
        top = max(top, (uint32_t)dpp_i<DPP_XOR2>((int)top));
        if (NG == 4) top = max(top, (uint32_t)dpp_i<DPP_HALF_MIRROR>((int)top));
        const _Float16 lim = __builtin_bit_cast(_Float16, (uint16_t)top) * (_Float16)0x1p-8f;
        far |= least < max((uint32_t)__builtin_bit_cast(uint16_t, lim), 1u) - 1u;
    };
    for (int r = r0 + RPL * (int)threadIdx.x; r - RPL * (int)threadIdx.x < r1; r += RPL * 512) {
        const int at = min(r, (r1 - 1) / RPL * RPL);            // (inside the plane; rows past the end count as 0)
        const u32x4_t x = *(gptr<const u32x4_t>)(k.scales + (size_t)at * NG);
        const u32x4_t y = *(gptr<const u32x4_t>)(v.scales + (size_t)at * NG);
        look(x, r);
        look(y, r);
    }
    return far;
}

// A block's range of k_q4_tile<BF> from the codes, 8 query rows at a time.
template <int NG, int STEP>
__device__ __forceinline__ void q4_tile_again(const Q4KvArgs& c, const Q4AttnArgs& a, float (*ow)[8][128], float (*mls)[8][2]) {
    uint32_t bx = blockIdx.x;
    __asm__ volatile("" : "+s"(bx));
    const int kh = bx % c.KH, rs = bx / c.KH, u = a.units - 1 - rs % a.units, sr = rs / a.units;
    CallUnit un;
    if (!call_unit(c, u, a.tp, un)) return;
    const int steps = (min(un.pos + un.n - 1, c.maxT - 1) + STEP) / STEP;
    const int t0 = (int)((long long)steps * sr / a.S) * (STEP / 32), t1 = (int)((long long)steps * (sr + 1) / a.S) * (STEP / 32);
    const int tp = 8 >> a.lq;
#pragma unroll 1
    for (int t = 0; t < un.n; t += tp) {
        const CallUnit x = {un.seq, un.tok + t, min(tp, un.n - t), un.pos + t};
        const int NT = (min(x.pos + x.n - 1, c.maxT - 1) + 32) / 32;
        q4_attn_unit<NG, true, 8>(c, a, x, kh, t0, min(t1, NT), u, sr, t << a.lq, ow, mls);
        __syncthreads();
    }
}

template <int NG, bool BF, int RG>
__global__ void __launch_bounds__(512, 2)
k_q4_tile(Q4KvArgs c, Q4AttnArgs a) {
    constexpr int HD = 128, QB = BF ? 2 : 1, PS = 8 / RG, STEP = 32 * PS, ROWS = 32 * QB * RG;
    constexpr int NI = STEP / 64;               // 16-byte code chunks a thread and step
    constexpr int PB = STEP * 512;              // bytes of a step's K and V
    __shared__ __align__(16) unsigned char kv[2][PB];
    __shared__ __align__(16) uint16_t sc[BF ? 1 : 2][2][BF ? 8 : STEP * NG];     // the step's scales (float32 queries)
    __shared__ float mls[8][32 * QB][2];
    // the second block of query rows of each row group (BF): with it in
    // registers too, the compiler spills
    __shared__ __align__(16) uint4 q1[BF ? RG : 1][8][64];
    __shared__ int eb[2][STEP / 16][2];         // (BF) exponents of the 16-row blocks' scales, K and V
    __shared__ uint32_t tn[8][32 * QB];
    __shared__ uint32_t apart[8];
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int rg = w % RG, ps = w / RG, n = lane & 31, h = lane >> 5;
    const int kh = blockIdx.x % c.KH, rs = blockIdx.x / c.KH;
    const int u = a.units - 1 - rs % a.units, sr = rs / a.units;        // the longest prefixes first
    CallUnit un;
    if (c.pos) {                                // the decoder's form: one prompt's tokens
        un.seq = 0;
        un.tok = u * a.tp;
        un.n = min(a.tp, c.N - un.tok);
        un.pos = 0;
    } else if (!call_unit(c, u, a.tp, un)) {
        return;
    }
    // this lane's query rows, and the last cache row that each sees
    int tok[QB], prow[QB], head[QB];
    bool live[QB];
    int pmax = -1, pmin = c.maxT;
#pragma unroll
    for (int b = 0; b < QB; b++) {
        const int r = 32 * (QB * rg + b) + n, t = r >> a.lq;
        live[b] = t < un.n;
        tok[b] = un.tok + min(t, un.n - 1);
        head[b] = kh * a.qpk + (r & (a.qpk - 1));
        prow[b] = c.pos ? c.pos[tok[b]] : un.pos + (tok[b] - un.tok);
        live[b] = live[b] && prow[b] < c.maxT;
        prow[b] = min(prow[b], c.maxT - 1);
    }
    for (int t = lane; t < un.n; t += 64) {     // (over the unit's tokens, the same in every wave)
        const int p = min(c.pos ? c.pos[un.tok + t] : un.pos + t, c.maxT - 1);
        pmax = max(pmax, p);
        pmin = min(pmin, p);
    }
#pragma unroll
    for (int o = 32; o; o >>= 1) {
        pmax = max(pmax, __shfl_xor(pmax, o, JM_WAVE));
        pmin = min(pmin, __shfl_xor(pmin, o, JM_WAVE));
    }
    pmax = __builtin_amdgcn_readfirstlane(pmax);
    pmin = __builtin_amdgcn_readfirstlane(pmin);
    // this block's range of the steps (none where no token sees a row)
    const int steps = (pmax + STEP) / STEP;
    const int step0 = (int)((long long)steps * sr / a.S), nstep = (int)((long long)steps * (sr + 1) / a.S);
    const Q4Head<NG> kk(q4_plane(c, un.seq, 0), kh, c.KH, c.R), vv(q4_plane(c, un.seq, 1), kh, c.KH, c.R);

    // ---- a step's codes and scales on their way, and into LDS
    struct Stage {
        u32x4_t code[NI];
        u32x4_t scl[NI][NG / 2];                // V: 4 rows' scales; K: the row's in the first words
    } sg;
    // (rows of a step by halves of 64, which lie in the plane as wholes: past the
    // end the last one again, whose rows are masked)
    auto half_row = [&](int i, int half) __attribute__((always_inline)) { return min(i * STEP + 64 * half, c.R - 64); };
    auto request = [&](int i) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < NI; j++) {
            // (wave-uniform: which of K and V, and which half)
            const int w8 = w + 8 * j;
            if (w8 < STEP / 16) {
                const int r0 = half_row(i, w8 / 4), r = 16 * (w8 % 4) + (lane >> 2);
                sg.code[j] = *(gptr<const u32x4_t>)(kk.codes + (size_t)r0 * 16 + (uint32_t)(16 * r + 4 * (lane & 3)));
                const gptr<const uint32_t> s = (gptr<const uint32_t>)(kk.scales + (size_t)r0 * NG) + (uint32_t)(r * NG / 2);
#pragma unroll
                for (int e = 0; e < NG / 2; e++) sg.scl[j][0][e] = s[e];
            } else {
                const int wv = w8 - STEP / 16, r0 = half_row(i, wv / 4), r = 16 * (wv % 4) + 4 * (lane >> 4);
                sg.code[j] = *(gptr<const u32x4_t>)(vv.codes + (size_t)r0 * 16 + (uint32_t)(16 * r + 4 * (lane & 15)));
#pragma unroll
                for (int e = 0; e < NG / 2; e++)
                    sg.scl[j][e] = ((gptr<const u32x4_t>)(vv.scales + (size_t)r0 * NG + (uint32_t)(r * NG)))[e];
            }
        }
    };
    // BF: the 16 rows of K or V that a wave stages are scaled by a power of two of
    // their own, which goes to the step's multipliers through eb: 2^e just above
    // their largest scale, and whether one of their scales is not finite (such
    // scales are 0 in LDS; `taint` has which of this lane's query rows saw one)
    uint32_t taint[QB] = {};
    const Q4Bits bits;
    const Q4Mix mix;
    auto stage = [&](int i) __attribute__((always_inline)) {
        const int buf = i & 1;
#pragma unroll
        for (int j = 0; j < NI; j++) {
            const int w8 = w + 8 * j;                           // (wave-uniform)
            const bool isk = w8 < STEP / 16;
            const int rb = isk ? w8 : w8 - STEP / 16;           // the 16-row block
            int ln = lane;
            __asm__ volatile("" : "+v"(ln));                    // (the addresses anew each step)
            f16x2 fe;
            if constexpr (BF) {
                constexpr int NW = 2 * NG;                      // V: words of scales, NG / 2 a row; K: the first NG / 2
                if (i * STEP + 16 * rb + 15 > pmax) {           // rows that nobody sees
                    const int row = i * STEP + 16 * rb + (isk ? ln >> 2 : 4 * (ln >> 4));
#pragma unroll
                    for (int e = 0; e < NW; e++)
                        if (row + (isk ? 0 : 2 * e / NG) > pmax) sg.scl[j][e / 4][e % 4] = 0;
                }
                auto largest = [&]() __attribute__((always_inline)) {
                    u16x2_t m = 0;
                    if (isk) {
#pragma unroll
                        for (int e = 0; e < NG / 2; e++)
                            m = __builtin_elementwise_max(m, __builtin_bit_cast(u16x2_t, sg.scl[j][0][e] & 0x7FFF7FFFu));
                    } else {
#pragma unroll
                        for (int e = 0; e < NW; e++)
                            m = __builtin_elementwise_max(m, __builtin_bit_cast(u16x2_t, sg.scl[j][e / 4][e % 4] & 0x7FFF7FFFu));
                    }
                    return wave_max_u(max(m.x, m.y));
                };
                uint32_t m = largest();
                const bool bad = m >= 0x7C00u;
                if (bad) {
#pragma unroll
                    for (int e = 0; e < NW; e++) {
                        uint32_t x = sg.scl[j][e / 4][e % 4];
                        if ((x & 0x7C00u) == 0x7C00u) x &= 0xFFFF0000u;
                        if ((x & 0x7C000000u) == 0x7C000000u) x &= 0xFFFFu;
                        sg.scl[j][e / 4][e % 4] = x;
                    }
                    m = largest();
                }
                const int e = (int)(m >> 10) - 15;
                fe = q4t_pow2(-e);
                if (lane == 0) eb[buf][rb][isk ? 0 : 1] = e + (bad ? 64 : 0);
            }
            if (isk) {
                const int r = 16 * rb + (ln >> 2), cc = ln & 3;
                Q4Scaled s2[NG];
                if constexpr (BF) {
#pragma unroll
                    for (int e = 0; e < NG; e++) {
                        const uint32_t x = sg.scl[j][0][e / 2];
                        s2[e].set(__builtin_bit_cast(f16x2, __builtin_amdgcn_perm(x, x, e & 1 ? 0x03020302u : 0x01000100u)) * fe);
                    }
                } else if (cc == 0) {
#pragma unroll
                    for (int e = 0; e < NG / 2; e++) *(uint32_t*)&sc[buf][0][r * NG + 2 * e] = sg.scl[j][0][e];
                }
                const int at = q4t_k(r, 4 * cc);
#pragma unroll
                for (int s = 0; s < 4; s++) {
                    const uint32_t d = sg.code[j][s], d8 = d >> 8;
                    uint32_t o[4];
                    if constexpr (BF) {
                        const Q4Scaled& x = s2[s * NG / 4];
                        o[0] = x.lo(d); o[1] = x.hi(d); o[2] = x.lo(d8); o[3] = x.hi(d8);
                    } else {
                        o[0] = bits.lo(d); o[1] = bits.hi(d); o[2] = bits.lo(d8); o[3] = bits.hi(d8);
                    }
                    *(uint4*)(kv[buf] + (at ^ (16 * s))) = make_uint4(o[0], o[1], o[2], o[3]);
                }
            } else {
                const int blk = 4 * rb + (ln >> 4), nn = ln & 15;
                // rows (0, 1) and (2, 3) of the block
                uint32_t lo[2], hi[2];
                Q4Scaled s2[2][NG];
#pragma unroll
                for (int q = 0; q < 2; q++) {
                    const uint32_t d0 = sg.code[j][2 * q], d1 = sg.code[j][2 * q + 1];
                    lo[q] = __builtin_amdgcn_perm(d1, d0, 0x05040100u);
                    hi[q] = __builtin_amdgcn_perm(d1, d0, 0x07060302u);
                    if constexpr (BF) {
#pragma unroll
                        for (int e = 0; e < NG; e++) {
                            const int a0 = (2 * q) * NG + e, a1 = a0 + NG;          // fp16 indices of the two rows
                            const uint32_t x0 = sg.scl[j][a0 / 8][(a0 % 8) / 2], x1 = sg.scl[j][a1 / 8][(a1 % 8) / 2];
                            s2[q][e].set(__builtin_bit_cast(f16x2, __builtin_amdgcn_perm(x1, x0, e & 1 ? 0x07060302u : 0x05040100u)) * fe);
                        }
                    }
                }
                if constexpr (!BF) {
                    if (nn == 0) {
#pragma unroll
                        for (int e = 0; e < NG / 2; e++) *(u32x4_t*)&sc[buf][1][4 * blk * NG + 8 * e] = sg.scl[j][e];
                    }
                }
                // block b of the tile's 8: chunk (s, h) = (b / 4, b % 2), its half (b / 2) % 2
                const int t = blk >> 3, b8 = blk & 7, sh = 2 * (b8 >> 2) + (b8 & 1), half = 8 * ((b8 >> 1) & 1);
                unsigned char* const at = kv[buf] + STEP * 256 + q4t_v(t, nn, sh) + half;
#pragma unroll
                for (int jn = 0; jn < 8; jn++) {
                    uint32_t o[2];
#pragma unroll
                    for (int q = 0; q < 2; q++) {
                        const uint32_t d = (jn < 4 ? lo[q] : hi[q]) >> (jn & 2 ? 8 : 0);
                        if constexpr (BF) o[q] = jn & 1 ? s2[q][jn * NG / 8].hi(d) : s2[q][jn * NG / 8].lo(d);
                        else o[q] = jn & 1 ? bits.hi(d) : bits.lo(d);
                    }
                    *(uint2*)(at + 1024 * jn) = make_uint2(o[0], o[1]);
                }
            }
        }
    };

    if (step0 < nstep) request(step0);
    if constexpr (BF) {
        const bool far = q4_rows_apart<NG>(kk, vv, step0 * STEP, min(nstep * STEP, pmax + 1));
        const bool any = __any(far);
        if (lane == 0) apart[w] = any;
        __syncthreads();
        uint32_t f = 0;
#pragma unroll
        for (int i = 0; i < 8; i++) f |= apart[i];
        if (__builtin_amdgcn_readfirstlane(f)) {
            q4_tile_again<NG, STEP>(c, a, (float (*)[8][HD])&kv[0][0], (float (*)[8][2])&mls[0][0][0]);
            return;
        }
    }

    // ---- the query rows
    f16x8 qh[8], ql[BF ? 1 : 8];
    float cs[QB];
#pragma unroll
    for (int b = 0; b < QB; b++) {
        const size_t qi = (size_t)(tok[b] * a.qts + head[b] * a.qhs);
        float x[8][8], top = 0.0f;
#pragma unroll
        for (int k = 0; k < 8; k++) {
            const int d = 32 * (k / 2) + 8 * (2 * (k % 2) + h);
            float y[4];
            load4<BF>(a.q, qi + d, y);
#pragma unroll
            for (int e = 0; e < 4; e++) x[k][e] = y[e];
            load4<BF>(a.q, qi + d + 4, y);
#pragma unroll
            for (int e = 0; e < 4; e++) x[k][4 + e] = y[e];
#pragma unroll
            for (int e = 0; e < 8; e++) top = fmaxf(top, fabsf(x[k][e]));
        }
        top = fmaxf(top, __shfl_xor(top, 32, JM_WAVE));
        // its largest value in [2^10, 2^11), with the score scale's sign
        const uint32_t ex = min(max(__float_as_uint(top) >> 23, 12u), 252u);
        const float f = __builtin_copysignf(__uint_as_float((264u - ex) << 23), a.scale2);
        // (a scale of 0, or one that underflows with q, as 2^-100: scores below 2^-48, as
        // they are, and masked ones still -inf behind it)
        cs[b] = __fmul_rn(__uint_as_float((ex - 10u) << 23), fabsf(a.scale2));
        if (BF) cs[b] = fmaxf(cs[b], 0x1p-100f);
#pragma unroll
        for (int k = 0; k < 8; k++) {
            uint32_t hi[4], lo[4];
#pragma unroll
            for (int e = 0; e < 4; e++) {
                split_f16x2(mix, __fmul_rn(x[k][e], f), __fmul_rn(x[k][e + 4], f), hi[e], lo[e]);
                if (!BF && (e & 1)) {           // codes 16 times too large
                    hi[e] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2, hi[e]) * (_Float16)0.0625f);
                    lo[e] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2, lo[e]) * (_Float16)0.0625f);
                }
            }
            if (b == 0) qh[k] = as_f16x8(hi[0], hi[1], hi[2], hi[3]);
            else if (ps == 0) q1[rg][k][lane] = make_uint4(hi[0], hi[1], hi[2], hi[3]);
            if (!BF) ql[k] = as_f16x8(lo[0], lo[1], lo[2], lo[3]);
        }
    }

    f32x16 O[QB][4];
    float ref[QB], l[QB];
#pragma unroll
    for (int b = 0; b < QB; b++) {
        ref[b] = -INFINITY;
        l[b] = 0.0f;
#pragma unroll
        for (int nt = 0; nt < 4; nt++)
#pragma unroll
            for (int v = 0; v < 16; v++) O[b][nt][v] = 0.0f;
    }
    // raise a column's reference so that z (the largest exponent met) is at most
    // 2^14 above it
    auto raise = [&](int b, float z) __attribute__((always_inline)) {
        if (__any(z > ref[b] + 14.0f)) {
            z = fmaxf(z, __shfl_xor(z, 32, JM_WAVE));
            const float nref = fmaxf(ref[b], z - 6.0f);
            const float f = ref[b] == -INFINITY ? 0.0f : pow2f(ref[b] - nref);
            l[b] *= f;
#pragma unroll
            for (int nt = 0; nt < 4; nt++)
#pragma unroll
                for (int v = 0; v < 16; v++) O[b][nt][v] *= f;
            ref[b] = nref;
        }
    };

    auto compute = [&](int i) __attribute__((always_inline)) {
        const int buf = i & 1;
        const int t0 = i * STEP + 32 * ps;
        if (t0 > pmax) return;
        // the operands' addresses from one each, an XOR at a time: kept in
        // registers over the steps, the compiler spills others for them
        int ka = buf * PB + ps * 8192 + q4t_k(n, 4 * h), va = buf * PB + STEP * 256 + q4t_v(ps, n, h);
        __asm__ volatile("" : "+v"(ka), "+v"(va));
        auto kop = [&](int k) __attribute__((always_inline)) {
            return *(const f16x8*)(&kv[0][0] + (ka ^ (16 * (8 * (k % 2) + k / 2))));
        };
        auto vop = [&](int nt, int s) __attribute__((always_inline)) {
            return *(const f16x8*)(&kv[0][0] + 2048 * nt + (va ^ (32 * s)));
        };
        if constexpr (BF) {
            // the exponents of the tile's two 16-row blocks (2^10 of the codes in LDS
            // goes into the scores here, and that of V into the end)
            int ek[2], ev[2];
#pragma unroll
            for (int q = 0; q < 2; q++) {
                ek[q] = __builtin_amdgcn_readfirstlane(eb[buf][2 * ps + q][0]);
                ev[q] = __builtin_amdgcn_readfirstlane(eb[buf][2 * ps + q][1]);
            }
            if (max(max(ek[0], ek[1]), max(ev[0], ev[1])) > 31) {
                // row by row: which of this lane's query rows see what is not finite
#pragma unroll 1
                for (int row = t0; row < t0 + 32 && row <= pmax; row++) {
                    uint32_t bits = 0;
#pragma unroll
                    for (int e = 0; e < NG; e++) {
                        if ((*kk.scale(row, e) & 0x7FFFu) >= 0x7C00u) bits = (1u << NG) - 1;
                        if ((*vv.scale(row, e) & 0x7FFFu) >= 0x7C00u) bits |= 1u << e;
                    }
#pragma unroll
                    for (int b = 0; b < QB; b++) taint[b] |= row <= prow[b] ? bits : 0u;
                }
#pragma unroll
                for (int q = 0; q < 2; q++) {
                    if (ek[q] > 31) ek[q] -= 64;
                    if (ev[q] > 31) ev[q] -= 64;
                }
            }
            f32x16 S[QB] = {f32x16(0.0f), f32x16(0.0f)};
#pragma unroll
            for (int k = 0; k < 8; k++) {
                const f16x8 xk = kop(k);
                S[0] = __builtin_amdgcn_mfma_f32_32x32x16_f16(xk, qh[k], S[0], 0, 0, 0);
                S[1] = __builtin_amdgcn_mfma_f32_32x32x16_f16(xk, *(const f16x8*)&q1[rg][k][lane], S[1], 0, 0, 0);
            }
            f16x8 P[QB][2];
#pragma unroll
            for (int b = 0; b < QB; b++) {
                if (t0 + 31 > pmin) {
                    const int lim = prow[b] - t0 - 4 * h;
#pragma unroll
                    for (int v = 0; v < 16; v++)
                        if (8 * (v / 4) + v % 4 > lim) S[b][v] = -INFINITY;
                }
                // lane registers 0..7 are rows of the first block, 8..15 of the second
                float cf[2], z[2];
#pragma unroll
                for (int q = 0; q < 2; q++) {
                    float m = S[b][8 * q];
#pragma unroll
                    for (int v = 1; v < 8; v++) m = fmaxf(m, S[b][8 * q + v]);
                    cf[q] = __fmul_rn(cs[b], __uint_as_float((uint32_t)(137 + ek[q]) << 23));
                    z[q] = __builtin_fmaf(m, cf[q], (float)ev[q]);
                }
                raise(b, fmaxf(z[0], z[1]));
#pragma unroll
                for (int s = 0; s < 2; s++) {
                    const float add = ref[b] == -INFINITY ? 0.0f : (float)ev[s] - ref[b];
                    float t = 0.0f;
                    uint32_t p[4];
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const float x0 = pow2f(__builtin_fmaf(S[b][8 * s + 2 * e], cf[s], add));
                        const float x1 = pow2f(__builtin_fmaf(S[b][8 * s + 2 * e + 1], cf[s], add));
                        t = __fadd_rn(t, __fadd_rn(x0, x1));
                        const f16x2 x2 = {(_Float16)x0, (_Float16)x1};
                        p[e] = __builtin_bit_cast(uint32_t, x2);
                    }
                    P[b][s] = as_f16x8(p[0], p[1], p[2], p[3]);
                    l[b] = __builtin_fmaf(t, __uint_as_float((uint32_t)(127 - ev[s]) << 23), l[b]);
                }
            }
#pragma unroll
            for (int k = 0; k < 8; k++) {
                const int s = k / 4, nt = k % 4;
                const f16x8 xv = vop(nt, s);
#pragma unroll
                for (int b = 0; b < QB; b++) O[b][nt] = __builtin_amdgcn_mfma_f32_32x32x16_f16(xv, P[b][s], O[b][nt], 0, 0, 0);
            }
        } else {
            // the scales of the lane's cache rows 8 q + 4 h + e, two a word
            const uint16_t* const s0 = &sc[buf][0][(32 * ps + 4 * h) * NG];
            auto load_scales = [&](int which, uint32_t (&x)[4][2 * NG]) __attribute__((always_inline)) {
#pragma unroll
                for (int q = 0; q < 4; q++)
#pragma unroll
                    for (int e = 0; e < NG / 2; e++) {
                        const uint4 y = *(const uint4*)(s0 + which * STEP * NG + 8 * q * NG + 8 * e);
                        x[q][4 * e] = y.x; x[q][4 * e + 1] = y.y; x[q][4 * e + 2] = y.z; x[q][4 * e + 3] = y.w;
                    }
            };
            auto scale = [&](const uint32_t (&x)[4][2 * NG], int v, int g) __attribute__((always_inline)) {
                const int at = (v % 4) * NG + g;
                return (float)__builtin_bit_cast(f16x2, x[v / 4][at / 2])[at % 2];
            };
            uint32_t sx[4][2 * NG];
            load_scales(0, sx);
            float y[16];
#pragma unroll
            for (int v = 0; v < 16; v++) y[v] = 0.0f;
#pragma unroll
            for (int g = 0; g < NG; g++) {
                f32x16 acc;
#pragma unroll
                for (int v = 0; v < 16; v++) acc[v] = 0.0f;
#pragma unroll
                for (int k = g * (8 / NG); k < (g + 1) * (8 / NG); k++) {
                    const f16x8 x = kop(k);
                    acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(x, ql[k], acc, 0, 0, 0);
                    acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(x, qh[k], acc, 0, 0, 0);
                }
#pragma unroll
                for (int v = 0; v < 16; v++) y[v] = __builtin_fmaf(scale(sx, v, g), acc[v], y[v]);
            }
            load_scales(1, sx);
#pragma unroll
            for (int v = 0; v < 16; v++) y[v] = __fmul_rn(y[v], cs[0]);
            if (t0 + 31 > pmin) {
                const int lim = prow[0] - t0 - 4 * h;
#pragma unroll
                for (int v = 0; v < 16; v++) {
                    const bool in = 8 * (v / 4) + v % 4 <= lim;
                    y[v] = in ? y[v] : -INFINITY;
#pragma unroll
                    for (int e = 0; e < NG / 2; e++) sx[v / 4][(v % 4) * NG / 2 + e] = in ? sx[v / 4][(v % 4) * NG / 2 + e] : 0u;
                }
            }
            float m = y[0];
            u16x2_t sm = 0;
#pragma unroll
            for (int v = 1; v < 16; v++) m = fmaxf(m, y[v]);
#pragma unroll
            for (int q = 0; q < 4; q++)
#pragma unroll
                for (int e = 0; e < 2 * NG; e++) sm = __builtin_elementwise_max(sm, __builtin_bit_cast(u16x2_t, sx[q][e]));
            if (__any(q4_weight_exp(m, sm) > ref[0] + 29.0f)) {     // (as in q4_attn_unit)
                float z = -INFINITY;
#pragma unroll
                for (int v = 0; v < 16; v++) z = fmaxf(z, q4_weight_exp<NG>(y[v], &sx[v / 4][(v % 4) * NG / 2]));
                raise(0, z - 15.0f);
            }
            const float r0 = ref[0] == -INFINITY ? 0.0f : ref[0];
#pragma unroll
            for (int v = 0; v < 16; v++) {
                y[v] = pow2f(__fsub_rn(y[v], r0));
                l[0] = __fadd_rn(l[0], y[v]);
            }
#pragma unroll
            for (int g = 0; g < NG; g++)
#pragma unroll
                for (int s = 0; s < 2; s++) {
                    uint32_t hi[4], lo[4];
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const int v = 8 * s + 2 * e;
                        split_f16x2(mix, __fmul_rn(y[v], scale(sx, v, g)), __fmul_rn(y[v + 1], scale(sx, v + 1, g)), hi[e], lo[e]);
                    }
                    const f16x8 ph = as_f16x8(hi[0], hi[1], hi[2], hi[3]), pl = as_f16x8(lo[0], lo[1], lo[2], lo[3]);
#pragma unroll
                    for (int nt = g * (4 / NG); nt < (g + 1) * (4 / NG); nt++) {
                        const f16x8 x = vop(nt, s);
                        O[0][nt] = __builtin_amdgcn_mfma_f32_32x32x16_f16(x, pl, O[0][nt], 0, 0, 0);
                        O[0][nt] = __builtin_amdgcn_mfma_f32_32x32x16_f16(x, ph, O[0][nt], 0, 0, 0);
                    }
                }
        }
    };

    // Step k is staged before the barrier that all waves pass before they multiply
    // it.  Of the two waves of a SIMD (w and w + 4) one stages step k + 1 before it
    // multiplies step k, the other after, so that the one's vector work falls to
    // the other's products; in its code the second meets the barrier between
    // staging k and multiplying it.
    const bool ahead = w < 4;
    auto meet = [&]() __attribute__((always_inline)) {
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup");
        __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup");
    };
    if (ahead) {
        if (step0 < nstep) stage(step0);
        if (step0 + 1 < nstep) request(step0 + 1);
        meet();
    }
#pragma unroll 1
    for (int k = step0; k < nstep; k++) {
        const int sk = ahead ? k + 1 : k;
        if (sk < nstep) {
            stage(sk);
            if (sk + 1 < nstep) request(sk + 1);
        }
        if (!ahead) meet();
        compute(k);
        if (ahead) meet();
    }
    if (!ahead) meet();

    // ---- the PS waves of each row group merged, 32 dimensions at a time
    float f[QB], inv[QB];
#pragma unroll
    for (int b = 0; b < QB; b++) {
        l[b] = __fadd_rn(l[b], __shfl_xor(l[b], 32, JM_WAVE));
        if (h == 0) {
            mls[w][32 * b + n][0] = ref[b];
            mls[w][32 * b + n][1] = l[b];
            if (BF) tn[w][32 * b + n] = taint[b];
        }
    }
    __syncthreads();
#pragma unroll
    for (int b = 0; b < QB; b++) {
        float M = -INFINITY, L = 0.0f;
#pragma unroll
        for (int q = 0; q < PS; q++) M = fmaxf(M, mls[q * RG + rg][32 * b + n][0]);
        const float m0 = M == -INFINITY ? 0.0f : M;
#pragma unroll
        for (int q = 0; q < PS; q++)
            L = __builtin_fmaf(mls[q * RG + rg][32 * b + n][1], pow2f(mls[q * RG + rg][32 * b + n][0] - m0), L);
        f[b] = pow2f(ref[b] - m0);
        inv[b] = prow[b] < 0 ? 0.0f : __fdiv_rn(1.0f, L);              // (as in k_q4_attn)
        if (a.S > 1) {
            inv[b] = 1.0f;
            float* const ml = a.part_ml + 2 * (((size_t)(u * c.KH + kh) * a.S + sr) * (a.qpk * a.tp) + 32 * (QB * rg + b) + n);
            if (ps == 0 && h == 0 && live[b]) *(float2*)ml = make_float2(M, L);
        }
        if constexpr (BF) {
#pragma unroll
            for (int q = 0; q < PS; q++) taint[b] |= tn[q * RG + rg][32 * b + n];
        }
    }
    float4* const mb = (float4*)&kv[0][0];                                 // [wave][QB][4][64 lanes]
    static_assert(8 * QB * 4 * 64 * 16 <= 2 * PB && 8 * 8 * HD * 4 <= 2 * PB, "the outputs of 32 dimensions, and of 8 rows, fit");
#pragma unroll
    for (int nt = 0; nt < 4; nt++) {
        if (nt) __syncthreads();
#pragma unroll
        for (int b = 0; b < QB; b++)
#pragma unroll
            for (int q = 0; q < 4; q++) {
                // BF: 2^10 of V's codes; float32: the odd nibbles' dimensions (the
                // upper 16 of 32) are 16 times too large
                const float s = BF ? f[b] * 1024.0f : q >= 2 ? f[b] * 0.0625f : f[b];
                mb[((w * QB + b) * 4 + q) * 64 + lane] = make_float4(O[b][nt][4 * q] * s, O[b][nt][4 * q + 1] * s,
                                                                     O[b][nt][4 * q + 2] * s, O[b][nt][4 * q + 3] * s);
            }
        __syncthreads();
#pragma unroll
        for (int b = 0; b < QB; b++)
#pragma unroll
            for (int q = 0; q < 4; q++) {
                if ((b * 4 + q) % PS != ps || !live[b]) continue;
                float4 s = mb[((rg * QB + b) * 4 + q) * 64 + lane];
#pragma unroll
                for (int p = 1; p < PS; p++) {
                    const float4 x = mb[(((p * RG + rg) * QB + b) * 4 + q) * 64 + lane];
                    s = make_float4(s.x + x.x, s.y + x.y, s.z + x.z, s.w + x.w);
                }
                s = make_float4(s.x * inv[b], s.y * inv[b], s.z * inv[b], s.w * inv[b]);
                if (BF && (taint[b] >> ((32 * nt) / (HD / NG)) & 1)) {
                    const float x = __uint_as_float(0x7FC00000u);
                    s = make_float4(x, x, x, x);
                }
                const int d = 32 * nt + 8 * q + 4 * h;
                if (a.S == 1) {
                    store_out<BF>(a.out, ((size_t)tok[b] * a.H + head[b]) * HD + d, s);
                } else {
                    const size_t row = ((size_t)(u * c.KH + kh) * a.S + sr) * (a.qpk * a.tp) + 32 * (QB * rg + b) + n;
                    *(float4*)(a.part_o + row * HD + d) = s;
                }
            }
    }
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
    const dim3 grid((unsigned)((((long long)c.N + 3) / 4 * c.KH + 3) / 4));
    JM_Q4_EACH(k_q4_write, grid, dim3(256), c, k, v, st4[0], st4[1], st4[2], st4[3]);
    return hipGetLastError();
}

hipError_t launch_q4_read(const Q4KvArgs& c, void* k, void* v, bool bf, hipStream_t st) {
    if (c.N == 0) return hipSuccess;
    const dim3 grid((unsigned)((((long long)c.N + 3) / 4 * c.KH + 3) / 4));
    JM_Q4_EACH(k_q4_read, grid, dim3(256), c, k, v);
    return hipGetLastError();
}

// How the attention of a call is cut: tokens a unit, units, ranges of rows;
// whether it takes k_q4_tile, and with how many row groups.
Q4AttnPlan q4_attn_plan(const Q4KvArgs& c, int H, bool bf, bool shared) {
    Q4AttnPlan p{};
    const int qpk = H / c.KH;
    const int n_seq = c.cu ? c.n_seq : shared ? 1 : c.N;
    auto cut = [&](int tp) {
        p.tp = tp;
        // (every sequence's tokens are rounded up to whole units)
        p.units = (int)std::min<long long>(c.N, ((long long)c.N + (long long)n_seq * (tp - 1)) / tp);
        return (long long)p.units * c.KH;
    };
    long long blocks;
    // up to `want` blocks while each has `rows` cache rows
    auto ranges = [&](long long want, int rows) {
        return std::min((want + blocks - 1) / blocks, ((long long)c.maxT + rows - 1) / rows);
    };
    // Tiles from 64 query rows a sequence (bf16: 96).  Both ways, us, float32 and
    // bf16, 8 query heads a KV head: 8 tokens behind 30000 rows (8 KV heads) tiles
    // 42 and 46, else 54 and 47; 16 tokens 57 and 48, else 93 and 80; 8 tokens behind
    // 2000 (4 sequences, 4 heads) 20 and 22, else 17 and 15; 16 tokens 27 and 24, else 25
    // and 22; 64 tokens behind 4000 (8 heads) 36 and 30, else 56 and 48.
    const long long rows = (long long)c.N * qpk;
    if (rows >= (bf ? 96ll : 64ll) * n_seq) {
        // 4 row groups share what a step stages, but take twice the rows for a block:
        // where the blocks are enough, or the prefixes may be long enough to be cut.
        // (us, with 2 and with 4, bf16, 8 KV heads: 64 tokens behind 4000 rows 30 and
        // 33, 256 tokens 69 and 64; behind 30000 rows 107 and 94, 358 and 296)
        const int unit = bf ? 256 : 128;
        p.rg = 4;
        blocks = cut(unit / qpk);
        if (rows < (long long)unit * n_seq || (blocks < 256 && blocks * c.maxT < 160000)) {
            p.rg = 2;
            blocks = cut(unit / 2 / qpk);
        }
        // (a block fills a CU; 256 tokens behind 30000 rows, bf16: 682 us uncut with 2.
        // By the rows that a cache has room for, here too: 509 float32 tokens in a cache
        // of 509 rows 21 us, of 4096 or 32768 28)
        p.S = (int)std::max(std::min(256 / blocks, ((long long)c.maxT + 255) / 256), 1ll);
    } else {
        blocks = cut(c.cu ? 8 / qpk : 1);
        // Ranges, for caches of more than 1024 rows (those it has room for: how many are
        // in use is in device memory.  1 token behind 777 rows 9.6 us in a cache of
        // 1024, 11.7 in one of 4096, 14.7 of 32768, 34 of 131072; 8 behind 2048 rows 11.4
        // in caches of 2049 and 4096, 15.8 of 32768): a block a CU while each has 128
        // rows (a tile a wave), up to 4 a CU while each has 512.  Up to there one
        // range is faster than a second launch and its workspace: 1 or 8 tokens behind
        // 777 float32 rows (4 KV heads) 10.0 us against 12.6, 23 in a captured graph,
        // where the workspace is a node; 1000 rows 10.9 and 12.8, 1500 rows 14.2 and
        // 12.6.  (Above, both kernels alone: 8 sequences of 2048 rows 11.6 us on 256
        // blocks, 14.6 on 1024; 6 sequences' drafts over up to 5000 rows 22.0 us on 256
        // blocks, 19.4 on 1024; bfloat16, 32 sequences of 16384: 115 us without a
        // split, 104 with 1024 blocks.)
        p.S = c.maxT <= 1024 ? 1 : (int)std::max(std::max(ranges(256, 128), ranges(1024, 512)), 1ll);
    }
    const size_t cols = (size_t)blocks * p.S * qpk * p.tp;
    p.o_floats = p.S > 1 ? cols * 128 : 0;
    p.ml_floats = p.S > 1 ? cols * 2 : 0;
    return p;
}

hipError_t launch_q4_attn(const Q4KvArgs& c, const Q4AttnPlan& p, const void* q, bool bf, long long qts, long long qhs,
                          int H, float scale, void* out, float* part_o, float* part_ml, hipStream_t st) {
    if (c.N == 0) return hipSuccess;
    Q4AttnArgs a{};
    a.q = q; a.qts = qts; a.qhs = qhs; a.H = H; a.qpk = H / c.KH; a.lq = __builtin_ctz((unsigned)a.qpk); a.tp = p.tp;
    a.scale2 = scale * 1.4426950408889634f;
    a.out = out; a.units = p.units; a.S = p.S; a.part_o = part_o; a.part_ml = part_ml;
    const dim3 grid((unsigned)c.KH * p.units * p.S);
    if (p.rg) {
#define JM_Q4_TILE(NGV, BFV) \
        if (c.group == 128 / NGV && bf == BFV) { \
            if (p.rg == 4) hipLaunchKernelGGL((k_q4_tile<NGV, BFV, 4>), grid, dim3(512), 0, st, c, a); \
            else hipLaunchKernelGGL((k_q4_tile<NGV, BFV, 2>), grid, dim3(512), 0, st, c, a); \
        }
        JM_Q4_TILE(2, false) JM_Q4_TILE(2, true) JM_Q4_TILE(4, false) JM_Q4_TILE(4, true)
#undef JM_Q4_TILE
    } else {
        JM_Q4_EACH(k_q4_attn, grid, dim3(256), c, a);
    }
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || p.S == 1) return e;
    const dim3 mg((unsigned)c.KH * p.units * ((a.qpk * a.tp + 7) / 8));
    if (bf) hipLaunchKernelGGL(k_q4_merge<true>, mg, dim3(256), 0, st, c, a);
    else hipLaunchKernelGGL(k_q4_merge<false>, mg, dim3(256), 0, st, c, a);
    return hipGetLastError();
}

}  // namespace jm
