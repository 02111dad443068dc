// Paged KV caches: new rows finished (norm, rotation) and written to their
// sequences' pages, and attention over the pages.
//
// The rows of a (page, KV head) are contiguous, [page][128]; pages hold at least 16
// rows, so 16 aligned rows always lie in one page.
#include <algorithm>
#include <climits>
#include <type_traits>

#include "jm_kernels.h"
#include "jm_tokens.h"

namespace jm {

// ---------------------------------------------------------------- new rows

// 16 lanes a head, 8 dimensions a lane (dimension d and its partner d + 64 lie 8 lanes
// apart); a block takes 16 NH heads of one token, NH a group of lanes: q heads, then k heads,
// then v heads.
//
// Bound by what it reads and writes, if the rotation's factors (1 KB of float32 a token, of
// which a head wants all) are not loaded anew for each head of 256 bytes, and if the heads are
// on their way before the token's place is known: 13374 bf16 tokens of 48 heads 65 us, 5 TB/s
// (NH = 3); NH = 1 76 (and 93 with the place first), NH = 2 78, NH = 4 66.  Few tokens wait
// for each load in turn: 8 of 40 heads 2.9 us (NH = 1) / 3.9 (NH = 3), 1805 of 48 8.1 / 7.8.
template <bool BF, int NH>
__global__ void __launch_bounds__(256)
k_paged_append(PagedArgs c, PagedRows r, int chunks) {
    constexpr int HD = 128;
    const int t = blockIdx.x / chunks, h0 = blockIdx.x % chunks * 16 * NH + (threadIdx.x >> 4), heads = r.H + 2 * c.KH;
    const int j = threadIdx.x & 15;
    float x[NH][8];
    int what[NH], head[NH];
#pragma unroll
    for (int i = 0; i < NH; i++) {
        const int hr = h0 + 16 * i;
        what[i] = hr < r.H ? 0 : hr < r.H + c.KH ? 1 : hr < heads ? 2 : 3;
        head[i] = what[i] == 0 ? hr : what[i] == 1 ? hr - r.H : hr - r.H - c.KH;
        const int w = what[i];
        if (w < 3) load8<BF>(w == 0 ? r.x[0] : w == 1 ? r.x[1] : r.x[2],
                             (size_t)(t * (w == 0 ? r.ts[0] : w == 1 ? r.ts[1] : r.ts[2]) + head[i] * (w == 0 ? r.hs[0] : w == 1 ? r.hs[1] : r.hs[2])) + 8 * j, x[i]);
    }
    int seq, pos;
    if (!call_place(c, t, seq, pos)) return;                // (block-uniform)
    const int page = c.table[seq * c.table_stride + (pos >> c.lp)];
    float cs[8], sn[8];
    if (r.cos && h0 < r.H + c.KH) {                         // (the group's first head is one to rotate)
        const size_t at = (size_t)pos * HD + 8 * j;
        load8<false>(r.cos, at, cs);
        load8<false>(r.sin, at, sn);
    }
#pragma unroll
    for (int i = 0; i < NH; i++) {
        if (what[i] == 3) return;                           // (whole rows of 16 lanes)
        const uint16_t* w = what[i] == 0 ? r.w[0] : what[i] == 1 ? r.w[1] : nullptr;
        if (w) {
            const uint4 u = *(const uint4*)(w + 8 * j);
            const uint32_t ww[4] = {u.x, u.y, u.z, u.w};
            float ss = 0.0f;
#pragma unroll
            for (int e = 0; e < 8; e++) ss = __builtin_fmaf(x[i][e], x[i][e], ss);
            ss = seg_sum<16>(ss);
            const float inv = __fdiv_rn(1.0f, __fsqrt_rn(__fadd_rn(ss * (1.0f / HD), r.eps)));
#pragma unroll
            for (int e = 0; e < 4; e++) {
                x[i][2 * e] = x[i][2 * e] * inv * __uint_as_float(ww[e] << 16);
                x[i][2 * e + 1] = x[i][2 * e + 1] * inv * __uint_as_float(ww[e] & 0xFFFF0000u);
            }
        }
        if (r.cos && what[i] < 2) {
            float y[8];
#pragma unroll
            for (int e = 0; e < 8; e++) y[e] = dpp_f<DPP_ROR8>(x[i][e]);
#pragma unroll
            for (int e = 0; e < 8; e++) x[i][e] = __builtin_fmaf(j < 8 ? -y[e] : y[e], sn[e], x[i][e] * cs[e]);
        }
        if (what[i] == 0) {
            store8<BF>(r.q_out, ((size_t)t * r.H + head[i]) * HD + 8 * j, x[i]);
            continue;
        }
        if ((unsigned)page >= (unsigned)c.n_pages) continue;
        char* const base = (char*)(what[i] == 1 ? c.k : c.v) + (size_t)page * c.page_stride;
        const size_t at = (((size_t)head[i] << c.lp) + (pos & ((1 << c.lp) - 1))) * HD + 8 * j;
        if (c.f32) store8<false>(base, at, x[i]);
        else store8<true>(base, at, x[i]);
    }
}

hipError_t launch_paged_append(const PagedArgs& c, const PagedRows& r, hipStream_t st) {
    if (c.N == 0) return hipSuccess;
    const int heads = r.H + 2 * c.KH, one = (heads + 15) / 16;
    const bool few = (long long)c.N * one <= 2048;          // (8 blocks a CU: all heads at once)
    const int chunks = few ? one : (heads + 47) / 48;
    const dim3 grid((unsigned)((long long)c.N * chunks));
#define JM_PAGED_APPEND(BFV, NHV) hipLaunchKernelGGL((k_paged_append<BFV, NHV>), grid, dim3(256), 0, st, c, r, chunks)
    if (r.bf) { if (few) JM_PAGED_APPEND(true, 1); else JM_PAGED_APPEND(true, 3); }
    else { if (few) JM_PAGED_APPEND(false, 1); else JM_PAGED_APPEND(false, 3); }
#undef JM_PAGED_APPEND
    return hipGetLastError();
}

// ------------------------------------------------------- few query tokens
//
// Block (KV head, unit of up to 16 query rows: tokens x heads of the KV head, range of
// the unit's rows), 4 waves that take the range's tiles in turn, with a softmax each,
// joined at the end; the ranges of a unit are joined by a second launch
// (k_paged_merge).  A tile (8 KB of K and of V: 32 bf16 rows, 16 float32 ones) goes
// straight to the lanes' registers in the order in which the matrix cores take it, the
// next tile's while one is multiplied; nothing passes through LDS.
//
//   scores  16 rows as A (lane l: row 4 (l % 4) + l % 16 / 4 of them and the dimensions
//           of its group l / 16), the query rows as B: lane (g, n) holds query row n
//           at rows 4 i + g, i = 0 .. 3.  bf16: v_mfma_f32_16x16x32, group g of step s
//           dimensions 32 s + 8 g ..; float32: v_mfma_f32_16x16x4, group g of step
//           (s, e) dimension 16 s + 4 g + e.
//   P . V   V^T as A, the weights as B from the lanes that formed them: of its
//           contraction, group g has the rows 4 i + g.  Product j has the dimensions 8 m
//           + j in its rows m, so that lane (g, m) wants 8 consecutive dimensions of each
//           of its rows, 16 or 32 bytes as they lie in memory: in float32 these are the
//           operands of the 8 products; in bf16 pairs of rows change places, one
//           v_perm_b32 a register.
//
// bf16 pages: float32 q and weights are three bf16 parts (24 bits, one product each),
// bf16 q is exact in one, its weights two parts; all their products with K and V are
// exact, sums float32.  float32 pages: float32 products.
//
// Bound by HBM where prefixes are long: one token behind 131001 rows (537 MB) 84 us and 6 to
// join, 6.0 TB/s; 32 behind up to 16 k rows 260, 5.9 TB/s.  (A large copy here: 4.95 TB/s,
// reads and writes.)  Short ones wait: 7 us for a block with 6 tiles a wave, most of it the
// launch and the loads that need one another (cu, start, table, rows), and 4 for the second
// launch.  Registers, not LDS, hold the tile that is on its way: 235 to 256 of them, two
// waves a SIMD.

typedef float f32x4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ float pow2f(float x) { return __builtin_amdgcn_exp2f(x); }

__device__ __forceinline__ bf16x8 as_bf16x8(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    return __builtin_bit_cast(bf16x8, make_uint4(a, b, c, d));
}

// a and b as NP bf16 parts, each the rest of those before it.  (An infinity's rest is
// NaN: so is every output that it enters.)
template <int NP>
__device__ __forceinline__ void parts_bf16(float a, float b, uint32_t (&p)[NP]) {
#pragma unroll
    for (int i = 0; i < NP; i++) {
        p[i] = pack_bf16x2(a, b);
        a = __fsub_rn(a, __uint_as_float(p[i] << 16));
        b = __fsub_rn(b, __uint_as_float(p[i] & 0xFFFF0000u));
    }
}

struct PagedAttnArgs {
    const void* q;              // strides qts, qhs
    long long qts, qhs;
    int H, qpk, tp;             // tp tokens a unit
    float scale2;               // score scale times log2(e)
    void* out;                  // [N][H][128]
    int units, S;
    float* part_o;              // [units][KH][S][qpk tp][128]: not divided by the sum
    float* part_ml;             // [units][KH][S][qpk tp][2]: reference, sum (-1: no row seen)
};

// The pages of a sequence in one KV head.
struct PagedSeq {
    const int* table;
    const char* k;              // this head's rows of page 0
    const char* v;
    __device__ __forceinline__ PagedSeq(const PagedArgs& c, int seq, int kh) {
        const size_t head = ((size_t)kh << c.lp) * (c.f32 ? 512 : 256);
        table = c.table + seq * c.table_stride;
        k = (const char*)c.k + head;
        v = (const char*)c.v + head;
    }
};

// Where a tile's 16-row groups lie (wave-uniform): bytes from page 0's rows, and the last
// row of the group that may be read.  A group without a page, or past the last row that
// anyone sees, reads the tile's other group in its place; a tile without either is not
// read (live false).
template <int NG>
struct PagedTile {
    size_t at[NG];
    int lim[NG];
    bool ok[NG];
    bool live;
};

// The pages of the wave's tiles: lane i holds those of its group i of the next 64.
template <bool F32>
struct PagedWalk {
    static constexpr int NG = F32 ? 1 : 2, TR = 16 * NG, ROWB = F32 ? 512 : 256, AHEAD = 64 / NG;
    const PagedArgs& c;
    const int* table;
    int last, t0, W;            // the last row anyone sees, the wave's first tile, tiles between
    int page, next;             // the batch at hand and the one behind it
    __device__ __forceinline__ int fetch(int batch) const {
        const int lane = threadIdx.x & 63;
        const long long row = ((long long)t0 + (long long)(batch * AHEAD + lane / NG) * W) * TR + 16 * (lane % NG);
        const int p = row <= last ? table[row >> c.lp] : -1;
        return (unsigned)p < (unsigned)c.n_pages ? p : -1;
    }
    __device__ __forceinline__ PagedWalk(const PagedArgs& c_, const int* tb, int last_, int t, int w)
        : c(c_), table(tb), last(last_), t0(t), W(w) {
        page = fetch(0);
        next = fetch(1);
    }
    // the wave's i-th tile (each i once, in order)
    __device__ __forceinline__ void tile(int i, PagedTile<NG>& x) {
        if (i && i % AHEAD == 0) {
            page = next;
            next = fetch(i / AHEAD + 1);
        }
        const int row0 = (t0 + i * W) * TR;
        x.live = false;
#pragma unroll
        for (int g = 0; g < NG; g++) {
            const int p = __builtin_amdgcn_readlane(page, i % AHEAD * NG + g);
            const int row = row0 + 16 * g;
            x.ok[g] = p >= 0;
            x.lim[g] = min(last - row, 15);
            x.at[g] = (size_t)(p >= 0 ? p : 0) * c.page_stride + (size_t)(row & ((1 << c.lp) - 1)) * ROWB;
            x.live |= x.ok[g];
        }
        if (NG == 2) {
            if (!x.ok[0]) { x.at[0] = x.at[NG - 1]; x.lim[0] = x.lim[NG - 1]; }
            else if (!x.ok[NG - 1]) { x.at[NG - 1] = x.at[0]; x.lim[NG - 1] = x.lim[0]; }
        }
    }
};

// A tile as a lane gets it: 8 pieces of 16 bytes of K and of V.
template <bool F32>
__device__ __forceinline__ void paged_load_k(const PagedSeq& s, const PagedTile<F32 ? 1 : 2>& x, u32x4_t (&k)[8]) {
    constexpr int ROWB = F32 ? 512 : 256, NG = F32 ? 1 : 2;
    const int lane = threadIdx.x & 63, g = lane >> 4, n = lane & 15;
    if (!x.live) return;
#pragma unroll
    for (int h = 0; h < NG; h++) {
        const gptr<const char> p = (gptr<const char>)(s.k + x.at[h]);
        const uint32_t r = (uint32_t)min(4 * (n & 3) + (n >> 2), x.lim[h]) * ROWB + 16 * g;
#pragma unroll
        for (int i = 0; i < 8 / NG; i++) k[8 / NG * h + i] = __builtin_nontemporal_load((gptr<const u32x4_t>)(p + r + 64 * i));
    }
}
template <bool F32>
__device__ __forceinline__ void paged_load_v(const PagedSeq& s, const PagedTile<F32 ? 1 : 2>& x, u32x4_t (&v)[8]) {
    constexpr int ROWB = F32 ? 512 : 256, NG = F32 ? 1 : 2;
    const int lane = threadIdx.x & 63, g = lane >> 4, n = lane & 15;
    if (!x.live) return;
#pragma unroll
    for (int h = 0; h < NG; h++) {
        const gptr<const char> p = (gptr<const char>)(s.v + x.at[h]);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const uint32_t r = (uint32_t)min(4 * i + g, x.lim[h]) * ROWB + ROWB / 16 * n;
#pragma unroll
            for (int j = 0; j < 2 / NG; j++) v[4 * h + 2 / NG * i + j] = __builtin_nontemporal_load((gptr<const u32x4_t>)(p + r + 16 * j));
        }
    }
}

// The weights p of the lane's rows as operands.
template <bool F32, int NP>
struct PagedWeights {
    uint32_t w[NP][4];
    __device__ __forceinline__ explicit PagedWeights(const float (&p)[8]) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            if (F32) {
                w[0][i] = __float_as_uint(p[i]);
                continue;
            }
            uint32_t x[NP];
            parts_bf16<NP>(p[2 * i], p[2 * i + 1], x);
#pragma unroll
            for (int k = 0; k < NP; k++) w[k][i] = x[k];
        }
    }
    // o + V^T's product j times the weights; v(e, d): dword d of piece e
    template <class V>
    __device__ __forceinline__ f32x4 times(V v, int j, f32x4 o) const {
        if (F32) {
#pragma unroll
            for (int i = 0; i < 4; i++)
                o = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(v(2 * i + j / 4, j % 4)), __uint_as_float(w[0][i]), o, 0, 0, 0);
            return o;
        }
        uint32_t a[4];
#pragma unroll
        for (int i = 0; i < 4; i++) a[i] = __builtin_amdgcn_perm(v(2 * i + 1, j / 2), v(2 * i, j / 2), j & 1 ? 0x07060302u : 0x05040100u);
        const bf16x8 x = as_bf16x8(a[0], a[1], a[2], a[3]);
#pragma unroll
        for (int k = NP - 1; k >= 0; k--)
            o = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x, as_bf16x8(w[k][0], w[k][1], w[k][2], w[k][3]), o, 0, 0, 0);
        return o;
    }
};

constexpr int PAGED_OW = 132;               // floats between the columns of a wave's outputs in LDS
constexpr int PAGED_W = 4;                  // waves of a block

// The query rows of one unit over tiles t0 .. t_end - 1 of its sequence; the waves joined,
// and the output, or (several ranges) the partial outputs.
template <bool F32, bool BF>
__global__ void __launch_bounds__(64 * PAGED_W, 2)
k_paged_attn(PagedArgs c, PagedAttnArgs a) {
    constexpr int HD = 128, W = PAGED_W, NG = F32 ? 1 : 2, TR = 16 * NG, NY = 4 * NG;
    constexpr int NQ = BF ? 1 : 3, NP = BF ? 2 : 3;         // parts of q, of the weights
    __shared__ __align__(16) float ow[W][16][PAGED_OW];
    __shared__ float mls[W][16][2];
    const int kh = blockIdx.x % c.KH, u = blockIdx.x / c.KH % a.units, s = blockIdx.x / c.KH / a.units;
    CallUnit un;
    if (!call_unit(c, u, a.tp, un)) return;                 // (block-uniform)
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int g = lane >> 4, n = lane & 15;
    const int last = min(un.pos + un.n - 1, c.maxT - 1);    // the last row any token sees
    const int NT = last < 0 ? 0 : last / TR + 1;
    const int t0 = (int)((long long)NT * s / a.S), t_end = (int)((long long)NT * (s + 1) / a.S);
    const int ncol = a.qpk * un.n;
    const int ct = min(n / a.qpk, un.n - 1), head = kh * a.qpk + n % a.qpk;
    const int crow = min(un.pos + ct, c.maxT - 1);          // the last row that this column sees

    const PagedSeq seq(c, un.seq, kh);
    const int mine = t_end - t0 > w ? (t_end - t0 - w + W - 1) / W : 0;     // this wave's tiles
    PagedWalk<F32> walk(c, seq.table, mine ? last : -1, t0 + w, W);
    PagedTile<NG> x, xn;
    u32x4_t ck[8], cv[8], nk[8], nv[8];
    x.live = xn.live = false;
    if (mine) {
        walk.tile(0, x);
        paged_load_k<F32>(seq, x, ck);
        paged_load_v<F32>(seq, x, cv);
    }

    // the query columns
    float qf[F32 ? 32 : 1];
    bf16x8 qb[F32 ? 1 : NQ][4];
    const size_t qi = (size_t)((un.tok + ct) * a.qts + head * a.qhs);
    if constexpr (F32) {
#pragma unroll
        for (int i = 0; i < 8; i++) {
            float y[4];
            load4<BF>(a.q, qi + 16 * i + 4 * g, y);
#pragma unroll
            for (int e = 0; e < 4; e++) qf[4 * i + e] = y[e];
        }
    } else {
#pragma unroll
        for (int st = 0; st < 4; st++) {
            float y[8];
            load8<BF>(a.q, qi + 32 * st + 8 * g, y);
            uint32_t z[NQ][4];
#pragma unroll
            for (int e = 0; e < 4; e++) {
                uint32_t p[NQ];
                parts_bf16<NQ>(y[2 * e], y[2 * e + 1], p);
#pragma unroll
                for (int k = 0; k < NQ; k++) z[k][e] = p[k];
            }
#pragma unroll
            for (int k = 0; k < NQ; k++) qb[k][st] = as_bf16x8(z[k][0], z[k][1], z[k][2], z[k][3]);
        }
    }

    f32x4 O[8];
    float ref = -INFINITY, l = 0.0f;
    int seen = 0;
#pragma unroll
    for (int j = 0; j < 8; j++) O[j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};

    for (int i = 0; i < mine; i++) {
        const bool more = i + 1 < mine;
        if (more) {
            walk.tile(i + 1, xn);
            paged_load_k<F32>(seq, xn, nk);
            paged_load_v<F32>(seq, xn, nv);
        }
        const int row0 = (t0 + w + i * W) * TR;
        float p[8];
        bool whole = row0 + TR - 1 <= un.pos;
        if (x.live) {
            // ---- scores
#pragma unroll
            for (int h = 0; h < NG; h++) {
                f32x4 S = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
                if constexpr (F32) {
                    f32x4 S2 = S;
#pragma unroll
                    for (int k = 0; k < 32; k += 2) {
                        S = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(ck[k / 4][k % 4]), qf[k], S, 0, 0, 0);
                        S2 = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(ck[k / 4][k % 4 + 1]), qf[k + 1], S2, 0, 0, 0);
                    }
                    S += S2;
                } else {
#pragma unroll
                    for (int k = NQ - 1; k >= 0; k--)
#pragma unroll
                        for (int st = 0; st < 4; st++)
                            S = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, ck[4 * h + st]), qb[k][st], S, 0, 0, 0);
                }
#pragma unroll
                for (int e = 0; e < 4; e++) p[4 * h + e] = __fmul_rn(S[e], a.scale2);
            }
            // rows that the column does not see: past its own, or without a page
#pragma unroll
            for (int h = 0; h < NG; h++) {
                whole &= x.ok[h];
                seen |= (int)x.ok[h] & (int)(row0 + 16 * h <= crow);
            }
            if (!whole) {
#pragma unroll
                for (int e = 0; e < NY; e++)
                    if (!x.ok[e / 4] || row0 + 16 * (e / 4) + 4 * (e % 4) + g > crow) p[e] = -INFINITY;
            }
            // ---- the reference: raised to the largest score when one passes it by 2^10
            float ym = p[0];
#pragma unroll
            for (int e = 1; e < NY; e++) ym = fmaxf(ym, p[e]);
            if (__any(ym > ref + 10.0f)) {
                ym = fmaxf(ym, swz_xor16_f(ym));
                ym = fmaxf(ym, __shfl_xor(ym, 32, JM_WAVE));
                const float nref = fmaxf(ref, ym);
                const float f = nref == -INFINITY ? 1.0f : pow2f(ref - nref);
                l *= f;
#pragma unroll
                for (int j = 0; j < 8; j++) O[j] *= f;
                ref = nref;
            }
            const float r0 = ref == -INFINITY ? 0.0f : ref;       // (a column that has seen nothing yet)
#pragma unroll
            for (int e = 0; e < NY; e++) {
                p[e] = pow2f(__fsub_rn(p[e], r0));
                l = __fadd_rn(l, p[e]);
            }
            // ---- P . V.  A weight of 0 does not hide a value that is not finite: where
            // some column does not see such a row, token by token, each with the rows that
            // it sees.
            bool apart = false;
            auto row_of = [&](int e) __attribute__((always_inline)) {       // of cv[e]; a group without a page holds another's
                const int h = F32 ? 0 : e / 4;
                return x.ok[h] ? row0 + 16 * h + 4 * (F32 ? e / 2 : e % 4) + g : INT_MAX;
            };
            if (!whole && un.n > 1) {
                uint32_t bad = 0;
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    uint32_t y = 0;
#pragma unroll
                    for (int d = 0; d < 4; d++) {
                        y |= (cv[e][d] & 0x7F800000u) == 0x7F800000u;
                        if (!F32) y |= (cv[e][d] & 0x7F80u) == 0x7F80u;
                    }
                    bad |= row_of(e) > un.pos ? y : 0u;
                }
                apart = __any(bad != 0);
            }
            if (!apart) {
                if constexpr (F32) {
                    // (a row at a time, so that a product never waits for the one before it)
#pragma unroll
                    for (int i = 0; i < 4; i++)
#pragma unroll
                        for (int j = 0; j < 8; j++)
                            O[j] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(cv[2 * i + j / 4][j % 4]), p[i], O[j], 0, 0, 0);
                } else {
                    const PagedWeights<F32, NP> pw(p);
#pragma unroll
                    for (int j = 0; j < 8; j++) O[j] = pw.times([&](int e, int d) { return cv[e][d]; }, j, O[j]);
                }
            } else {
#pragma unroll 1
                for (int t = 0; t < un.n; t++) {
                    float pt[8];
#pragma unroll
                    for (int e = 0; e < NY; e++) pt[e] = ct == t ? p[e] : 0.0f;
                    const PagedWeights<F32, NP> pw(pt);
#pragma unroll
                    for (int j = 0; j < 8; j++) {
                        const f32x4 T = pw.times([&](int e, int d) { return row_of(e) <= un.pos + t ? cv[e][d] : 0u; }, j,
                                                 f32x4{0.0f, 0.0f, 0.0f, 0.0f});
#pragma unroll
                        for (int i = 0; i < 4; i++) O[j][i] = ct == t ? O[j][i] + T[i] : O[j][i];
                    }
                }
            }
        }
#pragma unroll
        for (int e = 0; e < 8; e++) {
            ck[e] = nk[e];
            cv[e] = nv[e];
        }
        x = xn;
    }

    // ---- the wave's outputs: dimensions 32 g + 8 i + j of column 16 b + n
    l += swz_xor16_f(l);
    l += __shfl_xor(l, 32, JM_WAVE);
#pragma unroll
    for (int i = 0; i < 4; i++) {
        *(float4*)&ow[w][n][32 * g + 8 * i] = make_float4(O[0][i], O[1][i], O[2][i], O[3][i]);
        *(float4*)&ow[w][n][32 * g + 8 * i + 4] = make_float4(O[4][i], O[5][i], O[6][i], O[7][i]);
    }
    if (g == 0) {
        mls[w][n][0] = ref;
        mls[w][n][1] = seen ? l : -1.0f;
    }
    __syncthreads();

    // ---- the block's: thread = column, dimensions 4 (tid % 32) ..
    for (int oc = threadIdx.x >> 5; oc < ncol; oc += 2 * W) {
        const int od = 4 * (threadIdx.x & 31);
        float M = -INFINITY;
#pragma unroll
        for (int i = 0; i < W; i++) M = fmaxf(M, mls[i][oc][0]);
        float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        float L = 0.0f;
        bool any = false;
#pragma unroll
        for (int i = 0; i < W; i++) {
            if (mls[i][oc][1] == -1.0f) continue;
            any = true;
            const float f = pow2f(mls[i][oc][0] - M);
            const float4 y = *(const float4*)&ow[i][oc][od];
            v.x = __builtin_fmaf(y.x, f, v.x);
            v.y = __builtin_fmaf(y.y, f, v.y);
            v.z = __builtin_fmaf(y.z, f, v.z);
            v.w = __builtin_fmaf(y.w, f, v.w);
            L = __builtin_fmaf(mls[i][oc][1], f, L);
        }
        const int to = oc / a.qpk;
        if (un.pos + to >= c.maxT) continue;
        if (a.S == 1) {
            // a token that sees no row: 0.  (A sum of 0 elsewhere is that of scores that are
            // all -infinity: NaN.)
            const float inv = any ? __fdiv_rn(1.0f, L) : 0.0f;
            const size_t oi = ((size_t)(un.tok + to) * a.H + kh * a.qpk + oc % a.qpk) * HD + od;
            store_out<BF>(a.out, oi, make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv));
        } else {
            const size_t pi = (((size_t)u * c.KH + kh) * a.S + s) * (a.qpk * a.tp) + oc;
            if (any) *(float4*)(a.part_o + pi * HD + od) = v;
            if ((threadIdx.x & 31) == 0) *(float2*)(a.part_ml + 2 * pi) = make_float2(M, any ? L : -1.0f);
        }
    }
}

// The ranges of a (unit, KV head, query row) joined into the output, by 32 lanes, 4
// dimensions a lane (G = 1), or by 8 groups of them that take the ranges in turn and are
// added in order (G = 8).
template <bool BF, int G>
__global__ void __launch_bounds__(256)
k_paged_merge(PagedArgs c, PagedAttnArgs a) {
    constexpr int HD = 128;
    __shared__ __align__(16) float4 acc[G][32];
    __shared__ float ls[G];
    const int nc = a.qpk * a.tp;
    const int j = threadIdx.x & 31, gr = G == 1 ? 0 : threadIdx.x >> 5;
    // (a block's rows are of one unit: call_unit wants the same in every lane)
    const int nb = G == 1 ? (nc + 7) / 8 : nc, kh = blockIdx.x % c.KH, rs = blockIdx.x / c.KH, u = rs / nb;
    const int oc = G == 1 ? 8 * (rs % nb) + (threadIdx.x >> 5) : rs % nb;
    CallUnit un;
    if (!call_unit(c, u, a.tp, un)) return;
    const int to = oc / a.qpk;
    if (oc >= nc || to >= un.n || un.pos + to >= c.maxT) return;        // (with G = 8 block-uniform)
    const size_t p0 = ((size_t)u * c.KH + kh) * a.S * nc + oc;
    float M = -INFINITY;
    uint32_t any = 0;
    for (int s = j; s < a.S; s += 32) {
        const float2 x = *(const float2*)(a.part_ml + 2 * (p0 + (size_t)s * nc));
        M = fmaxf(M, x.x);
        any |= (uint32_t)(x.y != -1.0f);
    }
    M = seg_max<32>(M);
    any = (uint32_t)(__ballot(any != 0) >> (threadIdx.x & 32));
    float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    float L = 0.0f;
    for (int s0 = gr; s0 < a.S; s0 += 4 * G) {
        float4 x[4];
        float2 ml[4];
#pragma unroll
        for (int q = 0; q < 4; q++) {
            const size_t p = p0 + (size_t)min(s0 + G * q, a.S - 1) * nc;
            ml[q] = *(const float2*)(a.part_ml + 2 * p);
            x[q] = *(const float4*)(a.part_o + p * HD + 4 * j);
        }
#pragma unroll
        for (int q = 0; q < 4; q++) {
            if (s0 + G * q >= a.S || ml[q].y == -1.0f) continue;       // (a range without a row has no output)
            const float f = pow2f(ml[q].x - M);
            v.x = __builtin_fmaf(x[q].x, f, v.x);
            v.y = __builtin_fmaf(x[q].y, f, v.y);
            v.z = __builtin_fmaf(x[q].z, f, v.z);
            v.w = __builtin_fmaf(x[q].w, f, v.w);
            L = __builtin_fmaf(ml[q].y, f, L);
        }
    }
    if constexpr (G > 1) {
        acc[gr][j] = v;
        if (j == 0) ls[gr] = L;
        __syncthreads();
        if (gr) return;
#pragma unroll
        for (int i = 1; i < G; i++) {
            const float4 y = acc[i][j];
            v = make_float4(v.x + y.x, v.y + y.y, v.z + y.z, v.w + y.w);
            L += ls[i];
        }
    }
    const float inv = any ? __fdiv_rn(1.0f, L) : 0.0f;                  // (as in k_paged_attn)
    store_out<BF>(a.out, ((size_t)(un.tok + to) * a.H + kh * a.qpk + oc % a.qpk) * HD + 4 * j,
                  make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv));
}

// ------------------------------------------------------ many query tokens
//
// Prompts over bf16 pages: block (KV head, unit of 32 QB RG query rows, range of the
// unit's rows), 8 waves = RG row groups x PS position strides; in a step wave (rg, ps)
// takes the 32 cache rows ps of the step's 32 PS for its 32 QB query rows, with an online
// softmax, and the PS waves of a row group are joined at the end.  A step's rows go
// straight to LDS, those of the NS - 1 steps after it on their way.
//
//   scores   v_mfma_f32_32x32x16_bf16, cache rows as A (lane l: row l % 32, dimensions 16
//            kk + 8 (l / 32) ..), query rows as B: lane l holds query row l % 32 at cache
//            rows 8 (v / 4) + 4 (l / 32) + v % 4
//   P . V    V^T as A, read transposed from LDS (ds_read_b64_tr_b16: 4 rows of 16
//            dimensions), the weights as B from the registers that formed them:
//            contraction index j of half h in step s is row 16 s + 8 (j / 4) + 4 h + j % 4
//
// bf16 queries (BF): 64 query rows a wave (QB = 2), so that an operand read from LDS serves
// two products; q is exact, the weights are two bf16 parts.  float32 queries: q and the
// weights as three bf16 parts each.  Both as in k_paged_attn, so that a token gets the same
// precision whichever kernel its call takes.  (The weights of bf16 queries in one part: 2047
// tokens behind 4099 rows 190 us instead of 236, but two outputs in five come out another bf16
// number, and the error against float64 is 1.4 times that of the output's own rounding.)
//
// Bound by the issue of instructions: a step takes 5100 cycles for 3168 of products, as the two
// waves of a SIMD have 480 instructions each, of which a wave issues one in 5 to 7 cycles.  2047
// tokens behind 4099 rows (32 heads on 8) 236 us, 727 TFLOP/s of the formula's products, and
// 28% of it is the longest prefix's block against the mean one.  What brought it there
// (measured with weights of one part, 192 us): the two waves of a SIMD a phase apart instead of
// in step (206 to 232), a reference that is raised only where the weights' sum tells of a score
// far above it, loads to LDS as buffers (as flat ones every read of LDS waits for all before
// it), outputs through LDS in whole lines (200).

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

// 4 rows x 16 columns of bf16 in LDS, transposed over 16 lanes: lane i gives the address
// of 4 columns (4 (i % 4) ..) of row i / 4 and receives column i of rows 0 .. 3
__device__ __forceinline__ s16x4 paged_tr16(const uint16_t* p) {
    return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(void*)p);
}

// The phases of k_paged_tile: what must have completed is waited for explicitly, and
// nothing moves from one to the next.
__device__ __forceinline__ void paged_meet() {
    __builtin_amdgcn_sched_barrier(0);
    wave_meet();
    __builtin_amdgcn_sched_barrier(0);
}

template <bool BF, int RG>
__global__ void __launch_bounds__(512, 2)
k_paged_tile(PagedArgs c, PagedAttnArgs a) {
    constexpr int HD = 128, QB = BF ? 2 : 1, NQ = BF ? 1 : 3, NP = BF ? 2 : 3, PS = 8 / RG, STEP = 32 * PS, TILE = 32 * HD;
    constexpr int RW = 8 * (PS / 2);            // rows of a step that a wave stages, of K and of V
    constexpr int LPS = RW / 2;                 // its loads, 4 rows each
    constexpr int NROW = 32 * QB * RG, AHEAD = 2;
    constexpr int NS = PS == 2 ? 3 : 2;         // steps in LDS
    // PS tiles of K and of V of NS steps; at the end the outputs being joined
    __shared__ __align__(16) uint16_t kv[2][NS][PS * TILE];
    auto& kt = kv[0];
    auto& vt = kv[1];
    // the second block of query rows of each row group (BF)
    __shared__ __align__(16) uint4 q1[BF ? RG : 1][8][64];
    __shared__ float mls[8][32 * QB][2];
    // which dimensions met a V value of +inf (bit 0), -inf (bit 1) or NaN (both) that not
    // every query row of a wave sees, 16 dimensions a word
    __shared__ uint32_t taint[NROW][HD / 16];
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int rg = w % RG, ps = w / RG, n = lane & 31, h = lane >> 5;
    const int kh = blockIdx.x % c.KH, rs = blockIdx.x / c.KH;
    const int u = a.units - 1 - rs % a.units, sr = rs / a.units;        // the longest prefixes first
    CallUnit un;
    if (!call_unit(c, u, a.tp, un)) return;
    const PagedSeq seq(c, un.seq, kh);
    const int pmax = min(un.pos + un.n - 1, c.maxT - 1);
    // this block's range of the steps (none where no token sees a row)
    const int steps = pmax < 0 ? 0 : pmax / STEP + 1;
    const int step0 = (int)((long long)steps * sr / a.S), nstep = (int)((long long)steps * (sr + 1) / a.S) - step0;

    // this lane's query rows, and the last cache row that each sees
    int tok[QB], prow[QB], head[QB];
    bool live[QB];
#pragma unroll
    for (int b = 0; b < QB; b++) {
        const int r = 32 * (QB * rg + b) + n, t = r / a.qpk;
        live[b] = t < un.n && un.pos + t < c.maxT;
        tok[b] = min(t, un.n - 1);
        head[b] = kh * a.qpk + r % a.qpk;
        prow[b] = min(un.pos + tok[b], c.maxT - 1);
    }
    // ... the first of the wave's
    const int wmin = min(un.pos + min(32 * QB * rg / a.qpk, un.n - 1), c.maxT - 1);

    // ---- staging: of the half of a step that its four waves (w < 4, or the others)
    // multiply, wave w has rows RW (w % 4) ..: 8 or 16 rows of the tile that it multiplies
    // itself.  Lane 2 i + g of `page` has the page of the tile's 16-row group g in the i-th of
    // 32 steps.
    const int srow = STEP / 2 * (w >> 2) + RW * (w & 3), sgroup = (srow >> 4) & 1;
    auto fetch = [&](int batch) __attribute__((always_inline)) {
        const long long row = (long long)(step0 + 32 * batch + (lane >> 1)) * STEP + 32 * ps + 16 * (lane & 1);
        const int p = row <= pmax ? seq.table[row >> c.lp] : -1;
        return (unsigned)p < (unsigned)c.n_pages ? p : -1;
    };
    int page = fetch(0), next = fetch(1);
    // ---- the query rows' values on their way
    u32x4_a8 qv[QB][8][BF ? 1 : 2];
#pragma unroll
    for (int b = 0; b < QB; b++) {
        const size_t qi = (size_t)((un.tok + tok[b]) * a.qts + head[b] * a.qhs);
#pragma unroll
        for (int k = 0; k < 8; k++)
#pragma unroll
            for (int i = 0; i < (BF ? 1 : 2); i++)
                qv[b][k][i] = BF ? *(const u32x4_a8*)((const uint16_t*)a.q + qi + 16 * k + 8 * h) : *(const u32x4_a8*)((const float*)a.q + qi + 16 * k + 8 * h + 4 * i);
    }
    // where a lane's first load of a step lies within its rows (load j: 4 j rows on; of K
    // another chunk of them)
    const int r0 = lane >> 4;
    const int koff = 256 * r0 + 16 * ((lane & 15) ^ ((srow + r0) & 15)), voff = 256 * r0 + 16 * ((lane & 15) ^ (4 * r0));
    // the wave's rows of K or V of a step into `to`: `at` bytes from page 0's rows, lim + 1 of
    // them to be read (none: no page)
    auto request = [&](auto full, const char* src, bool isk, size_t at, int lim, uint16_t* to) __attribute__((always_inline)) {
        // (as a number: the compiler would have every read of LDS wait for these loads, which
        // are waited for below; and as a buffer: behind a load from a global address to LDS,
        // which counts as both, it lets no read of LDS be outstanding when it waits for one)
        uint32_t num = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(__attribute__((address_space(3))) void*)(to + srow * HD));
        __asm__ volatile("" : "+s"(num));
        const auto dst = (__attribute__((address_space(3))) uint16_t*)(uintptr_t)num;
        const auto base = __builtin_amdgcn_make_buffer_rsrc((void*)(src + at), 0, RW * 256, 0x00020000);
        if (decltype(full)::value || lim >= RW - 1) {
#pragma unroll
            for (int j = 0; j < RW / 4; j++)
                __builtin_amdgcn_raw_ptr_buffer_load_lds(base, (__attribute__((address_space(3))) void*)(dst + 4 * j * HD), 16,
                                                         isk ? koff ^ (64 * j) : voff, 1024 * j, 0, 0);
        } else if (lim >= 0) {
            // (rows past the prefixes repeat the last one; their weights are 0)
#pragma unroll
            for (int j = 0; j < RW / 4; j++) {
                const int r = 4 * j + r0, x = isk ? (srow + r) & 15 : 4 * r0;
                __builtin_amdgcn_raw_ptr_buffer_load_lds(base, (__attribute__((address_space(3))) void*)(dst + 4 * j * HD), 16,
                                                         min(r, lim) * 256 + 16 * ((lane & 15) ^ x), 0, 0, 0);
            }
        } else if (!isk) {
#pragma unroll
            for (int j = 0; j < RW / 4; j++) *(uint4*)(to + (srow + 4 * j) * HD + 8 * lane) = make_uint4(0, 0, 0, 0);
        }
    };
    // where the rows of K of the step to be requested next lie, and those of V, of the step
    // before it; has: whether the tile's groups have pages, two bits a step, the latest lowest
    int klim = -1, vlim = -1;
    size_t kat = 0, vat = 0;
    uint32_t has = 0;
    auto locate = [&](int t) __attribute__((always_inline)) {
        vat = kat;
        vlim = klim;
        if (t && t % 32 == 0) {
            page = next;
            next = fetch(t / 32 + 1);
        }
        const int p0 = __builtin_amdgcn_readlane(page, 2 * (t % 32)), p1 = __builtin_amdgcn_readlane(page, 2 * (t % 32) + 1);
        has = has << 2 | (p0 >= 0 ? 1u : 0u) | (p1 >= 0 ? 2u : 0u);
        const int p = sgroup ? p1 : p0, row = (step0 + t) * STEP + srow;
        klim = p >= 0 ? min(pmax - row, RW - 1) : -1;
        kat = (size_t)(klim >= 0 ? p : 0) * c.page_stride + (uint32_t)((row & ((1 << c.lp) - 1)) * 256);
    };
    constexpr std::true_type yes{};
    constexpr std::false_type no{};
#pragma unroll 1
    for (int t = 0; t < NS; t++) {
        locate(t);
        if (t < nstep) request(no, seq.k, true, kat, klim, kt[t]);
        if (t < nstep && t < NS - 1) request(no, seq.v, false, kat, klim, vt[t]);
    }
    locate(NS);

    // ---- the query rows, with the score scale's sign (a scale of 0 as 2^-149, of which the
    // largest score makes 2^-21: masked scores stay -inf behind it)
    const float cs = fmaxf(fabsf(a.scale2), 0x1p-149f);
    const uint32_t sign = a.scale2 < 0.0f ? 0x80008000u : 0u;
    bf16x8 qr[NQ][8];
#pragma unroll
    for (int b = 0; b < QB; b++)
#pragma unroll
        for (int k = 0; k < 8; k++) {
            uint32_t y[NQ][4];
#pragma unroll
            for (int e = 0; e < 4; e++) {
                if (BF) {
                    y[0][e] = qv[b][k][0][e] ^ sign;
                } else {
                    uint32_t p[NQ];
                    const u32x4_a8 x = qv[b][k][BF ? 0 : e / 2];
                    parts_bf16<NQ>(__uint_as_float(x[2 * (e & 1)]), __uint_as_float(x[2 * (e & 1) + 1]), p);
#pragma unroll
                    for (int i = 0; i < NQ; i++) y[i][e] = p[i] ^ sign;
                }
            }
            if (b == 0) {
#pragma unroll
                for (int i = 0; i < NQ; i++) qr[i][k] = as_bf16x8(y[i][0], y[i][1], y[i][2], y[i][3]);
            } else if (ps == 0) {
                q1[rg][k][lane] = make_uint4(y[0][0], y[0][1], y[0][2], y[0][3]);
            }
        }
    for (int i = tid; i < NROW * (HD / 16); i += 512) (&taint[0][0])[i] = 0;

    f32x16 O[QB][4];
    float ref[QB], l[QB];
    int seen[QB];                               // whether the lane's query rows saw a row; all: all of them did
    bool all = false;
    f32x16 S[QB];
    u32x4_t P[QB][NP][2];
#pragma unroll
    for (int b = 0; b < QB; b++) {
        ref[b] = -INFINITY;
        l[b] = 0.0f;
        seen[b] = 0;
#pragma unroll
        for (int nt = 0; nt < 4; nt++) O[b][nt] = f32x16(0.0f);
    }
    const int ko = (32 * ps + n) * HD + 8 * (h ^ (n & 15));     // K row n: dimensions 16 kk + 8 h .. at chunk (2 kk) ^ h ^ (n % 16)
    // this lane's part of a transposed read: row 4 h + i / 4, 4 columns 16 (l / 16 % 2) + 4 (i
    // % 4) of a 32-column block, i = l % 16; chunk c of V row r sits at c ^ 4 (r % 4)
    const int vrow = (lane & 15) >> 2;
    const int vo = (32 * ps + 4 * h + vrow) * HD + 32 * vrow + 8 * (2 * ((lane >> 4) & 1) + ((lane >> 1) & 1)) + 4 * (lane & 1);

    // ---- a wave's weights of a step: of lane registers 8 s + 2 e, + 1 of its scores
    auto weights = [&](int s, int e) __attribute__((always_inline)) {
#pragma unroll
        for (int b = 0; b < QB; b++) {
            const float r0 = ref[b] == -INFINITY ? 0.0f : ref[b];
            const float x0 = pow2f(__builtin_fmaf(S[b][8 * s + 2 * e], cs, -r0));
            const float x1 = pow2f(__builtin_fmaf(S[b][8 * s + 2 * e + 1], cs, -r0));
            uint32_t p[NP];
            parts_bf16<NP>(x0, x1, p);
#pragma unroll
            for (int q = 0; q < NP; q++) P[b][q][s][e] = p[q];
            l[b] += x0 + x1;
        }
    };
    // The vector work of a phase: of step t, the scores that are not seen, the weights, the
    // reference.
    auto weigh = [&](int t) __attribute__((always_inline)) {
        const int t0 = (step0 + t) * STEP + 32 * ps;
        const uint32_t ok = has >> (2 * NS) & 3u;
        if (ok == 3u && t0 + 31 <= wmin) {
            all = true;
        } else {
#pragma unroll
            for (int b = 0; b < QB; b++) {
                const int lim = prow[b] - t0;
                seen[b] |= (int)(ok & 1u) & (int)(lim >= 0);
                seen[b] |= (int)(ok >> 1) & (int)(lim >= 16);
#pragma unroll
                for (int v = 0; v < 16; v++) {
                    const int see = ok & (v < 8 ? 1u : 2u) ? lim - 4 * h : -1;
                    S[b][v] = 8 * (v / 4) + v % 4 > see ? -INFINITY : S[b][v];
                }
            }
        }
        // The weights by the reference as it is, and a new one only where their sum says that one
        // has passed it by far (or where there is none yet): the largest score is not looked for
        // otherwise.
        float before[QB];
#pragma unroll
        for (int b = 0; b < QB; b++) before[b] = l[b];
#pragma unroll
        for (int e = 0; e < 8; e++) weights(e / 4, e % 4);
        bool high = false;
#pragma unroll
        for (int b = 0; b < QB; b++) high |= l[b] > before[b] + 4096.0f || ref[b] == -INFINITY;
        if (__any(high)) {
#pragma unroll
            for (int b = 0; b < QB; b++) {
                float m = S[b][0];
#pragma unroll
                for (int v = 1; v < 16; v++) m = fmaxf(m, S[b][v]);
                m = fmaxf(m, __shfl_xor(m, 32, JM_WAVE)) * cs;
                const float nref = fmaxf(ref[b], m);
                const float f = nref == -INFINITY ? 1.0f : pow2f(ref[b] - nref);
                l[b] = before[b] * f;
#pragma unroll
                for (int nt = 0; nt < 4; nt++) O[b][nt] *= f;
                ref[b] = nref;
            }
#pragma unroll
            for (int e = 0; e < 8; e++) weights(e / 4, e % 4);
        }
        // (here and now: the compiler would put them off to where they are used, among the
        // products)
#pragma unroll
        for (int b = 0; b < QB; b++) {
#pragma unroll
            for (int q = 0; q < NP; q++) __asm__ volatile("" : "+v"(P[b][q][0]), "+v"(P[b][q][1]));
            __asm__ volatile("" : "+v"(l[b]));
        }
    };

    // ---- the products of a phase: the weights of step t times its V, the scores of the step
    // after it.  (Operands AHEAD products ahead of their use, in an order
    // that the compiler keeps: left to it, every product waits for its own.  Their
    // addresses from one each, an XOR at a time: those of all steps in LDS kept in
    // registers, others spill.)
    auto multiply = [&](auto has_v, int t, uint16_t* v, const uint16_t* kk) __attribute__((always_inline)) {
        constexpr bool V = decltype(has_v)::value;
        const int t0 = (step0 + t) * STEP + 32 * ps;
        int va = vo;
        __asm__ volatile("" : "+v"(va));
        auto vop = [&](int k) __attribute__((always_inline)) {
            const uint16_t* const p = v + (va ^ (32 * (k % 4))) + 16 * (k / 4) * HD;
            return __builtin_bit_cast(bf16x8, __builtin_shufflevector(paged_tr16(p), paged_tr16(p + 8 * HD), 0, 1, 2, 3, 4, 5, 6, 7));
        };
        // A weight of 0 does not hide a value that is not finite.  Where not all of the
        // wave's query rows see the tile, such values go into `taint`, for all of the
        // block's rows that see them, and out of the tile.  (The other waves that multiply it
        // find them there or in `taint`: either is right.)
        if (V && t0 + 31 > wmin) {
            uint16_t* const tile = v + ps * TILE;
            uint32_t nf = 0;
#pragma unroll 2
            for (int j = 0; j < 8; j++) {
                const uint4 y = *(const uint4*)(tile + 8 * (64 * j + lane));
                const uint32_t x[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
                for (int e = 0; e < 4; e++)
                    nf |= (uint32_t)((x[e] & 0x7F80u) == 0x7F80u) | (uint32_t)((x[e] & 0x7F800000u) == 0x7F800000u);
            }
            if (__any(nf != 0)) {
#pragma unroll 1
                for (int e = lane; e < TILE; e += 64) {
                    const int r = e / HD, dim = (e % HD) ^ (32 * (r & 3));
                    const uint32_t x = tile[e];
                    if ((x & 0x7F80u) != 0x7F80u) continue;
                    const uint32_t bits = (x & 0x7Fu) ? 3u : (x >> 15) ? 2u : 1u;
                    if (t0 + r <= pmax) {               // (a row past the prefixes holds the last one again)
#pragma unroll 1
                        for (int q = 0; q < NROW; q++)
                            if (t0 + r <= un.pos + min(q / a.qpk, un.n - 1)) atomicOr(&taint[q][dim / 16], bits << (2 * (dim % 16)));
                    }
                    tile[e] = 0;
                }
                __builtin_amdgcn_s_waitcnt(0xC07F);     // lgkmcnt(0)
                __asm__ volatile("" : : : "memory");
            }
        }
        int ka = ko;
        __asm__ volatile("" : "+v"(ka));
        auto kop = [&](int k) __attribute__((always_inline)) { return *(const bf16x8*)(kk + (ka ^ (16 * k))); };
        auto qop = [&](int k) __attribute__((always_inline)) { return *(const bf16x8*)&q1[BF ? rg : 0][k][lane]; };
        constexpr int first = V ? 0 : 8, end = 16;
        bf16x8 x[16], y[16];
#pragma unroll
        for (int k = first; k < end + AHEAD; k++) {
            if (k < end) {
                x[k] = k < 8 ? vop(k) : kop(k - 8);
                if (QB == 2 && k >= 8) y[k] = qop(k - 8);
            }
            if (k < first + AHEAD) continue;
            __builtin_amdgcn_sched_barrier(0);
            const int j = k - AHEAD;
            if (j == 8) {
#pragma unroll
                for (int b = 0; b < QB; b++) S[b] = f32x16(0.0f);
            }
            if (j < 8) {
#pragma unroll
                for (int q = NP - 1; q >= 0; q--)
#pragma unroll
                    for (int b = 0; b < QB; b++)
                        O[b][j % 4] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(x[j], __builtin_bit_cast(bf16x8, P[b][q][j / 4]), O[b][j % 4], 0, 0, 0);
                if (j == 4) locate(t + 1 + NS);
            } else {
#pragma unroll
                for (int p = NQ - 1; p >= 0; p--) S[0] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(x[j], qr[p][j - 8], S[0], 0, 0, 0);
                if (QB == 2) S[QB - 1] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(x[j], y[j], S[QB - 1], 0, 0, 0);
            }
        }
    };
    // ---- The two waves of a SIMD (w and w + 4) are one phase apart: while one multiplies,
    // the other weighs.  In the phase in which a wave weighs step t it requests K of step t +
    // NS and V of step t + NS - 1, into the rows that its half multiplied in the phase
    // before; it waits for them by the end of the phase in which it weighs step t + NS - 1,
    // behind which they are multiplied.
    __builtin_amdgcn_s_waitcnt(0x0070);         // vmcnt(0), lgkmcnt(0)
    paged_meet();
    if (w >= 4) paged_meet();
    multiply(std::false_type{}, 0, vt[0], kt[0]);
    __builtin_amdgcn_s_waitcnt(0xC07F);         // lgkmcnt(0): this wave's reads are done
    paged_meet();
    int slot = 0;                               // t % NS
#pragma unroll 1
    for (int t = 0; t < nstep; t++) {
        weigh(t);
        const int before = slot ? slot - 1 : NS - 1, after = slot < NS - 1 ? slot + 1 : 0;
        if (t + NS < nstep && min(klim, vlim) == RW - 1) {
            request(yes, seq.v, false, vat, vlim, vt[before]);
            request(yes, seq.k, true, kat, klim, kt[slot]);
            static_assert((NS - 1) * LPS == 8, "the loads that may be on their way");
            __builtin_amdgcn_s_waitcnt(0x0078); // vmcnt(8), lgkmcnt(0)
        } else {
            if (t + NS <= nstep) request(no, seq.v, false, vat, vlim, vt[before]);
            if (t + NS < nstep) request(no, seq.k, true, kat, klim, kt[slot]);
            __builtin_amdgcn_s_waitcnt(0x0070);
        }
        paged_meet();
        multiply(std::true_type{}, t, vt[slot], kt[after]);     // (behind the last step: scores that nobody takes)
        __builtin_amdgcn_s_waitcnt(0xC07F);
        paged_meet();
        slot = after;
    }
    if (w < 4) paged_meet();

    // ---- the PS waves of each row group joined, 32 dimensions of 32 rows at a time
    float f[QB], inv[QB];
#pragma unroll
    for (int b = 0; b < QB; b++) {
        seen[b] |= all;
        l[b] += __shfl_xor(l[b], 32, JM_WAVE);
        if (h == 0) {
            mls[w][32 * b + n][0] = ref[b];
            mls[w][32 * b + n][1] = seen[b] ? l[b] : -1.0f;
        }
    }
    __syncthreads();
#pragma unroll
    for (int b = 0; b < QB; b++) {
        float M = -INFINITY, L = 0.0f;
        bool any = false;
#pragma unroll
        for (int q = 0; q < PS; q++) M = fmaxf(M, mls[q * RG + rg][32 * b + n][0]);
#pragma unroll
        for (int q = 0; q < PS; q++) {
            const float lq = mls[q * RG + rg][32 * b + n][1];
            if (lq == -1.0f) continue;
            any = true;
            L = __builtin_fmaf(lq, pow2f(mls[q * RG + rg][32 * b + n][0] - M), L);
        }
        f[b] = seen[b] ? pow2f(ref[b] - M) : 0.0f;
        inv[b] = any ? __fdiv_rn(1.0f, L) : 0.0f;                           // (as in k_paged_attn)
        if (a.S > 1) {
            inv[b] = 1.0f;
            float* const ml = a.part_ml + 2 * (((size_t)(u * c.KH + kh) * a.S + sr) * (a.qpk * a.tp) + 32 * (QB * rg + b) + n);
            if (ps == 0 && h == 0 && live[b]) *(float2*)ml = make_float2(M, any ? L : -1.0f);
        }
    }
    // of a row block's 4 pieces of 32 dimensions a wave keeps one in PS, which it finishes, and
    // hands the others on (piece nt of wave w at [w][which(nt)])
    constexpr int HAND = 4 - 4 / PS;
    auto which = [](int nt, int p) { return PS == 2 ? nt >> 1 : nt - (nt > p); };
    float4* const mb = (float4*)&kt[0][0] + lane;
    static_assert(8 * HAND * 4096 <= sizeof(kt) + sizeof(vt), "what the waves hand on fits");
#pragma unroll
    for (int b = 0; b < QB; b++) {
        if (b) __syncthreads();
#pragma unroll
        for (int nt = 0; nt < 4; nt++)
            if (nt % PS != ps)
#pragma unroll
                for (int q = 0; q < 4; q++)
                    mb[((w * HAND + which(nt, ps)) * 4 + q) * 64] = make_float4(O[b][nt][4 * q] * f[b], O[b][nt][4 * q + 1] * f[b],
                                                                                O[b][nt][4 * q + 2] * f[b], O[b][nt][4 * q + 3] * f[b]);
        __syncthreads();
#pragma unroll
        for (int nt = 0; nt < 4; nt++) {
            if (nt % PS != ps) continue;
#pragma unroll
            for (int q = 0; q < 4; q++) {
                float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
                for (int i = 1; i < PS; i++) {
                    const int p = (ps + i) % PS;
                    const float4 y = mb[(((p * RG + rg) * HAND + which(nt, p)) * 4 + q) * 64];
                    x = make_float4(x.x + y.x, x.y + y.y, x.z + y.z, x.w + y.w);
                }
                O[b][nt][4 * q] = (O[b][nt][4 * q] * f[b] + x.x) * inv[b];
                O[b][nt][4 * q + 1] = (O[b][nt][4 * q + 1] * f[b] + x.y) * inv[b];
                O[b][nt][4 * q + 2] = (O[b][nt][4 * q + 2] * f[b] + x.z) * inv[b];
                O[b][nt][4 * q + 3] = (O[b][nt][4 * q + 3] * f[b] + x.w) * inv[b];
            }
            const uint32_t* const tn = &taint[32 * (QB * rg + b) + n][2 * nt];
            if (__any(tn[0] | tn[1])) {
#pragma unroll
                for (int v = 0; v < 16; v++) {
                    // dimension 8 (v / 4) + 4 h + v % 4
                    const uint32_t x = tn[v / 8] >> (16 * (v / 4 % 2) + 8 * h + 2 * (v % 4)) & 3u;
                    const uint32_t bits = (x ? 0x7F800000u : 0u) | (x == 2u ? 0x80000000u : 0u) | (x == 3u ? 0x400000u : 0u);
                    O[b][nt][v] += __uint_as_float(bits);
                }
            }
        }
    }
    if (a.S > 1) {
#pragma unroll
        for (int b = 0; b < QB; b++)
#pragma unroll
            for (int nt = 0; nt < 4; nt++) {
                if (nt % PS != ps || !live[b]) continue;
                const size_t row = ((size_t)(u * c.KH + kh) * a.S + sr) * (a.qpk * a.tp) + 32 * (QB * rg + b) + n;
#pragma unroll
                for (int q = 0; q < 4; q++)
                    *(float4*)(a.part_o + row * HD + 32 * nt + 8 * q + 4 * h) =
                        make_float4(O[b][nt][4 * q], O[b][nt][4 * q + 1], O[b][nt][4 * q + 2], O[b][nt][4 * q + 3]);
            }
        return;
    }
    // the rows through LDS, so that they leave in whole lines: 16-byte chunk x of row r at x ^ (r
    // % 8), where each row goes in `to`
    constexpr int OB = BF ? 2 : 4, CH = HD * OB / 16;
    static_assert(NROW * HD * OB + NROW * 8 <= sizeof(kt) + sizeof(vt), "the rows fit");
    char* const rows = (char*)&kt[0][0];
    long long* const to = (long long*)(rows + NROW * HD * OB);
    __syncthreads();
#pragma unroll
    for (int b = 0; b < QB; b++) {
        const int r = 32 * (QB * rg + b) + n;
        if (ps == 0 && h == 0) to[r] = live[b] ? (long long)(un.tok + tok[b]) * a.H + head[b] : -1;
#pragma unroll
        for (int nt = 0; nt < 4; nt++) {
            if (nt % PS != ps) continue;
#pragma unroll
            for (int q = 0; q < 4; q++) {
                const float4 v = make_float4(O[b][nt][4 * q], O[b][nt][4 * q + 1], O[b][nt][4 * q + 2], O[b][nt][4 * q + 3]);
                const int x = BF ? 4 * nt + q : 8 * nt + 2 * q + h;
                store_out<BF>(rows + (size_t)r * HD * OB + 16 * (x ^ (r & 7)) + (BF ? 8 * h : 0), 0, v);
            }
        }
    }
    __syncthreads();
    for (int i = tid; i < NROW * CH; i += 512) {
        const int r = i / CH, x = i % CH;
        const long long row = to[r];
        if (row >= 0) {
            const uint4 v = *(const uint4*)(rows + (size_t)r * HD * OB + 16 * (x ^ (r & 7)));
            *(u32x4_a8*)((char*)a.out + (size_t)row * HD * OB + 16 * x) = u32x4_a8{v.x, v.y, v.z, v.w};
        }
    }
}

// The same over float32 pages, in float32 products (v_mfma_f32_16x16x4): block (KV head, unit
// of 32 query rows, range of the unit's rows), 8 waves = RG = 2 row groups of 16 x PS = 4
// position strides; a step is 64 rows, of which a wave takes 16.  The products are those of
// k_paged_attn, but for the dimensions of a lane's V: pieces m and m + 16 of a row.  Chunk x
// (16 bytes) of row r sits at x ^ (r % 16) in LDS.
//
// Bound by the float32 products (32 cycles each, 64 for a wave's 16 rows).  More position
// strides and fewer row groups win because a step's fixed part (barrier, staging, softmax) is
// shared by more rows, although each row read from memory serves fewer query rows: two prompts
// of 1021 tokens behind 260 rows, 16 heads: RG = 2 95 us, RG = 4 120, row groups only (2, 4,
// 8 waves) 146, 135, 135; k_paged_attn 126.
template <bool BF>
__global__ void __launch_bounds__(512, 2)
k_paged_tile_f32(PagedArgs c, PagedAttnArgs a) {
    constexpr int HD = 128, RG = 2, PS = 8 / RG, STEP = 16 * PS, RW = STEP / 8;
    __shared__ __align__(16) float kv[2][2][STEP * HD];     // [step % 2][K, V][row][dimension]
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int rg = w % RG, ps = w / RG, g = lane >> 4, n = lane & 15;
    const int kh = blockIdx.x % c.KH, rs = blockIdx.x / c.KH;
    const int u = a.units - 1 - rs % a.units, sr = rs / a.units;        // the longest prefixes first
    CallUnit un;
    if (!call_unit(c, u, a.tp, un)) return;
    const PagedSeq seq(c, un.seq, kh);
    const int pmax = min(un.pos + un.n - 1, c.maxT - 1);
    const int steps = pmax < 0 ? 0 : pmax / STEP + 1;
    const int step0 = (int)((long long)steps * sr / a.S), nstep = (int)((long long)steps * (sr + 1) / a.S) - step0;
    // this lane's query row, and the last cache row that it sees; of the wave's, the first
    // token and how many there are
    const int r = 16 * rg + n, ct = min(r / a.qpk, un.n - 1), head = kh * a.qpk + r % a.qpk;
    const int crow = min(un.pos + ct, c.maxT - 1);
    const bool live = r / a.qpk < un.n && un.pos + ct < c.maxT;
    const int wt0 = min(16 * rg / a.qpk, un.n - 1), wt1 = min((16 * rg + 15) / a.qpk, un.n - 1), wmin = min(un.pos + wt0, c.maxT - 1);

    // ---- staging: wave w has rows RW w .. of each step, 2 rows a load.  Lane PS i + g of `page`
    // has the page of 16-row group g in the i-th of 64 / PS steps.
    auto fetch = [&](int batch) __attribute__((always_inline)) {
        const long long row = (long long)(step0 + 64 / PS * batch) * STEP + 16 * lane;
        const int p = row <= pmax ? seq.table[row >> c.lp] : -1;
        return (unsigned)p < (unsigned)c.n_pages ? p : -1;
    };
    int page = fetch(0), next = fetch(1);
    bool has = false, had = false;              // whether this wave's group of the step staged last, and before, has a page
    auto stage = [&](int t, int slot) __attribute__((always_inline)) {
        const int i0 = t % (64 / PS) * PS;
        if (t && i0 == 0) {
            page = next;
            next = fetch(t / (64 / PS) + 1);
        }
        had = has;
        has = __builtin_amdgcn_readlane(page, i0 + ps) >= 0;
        const int p = __builtin_amdgcn_readlane(page, i0 + RW * w / 16), row = (step0 + t) * STEP + RW * w, lim = pmax - row;
        const size_t at = (size_t)max(p, 0) * c.page_stride + (uint32_t)((row & ((1 << c.lp) - 1)) * 512);
#pragma unroll
        for (int v = 0; v < 2; v++) {
            float* const to = kv[slot][v] + RW * w * HD;
            if (p >= 0 && lim >= 0) {
                uint32_t num = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(__attribute__((address_space(3))) void*)to);
                __asm__ volatile("" : "+s"(num));           // (as in k_paged_tile)
                const auto dst = (__attribute__((address_space(3))) float*)(uintptr_t)num;
                const auto base = __builtin_amdgcn_make_buffer_rsrc((void*)((v ? seq.v : seq.k) + at), 0, RW * 512, 0x00020000);
#pragma unroll
                for (int j = 0; j < RW / 2; j++) {
                    const int i = 2 * j + (lane >> 5);      // (rows past the prefixes repeat the last one)
                    __builtin_amdgcn_raw_ptr_buffer_load_lds(base, (__attribute__((address_space(3))) void*)(dst + 2 * j * HD), 16,
                                                             min(i, lim) * 512 + 16 * ((lane & 31) ^ ((RW * w + i) & 15)), 0, 0, 0);
                }
            } else if (v) {
#pragma unroll
                for (int j = 0; j < RW / 2; j++) *(float4*)(to + 2 * j * HD + 4 * lane) = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            }
        }
    };

    float qf[32];
    const size_t qi = (size_t)((un.tok + ct) * a.qts + head * a.qhs);
#pragma unroll
    for (int i = 0; i < 8; i++) {
        float y[4];
        load4<BF>(a.q, qi + 16 * i + 4 * g, y);
#pragma unroll
        for (int e = 0; e < 4; e++) qf[4 * i + e] = y[e];
    }
    if (nstep > 0) stage(0, 0);

    f32x4 O[8];
#pragma unroll
    for (int j = 0; j < 8; j++) O[j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    float ref = -INFINITY, l = 0.0f;
    int seen = 0;
#pragma unroll 1
    for (int t = 0; t < nstep; t++) {
        // this wave's rows of the step have arrived and its reads of the step before are done,
        // then everyone's
        __builtin_amdgcn_s_waitcnt(0x0070);
        wave_meet();
        if (t + 1 < nstep) stage(t + 1, (t + 1) & 1);
        const int row0 = (step0 + t) * STEP + 16 * ps;
        if ((t + 1 < nstep ? had : has) && row0 <= min(un.pos + wt1, c.maxT - 1)) {            // (wave-uniform)
            const float* const kt = kv[t & 1][0] + 16 * ps * HD;
            const float* const vt = kv[t & 1][1] + 16 * ps * HD;
            // ---- scores (lane (g, n): query row n at rows 4 i + g)
            f32x4 S = f32x4{0.0f, 0.0f, 0.0f, 0.0f}, S2 = S;
            int kr = 4 * (n & 3) + (n >> 2), gg = g;
            __asm__ volatile("" : "+v"(kr), "+v"(gg));      // (the addresses anew each time: kept, others spill)
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const float4 x = *(const float4*)(kt + kr * HD + 4 * ((4 * i + gg) ^ kr));
                S = __builtin_amdgcn_mfma_f32_16x16x4f32(x.x, qf[4 * i], S, 0, 0, 0);
                S2 = __builtin_amdgcn_mfma_f32_16x16x4f32(x.y, qf[4 * i + 1], S2, 0, 0, 0);
                S = __builtin_amdgcn_mfma_f32_16x16x4f32(x.z, qf[4 * i + 2], S, 0, 0, 0);
                S2 = __builtin_amdgcn_mfma_f32_16x16x4f32(x.w, qf[4 * i + 3], S2, 0, 0, 0);
            }
            float p[4];
            const bool whole = row0 + 15 <= wmin;
            seen |= (int)(row0 <= crow);
#pragma unroll
            for (int e = 0; e < 4; e++) {
                p[e] = __fmul_rn(S[e] + S2[e], a.scale2);
                if (!whole && row0 + 4 * e + g > crow) p[e] = -INFINITY;
            }
            // ---- the reference and the weights, as in k_paged_attn
            float m = fmaxf(fmaxf(p[0], p[1]), fmaxf(p[2], p[3]));
            if (__any(m > ref + 10.0f)) {
                m = fmaxf(m, swz_xor16_f(m));
                m = fmaxf(m, __shfl_xor(m, 32, JM_WAVE));
                const float nref = fmaxf(ref, m);
                const float f = nref == -INFINITY ? 1.0f : pow2f(ref - nref);
                l *= f;
#pragma unroll
                for (int j = 0; j < 8; j++) O[j] *= f;
                ref = nref;
            }
            const float r0 = ref == -INFINITY ? 0.0f : ref;
#pragma unroll
            for (int e = 0; e < 4; e++) {
                p[e] = pow2f(__fsub_rn(p[e], r0));
                l = __fadd_rn(l, p[e]);
            }
            // ---- P . V; token by token where some query row of the wave does not see a row
            // whose V is not finite
            uint32_t bad = 0;
            if (!whole) {
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const int vr = 4 * i + g;
#pragma unroll
                    for (int d = 0; d < 2; d++) {
                        const uint4 x = *(const uint4*)(vt + vr * HD + 4 * ((n + 16 * d) ^ vr));
                        const uint32_t y = (uint32_t)((x.x & 0x7F800000u) == 0x7F800000u) | (uint32_t)((x.y & 0x7F800000u) == 0x7F800000u) |
                                           (uint32_t)((x.z & 0x7F800000u) == 0x7F800000u) | (uint32_t)((x.w & 0x7F800000u) == 0x7F800000u);
                        bad |= row0 + vr > wmin ? y : 0u;
                    }
                }
            }
            if (!__any(bad != 0)) {
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const int vr = 4 * i + g;
#pragma unroll
                    for (int d = 0; d < 2; d++) {
                        const float4 x = *(const float4*)(vt + vr * HD + 4 * ((n + 16 * d) ^ vr));
                        O[4 * d] = __builtin_amdgcn_mfma_f32_16x16x4f32(x.x, p[i], O[4 * d], 0, 0, 0);
                        O[4 * d + 1] = __builtin_amdgcn_mfma_f32_16x16x4f32(x.y, p[i], O[4 * d + 1], 0, 0, 0);
                        O[4 * d + 2] = __builtin_amdgcn_mfma_f32_16x16x4f32(x.z, p[i], O[4 * d + 2], 0, 0, 0);
                        O[4 * d + 3] = __builtin_amdgcn_mfma_f32_16x16x4f32(x.w, p[i], O[4 * d + 3], 0, 0, 0);
                    }
                }
            } else {
#pragma unroll 1
                for (int tt = wt0; tt <= wt1; tt++) {
#pragma unroll
                    for (int j = 0; j < 8; j++) {
                        f32x4 T = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                        for (int i = 0; i < 4; i++) {
                            const int vr = 4 * i + g;
                            const float x = row0 + vr <= un.pos + tt ? vt[vr * HD + 4 * ((n + 16 * (j / 4)) ^ vr) + j % 4] : 0.0f;
                            T = __builtin_amdgcn_mfma_f32_16x16x4f32(x, ct == tt ? p[i] : 0.0f, T, 0, 0, 0);
                        }
#pragma unroll
                        for (int i = 0; i < 4; i++) O[j][i] = ct == tt ? O[j][i] + T[i] : O[j][i];
                    }
                }
            }
        }
    }

    // ---- the PS waves of each row group joined by the first of them
    l += swz_xor16_f(l);
    l += __shfl_xor(l, 32, JM_WAVE);
    __shared__ float mls[8][16][2];
    float4* const ow = (float4*)&kv[0][0][0] + lane;        // [wave, those of ps = 0 left out][8][64 lanes]
    static_assert((8 - RG) * 8 * 64 * 16 <= sizeof(kv), "the outputs of the others fit");
    __syncthreads();
    if (g == 0) {
        mls[w][n][0] = ref;
        mls[w][n][1] = seen ? l : -1.0f;
    }
    if (ps) {
#pragma unroll
        for (int j = 0; j < 8; j++) ow[((w - RG) * 8 + j) * 64] = make_float4(O[j][0], O[j][1], O[j][2], O[j][3]);
    }
    __syncthreads();
    if (ps || !live) return;
    float M = -INFINITY, L = 0.0f;
    bool any = false;
#pragma unroll
    for (int q = 0; q < PS; q++) M = fmaxf(M, mls[q * RG + rg][n][0]);
    const float f0 = seen ? pow2f(ref - M) : 0.0f;
#pragma unroll
    for (int j = 0; j < 8; j++) O[j] *= f0;
#pragma unroll
    for (int q = 0; q < PS; q++) {
        const float lq = mls[q * RG + rg][n][1];
        if (lq == -1.0f) continue;
        any = true;
        const float f = pow2f(mls[q * RG + rg][n][0] - M);
        L = __builtin_fmaf(lq, f, L);
        if (q == 0) continue;
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const float4 x = ow[((q * RG + rg - RG) * 8 + j) * 64];
            O[j] += f32x4{x.x, x.y, x.z, x.w} * f;
        }
    }
    // dimensions 64 d + 16 g + 4 i + e (register i of product 4 d + e) of the lane's query row
    const float inv = a.S > 1 ? 1.0f : any ? __fdiv_rn(1.0f, L) : 0.0f;         // (as in k_paged_attn)
    const size_t row = ((size_t)(u * c.KH + kh) * a.S + sr) * (a.qpk * a.tp) + r;
    if (a.S > 1 && g == 0) *(float2*)(a.part_ml + 2 * row) = make_float2(M, any ? L : -1.0f);
    const size_t oi = ((size_t)(un.tok + ct) * a.H + head) * HD;
#pragma unroll
    for (int d = 0; d < 2; d++)
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float4 v = make_float4(O[4 * d][i] * inv, O[4 * d + 1][i] * inv, O[4 * d + 2][i] * inv, O[4 * d + 3][i] * inv);
            const int dim = 64 * d + 16 * g + 4 * i;
            if (a.S > 1) *(float4*)(a.part_o + row * HD + dim) = v;
            else store_out<BF>(a.out, oi + dim, v);
        }
}

// How a call is cut, by sizes and types alone: the host does not know cu, and takes the
// tokens as spread evenly over all sequences, idle ones too.  What that costs where they are
// not (bf16): 2047 tokens behind 4099 rows take 243 us alone and in a set of up to 128
// sequences, 979 in one of 256, where k_paged_attn gets them; 512 tokens 81 alone, 99 in a set
// of 64, 173 from 128 on.  A prompt of 2048 (80) beside 63 single tokens behind 16000 rows
// (611) 1340, as each of those goes through the tiles.
//
// Times are of 32 query heads on 8 KV heads, "T tokens behind R rows, B sequences" (us).
//
// Which kernel: a block of k_paged_attn has 16 query rows, so that the cache is multiplied
// once for each 16, but is done in 8 us; k_paged_tile takes 15 us to begin and end.  The
// blocks times their rows (512 at least) decide.  bf16 q and pages, k_paged_attn /
// k_paged_tile: 64 tokens behind 2000 rows (264 k) 21 / 31, 2 such sequences (528 k) 28 / 34,
// 600 behind none (614 k) 28 / 28, 40 behind 2000, 4 sequences (653 k) 44 / 34, 700 behind
// none (717 k) 34 / 32, 16 behind 2000, 16 sequences (1 M) 62 / 52.  float32 q over bf16
// pages: 100 behind 2000 (420 k) 29 / 29, 400 behind none (410 k) 25 / 23, 200 behind 1000 (480
// k) 33 / 30, 16 behind 2000, 16 sequences (1 M) 76 / 46.  float32 pages, k_paged_attn /
// k_paged_tile_f32: 16 behind 2000 (64 k) 21 / 23, 32 behind 2000 (130 k) 27 / 24, 8 behind
// 2000, 4 sequences (128 k) 49 / 27, 16 sequences of 16 (1 M) 162 / 120.
//
// (A sequence with 17 query rows over float32 pages, the second unit of k_paged_attn, goes to
// the tiles: 5 tokens behind 4000 rows, 8 sequences 94 / 75.)
//
// Units and ranges of the tiles, by what they take: a step (2.5 us at most), a block's beginning
// and end 6 steps, 256 blocks at once, the longest prefix bounding all; joined ranges 2 steps
// and what their partial outputs are to move.  661 tokens behind 3761 float32 rows, 2
// sequences of 4 heads on one 142 us (468 blocks of a third of the rows), 209 (156 blocks).
// RG 2 reads the cache twice as often as RG 4: it has to be a tenth below.  RG 4 / RG 2: 777
// tokens behind none 41 / 34, 800 behind 2000 75 / 67, 2047 behind none 80 / 75, 2047 behind
// 4099 236 / 247, 4 sequences of 300 behind 500 43 / 59, of 700 94 / 105, 5 of 1201 (28 heads on
// 4) 120 / 166.  512 rows a range at least against 256: 300 tokens behind 1000 rows 37 / 37, 150
// behind 2000 34 / 33; of float32 pages 32 behind 2000 35 / 26.
//
// Ranges of k_paged_attn: a block of each CU in turn, each as long as its rows and 160 more; a
// quarter of a block behind the last, as the prefixes differ; joining them 750 rows (of
// float32, which take twice as long, 200).  One token: 500 rows 8.9 (one range) / 11.5 (four),
// 1000 rows 13.2 / 11.4, of float32 300 rows 16.6 / 12.3; 1000 rows of 32 sequences 23 / 27
// (two), 1500 of 40 53 / 46 (three); 3000 of 12 31 (five: 480 blocks), 35 (six), 33 (ten); up
// to 2048 float32 rows of 8 sequences on 4 heads 24 (eight: 256 blocks) / 31 (nine).
PagedPlan paged_plan(const PagedArgs& c, int H, bool bf, int rows) {
    PagedPlan p{};
    const int qpk = H / c.KH;
    rows = std::min(rows, c.maxT);
    const long long qrows = (long long)c.N * qpk, each = c.cu && c.n_seq ? ((long long)c.N + c.n_seq - 1) / c.n_seq : 1;
    long long likely = 0;
    // units of tp tokens: every sequence's tokens are rounded up to whole ones; `likely`
    // blocks where the sequences have about as many each
    auto cut = [&](int tp) {
        p.tp = tp;
        p.units = c.cu ? (int)std::min<long long>(c.N, ((long long)c.N + (long long)c.n_seq * (tp - 1)) / tp) : c.N;
        likely = std::min<long long>(p.units, c.n_seq * ((each + tp - 1) / tp)) * c.KH;
    };
    // ranges of at least `least` rows for up to `want` blocks
    auto ranges = [&](int want, int least) {
        return (int)std::max(std::min(want / likely, ((long long)rows + least - 1) / least), 1ll);
    };
    cut(c.cu ? 16 / qpk : 1);
    if (likely == 0) return p;
    if (c.cu && qrows >= (c.f32 ? 17ll : 32ll) * c.n_seq && likely * std::max(rows, 512) >= (c.f32 ? 100000 : bf ? 620000 : 450000)) {
        // the cut into units of tp tokens and steps of `step` rows: what it takes, in steps
        auto tiles = [&](int tp, int step, int least) {
            long long best = LLONG_MAX;
            cut(tp);
            for (int k = 0; k <= 4; k++) {                  // (as many ranges as fit k rounds; one)
                const long long S = k ? ranges(256 * k, least) : 1;
                const long long most = rows / step / S + 6, mean = std::max(rows - each / 2, 0ll) / step / S + 6;
                const long long all = std::max(most, (likely * S + 255) / 256 * mean) + (S > 1 ? 2 + c.N * S * H / 8192 : 0);
                if (all < best) {
                    best = all;
                    p.S = (int)S;
                }
            }
            return best;
        };
        if (c.f32) {
            p.rg = 1;
            tiles(32 / qpk, 64, 256);
        } else {
            const int tp = (bf ? 64 : 32) * 2 / qpk;
            const long long two = tiles(tp, 128, 512), four = tiles(2 * tp, 64, 512);
            p.rg = 4;
            if (10 * two < 9 * four) {
                p.rg = 2;
                tiles(tp, 128, 512);
            }
        }
    } else {
        // what S ranges take, in rows that a block passes over, times 4
        auto cost = [&](long long S) {
            return (4 * ((likely * S + 255) / 256) + 1) * ((rows + S - 1) / S + 160) + (S == 1 ? 0 : c.f32 ? 800 : 3000);
        };
        p.S = 1;
        for (int k = 1; k <= 8; k++) {                      // (as many ranges as fit k rounds)
            const int S = ranges(256 * k, 128);
            if (cost(S) < cost(p.S)) p.S = S;
        }
    }
    const size_t cols = (size_t)p.units * c.KH * p.S * qpk * p.tp;
    p.o_floats = p.S > 1 ? cols * 128 : 0;
    p.ml_floats = p.S > 1 ? cols * 2 : 0;
    return p;
}

hipError_t launch_paged_attn(const PagedArgs& c, const PagedPlan& p, const void* q, bool bf, long long qts, long long qhs,
                             int H, float scale, void* out, float* part_o, float* part_ml, hipStream_t st) {
    if (c.N == 0) return hipSuccess;
    PagedAttnArgs a{};
    a.q = q; a.qts = qts; a.qhs = qhs; a.H = H; a.qpk = H / c.KH; a.tp = p.tp;
    a.scale2 = scale * 1.4426950408889634f;
    a.out = out; a.units = p.units; a.S = p.S; a.part_o = part_o; a.part_ml = part_ml;
    const dim3 grid((unsigned)c.KH * p.units * p.S);
    if (p.rg == 1) {
        if (bf) hipLaunchKernelGGL(k_paged_tile_f32<true>, grid, dim3(512), 0, st, c, a);
        else hipLaunchKernelGGL(k_paged_tile_f32<false>, grid, dim3(512), 0, st, c, a);
    } else if (p.rg) {
#define JM_PAGED_TILE(BFV, RGV) \
        if (bf == BFV && p.rg == RGV) hipLaunchKernelGGL((k_paged_tile<BFV, RGV>), grid, dim3(512), 0, st, c, a)
        JM_PAGED_TILE(false, 2); else JM_PAGED_TILE(false, 4); else JM_PAGED_TILE(true, 2); else JM_PAGED_TILE(true, 4);
#undef JM_PAGED_TILE
    } else {
#define JM_PAGED(F32V, BFV) \
        if ((c.f32 != 0) == F32V && bf == BFV) hipLaunchKernelGGL((k_paged_attn<F32V, BFV>), grid, dim3(64 * PAGED_W), 0, st, c, a)
        JM_PAGED(false, false); else JM_PAGED(false, true); else JM_PAGED(true, false); else JM_PAGED(true, true);
#undef JM_PAGED
    }
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || p.S == 1) return e;
    // (few ranges: more groups a row only leave lanes without work; 32 tokens behind 2000 rows,
    // 16 sequences in 2 ranges 53 us against 78.  Many: 64 ranges of one token 12.8 against 17.)
    const bool apart = p.S < 16;
    const int nc = a.qpk * a.tp;
    const dim3 mg((unsigned)c.KH * p.units * (unsigned)(apart ? (nc + 7) / 8 : nc));
#define JM_PAGED_MERGE(BFV, GV) hipLaunchKernelGGL((k_paged_merge<BFV, GV>), mg, dim3(256), 0, st, c, a)
    if (bf) { if (apart) JM_PAGED_MERGE(true, 1); else JM_PAGED_MERGE(true, 8); }
    else { if (apart) JM_PAGED_MERGE(false, 1); else JM_PAGED_MERGE(false, 8); }
#undef JM_PAGED_MERGE
    return hipGetLastError();
}

}  // namespace jm
