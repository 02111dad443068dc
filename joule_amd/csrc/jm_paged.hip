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
// apart), 16 heads of one token a block: q heads, then k heads, then v heads.
template <bool BF>
__global__ void __launch_bounds__(256)
k_paged_append(PagedArgs c, PagedRows r, int chunks) {
    constexpr int HD = 128;
    const int t = blockIdx.x / chunks, hr = blockIdx.x % chunks * 16 + (threadIdx.x >> 4);
    const int j = threadIdx.x & 15;
    int seq, pos;
    if (!call_place(c, t, seq, pos)) return;                // (block-uniform)
    if (hr >= r.H + 2 * c.KH) return;                       // (whole rows of 16 lanes)
    const int what = hr < r.H ? 0 : hr < r.H + c.KH ? 1 : 2;
    const int head = what == 0 ? hr : what == 1 ? hr - r.H : hr - r.H - c.KH;
    float x[8];
    load8<BF>(r.x[what], (size_t)(t * r.ts[what] + head * r.hs[what]) + 8 * j, x);
    const uint16_t* w = what < 2 ? r.w[what] : nullptr;
    if (w) {
        const uint4 u = *(const uint4*)(w + 8 * j);
        const uint32_t ww[4] = {u.x, u.y, u.z, u.w};
        float ss = 0.0f;
#pragma unroll
        for (int e = 0; e < 8; e++) ss = __builtin_fmaf(x[e], x[e], ss);
        ss = seg_sum<16>(ss);
        const float inv = __fdiv_rn(1.0f, __fsqrt_rn(__fadd_rn(ss * (1.0f / HD), r.eps)));
#pragma unroll
        for (int e = 0; e < 4; e++) {
            x[2 * e] = x[2 * e] * inv * __uint_as_float(ww[e] << 16);
            x[2 * e + 1] = x[2 * e + 1] * inv * __uint_as_float(ww[e] & 0xFFFF0000u);
        }
    }
    if (r.cos && what < 2) {
        const size_t at = (size_t)pos * HD + 8 * j;
        float cs[8], sn[8];
        load8<false>(r.cos, at, cs);
        load8<false>(r.sin, at, sn);
        float y[8];
#pragma unroll
        for (int e = 0; e < 8; e++) y[e] = dpp_f<DPP_ROR8>(x[e]);
#pragma unroll
        for (int e = 0; e < 8; e++) x[e] = __builtin_fmaf(j < 8 ? -y[e] : y[e], sn[e], x[e] * cs[e]);
    }
    if (what == 0) {
        store8<BF>(r.q_out, ((size_t)t * r.H + head) * HD + 8 * j, x);
        return;
    }
    const int page = c.table[seq * c.table_stride + (pos >> c.lp)];
    if ((unsigned)page >= (unsigned)c.n_pages) return;
    char* const base = (char*)(what == 1 ? c.k : c.v) + (size_t)page * c.page_stride;
    const size_t at = (((size_t)head << c.lp) + (pos & ((1 << c.lp) - 1))) * HD + 8 * j;
    if (c.f32) store8<false>(base, at, x);
    else store8<true>(base, at, x);
}

hipError_t launch_paged_append(const PagedArgs& c, const PagedRows& r, hipStream_t st) {
    if (c.N == 0) return hipSuccess;
    const int chunks = (r.H + 2 * c.KH + 15) / 16;
    const dim3 grid((unsigned)((long long)c.N * chunks));
    if (r.bf) hipLaunchKernelGGL(k_paged_append<true>, grid, dim3(256), 0, st, c, r, chunks);
    else hipLaunchKernelGGL(k_paged_append<false>, grid, dim3(256), 0, st, c, r, chunks);
    return hipGetLastError();
}

// ------------------------------------------------------- few query tokens
//
// Block (KV head, unit of up to 16 query rows: tokens x heads of the KV head, range of
// the unit's rows), W waves that take the range's tiles in turn, with a softmax each,
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

// A tile as a lane gets it.
struct PagedRegs {
    u32x4_t k[8], v[8];
};

template <bool F32>
__device__ __forceinline__ void paged_load(const PagedSeq& s, const PagedTile<F32 ? 1 : 2>& x, PagedRegs& r) {
    constexpr int ROWB = F32 ? 512 : 256;
    const int lane = threadIdx.x & 63, g = lane >> 4, n = lane & 15;
    if (!x.live) return;
    if (F32) {
        const gptr<const char> k = (gptr<const char>)(s.k + x.at[0]), v = (gptr<const char>)(s.v + x.at[0]);
        const uint32_t kr = (uint32_t)min(4 * (n & 3) + (n >> 2), x.lim[0]) * ROWB + 16 * g;
#pragma unroll
        for (int i = 0; i < 8; i++) r.k[i] = __builtin_nontemporal_load((gptr<const u32x4_t>)(k + kr + 64 * i));
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const uint32_t vr = (uint32_t)min(4 * i + g, x.lim[0]) * ROWB + 32 * n;
            r.v[2 * i] = __builtin_nontemporal_load((gptr<const u32x4_t>)(v + vr));
            r.v[2 * i + 1] = __builtin_nontemporal_load((gptr<const u32x4_t>)(v + vr + 16));
        }
    } else {
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const gptr<const char> k = (gptr<const char>)(s.k + x.at[F32 ? 0 : h]), v = (gptr<const char>)(s.v + x.at[F32 ? 0 : h]);
            const int lim = x.lim[F32 ? 0 : h];
            const uint32_t kr = (uint32_t)min(4 * (n & 3) + (n >> 2), lim) * ROWB + 16 * g;
#pragma unroll
            for (int i = 0; i < 4; i++) r.k[4 * h + i] = __builtin_nontemporal_load((gptr<const u32x4_t>)(k + kr + 64 * i));
#pragma unroll
            for (int i = 0; i < 4; i++)
                r.v[4 * h + i] = __builtin_nontemporal_load((gptr<const u32x4_t>)(v + ((uint32_t)min(4 * i + g, lim) * ROWB + 16 * n)));
        }
    }
}

// O[j] += V^T's product j times the weights p of the lane's rows.
template <bool F32, int NP>
__device__ __forceinline__ void paged_pv(const u32x4_t (&v)[8], const float (&p)[8], f32x4 (&O)[8]) {
    if (F32) {
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
            for (int j = 0; j < 8; j++)
                O[j] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(v[2 * i + j / 4][j % 4]), p[i], O[j], 0, 0, 0);
    } else {
        uint32_t w[NP][4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            uint32_t x[NP];
            parts_bf16<NP>(p[2 * i], p[2 * i + 1], x);
#pragma unroll
            for (int k = 0; k < NP; k++) w[k][i] = x[k];
        }
#pragma unroll
        for (int j = 0; j < 8; j++) {
            uint32_t a[4];
#pragma unroll
            for (int i = 0; i < 4; i++)
                a[i] = __builtin_amdgcn_perm(v[2 * i + 1][j / 2], v[2 * i][j / 2], j & 1 ? 0x07060302u : 0x05040100u);
            const bf16x8 x = as_bf16x8(a[0], a[1], a[2], a[3]);
#pragma unroll
            for (int k = NP - 1; k >= 0; k--)
                O[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x, as_bf16x8(w[k][0], w[k][1], w[k][2], w[k][3]), O[j], 0, 0, 0);
        }
    }
}

constexpr int PAGED_OW = 132;               // floats between the columns of a wave's outputs in LDS

// The query rows of one unit over tiles t0 .. t_end - 1 of its sequence; the waves joined,
// and the output, or (several ranges) the partial outputs.
template <bool F32, bool BF, int W>
__global__ void __launch_bounds__(64 * W, W >= 8 ? 1 : 2)
k_paged_attn(PagedArgs c, PagedAttnArgs a) {
    constexpr int HD = 128, NG = F32 ? 1 : 2, TR = 16 * NG, NY = 4 * NG;
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
    PagedRegs cur, nxt;
    x.live = false;
    if (mine) {
        walk.tile(0, x);
        paged_load<F32>(seq, x, cur);
    }

    // the query columns
    const size_t qi = (size_t)((un.tok + ct) * a.qts + head * a.qhs);
    float qf[F32 ? 32 : 1];
    bf16x8 qb[F32 ? 1 : NQ][4];
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
            uint32_t b[NQ][4];
#pragma unroll
            for (int e = 0; e < 4; e++) {
                uint32_t p[NQ];
                parts_bf16<NQ>(y[2 * e], y[2 * e + 1], p);
#pragma unroll
                for (int k = 0; k < NQ; k++) b[k][e] = p[k];
            }
#pragma unroll
            for (int k = 0; k < NQ; k++) qb[k][st] = as_bf16x8(b[k][0], b[k][1], b[k][2], b[k][3]);
        }
    }

    f32x4 O[8];
#pragma unroll
    for (int j = 0; j < 8; j++) O[j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    float ref = -INFINITY, l = 0.0f;
    bool seen = false;

    for (int i = 0; i < mine; i++) {
        if (i + 1 < mine) {
            walk.tile(i + 1, xn);
            paged_load<F32>(seq, xn, nxt);
        }
        if (x.live) {
            const int row0 = (t0 + w + i * W) * TR;
            // ---- scores
            float y[8];
#pragma unroll
            for (int h = 0; h < NG; h++) {
                f32x4 S = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
                if constexpr (F32) {
                    f32x4 S2 = S;
#pragma unroll
                    for (int k = 0; k < 32; k += 2) {
                        S = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(cur.k[k / 4][k % 4]), qf[k], S, 0, 0, 0);
                        S2 = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(cur.k[k / 4][k % 4 + 1]), qf[k + 1], S2, 0, 0, 0);
                    }
                    S += S2;
                } else {
#pragma unroll
                    for (int k = NQ - 1; k >= 0; k--)
#pragma unroll
                        for (int st = 0; st < 4; st++)
                            S = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, cur.k[4 * h + st]), qb[k][st], S, 0, 0, 0);
                }
#pragma unroll
                for (int e = 0; e < 4; e++) y[4 * h + e] = __fmul_rn(S[e], a.scale2);
            }
            // rows that the column does not see: past its own, or without a page
            bool whole = row0 + TR - 1 <= un.pos;
#pragma unroll
            for (int h = 0; h < NG; h++) {
                whole &= x.ok[h];
                seen |= x.ok[h] && row0 + 16 * h <= crow;
            }
            if (!whole) {
#pragma unroll
                for (int e = 0; e < NY; e++)
                    if (!x.ok[e / 4] || row0 + 16 * (e / 4) + 4 * (e % 4) + g > crow) y[e] = -INFINITY;
            }
            // ---- the reference: raised to the largest score when one passes it by 2^10
            float ym = y[0];
#pragma unroll
            for (int e = 1; e < NY; e++) ym = fmaxf(ym, y[e]);
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
            const float r0 = ref == -INFINITY ? 0.0f : ref;     // (a column that has seen nothing yet)
            float p[8];
#pragma unroll
            for (int e = 0; e < NY; e++) {
                p[e] = pow2f(__fsub_rn(y[e], r0));
                l = __fadd_rn(l, p[e]);
            }
            // ---- P . V.  A weight of 0 does not hide a value that is not finite: where
            // some column does not see such a row, token by token, each with the rows that
            // it sees.
            bool apart = false;
            auto row_of = [&](int e) __attribute__((always_inline)) {       // of v[e]; a group without a page holds another's
                const int h = F32 ? 0 : e / 4;
                return x.ok[h] ? row0 + 16 * h + 4 * (F32 ? e / 2 : e % 4) + g : INT_MAX;
            };
            if (!whole && un.n > 1) {
                uint32_t bad = 0;
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    uint32_t b = 0;
#pragma unroll
                    for (int d = 0; d < 4; d++) {
                        b |= (cur.v[e][d] & 0x7F800000u) == 0x7F800000u;
                        if (!F32) b |= (cur.v[e][d] & 0x7F80u) == 0x7F80u;
                    }
                    bad |= row_of(e) > un.pos ? b : 0u;
                }
                apart = __any(bad != 0);
            }
            if (!apart) {
                paged_pv<F32, NP>(cur.v, p, O);
            } else {
#pragma unroll 1
                for (int t = 0; t < un.n; t++) {
                    u32x4_t v[8];
                    float pt[8];
                    f32x4 T[8];
#pragma unroll
                    for (int e = 0; e < 8; e++) {
                        v[e] = row_of(e) <= un.pos + t ? cur.v[e] : u32x4_t{0u, 0u, 0u, 0u};
                        T[e] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
                        if (e < NY) pt[e] = ct == t ? p[e] : 0.0f;
                    }
                    paged_pv<F32, NP>(v, pt, T);
#pragma unroll
                    for (int j = 0; j < 8; j++)
                        if (ct == t) O[j] += T[j];
                }
            }
        }
        x = xn;
        cur = nxt;
    }

    // ---- the wave's outputs: dimensions 32 g + 8 i + j of column n
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

// The ranges of one (unit, KV head, query row) joined into the output: 8 groups of 32
// lanes take the ranges in turn, 4 dimensions a lane, and are added in order.
template <bool BF>
__global__ void __launch_bounds__(256)
k_paged_merge(PagedArgs c, PagedAttnArgs a) {
    constexpr int HD = 128;
    __shared__ __align__(16) float4 acc[8][32];
    __shared__ float ls[8];
    const int nc = a.qpk * a.tp;
    const int kh = blockIdx.x % c.KH, oc = blockIdx.x / c.KH % nc, u = blockIdx.x / c.KH / nc;
    CallUnit un;
    if (!call_unit(c, u, a.tp, un)) return;
    const int to = oc / a.qpk;
    if (to >= un.n || un.pos + to >= c.maxT) return;        // (block-uniform)
    const size_t p0 = ((size_t)u * c.KH + kh) * a.S * nc + oc;
    const int j = threadIdx.x & 31, gr = threadIdx.x >> 5;
    float M = -INFINITY;
    bool any = false;
    for (int s = j; s < a.S; s += 32) {
        const float2 x = *(const float2*)(a.part_ml + 2 * (p0 + (size_t)s * nc));
        M = fmaxf(M, x.x);
        any |= x.y != -1.0f;
    }
    M = seg_max<32>(M);
    any = __any(any);
    float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    float L = 0.0f;
    for (int s0 = gr; s0 < a.S; s0 += 32) {
        float4 x[4];
        float2 ml[4];
#pragma unroll
        for (int q = 0; q < 4; q++) {
            const size_t p = p0 + (size_t)min(s0 + 8 * q, a.S - 1) * nc;
            ml[q] = *(const float2*)(a.part_ml + 2 * p);
            x[q] = *(const float4*)(a.part_o + p * HD + 4 * j);
        }
#pragma unroll
        for (int q = 0; q < 4; q++) {
            if (s0 + 8 * q >= a.S || ml[q].y == -1.0f) continue;       // (a range without a row has no output)
            const float f = pow2f(ml[q].x - M);
            v.x = __builtin_fmaf(x[q].x, f, v.x);
            v.y = __builtin_fmaf(x[q].y, f, v.y);
            v.z = __builtin_fmaf(x[q].z, f, v.z);
            v.w = __builtin_fmaf(x[q].w, f, v.w);
            L = __builtin_fmaf(ml[q].y, f, L);
        }
    }
    acc[gr][j] = v;
    if (j == 0) ls[gr] = L;
    __syncthreads();
    if (gr) return;
#pragma unroll
    for (int i = 1; i < 8; i++) {
        const float4 y = acc[i][j];
        v = make_float4(v.x + y.x, v.y + y.y, v.z + y.z, v.w + y.w);
        L += ls[i];
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
// straight to LDS (global_load_lds), the steps after it on their way.
//
//   scores   v_mfma_f32_32x32x16_bf16, cache rows as A (lane l: row l % 32, dimensions 16
//            kk + 8 (l / 32) ..), query rows as B: lane l holds query row l % 32 at cache
//            rows 8 (v / 4) + 4 (l / 32) + v % 4
//   P . V    V^T as A, read transposed from LDS (ds_read_b64_tr_b16: 4 rows of 16
//            dimensions), the weights as B from the registers that formed them:
//            contraction index j of half h in step s is row 16 s + 8 (j / 4) + 4 h + j % 4
//
// bf16 queries (BF): 64 query rows a wave (QB = 2), so that an operand read from LDS serves
// two products; q is exact, a weight is rounded to bf16 once, and the sum is of the
// rounded weights, so that the output stays a mean of values of V.  float32 queries: q and
// the weights as three bf16 parts each, as in k_paged_attn.

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

// 4 rows x 16 columns of bf16 in LDS, transposed over 16 lanes: lane i gives the address
// of 4 columns (4 (i % 4) ..) of row i / 4 and receives column i of rows 0 .. 3
__device__ __forceinline__ s16x4 paged_tr16(const uint16_t* p) {
    return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(void*)p);
}

#ifndef PAGED_AHEAD
#define PAGED_AHEAD 2
#endif
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
    constexpr int HD = 128, QB = BF ? 2 : 1, NQ = BF ? 1 : 3, PS = 8 / RG, STEP = 32 * PS, TILE = 32 * HD;
    constexpr int RW = 8 * (PS / 2);            // rows of a step that a wave stages, of K and of V
    constexpr int LPS = RW / 2;                 // its loads, 4 rows each
    constexpr int NROW = 32 * QB * RG, AHEAD = PAGED_AHEAD;
    constexpr int NS = PS == 2 ? 3 : 2;         // steps in LDS
    // PS tiles of K and of V of NS steps; at the end the outputs being joined
    __shared__ __align__(16) uint16_t kv[2][NS][PS * TILE];
    auto& kt = kv[0];
    auto& vt = kv[1];
    // the second block of query rows of each row group (BF)
    __shared__ __align__(16) uint4 q1[BF ? RG : 1][8][64];
    __shared__ float mls[8][32 * QB][2];
    __shared__ uint8_t okf[NS][2 * PS];          // whether a step's 16-row groups have pages
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

    // ---- the query rows, with the score scale's sign (a scale of 0, or a smaller one, as
    // 2^-100: masked scores stay -inf behind it)
    const float cs = fmaxf(fabsf(a.scale2), 0x1p-100f);
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
    u32x4_t P[QB][NQ][2];
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
            uint32_t p[NQ];
            parts_bf16<NQ>(x0, x1, p);
#pragma unroll
            for (int q = 0; q < NQ; q++) P[b][q][s][e] = p[q];
            if (BF) l[b] = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2_t, p[0]), __builtin_bit_cast(bf16x2_t, 0x3F803F80u), l[b], false);
            else l[b] += x0 + x1;
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
            for (int q = 0; q < NQ; q++) __asm__ volatile("" : "+v"(P[b][q][0]), "+v"(P[b][q][1]));
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
                for (int b = 0; b < QB; b++)
#pragma unroll
                    for (int q = NQ - 1; q >= 0; q--)
                        O[b][j % 4] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(x[j], __builtin_bit_cast(bf16x8, P[b][q][j / 4]), O[b][j % 4], 0, 0, 0);
                if (j == 4) locate(t + 1 + NS);
            } else {
#pragma unroll
                for (int p = NQ - 1; p >= 0; p--) S[0] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(x[j], qr[p][j - 8], S[0], 0, 0, 0);
                if (QB == 2) S[QB - 1] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(x[j], y[j], S[QB - 1], 0, 0, 0);
            }
        }
    };
    // ---- the vector work of a phase: the weights of step t
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

PagedPlan paged_plan(const PagedArgs& c, int H, bool bf, int rows) {
    PagedPlan p{};
    const int qpk = H / c.KH;
    rows = std::min(rows, c.maxT);
    long long blocks;
    auto cut = [&](int tp) {
        p.tp = tp;
        // (every sequence's tokens are rounded up to whole units)
        p.units = c.cu ? (int)std::min<long long>(c.N, ((long long)c.N + (long long)c.n_seq * (tp - 1)) / tp) : c.N;
        blocks = (long long)p.units * c.KH;
    };
    // up to `want` blocks while each has `least` rows
    auto ranges = [&](long long want, int least) {
        return std::min((want + blocks - 1) / blocks, ((long long)rows + least - 1) / least);
    };
    const long long qrows = (long long)c.N * qpk;
    if (!c.f32 && c.cu && qrows >= 64ll * c.n_seq) {
        const int unit = bf ? 256 : 128;
        p.rg = 4;
        cut(unit / qpk);
        if (qrows < (long long)unit * c.n_seq || (blocks < 256 && blocks * rows < 160000)) {
            p.rg = 2;
            cut(unit / 2 / qpk);
        }
        p.S = (int)std::max(std::min(256 / blocks, ((long long)rows + 255) / 256), 1ll);
    } else {
        cut(c.cu ? 16 / qpk : 1);
        p.S = rows <= 1024 ? 1 : (int)std::max(std::max(ranges(256, 128), ranges(1024, 512)), 1ll);
    }
    const size_t cols = (size_t)blocks * p.S * qpk * p.tp;
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
    if (p.rg) {
#define JM_PAGED_TILE(BFV, RGV) \
        if (bf == BFV && p.rg == RGV) hipLaunchKernelGGL((k_paged_tile<BFV, RGV>), grid, dim3(512), 0, st, c, a)
        JM_PAGED_TILE(false, 2); else JM_PAGED_TILE(false, 4); else JM_PAGED_TILE(true, 2); else JM_PAGED_TILE(true, 4);
#undef JM_PAGED_TILE
    } else {
#define JM_PAGED(F32V, BFV) \
        if ((c.f32 != 0) == F32V && bf == BFV) hipLaunchKernelGGL((k_paged_attn<F32V, BFV, 4>), grid, dim3(256), 0, st, c, a)
        JM_PAGED(false, false); else JM_PAGED(false, true); else JM_PAGED(true, false); else JM_PAGED(true, true);
#undef JM_PAGED
    }
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || p.S == 1) return e;
    const dim3 mg((unsigned)c.KH * p.units * (unsigned)(a.qpk * a.tp));
    if (bf) hipLaunchKernelGGL(k_paged_merge<true>, mg, dim3(256), 0, st, c, a);
    else hipLaunchKernelGGL(k_paged_merge<false>, mg, dim3(256), 0, st, c, a);
    return hipGetLastError();
}

}  // namespace jm
