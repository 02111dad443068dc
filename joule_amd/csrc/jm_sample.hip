// Sampling of the next token (jm_sample): temperature, top-k, top-p and min-p
// from one random number a row.
//
// Every filter keeps a prefix of the tokens in the order (logit descending,
// index ascending), so that the kept set is the shortest of three prefixes and
// all that is ever needed is "the weight of the first n tokens" and "the token
// at which the running weight passes x".  With whole-number weights
// w = round(2^40 exp((l - max) / T)) both are exact in any order of summation,
// so no sort of the vocabulary is needed, only histograms:
//
//   k_sample_max     each row's maximum and minimum, by chunks
//   k_sample_hist    weights (and, for top-k, counts) of SM_BINS equal steps of l
//                    from the maximum to the minimum, or to where weights end,
//                    by chunks; the row's last chunk adds them up and marks the
//                    few bins in which a border (of top-k, top-p, min-p or the
//                    draw itself) can lie
//   k_sample_pick    the tokens of the marked bins, listed; the row's last chunk
//                    sorts the list, finds the borders in it one after the other
//                    and the token
//
// A row whose marked bins hold more than SM_CAP tokens (many equal logits, a
// very high temperature) is selected by its keys instead, in the last kernel.
//
// Bound: the logits are read three times, the first time from memory, 20 float64
// operations and a 64-bit LDS addition a token in the histogram; a row takes three
// launches and two hand-overs between its chunks however short it is.  Measured
// (151936 float32 logits a row; kernels alone): one row 3.4 + 9.7 + 9.6 us, 7 rows of
// 50304 3.4 + 12.8 + 8.8, 128 rows with settings of their own 13.7 + 42.6 + 34.1 (read
// once at the rate of a copy: 16).
#include <algorithm>

#include "jm_device.h"
#include "jm_kernels.h"

namespace jm {

constexpr unsigned long long SM_ONE = 1ull << 40;      // the largest logit's weight
constexpr int SM_T = 1024;                             // threads a block
constexpr int SM_BINS = 1024;
constexpr int SM_CAP = 4096;                           // tokens a row's list holds
// past this (max - l) / T a weight is 0: 41 ln 2, and a bin more for rounding
constexpr float SM_SPAN = 28.45f;

// What the histogram's last chunk leaves for the row.
struct SmPlan {
    uint32_t mark[SM_BINS / 32];
    unsigned long long m1;      // the weight that top-k keeps, where it is known (0: the list tells)
    int mbin;                   // min-p: the first of the marked bins around its border
    unsigned long long m3_before;   // the weight before that bin
    int none;                   // a row with nothing to draw
};

// A row's part of the workspace.
struct SmRow {
    unsigned* ticket;           // [2] chunks done of the two kernels that hand over; [2]: the list's length
    float2* cmm;                // [SP] largest and smallest logit of the chunk
    float* wmx;                 // [SP][SM_T / 64] largest of each wave's
    SmPlan* plan;
    unsigned long long* umass;  // [SM_BINS] weight of the unmarked bins before a bin
    unsigned* ucnt;             // [SM_BINS]
    unsigned long long* hmass;  // [SP][SM_BINS]
    unsigned* hcnt;
    ulonglong2* list;           // [SM_CAP] key, weight
};

__host__ __device__ __forceinline__ size_t sm_row_bytes(int SP) {
    return 16 + ((size_t)SP * 8 + 15) / 16 * 16 + (size_t)SP * (SM_T / 16) + (sizeof(SmPlan) + 15) / 16 * 16 + (size_t)SM_BINS * 12 * (1 + SP) +
           (size_t)SM_CAP * 16;
}

__device__ __forceinline__ SmRow sm_row(char* ws, int b, int SP) {
    SmRow r;
    char* p = ws + (size_t)b * sm_row_bytes(SP);
    r.ticket = (unsigned*)p; p += 16;
    r.cmm = (float2*)p; p += ((size_t)SP * 8 + 15) / 16 * 16;
    r.wmx = (float*)p; p += (size_t)SP * (SM_T / 16);
    r.plan = (SmPlan*)p; p += (sizeof(SmPlan) + 15) / 16 * 16;
    r.list = (ulonglong2*)p; p += (size_t)SM_CAP * 16;
    r.umass = (unsigned long long*)p; p += (size_t)SM_BINS * 8;
    r.hmass = (unsigned long long*)p; p += (size_t)SM_BINS * 8 * SP;
    r.ucnt = (unsigned*)p; p += (size_t)SM_BINS * 4;
    r.hcnt = (unsigned*)p;
    return r;
}

// The order of the logits as unsigned integers (larger first): NaN below
// everything, -0 as +0.
__device__ __forceinline__ uint32_t sm_key(float l) {
    if (l != l) return 0;
    const uint32_t b = __float_as_uint(l + 0.0f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}

__device__ __forceinline__ float sm_unkey(uint32_t k) {
    return __uint_as_float(k & 0x80000000u ? k & 0x7FFFFFFFu : ~k);
}

__device__ __forceinline__ unsigned long long sm_key64(float l, int i) {
    return ((unsigned long long)sm_key(l) << 32) | (uint32_t)~i;
}

// round(2^40 2^t) for t <= 0: 2^f by its series on |f| <= 1/2 (the first term
// left out is below 2^-52), rounded to a whole number by adding 2^52.
__device__ __forceinline__ unsigned long long sm_exp2(double t) {
    const double k = rint(t), f = t - k;
    double p = 2.5678435993488196e-11;
    p = __builtin_fma(f, p, 4.4455382718708101e-10);
    p = __builtin_fma(f, p, 7.0549116208011209e-09);
    p = __builtin_fma(f, p, 1.0178086009239696e-07);
    p = __builtin_fma(f, p, 1.3215486790144305e-06);
    p = __builtin_fma(f, p, 1.5252733804059838e-05);
    p = __builtin_fma(f, p, 0.00015403530393381606);
    p = __builtin_fma(f, p, 0.0013333558146428441);
    p = __builtin_fma(f, p, 0.0096181291076284769);
    p = __builtin_fma(f, p, 0.055504108664821576);
    p = __builtin_fma(f, p, 0.24022650695910069);
    p = __builtin_fma(f, p, 0.69314718055994529);
    p = __builtin_fma(f, p, 1.0);
    p = ldexp(p, (int)k + 40) + 4503599627370496.0;
    return (unsigned long long)__double_as_longlong(p) & ((1ull << 52) - 1);
}

// A row's settings.
struct SmHow {
    float mx;                   // the largest logit
    double c;                   // log2(e) / T
    float cb;                   // bins a unit of l
    float T;
    int k;                      // 0: all
    float p, mp, u;
};

__device__ __forceinline__ void sm_how(SmHow& h, const SampleArgs& a, int b, const SmRow& r, int SP) {
    float T = a.temperature_b ? a.temperature_b[b] : a.temperature;
    h.k = a.top_k_b ? a.top_k_b[b] : a.top_k;
    h.p = a.top_p_b ? a.top_p_b[b] : a.top_p;
    h.mp = a.min_p_b ? a.min_p_b[b] : a.min_p;
    h.u = a.u[b];
    if (!(T > 0.0f)) { T = 1.0f; h.k = 1; }
    h.c = 1.4426950408889634 / (double)T;
    float mx = -INFINITY, mn = INFINITY;
    for (int i = threadIdx.x & 63; i < SP; i += 64) {
        const float2 v = r.cmm[i];
        mx = fmaxf(mx, v.x);
        mn = fminf(mn, v.y);
    }
    h.mx = seg_max<64>(mx);
    // (0 / 0 where all are alike: no span)
    const float span = fminf(__fsub_rn(h.mx, -seg_max<64>(-mn)), __fmul_rn(SM_SPAN, T));
    h.cb = fminf(__fdiv_rn((float)SM_BINS, span), 3.0e38f);
    h.T = T;
}

__device__ __forceinline__ unsigned long long sm_weight(const SmHow& h, float l) {
    if (l == h.mx) return SM_ONE;
    const double t = ((double)l - (double)h.mx) * h.c;
    return t >= -41.5 ? sm_exp2(t) : 0ull;             // (NaN: 0)
}

// The running weight that the drawn token is the first to pass, of a kept sum M.
__device__ __forceinline__ unsigned long long sm_target(float u, unsigned long long M) {
    if (!(u < 1.0f) && u == u) return M - 1;
    return min((unsigned long long)((double)(u > 0.0f ? u : 0.0f) * (double)M), M - 1);
}

// The bin of a logit: monotone in l, each step being so.
__device__ __forceinline__ int sm_bin(const SmHow& h, float l) {
    if (l == h.mx) return 0;
    return (int)fminf(__fmul_rn(__fsub_rn(h.mx, l), h.cb), (float)(SM_BINS - 1));
}

__device__ __forceinline__ float sm_logit(const SampleArgs& a, size_t row, int i) {
    return a.bf ? bf16_bits_to_f32(((const uint16_t*)a.logits)[row + i]) : ((const float*)a.logits)[row + i];
}

// What the chunks of a row hand to its last one in the same launch is written
// through the XCD's L2 and read past it (device scope), so that no cache has to
// be written back or emptied: with fences that do, 512 blocks took 12 us more.
template <typename T>
__device__ __forceinline__ void sm_put(T* p, T v) {
    __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
template <typename T>
__device__ __forceinline__ T sm_get(T* p) {
    return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// Whether this block is the last of the row's to come here; what the others
// put before is then there for sm_get.
__device__ __forceinline__ bool sm_last(unsigned* ticket, int SP, unsigned* flag) {
    __asm__ volatile("s_waitcnt vmcnt(0)" : : : "memory");     // this wave's stores are through
    __syncthreads();
    if (threadIdx.x == 0) *flag = atomicAdd(ticket, 1u) == (unsigned)SP - 1;
    __syncthreads();
    __asm__ volatile("" : : : "memory");
    return *flag;
}

__global__ void __launch_bounds__(SM_T)
k_sample_max(SampleArgs a, char* ws, int SP, int chunk) {
    __shared__ float red[2][SM_T / 64];
    const int b = blockIdx.x / SP, s = blockIdx.x % SP, tid = threadIdx.x;
    const size_t row = (size_t)b * a.ld;
    const int i1 = min((s + 1) * chunk, a.V);
    float mx = -INFINITY, mn = INFINITY;
    for (int i0 = s * chunk + tid; i0 < i1; i0 += 8 * SM_T) {
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; e++) v[e] = sm_logit(a, row, min(i0 + e * SM_T, i1 - 1));
#pragma unroll
        for (int e = 0; e < 8; e++) {
            // (each logit counts once: sm_kth_part takes the waves' maxima for parts)
            const bool in = i0 + e * SM_T < i1;
            mx = fmaxf(mx, in ? v[e] : -INFINITY);
            mn = fminf(mn, in && v[e] > -INFINITY ? v[e] : INFINITY);
        }
    }
    mx = seg_max<64>(mx);
    mn = -seg_max<64>(-mn);
    if ((tid & 63) == 0) {
        red[0][tid >> 6] = mx;
        red[1][tid >> 6] = mn;
    }
    const SmRow r = sm_row(ws, b, SP);
    if ((tid & 63) == 0) r.wmx[s * (SM_T / 64) + (tid >> 6)] = mx;
    __syncthreads();
    if (tid == 0) {
        for (int i = 1; i < SM_T / 64; i++) {
            mx = fmaxf(mx, red[0][i]);
            mn = fminf(mn, red[1][i]);
        }
        r.cmm[s] = make_float2(mx, mn);
    }
    if (s == 0 && tid < 3) r.ticket[tid] = 0;
}

// Running sum over the lanes (DPP: within rows of 16, then row ends onto the
// rows behind), 64 bits.
template <int CTRL, int ROWS>
__device__ __forceinline__ unsigned long long sm_dpp_add(unsigned long long v) {
    const unsigned lo = (unsigned)__builtin_amdgcn_update_dpp(0, (int)(unsigned)v, CTRL, ROWS, 0xF, false);
    const unsigned hi = (unsigned)__builtin_amdgcn_update_dpp(0, (int)(unsigned)(v >> 32), CTRL, ROWS, 0xF, false);
    return v + (((unsigned long long)hi << 32) | lo);
}
__device__ __forceinline__ unsigned long long sm_wave_scan(unsigned long long v) {
    v = sm_dpp_add<0x111, 0xF>(v);          // row_shr 1, 2, 4, 8
    v = sm_dpp_add<0x112, 0xF>(v);
    v = sm_dpp_add<0x114, 0xF>(v);
    v = sm_dpp_add<0x118, 0xF>(v);
    v = sm_dpp_add<0x142, 0xA>(v);          // lane 15 onto row 1, 47 onto row 3
    v = sm_dpp_add<0x143, 0xC>(v);          // lane 31 onto rows 2 and 3
    return v;
}
// ... over the block's threads; tot: 16 words of LDS that nothing else uses
__device__ __forceinline__ unsigned long long sm_block_scan(unsigned long long v, unsigned long long* tot) {
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    v = sm_wave_scan(v);
    __syncthreads();
    if (lane == 63) tot[w] = v;
    __syncthreads();
    const unsigned long long t = sm_wave_scan(lane < SM_T / 64 ? tot[lane] : 0ull);
    const int from = __builtin_amdgcn_readfirstlane(w) - 1;
    if (from < 0) return v;
    return v + (((unsigned long long)(unsigned)__builtin_amdgcn_readlane((int)(unsigned)(t >> 32), from) << 32) |
                (unsigned)__builtin_amdgcn_readlane((int)(unsigned)t, from));
}

// Thread i tells the first bin at which pass (monotone) holds, through *out,
// which starts as SM_BINS - 1; read it after a barrier.
template <typename F>
__device__ __forceinline__ void sm_find(F pass, int* out) {
    const int i = (int)threadIdx.x;
    if (pass(i) && (i == 0 || !pass(i - 1))) *out = i;
}
static_assert(SM_BINS == SM_T, "a bin a thread");

// A logit that at least k <= 64 of the row's are not below: the k-th of the
// maxima of 64 parts of it (or fewer); by one wave.
__device__ __forceinline__ float sm_kth_part(const SmRow& r, int SP, int k) {
    const int lane = threadIdx.x & 63;
    float m = -INFINITY;
    for (int i = lane; i < SP * (SM_T / 64); i += 64) m = fmaxf(m, r.wmx[i]);
    int above = 0;
#pragma unroll
    for (int i = 0; i < 64; i++) {
        const float x = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(m), i));
        above += x > m || (x == m && i < lane);
    }
    return __shfl(m, __builtin_ctzll(__ballot(above == k - 1)), JM_WAVE);
}

__global__ void __launch_bounds__(SM_T, 8)
k_sample_hist(SampleArgs a, char* ws, int SP, int chunk) {
    __shared__ unsigned long long mass[SM_BINS], incl[SM_BINS], wtot[16];
    __shared__ unsigned cnt[SM_BINS], cincl[SM_BINS], flag, mark[SM_BINS / 32];
    __shared__ int found[5];
    __shared__ float least;
    const int b = blockIdx.x / SP, s = blockIdx.x % SP, tid = threadIdx.x, lane = tid & 63;
    const size_t row = (size_t)b * a.ld;
    const int i1 = min((s + 1) * chunk, a.V);
    const SmRow r = sm_row(ws, b, SP);
    SmHow h;
    sm_how(h, a, b, r, SP);
    // (block-uniform) top-k matters; few enough that all it keeps fits the
    // list, where weights are formed: then only counts are needed here
    const bool counts = h.k > 0 && h.k < a.V, few = counts && h.k <= SM_CAP / 4;
    mass[tid] = 0;
    cnt[tid] = 0;
    // What is below the k-th largest need not be counted: worth its finding, 1.5 us,
    // where a thread has many tokens (top-k 50 of 151936: 128 rows 64 us without, 60
    // with it; one row, 8 tokens a thread, 24.7 and 27.0).
    if (few && tid < 64) {
        const float x = h.k <= 64 && chunk >= 16 * SM_T ? sm_kth_part(r, SP, h.k) : -INFINITY;
        if (tid == 0) least = x;
    }
    __syncthreads();
    if (h.mx > -INFINITY)
        for (int i0 = s * chunk + tid; i0 - tid < i1; i0 += 8 * SM_T) {
            float v[8];
#pragma unroll
            for (int e = 0; e < 8; e++) v[e] = sm_logit(a, row, min(i0 + e * SM_T, i1 - 1));
#pragma unroll
            for (int e = 0; e < 8; e++) v[e] = i0 + e * SM_T < i1 ? v[e] : -INFINITY;
            if (few) {
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    // (the last bin, where everything far below piles up, is
                    // what is taken if the others do not reach k)
                    if (!(v[e] >= least)) continue;
                    const int bin = sm_bin(h, v[e]);
                    if (bin < SM_BINS - 1) atomicAdd(&cnt[bin], 1u);
                }
                continue;
            }
            unsigned long long w[8];
#pragma unroll
            for (int e = 0; e < 8; e++) w[e] = sm_weight(h, v[e]);
#pragma unroll
            for (int e = 0; e < 8; e++) {
                if (!w[e]) continue;
                const int bin = sm_bin(h, v[e]);
                atomicAdd(&mass[bin], w[e]);
                if (counts) atomicAdd(&cnt[bin], 1u);
            }
        }
    __syncthreads();
    if (SP > 1) {
        if (!few) sm_put(&r.hmass[(size_t)s * SM_BINS + tid], mass[tid]);
        if (counts) sm_put(&r.hcnt[(size_t)s * SM_BINS + tid], cnt[tid]);
        if (!sm_last(r.ticket, SP, &flag)) return;
        unsigned long long m = 0;
        unsigned n = 0;
        // (the other chunks' lines come from memory: 16 requests at a time)
        for (int i0 = 0; i0 < SP; i0 += 16) {
            unsigned long long mv[16];
            unsigned nv[16];
#pragma unroll
            for (int i = 0; i < 16; i++) {
                const size_t at = (size_t)min(i0 + i, SP - 1) * SM_BINS + tid;
                mv[i] = few ? 0ull : sm_get(&r.hmass[at]);
                nv[i] = counts ? sm_get(&r.hcnt[at]) : 0;
            }
#pragma unroll
            for (int i = 0; i < 16; i++)
                if (i0 + i < SP) {
                    m += mv[i];
                    n += nv[i];
                }
        }
        mass[tid] = m;
        cnt[tid] = n;
    }
    if (h.mx == -INFINITY) {
        if (tid == 0) r.plan->none = 1;
        return;
    }
    const unsigned long long my_m = mass[tid];
    const unsigned my_n = cnt[tid];
    if (tid < SM_BINS / 32) mark[tid] = 0;
    if (tid < 5) found[tid] = SM_BINS - 1;
    if (few) {
        // every token up to top-k's border goes on the list
        cincl[tid] = (unsigned)sm_block_scan(my_n, wtot);
        __syncthreads();
        sm_find([&](int j) { return cincl[j] >= (unsigned)h.k; }, &found[0]);
        __syncthreads();
        const int last = found[0];
        r.umass[tid] = 0;
        r.ucnt[tid] = 0;
        if (tid < SM_BINS / 32) {
            const int n = last + 1 - 32 * tid;
            r.plan->mark[tid] = n <= 0 ? 0u : n >= 32 ? 0xFFFFFFFFu : (1u << n) - 1;
        }
        if (tid == 0) {
            r.plan->m1 = 0;
            r.plan->mbin = 0;
            r.plan->m3_before = 0;
            r.plan->none = 0;
        }
        return;
    }
    incl[tid] = sm_block_scan(my_m, wtot);
    if (counts) cincl[tid] = (unsigned)sm_block_scan(my_n, wtot);
    __syncthreads();
    auto before = [&](int i) { return i > 0 ? incl[i - 1] : 0ull; };
    const unsigned long long total = incl[SM_BINS - 1];
    auto set = [&](int lo, int hi) {
        if (tid >= lo && tid <= hi) atomicOr(&mark[tid >> 5], 1u << (tid & 31));
    };
    // top-k
    unsigned long long m1lo = total, m1hi = total;
    if (counts && (unsigned)h.k < cincl[SM_BINS - 1]) {
        const unsigned k = (unsigned)h.k;
        sm_find([&](int j) { return cincl[j] >= k; }, &found[0]);
        __syncthreads();
        const int i = found[0];
        m1hi = m1lo = incl[i];
        if (cincl[i] > k) {
            m1lo = before(i);
            set(i, i);
        }
    }
    unsigned long long lo = m1lo, hi = m1hi;
    if (h.p < 1.0f) {
        const double xl = (double)h.p * (double)m1lo, xh = (double)h.p * (double)m1hi;
        sm_find([&](int j) { return (double)incl[j] >= xl; }, &found[1]);
        sm_find([&](int j) { return (double)incl[j] >= xh; }, &found[2]);
        __syncthreads();
        const int il = found[1], ih = found[2];
        set(il, ih);
        lo = min(lo, before(il));
        hi = min(hi, incl[ih]);
    }
    int mbin = 0;
    if (h.mp > 0.0f) {
        // the bin where weights pass the border (rounded ones: half a unit below it),
        // and its neighbours, which rounding here may mean; in float64, as next to a
        // min_p of 1 the border is 2^-41 of (max - l) / T, and the last bin where a high
        // temperature puts it past all logits.  (cb is 0 where logits differ by more
        // than float32 holds: two bins for all, the border in either.)
        const double wmin = fmin(ceil((double)h.mp * (double)SM_ONE), (double)SM_ONE);
        const double z = -log((wmin - 0.5) / (double)SM_ONE) * (double)h.T * (double)h.cb;
        const int i = z < (double)(SM_BINS - 1) ? (int)z : SM_BINS - 1;
        mbin = h.cb > 0.0f ? max(i - 1, 0) : 0;
        const int mh = h.cb > 0.0f ? min(i + 1, SM_BINS - 1) : SM_BINS - 1;
        set(mbin, mh);
        lo = min(lo, before(mbin));
        hi = min(hi, incl[mh]);
    }
    const unsigned long long tl = sm_target(h.u, max(lo, SM_ONE)), th = sm_target(h.u, max(hi, SM_ONE));
    sm_find([&](int j) { return incl[j] > tl; }, &found[3]);
    sm_find([&](int j) { return incl[j] > th; }, &found[4]);
    __syncthreads();
    set(found[3], found[4]);
    __syncthreads();
    const bool marked = mark[tid >> 5] >> (tid & 31) & 1;
    r.umass[tid] = sm_block_scan(marked ? 0ull : my_m, wtot);
    if (counts) r.ucnt[tid] = (unsigned)sm_block_scan(marked ? 0u : my_n, wtot);
    if (tid < SM_BINS / 32) r.plan->mark[tid] = mark[tid];
    if (tid == 0) {
        r.plan->m1 = m1lo == m1hi ? m1hi : 0;
        r.plan->mbin = mbin;
        r.plan->m3_before = before(mbin);
        r.plan->none = 0;
    }
}

// The borders and the token of a row from its list in descending order: each(f)
// calls f(key, weight, running weight, running count) for every entry of this
// thread; one entry at most answers to each question.
template <typename E>
__device__ __forceinline__ void sm_finish(const SampleArgs& a, int b, const SmHow& h, const SmPlan& plan, int n, E each,
                                          unsigned long long* sh, unsigned long long* tot) {
    const int tid = threadIdx.x;
    unsigned long long M = plan.m1;
    if (!M) {
        // (fewer than k on the list: those are all there are)
        each([&](int i, unsigned long long, unsigned long long, unsigned long long run, unsigned c) {
            if (c == (unsigned)h.k || (i == n - 1 && c < (unsigned)h.k)) sh[0] = run;
        });
        __syncthreads();
        M = sh[0];
    }
    if (h.p < 1.0f) {
        const double x = fmax((double)h.p * (double)M, 0.5);
        each([&](int, unsigned long long, unsigned long long w, unsigned long long run, unsigned) {
            if ((double)run >= x && (double)(run - w) < x) sh[1] = run;
        });
        __syncthreads();
        M = min(M, sh[1]);
    }
    if (h.mp > 0.0f) {
        const double wmin = ceil((double)h.mp * (double)SM_ONE);
        unsigned long long t = 0;
        each([&](int, unsigned long long key, unsigned long long w, unsigned long long, unsigned) {
            if ((double)w >= wmin && sm_bin(h, sm_unkey((uint32_t)(key >> 32))) >= plan.mbin) t += w;
        });
        t = sm_block_scan(t, tot);
        if (tid == SM_T - 1) sh[2] = t;
        __syncthreads();
        M = min(M, wmin > (double)SM_ONE ? SM_ONE : plan.m3_before + sh[2]);
    }
    M = max(M, SM_ONE);
    const unsigned long long t = sm_target(h.u, M);
    each([&](int, unsigned long long key, unsigned long long w, unsigned long long run, unsigned) {
        if (run > t && run - w <= t) {
            a.out_tok[b] = (int)~(uint32_t)key;
            if (a.out_p) a.out_p[b] = (float)((double)w / (double)M);
        }
    });
}

// The row selected by its keys, 11 bits at a time from the top: a histogram of
// the tokens that share the prefix found so far, then the digit at which the
// running sum (of weights, or of tokens) passes the target.  Six passes over the
// row a border, in one block: for rows whose list would be too long.
__device__ __forceinline__ void sm_by_keys(const SampleArgs& a, int b, const SmHow& h, const SmPlan& plan,
                                           unsigned long long* hist, unsigned long long* sh, unsigned long long* tot) {
    constexpr int BITS = 11, ND = 1 << BITS;
    const int tid = threadIdx.x, lane = tid & 63;
    const size_t row = (size_t)b * a.ld;
    auto each = [&](auto f) {
        for (int i0 = tid; i0 < a.V; i0 += 4 * SM_T) {
            float v[4];
#pragma unroll
            for (int e = 0; e < 4; e++) v[e] = sm_logit(a, row, min(i0 + e * SM_T, a.V - 1));
#pragma unroll
            for (int e = 0; e < 4; e++)
                if (i0 + e * SM_T < a.V) f(i0 + e * SM_T, v[e]);
        }
    };
    // the key found; sh[0]: the sum before it
    auto select = [&](bool counting, unsigned long long target) {
        unsigned long long prefix = 0, before = 0;
        for (int top = 64; top > 0;) {
            const int bits = min(top, BITS), low = top - bits;
            __syncthreads();
            for (int i = tid; i < ND; i += SM_T) hist[i] = 0;
            __syncthreads();
            each([&](int i, float l) {
                const unsigned long long key = sm_key64(l, i);
                if (top < 64 && (key >> top) != (prefix >> top)) return;
                const unsigned long long w = sm_weight(h, l);
                if (w) atomicAdd(&hist[(key >> low) & (ND - 1)], counting ? 1ull : w);
            });
            __syncthreads();
            // from the largest digit down: wave 0, 32 digits a lane
            if (tid < 64) {
                unsigned long long own = 0;
                for (int i = 0; i < ND / 64; i++) own += hist[ND - 1 - (lane * (ND / 64) + i)];
                unsigned long long upto = own;
                for (int o = 1; o < 64; o <<= 1) {
                    const unsigned long long t = __shfl_up(upto, o, JM_WAVE);
                    if (lane >= o) upto += t;
                }
                unsigned long long run = before + upto - own;
                if (run + own > target && run <= target)
                    for (int i = 0; i < ND / 64; i++) {
                        const int d = ND - 1 - (lane * (ND / 64) + i);
                        if (run + hist[d] > target) {
                            sh[0] = run;
                            sh[1] = (unsigned long long)d;
                            break;
                        }
                        run += hist[d];
                    }
            }
            __syncthreads();
            before = sh[0];
            prefix |= sh[1] << low;
            top = low;
        }
        return prefix;
    };
    auto weight_of = [&](unsigned long long key) { return sm_weight(h, sm_unkey((uint32_t)(key >> 32))); };
    // a count's border: the weight up to and with that token
    auto sum_if = [&](auto take) {
        unsigned long long t = 0;
        each([&](int i, float l) {
            const unsigned long long w = sm_weight(h, l);
            if (take(sm_key64(l, i), w)) t += w;
        });
        t = sm_block_scan(t, tot);
        if (tid == SM_T - 1) sh[2] = t;
        __syncthreads();
        return sh[2];
    };
    unsigned long long M = plan.m1;
    if (!M) {
        const unsigned long long key = select(true, (unsigned long long)h.k - 1);
        M = sum_if([&](unsigned long long k, unsigned long long) { return k >= key; });
    }
    if (h.p < 1.0f) {
        const double x = ceil((double)h.p * (double)M);
        const unsigned long long key = select(false, x > 1.0 ? (unsigned long long)x - 1 : 0ull);
        M = min(M, sh[0] + weight_of(key));
    }
    if (h.mp > 0.0f) {
        const double x = ceil((double)h.mp * (double)SM_ONE);
        M = min(M, x > (double)SM_ONE ? SM_ONE : sum_if([&](unsigned long long, unsigned long long w) { return (double)w >= x; }));
    }
    M = max(M, SM_ONE);
    const unsigned long long t = sm_target(h.u, M);
    const unsigned long long key = select(false, t);
    if (tid == 0) {
        a.out_tok[b] = (int)~(uint32_t)key;
        if (a.out_p) a.out_p[b] = (float)((double)weight_of(key) / (double)M);
    }
}

__global__ void __launch_bounds__(SM_T, 8)
k_sample_pick(SampleArgs a, char* ws, int SP, int chunk) {
    __shared__ unsigned long long key[SM_CAP], wt[SM_CAP], sh[4], wtot[16];
    __shared__ unsigned flag, have, mark[SM_BINS / 32], bucket[2 * SM_T + 1], mbefore[SM_BINS / 32 + 1];
    const int b = blockIdx.x / SP, s = blockIdx.x % SP, tid = threadIdx.x, lane = tid & 63;
    const size_t row = (size_t)b * a.ld;
    const int i1 = min((s + 1) * chunk, a.V);
    const SmRow r = sm_row(ws, b, SP);
    SmHow h;
    sm_how(h, a, b, r, SP);
    if (r.plan->none) {
        if (s == 0 && tid == 0) {
            a.out_tok[b] = -1;
            if (a.out_p) a.out_p[b] = 0.0f;
        }
        return;
    }
    if (tid < SM_BINS / 32) mark[tid] = r.plan->mark[tid];
    if (tid == 0) have = 0;
    __syncthreads();
    // the first and the end of the marked bins; most tokens are outside
    const uint32_t mw = lane < SM_BINS / 32 ? mark[lane] : 0u;
    const unsigned long long mb = __ballot(mw != 0);
    const int wa = mb ? __builtin_ctzll(mb) : 0, wz = mb ? 63 - __builtin_clzll(mb) : 0;
    const uint32_t ma = (uint32_t)__builtin_amdgcn_readlane((int)mw, wa), mz = (uint32_t)__builtin_amdgcn_readlane((int)mw, wz);
    const float za = ma ? (float)(32 * wa + __builtin_ctz(ma)) : 0.0f;
    const int be = mz ? 32 * wz + 32 - __builtin_clz(mz) : 0;
    const float zz = be < SM_BINS ? (float)be : __uint_as_float(0x7FC00000u);     // (the last bin has no end)
    for (int i0 = s * chunk + tid; i0 - tid < i1; i0 += 8 * SM_T) {
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; e++) v[e] = sm_logit(a, row, min(i0 + e * SM_T, i1 - 1));
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const float z = __fmul_rn(__fsub_rn(h.mx, v[e]), h.cb);
            if (!__any(!(z < za || z >= zz))) continue;
            const int bin = sm_bin(h, v[e]);
            bool in = i0 + e * SM_T < i1 && (mark[bin >> 5] >> (bin & 31) & 1);
            if (!__any(in)) continue;
            const unsigned long long w = in ? sm_weight(h, v[e]) : 0ull;
            in = w != 0;
            const unsigned long long who = __ballot(in);
            if (!who) continue;
            unsigned at = 0;
            if (lane == 0) at = atomicAdd(&have, (unsigned)__popcll(who));
            at = __builtin_amdgcn_readfirstlane(at) + __popcll(who & ((1ull << lane) - 1));
            if (in && at < SM_CAP) {
                key[at] = sm_key64(v[e], i0 + e * SM_T);
                wt[at] = w;
            }
        }
    }
    __syncthreads();
    const unsigned mine = have;
    if (tid == 0) flag = mine ? atomicAdd(&r.ticket[2], mine) : 0u;
    __syncthreads();
    const unsigned base = flag;
    for (unsigned i = tid; i < min(mine, (unsigned)SM_CAP) && base + i < SM_CAP; i += SM_T) {
        sm_put(&r.list[base + i].x, key[i]);
        sm_put(&r.list[base + i].y, wt[i]);
    }
    if (!sm_last(r.ticket + 1, SP, &flag)) return;
    const SmPlan& plan = *r.plan;
    const int n = (int)sm_get(&r.ticket[2]);         // tokens met, listed or not
    if (n > SM_CAP) {
        sm_by_keys(a, b, h, plan, key, sh, wtot);
        return;
    }
    // The list in descending order of its keys: a bucket for each part of each
    // marked bin, then each token's rank in its bucket.  (Equal parts of the
    // keys' range would put a bin into one bucket where the range spans 0: 50 us
    // for 2000 tokens.)
    constexpr int E = SM_CAP / SM_T, NB = 2 * SM_T;
    if (tid == 0) {
        unsigned t = 0;
        for (int i = 0; i < SM_BINS / 32; i++) {
            mbefore[i] = t;
            t += (unsigned)__popc(mark[i]);
        }
        mbefore[SM_BINS / 32] = t;
    }
    bucket[tid] = bucket[tid + SM_T] = 0;
    __syncthreads();
    const int parts = NB / (int)mbefore[SM_BINS / 32];
    ulonglong2 x[E];
    unsigned at[E], bk[E];
#pragma unroll
    for (int e = 0; e < E; e++)
        if (tid + e * SM_T < n) {
            x[e] = make_ulonglong2(sm_get(&r.list[tid + e * SM_T].x), sm_get(&r.list[tid + e * SM_T].y));
            const float l = sm_unkey((uint32_t)(x[e].x >> 32));
            const int bin = sm_bin(h, l);
            // where in its bin (exact: monotone as the bin itself is)
            const float z = l == h.mx ? 0.0f : __fmul_rn(__fsub_rn(h.mx, l), h.cb);
            const int part = (int)fminf(__fmul_rn(__fsub_rn(z, (float)bin), (float)parts), (float)(parts - 1));
            bk[e] = (mbefore[bin >> 5] + (unsigned)__popc(mark[bin >> 5] & ((1u << (bin & 31)) - 1))) * parts + part;
            at[e] = atomicAdd(&bucket[bk[e]], 1u);
        }
    __syncthreads();
    const unsigned b0 = bucket[2 * tid], b1 = bucket[2 * tid + 1];
    const unsigned upto_b = (unsigned)sm_block_scan(b0 + b1, wtot);
    bucket[2 * tid] = upto_b - b0 - b1;         // the buckets' first places
    bucket[2 * tid + 1] = upto_b - b1;
    if (tid == 0) bucket[NB] = (unsigned)n;
    __syncthreads();
#pragma unroll
    for (int e = 0; e < E; e++)
        if (tid + e * SM_T < n) key[bucket[bk[e]] + at[e]] = x[e].x;
    __syncthreads();
#pragma unroll
    for (int e = 0; e < E; e++)
        if (tid + e * SM_T < n) {
            const unsigned first = bucket[bk[e]], end = bucket[bk[e] + 1];
            at[e] = first;
            for (unsigned i = first; i < end; i++) at[e] += key[i] > x[e].x;
        }
    __syncthreads();
#pragma unroll
    for (int e = 0; e < E; e++)
        if (tid + e * SM_T < n) {
            key[at[e]] = x[e].x;
            wt[at[e]] = x[e].y;
        }
    __syncthreads();
    // running sums: 4 consecutive entries a thread
    unsigned long long run[E], t = 0;
#pragma unroll
    for (int e = 0; e < E; e++) {
        if (E * tid + e < n) t += wt[E * tid + e];
        run[e] = t;
    }
    const unsigned long long upto = sm_block_scan(t, wtot);
    const bool counts = h.k > 0 && h.k < a.V;
    unsigned cnt[E];
#pragma unroll
    for (int e = 0; e < E; e++) {
        const int i = E * tid + e;
        cnt[e] = 0;
        if (i >= n) continue;
        const int bin = sm_bin(h, sm_unkey((uint32_t)(key[i] >> 32)));
        run[e] += upto - t + r.umass[bin];
        cnt[e] = i + 1 + (counts ? r.ucnt[bin] : 0u);
    }
    sm_finish(a, b, h, plan, n, [&](auto f) {
#pragma unroll
        for (int e = 0; e < E; e++)
            if (E * tid + e < n) f(E * tid + e, key[E * tid + e], wt[E * tid + e], run[e], cnt[e]);
    }, sh, wtot);
}

// Chunks of a row: two blocks a CU over all rows (128 rows: 94 us; one 105, four
// 98, eight 115), at least 8 tokens a thread.
static int sm_chunks(int B, int V) {
    return std::max(1, std::min(512 / B, (V + 8 * SM_T - 1) / (8 * SM_T)));
}

// Rows a launch takes: more would fill the card no better, and the workspace is
// some 90 KB a row.
constexpr int SM_ROWS = 1024;

size_t sample_ws_bytes(int B, int V) {
    B = std::min(B, SM_ROWS);
    return (size_t)B * sm_row_bytes(sm_chunks(B, V));
}

hipError_t launch_sample(const SampleArgs& all, void* ws, hipStream_t st) {
    for (int b0 = 0; b0 < all.B; b0 += SM_ROWS) {
        SampleArgs a = all;
        a.B = std::min(all.B - b0, SM_ROWS);
        a.logits = (const char*)all.logits + (size_t)b0 * all.ld * (all.bf ? 2 : 4);
        a.u += b0;
        a.out_tok += b0;
        if (a.out_p) a.out_p += b0;
        if (a.temperature_b) a.temperature_b += b0;
        if (a.top_k_b) a.top_k_b += b0;
        if (a.top_p_b) a.top_p_b += b0;
        if (a.min_p_b) a.min_p_b += b0;
        // (as many chunks as the workspace has room for)
        const int SP = sm_chunks(std::min(all.B, SM_ROWS), a.V), chunk = (a.V + SP - 1) / SP;
        const dim3 grid((unsigned)a.B * SP);
        hipLaunchKernelGGL(k_sample_max, grid, dim3(SM_T), 0, st, a, (char*)ws, SP, chunk);
        hipLaunchKernelGGL(k_sample_hist, grid, dim3(SM_T), 0, st, a, (char*)ws, SP, chunk);
        hipLaunchKernelGGL(k_sample_pick, grid, dim3(SM_T), 0, st, a, (char*)ws, SP, chunk);
        if (const hipError_t e = hipGetLastError()) return e;
    }
    return hipSuccess;
}

}  // namespace jm
