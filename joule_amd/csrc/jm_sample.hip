// Sampling of the next token (jm_sample): temperature, top-k, top-p and min-p
// from one random number a row.
//
// Every filter keeps a prefix of the tokens in the order (logit descending,
// index ascending), so that the kept set is the shortest of three prefixes and
// all that is ever needed is "the weight of the first n tokens" and "the token
// at which the running weight passes x".  With whole-number weights
// w = round(2^40 exp((l - max) / T)) both are exact in any order of summation.
#include "jm_device.h"
#include "jm_kernels.h"

namespace jm {

constexpr unsigned long long SM_ONE = 1ull << 40;      // the largest logit's weight

// The order of the logits as unsigned integers (larger first): NaN below
// everything, -0 as +0.
__device__ __forceinline__ uint32_t sm_key(float l) {
    if (l != l) return 0;
    const uint32_t b = __float_as_uint(l + 0.0f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}

__device__ __forceinline__ unsigned long long sm_weight(float l, float mx, double inv_t) {
    if (l == mx) return SM_ONE;
    if (!(l > -INFINITY)) return 0;
    return (unsigned long long)rint(exp(((double)l - (double)mx) * inv_t) * (double)SM_ONE);
}

__device__ __forceinline__ float sm_logit(const SampleArgs& a, size_t row, int i) {
    return a.bf ? bf16_bits_to_f32(((const uint16_t*)a.logits)[row + i]) : ((const float*)a.logits)[row + i];
}

// One block per row.  A selection walks down the 64-bit keys (logit order, then
// the index from the top) 8 bits at a time: a histogram of the elements that
// share the prefix found so far, then the digit at which the running sum
// passes the target.
__global__ void __launch_bounds__(1024)
k_sample_row(SampleArgs a) {
    __shared__ unsigned long long hist[256], sh[20];
    __shared__ float smax[16];
    const int tid = threadIdx.x, b = blockIdx.x;
    const size_t row = (size_t)b * a.ld;
    float T = a.temperature_b ? a.temperature_b[b] : a.temperature;
    int k = a.top_k_b ? a.top_k_b[b] : a.top_k;
    const float p = a.top_p_b ? a.top_p_b[b] : a.top_p, mp = a.min_p_b ? a.min_p_b[b] : a.min_p;
    if (!(T > 0.0f)) { T = 1.0f; k = 1; }
    const double inv_t = 1.0 / (double)T;
    float mx = -INFINITY;
    for (int i = tid; i < a.V; i += 1024) mx = fmaxf(mx, sm_logit(a, row, i));
    mx = seg_max<64>(mx);
    if ((tid & 63) == 0) smax[tid >> 6] = mx;
    __syncthreads();
    for (int i = 0; i < 16; i++) mx = fmaxf(mx, smax[i]);
    if (mx == -INFINITY) {
        if (tid == 0) {
            a.out_tok[b] = -1;
            if (a.out_p) a.out_p[b] = 0.0f;
        }
        return;
    }
    // the running weight (or, counting, the number of elements) passes
    // `target`: the key of that element and the weight up to and with it
    auto select = [&](bool counting, unsigned long long target, unsigned long long& key) {
        unsigned long long prefix = 0, before = 0, wsum = 0;
        for (int level = 0; level < 8; level++) {
            const int sh8 = 56 - 8 * level;
            __syncthreads();
            if (tid < 256) hist[tid] = 0;
            __syncthreads();
            for (int i = tid; i < a.V; i += 1024) {
                const float l = sm_logit(a, row, i);
                const unsigned long long w = sm_weight(l, mx, inv_t);
                if (!w) continue;
                const unsigned long long kk = ((unsigned long long)sm_key(l) << 32) | (uint32_t)~i;
                if (level && (kk >> (sh8 + 8)) != (prefix >> (sh8 + 8))) continue;
                atomicAdd(&hist[(kk >> sh8) & 255], counting ? 1ull : w);
            }
            __syncthreads();
            if (tid == 0) {
                unsigned long long run = before;
                int d = 255;
                for (; d > 0; d--) {
                    if (run + hist[d] > target) break;
                    run += hist[d];
                }
                sh[0] = run;
                sh[1] = d;
            }
            __syncthreads();
            before = sh[0];
            prefix |= sh[1] << sh8;
        }
        key = prefix;
        (void)wsum;
        return before;
    };
    auto sum_from = [&](unsigned long long key, unsigned long long wmin) {
        unsigned long long s = 0;
        for (int i = tid; i < a.V; i += 1024) {
            const float l = sm_logit(a, row, i);
            const unsigned long long w = sm_weight(l, mx, inv_t);
            const unsigned long long kk = ((unsigned long long)sm_key(l) << 32) | (uint32_t)~i;
            if (kk >= key && w >= wmin) s += w;
        }
        __syncthreads();
        if (tid == 0) sh[2] = 0;
        __syncthreads();
        atomicAdd(&sh[2], s);
        __syncthreads();
        const unsigned long long r = sh[2];
        return r;
    };
    unsigned long long key = 0, M;
    if (k > 0 && k < a.V) {
        select(true, (unsigned long long)k - 1, key);
        M = sum_from(key, 0);
    } else {
        M = sum_from(0, 0);
    }
    if (p < 1.0f) {
        const double x = (double)p * (double)M;
        unsigned long long kp;
        // the first element whose running weight reaches x
        const unsigned long long c = x > 0.0 ? (unsigned long long)ceil(x) : 0ull;
        select(false, c ? c - 1 : 0ull, kp);
        M = min(M, sum_from(kp, 0));
    }
    if (mp > 0.0f) {
        const double x = ceil((double)mp * (double)SM_ONE);
        M = min(M, x > (double)SM_ONE ? SM_ONE : sum_from(0, (unsigned long long)x));
        M = max(M, SM_ONE);
    }
    float u = a.u[b];
    u = u > 0.0f ? u : 0.0f;
    unsigned long long t = u < 1.0f ? (unsigned long long)floor((double)u * (double)M) : M - 1;
    t = min(t, M - 1);
    select(false, t, key);
    if (tid == 0) {
        const int i = (int)~(uint32_t)key;
        a.out_tok[b] = i;
        if (a.out_p) a.out_p[b] = (float)((double)sm_weight(sm_logit(a, row, i), mx, inv_t) / (double)M);
    }
}

hipError_t launch_sample(const SampleArgs& a, hipStream_t st) {
    if (a.B == 0) return hipSuccess;
    hipLaunchKernelGGL(k_sample_row, dim3((unsigned)a.B), dim3(1024), 0, st, a);
    return hipGetLastError();
}

}  // namespace jm
