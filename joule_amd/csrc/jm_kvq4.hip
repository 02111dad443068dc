// The 4-bit KV cache's operators: rows quantised as they are written, read
// back, and attended over (jm_q4kv.h has the layout).
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

// Attention, one block per (head, token): wave w takes every fourth row up to
// the token's own with a running maximum and sum, lane l dimensions 2 l and
// 2 l + 1; the waves merge at the end.  Float32 throughout.
template <int NG, bool BF>
__global__ void __launch_bounds__(256)
k_q4_attn_row(Q4KvArgs c, const void* __restrict__ q, long long qts, long long qhs, int H, float scale,
              void* __restrict__ out) {
    __shared__ float mls[4][2], ol[4][128];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, t = blockIdx.y, hd = blockIdx.x;
    const int kh = hd / (H / c.KH);
    int seq, pos;
    const bool in = q4_place(c, t, seq, pos);
    if (!in && (seq < 0 || seq >= c.n_seq || pos >= c.maxT)) return;
    float o0 = 0.0f, o1 = 0.0f, m = -INFINITY, l = 0.0f;
    if (in) {
        const Q4Head<NG> kk(q4_plane(c, seq, 0), kh, c.KH, c.R), vv(q4_plane(c, seq, 1), kh, c.KH, c.R);
        const size_t qi = (size_t)(t * qts + hd * qhs) + 2 * lane;
        const float q0 = BF ? bf16_bits_to_f32(((const uint16_t*)q)[qi]) : ((const float*)q)[qi];
        const float q1 = BF ? bf16_bits_to_f32(((const uint16_t*)q)[qi + 1]) : ((const float*)q)[qi + 1];
        const int g = lane / (64 / NG), od = lane >> 2, kp = 4 * (od & 3) + (od >> 2), ks = 8 * (lane & 3);
        const int n = (2 * lane) & 15, vs = 4 * (lane >> 3);
        for (int r = w; r <= pos; r += 4) {
            const uint32_t kd = *kk.k_dword(r, kp) >> ks;
            const uint32_t v0 = *vv.v_dword(r, n) >> vs, v1 = *vv.v_dword(r, n + 1) >> vs;
            const float sk = fp16_hw(*kk.scale(r, g)), sv = fp16_hw(*vv.scale(r, g));
            const float d = __builtin_fmaf(q0, (float)((int)(kd & 15u) - 8), q1 * (float)((int)((kd >> 4) & 15u) - 8));
            const float s = seg_sum<64>(d * sk) * scale;
            const float mn = fmaxf(m, s), mref = mn == -INFINITY ? 0.0f : mn;
            const float f = expf(m - mref), p = expf(s - mref);
            o0 = __builtin_fmaf(o0, f, p * sv * (float)((int)(v0 & 15u) - 8));
            o1 = __builtin_fmaf(o1, f, p * sv * (float)((int)(v1 & 15u) - 8));
            l = __builtin_fmaf(l, f, p);
            m = mn;
        }
    }
    if (lane == 0) { mls[w][0] = m; mls[w][1] = l; }
    ol[w][2 * lane] = o0;
    ol[w][2 * lane + 1] = o1;
    __syncthreads();
    if (w) return;
    float M = fmaxf(fmaxf(mls[0][0], mls[1][0]), fmaxf(mls[2][0], mls[3][0]));
    if (M == -INFINITY) M = 0.0f;
    float L = 0.0f, a = 0.0f, b = 0.0f;
    for (int i = 0; i < 4; i++) {
        const float f = expf(mls[i][0] - M);
        L += mls[i][1] * f;
        a += ol[i][2 * lane] * f;
        b += ol[i][2 * lane + 1] * f;
    }
    if (in) { a /= L; b /= L; }              // a token with no row to see: 0
    const size_t oi = ((size_t)t * H + hd) * 128 + 2 * lane;
    if (BF) *(uint32_t*)((uint16_t*)out + oi) = pack_bf16x2(a, b);
    else *(float2*)((float*)out + oi) = make_float2(a, b);
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

hipError_t launch_q4_attn(const Q4KvArgs& c, const void* q, bool bf, long long qts, long long qhs, int H, float scale,
                          void* out, hipStream_t st) {
    if (c.N == 0) return hipSuccess;
    const dim3 grid((unsigned)H, (unsigned)c.N);
    JM_Q4_EACH(k_q4_attn_row, grid, dim3(256), c, q, qts, qhs, H, scale, out);
    return hipGetLastError();
}

}  // namespace jm
