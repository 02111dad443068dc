// The tokens of a call over caches: their values, and which sequence and cache row each
// has.  C is the call's arguments (Q4KvArgs, PagedArgs): n_seq, N, maxT, start and cu
// (NULL: token t is sequence t's only one).
#pragma once

#include "jm_device.h"

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

// 8 of them (aligned to 4).
typedef uint32_t u32x4_a8 __attribute__((ext_vector_type(4), aligned(8)));
template <bool BF>
__device__ __forceinline__ void load8(const void* p, size_t i, float (&v)[8]) {
    if (BF) {
        const u32x4_a8 u = *(const u32x4_a8*)((const uint16_t*)p + i);
#pragma unroll
        for (int e = 0; e < 4; e++) {
            v[2 * e] = __uint_as_float(u[e] << 16);
            v[2 * e + 1] = __uint_as_float(u[e] & 0xFFFF0000u);
        }
    } else {
#pragma unroll
        for (int e = 0; e < 8; e += 4) {
            const float4 u = *(const float4*)((const float*)p + i + e);
            v[e] = u.x; v[e + 1] = u.y; v[e + 2] = u.z; v[e + 3] = u.w;
        }
    }
}

template <bool BF>
__device__ __forceinline__ void store8(void* p, size_t i, const float (&v)[8]) {
    if (BF) {
        u32x4_a8 u;
#pragma unroll
        for (int e = 0; e < 4; e++) u[e] = pack_bf16x2(v[2 * e], v[2 * e + 1]);
        __builtin_nontemporal_store(u, (u32x4_a8*)((uint16_t*)p + i));
    } else {
#pragma unroll
        for (int e = 0; e < 8; e += 4)
            __builtin_nontemporal_store(u32x4_t{__float_as_uint(v[e]), __float_as_uint(v[e + 1]), __float_as_uint(v[e + 2]),
                                                __float_as_uint(v[e + 3])}, (u32x4_t*)((float*)p + i + e));
    }
}

// 4 values to a contiguous output.
template <bool BF>
__device__ __forceinline__ void store_out(void* p, size_t i, float4 v) {
    if (BF) *(uint2*)((uint16_t*)p + i) = make_uint2(pack_bf16x2(v.x, v.y), pack_bf16x2(v.z, v.w));
    else *(float4*)((float*)p + i) = v;
}

// The sequence and cache row of the four tokens t0 .. t0 + 3 of a call (not the
// decoder's form) in the wave's four rows of 16 lanes: each lane gets its row's
// token's; false for a token that has none (behind the last sequence, or a row
// outside the cache).
template <class C>
__device__ __forceinline__ bool call_places(const C& c, int t0, int& seq, int& pos) {
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

// The same for one token, alike in every lane.
template <class C>
__device__ __forceinline__ bool call_place(const C& c, int t, int& seq, int& pos) {
    const int lane = threadIdx.x & 63;
    seq = t;
    int first = t;
    if (c.cu) {
        int n = 0;
        for (int s = 0; s <= c.n_seq; s += 64)
            n += __popcll(__ballot(s + lane <= c.n_seq && c.cu[min(s + lane, c.n_seq)] <= t));
        seq = n - 1;
        if (seq < 0 || seq >= c.n_seq) return false;
        first = c.cu[seq];
    }
    const long long p = (long long)c.start[seq] + (t - first);
    pos = (int)(p < 0 ? -1 : p >= c.maxT ? c.maxT : p);
    return p >= 0 && p < c.maxT;
}

// The KV head's query rows of one unit: which sequence, its first token, how
// many tokens, the first token's cache row.
struct CallUnit {
    int seq, tok, n, pos;
};

// The cache row of token u where tokens have a sequence each (call_unit without cu).
template <class C>
__device__ __forceinline__ int call_row(const C& c, int u) { return c.start[u]; }

// Unit u of the call for tp tokens a unit (without cu and in the decoder's form:
// token u alone); false if there is none.  The same in every lane.
template <class C>
__device__ __forceinline__ bool call_unit(const C& c, int u, int tp, CallUnit& q) {
    if (!c.cu) {
        q.seq = q.tok = u;
        q.n = 1;
        q.pos = min(call_row(c, u), c.maxT);                // (so that sums with q.n stay within an int)
        return true;
    }
    const int lane = threadIdx.x & 63;
    int base = 0;
    for (int s0 = 0; s0 < c.n_seq; s0 += 64) {
        const int s = s0 + lane;
        const int t0 = c.cu[min(s, c.n_seq)], t1 = c.cu[min(s + 1, c.n_seq)];
        const int n = s < c.n_seq ? max(t1 - t0, 0) : 0, p0 = c.start[min(s, c.n_seq - 1)];
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
            const long long p = (long long)__builtin_amdgcn_readlane(p0, l) + k * tp;
            q.pos = (int)(p < -c.N ? -c.N : p > c.maxT ? c.maxT : p);
            return q.n > 0 && q.tok >= 0;
        }
        base = all;
    }
    return false;
}

}  // namespace jm
