// What the two log-probability operators (logprobs.cu, linear_logprobs.cu) share: their outputs, the running softmax
// statistics of a row and how two parts of a row join.
#pragma once
#include "common.cuh"
#include "logprobs.h"

namespace mmz {

// Over a set of logits x: m the largest, s = sum e^(x - m), u = sum e^(x - m) (x - m). Then
//   lse = m + log s,   entropy = log s - u / s,   log p(t) = x_t - lse.
// The empty set, and one of -infinities only, has m = -inf and s = u = 0; a NaN makes s NaN.
struct RowStat {
    float m, s, u;
};

__device__ __forceinline__ RowStat stat_none() { return {-INFINITY, 0.f, 0.f}; }

constexpr float LOWEST = -3.402823466e38f, LOG2E = 1.4426950408889634f;

__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

// a thread's running maximum and sums; m starts at the lowest finite number, so that -inf adds e^(-inf) = 0 to every sum
struct Run {
    float m;
    float2 s, u;
    __device__ __forceinline__ void raise(float to) {
        if (to > m) {
            const float d = fmaxf(m - to, -200.f), e = ex2_approx(d * LOG2E);  // below e^-200 nothing is left
            u = ffma2(make_float2(d, d), s, u);
            u = make_float2(u.x * e, u.y * e);
            s = make_float2(s.x * e, s.y * e);
            m = to;
        }
    }
    __device__ __forceinline__ void add2(float a, float b) {
        float2 d = fadd2(make_float2(a, b), make_float2(-m, -m));
        d.x = max_nan(d.x, -200.f), d.y = max_nan(d.y, -200.f);  // a NaN stays; e = 0 for all that is cut
        const float2 e = make_float2(ex2_approx(d.x * LOG2E), ex2_approx(d.y * LOG2E));
        s = fadd2(s, e);
        u = ffma2(e, d, u);
    }
    // K pieces of N logits: one look at the maximum, two sets of sums
    template <int K, int N>
    __device__ __forceinline__ void add(const float (&x)[K][N], float h) {  // h: the largest of x
        raise(h);
        // the pieces' sums apart from the running ones, which so take one step for all of them (fp32 rounding)
        Run one{m, make_float2(0.f, 0.f), make_float2(0.f, 0.f)}, other = one;
#pragma unroll
        for (int k = 0; k < K; k++)
#pragma unroll
            for (int i = 0; i < N; i += 4) {
                one.add2(x[k][i], x[k][i + 1]);
                other.add2(x[k][i + 2], x[k][i + 3]);
            }
        s = fadd2(s, fadd2(one.s, other.s));
        u = fadd2(u, fadd2(one.u, other.u));
    }
};
// Whole warp: the lanes' statistics joined, in every lane. e^(x - M) (x - M) = e^(x - m) e^(m - M) ((x - m) + (m - M));
// nothing where e is 0 (a NaN stays in s)
__device__ __forceinline__ RowStat stat_warp(const RowStat& a) {
    float M = a.m;
#pragma unroll
    for (int w = 16; w; w >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffff, M, w));
    const float d = M == -INFINITY ? 0.f : a.m - M, e = __expf(d);
    float s = e * a.s, u = e > 0.f ? e * (a.u + d * a.s) : 0.f;
#pragma unroll
    for (int w = 16; w; w >>= 1) {
        s += __shfl_xor_sync(0xffffffff, s, w);
        u += __shfl_xor_sync(0xffffffff, u, w);
    }
    return {M, s, u};
}

// (value, lower id first) as one unsigned comparison; 0 stands for no candidate. -0 counts as +0. A NaN and -inf are no
// candidates.
__device__ __forceinline__ unsigned long long top_key(float v, int id) {
    if (!(v > -INFINITY)) return 0ull;
    uint32_t u = __float_as_uint(v + 0.f);
    u = (u & 0x80000000u) ? ~u : (u | 0x80000000u);
    return ((unsigned long long)u << 32) | (0xffffffffu - (uint32_t)id);
}
__device__ __forceinline__ int key_id(unsigned long long k) { return (int)(0xffffffffu - (uint32_t)k); }
__device__ __forceinline__ float key_value(unsigned long long k) {
    const uint32_t u = (uint32_t)(k >> 32);
    return __uint_as_float((u & 0x80000000u) ? (u & 0x7fffffffu) : ~u);
}

// The row's outputs except its alternatives; tgt: the target's logit (read only where the target is in [0, V)). Returns
// log s: a log probability is (x - m) - log s, which loses less than x - lse where it is close to 0
__device__ __forceinline__ float store_row(const LogpOut& o, long at, const RowStat& a, bool has_target, float tgt) {
    const bool none = a.m == -INFINITY && a.s == 0.f;
    const float ls = logf(a.m == INFINITY ? NAN : a.s), lse = none ? -INFINITY : a.m + ls;
    if (o.logp) o.logp[at] = !has_target ? 0.f : (tgt == -INFINITY && lse == lse) ? -INFINITY : (tgt - a.m) - ls;
    if (o.entropy) o.entropy[at] = none ? 0.f : ls - a.u / a.s;
    if (o.lse) o.lse[at] = lse;
    return ls;
}
// the index of row r's outputs; -1 where the column counter points outside them
__device__ __forceinline__ long row_at(const LogpOut& o, long r) {
    const int c = o.col ? *o.col : 0;
    return c >= 0 && c < o.ld ? r * o.ld + c : -1;
}
// one alternative of the row at `at`; key 0: none
__device__ __forceinline__ void store_top(const LogpOut& o, long at, int i, unsigned long long key, float m, float ls) {
    if (o.top_id) o.top_id[at * o.top + i] = key ? key_id(key) : -1;
    if (o.top_logp) o.top_logp[at * o.top + i] = key ? (key_value(key) - m) - ls : -INFINITY;
}

}  // namespace mmz
