// Writing and reading the 8-bit key/value cache, for sm_100a. No counterpart in the reference, whose caches are fp16
// (src/model.rs:440-446). The cache holds, per sequence and head, `cap` rows of 64 one-byte codes and one fp32 scale
// for every `block` of them: value = code * scale.
//
// kv8_write, tokens x at positions pos .. pos + n: for each block touched
//     a = max |x| over the block's new tokens,  s = a / Q  (Q = 127 for int8, 448 for e4m3)
//     s = max(s, the block's earlier scale)  where the block has tokens before pos
//     code = round_to_even(x / s)  (0 where s is 0: an all-zero block)
// and, where s grew, the earlier tokens' codes become round_to_even(code * s_old / s): a scale only grows while its
// block fills, so a code is rounded again at most as often as the block's maximum grows. x / s is the quotient by the
// unrounded scale, x Q / a (or by the block's earlier scale where that stays), rounded to fp32 once: 1 / s is kept as
// r + rl, and x / s = x r + x rl with one rounding that counts. (fp16 values often lie halfway between two codes exactly; a
// product by a rounded 1 / s misses so many of them that 1 code in 22 thousand is the wrong one, a whole step off.)
//
// Bound by memory: 2 bytes read and 1 written per value (and the reverse to read). 32 x 20 heads x 1500 tokens, keys and
// values: written in 71 us = 5.2 TB/s, read back in 55 to 59 us (369 MB, of whose 246 MB written 58 are still in L2 at the
// end: no memory rate). A warp takes 32 tokens of one block (8 lanes to a token, 16 bytes each), so that its 8 loads are all
// in flight before the maximum is known and the values are read once; blocks of 64 and 128 tokens are shared by 2 and 4
// warps of the CTA, which exchange their maxima in shared memory.
#include "fp8_cache.cuh"
#include "launch.h"

namespace mmz {
namespace kv8 {
constexpr int NT = 128;

// where a cache's codes (bytes) and scales (floats) of sequence b and head h start
struct Cache {
    uint8_t *k, *v;
    float *ks, *vs;
    long c_seq, c_head, s_seq, s_head;
};

__device__ __forceinline__ float finite(float x) {  // fp16 infinities count as the largest finite number
    return fabsf(x) > 65504.f ? copysignf(65504.f, x) : x;
}
}  // namespace kv8
using namespace kv8;

// grid: items / (4 / W) CTAs, an item = one (sequence, head, k or v, block); W warps to an item
template <int KIND>
__global__ void __launch_bounds__(NT) kv8_write_kernel(const h16* k, const h16* v, long x_seq,
                                                       long x_tok, long x_head, Cache c, const int* pos,
                                                       int heads, int n, int cap, int block, int nblk, unsigned items) {
    __shared__ float wmax[4];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int W = block <= 32 ? 1 : block / 32, tw = block < 32 ? block : 32;  // warps to an item, tokens to a warp
    const unsigned item = blockIdx.x * (4 / W) + warp / W;
    griddep_wait();
    griddep_launch_dependents();
    const bool live = item < items;
    const unsigned rest = live ? item / nblk : 0, pair = rest >> 1;
    const int ib = live ? (int)(item - rest * nblk) : 0, isv = rest & 1, hd = pair % heads;
    const long b = pair / heads;
    const int p0 = pos ? pos[b] : 0;
    // the first block with a new token at a position >= 0; blocks past the capacity or the last token have nothing
    const long first = p0 > 0 ? p0 / block : 0;
    const long blk = first + ib;
    const long t0 = blk * block + (warp % W) * tw;  // this warp's first position
    const long end = min((long)p0 + n, (long)cap);
    const bool any = live && blk * block < end;
    const h16* x = (isv ? v : k) + b * x_seq + hd * x_head;
    uint8_t* codes = (isv ? c.v : c.k) + b * c.c_seq + hd * c.c_head;
    float* scale = (isv ? c.vs : c.ks) + b * c.s_seq + hd * c.s_head + blk;
    const int sub = lane >> 3, d0 = (lane & 7) * 8;
    uint4 val[8];
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const long j = t0 + 4 * i + sub;
        val[i] = make_uint4(0, 0, 0, 0);
        if (any && 4 * i < tw && j >= p0 && j < end) val[i] = *reinterpret_cast<const uint4*>(x + (j - p0) * x_tok + d0);
    }
    // the largest magnitude, in fp16; a NaN or an infinity among the CTA's values is rare, and asked for only once
    __half2 big = __half2half2(__ushort_as_half(0));
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const __half2* w = reinterpret_cast<const __half2*>(&val[i]);
#pragma unroll
        for (int q = 0; q < 4; q++) big = __hmax2_nan(big, __habs2(w[q]));
    }
    float amax = __half2float(__hmax_nan(__low2half(big), __high2half(big)));
    const bool odd = __any_sync(0xffffffff, !(amax <= 65504.f));
    if (odd) {
        amax = 0.f;
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const uint32_t w[4] = {val[i].x, val[i].y, val[i].z, val[i].w};
#pragma unroll
            for (int q = 0; q < 4; q++) {
                const float2 p = h2_to_f2(w[q]);
                amax = fmaxf(amax, fmaxf(fabsf(finite(p.x)), fabsf(finite(p.y))));  // fmaxf drops a NaN
            }
        }
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffff, amax, o));
    const bool older = any && blk * block < p0;
    const float s_old = older ? *scale : 0.f;
    if (W > 1) {
        if (lane == 0) wmax[warp] = amax;
        __syncthreads();  // every warp of the CTA comes here; the earlier scale is read before it and written after it
        const int w0 = warp / W * W;
        for (int i = 0; i < W; i++) amax = fmaxf(amax, wmax[w0 + i]);
    } else {
        __syncwarp();
    }
    if (!any) return;
    const float s_new = __fdiv_rn(amax, kv8_top<KIND>());
    const bool kept = s_old > s_new;  // the earlier scale stays
    const float s = kept ? s_old : s_new, num = kept ? 1.f : kv8_top<KIND>(), den = kept ? s_old : amax;
    const float r = s > 0.f ? __fdiv_rn(num, den) : 0.f, rl = r > 0.f ? __fdiv_rn(__fmaf_rn(-r, den, num), den) : 0.f;
    auto over = [&](float x) { return __fmaf_rn(x, r, __fmul_rn(x, rl)); };
    if (lane == 0 && warp % W == 0) *scale = s;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const long j = t0 + 4 * i + sub;
        if (4 * i >= tw || j < p0 || j >= end) continue;
        const uint32_t w[4] = {val[i].x, val[i].y, val[i].z, val[i].w};
        uint2 o;
        uint32_t* op = &o.x;
#pragma unroll
        for (int q = 0; q < 2; q++) {
            const float2 a = h2_to_f2(w[2 * q]), e = h2_to_f2(w[2 * q + 1]);
            if (!odd) {
                op[q] = kv8_store4_finite<KIND>(make_float2(over(a.x), over(a.y)), make_float2(over(e.x), over(e.y)));
                continue;
            }
            const float y[4] = {over(finite(a.x)), over(finite(a.y)), over(finite(e.x)), over(finite(e.y))};
            op[q] = kv8_store4<KIND>(y);
        }
        *reinterpret_cast<uint2*>(codes + j * HD + d0) = o;
    }
    if (older && s != s_old) {  // the scale grew: the block's earlier codes on the new one
        const float f = __fmul_rn(s_old, r), fl = __fmaf_rn(s_old, rl, __fmaf_rn(s_old, r, -f));
        for (long j = t0 + sub; j < min(t0 + tw, (long)p0); j += 4) {
            uint2* at = reinterpret_cast<uint2*>(codes + j * HD + d0);
            uint2 o = *at;
            uint32_t* op = &o.x;
#pragma unroll
            for (int q = 0; q < 2; q++) {
                float y[4];
                kv8_load4<KIND>(op[q], y);
#pragma unroll
                for (int e = 0; e < 4; e++) y[e] = __fmaf_rn(y[e], f, __fmul_rn(y[e], fl));
                op[q] = kv8_store4<KIND>(y);
            }
            *at = o;
        }
    }
}

// CTA: 128 tokens of one (sequence, head, k or v); 8 lanes to a token, 4 tokens of a thread in flight
template <int KIND>
__global__ void __launch_bounds__(256) kv8_read_kernel(Cache c, h16* k, h16* v, long y_seq, long y_tok, long y_head,
                                                       const int* pos, const int* lens, int heads, int n, int cap,
                                                       int shift, unsigned tiles) {
    const unsigned rest = blockIdx.x / tiles, tile = blockIdx.x - rest * tiles, pair = rest >> 1;
    const int isv = rest & 1, hd = pair % heads, d0 = (threadIdx.x & 7) * 8;
    const long b = pair / heads;
    griddep_wait();
    griddep_launch_dependents();
    const long p0 = pos ? pos[b] : 0;
    const int end = lens ? min(lens[b], cap) : cap;
    const uint8_t* codes = (isv ? c.v : c.k) + b * c.c_seq + hd * c.c_head + d0;
    const float* scale = (isv ? c.vs : c.ks) + b * c.s_seq + hd * c.s_head;
    h16* y = (isv ? v : k) + b * y_seq + hd * y_head + d0;
    const int t0 = (int)tile * 128 + (threadIdx.x >> 3);
    uint2 w[4];
    float s[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const long j = p0 + t0 + 32 * i;
        w[i] = make_uint2(0, 0), s[i] = 0.f;
        if (t0 + 32 * i < n && j >= 0 && j < end) {
            w[i] = *reinterpret_cast<const uint2*>(codes + j * HD);
            s[i] = scale[j >> shift];
        }
    }
#pragma unroll
    for (int i = 0; i < 4; i++) {
        if (t0 + 32 * i >= n) break;
        uint4 o;
        float x[4];
        __half2* op = reinterpret_cast<__half2*>(&o);
#pragma unroll
        for (int q = 0; q < 2; q++) {
            kv8_load4<KIND>(q ? w[i].y : w[i].x, x);
            op[2 * q] = __floats2half2_rn(__fmul_rn(x[0], s[i]), __fmul_rn(x[1], s[i]));
            op[2 * q + 1] = __floats2half2_rn(__fmul_rn(x[2], s[i]), __fmul_rn(x[3], s[i]));
        }
        *reinterpret_cast<uint4*>(y + (t0 + 32 * i) * y_tok) = o;
    }
}

// what both calls ask of their arguments; 0 or the last error set
static int kv8_check(const char* what, const void* k, const void* v, const void* k8, const void* v8, const void* ks,
                     const void* vs, long long x_seq, long long x_tok, long long x_head, long long c_seq,
                     long long c_head, int batch, int heads, int n, int cap, int block, int kind) {
    if (batch < 0 || heads < 1 || n < 0 || cap < 1) return failf("%s: batch >= 0, heads >= 1, n >= 0, cap >= 1", what);
    if (cap > 0x7fff0000) return failf("%s: cap up to 2^31 - 65536", what);
    if (!kv8_block_ok(block)) return failf("%s: block is 16, 32, 64 or 128", what);
    if (kind != KV8_INT8 && kind != KV8_E4M3) return failf("%s: kind is 0 (int8) or 1 (e4m3)", what);
    if (batch == 0 || n == 0) return 0;
    if (!k || !v || !k8 || !v8 || !ks || !vs) return failf("%s: null pointer", what);
    if (((uintptr_t)k | (uintptr_t)v | (uintptr_t)k8 | (uintptr_t)v8) & 15)
        return failf("%s: k, v and the cache 16-byte aligned", what);
    if ((x_seq | x_tok | x_head) & 7) return failf("%s: strides of k and v multiples of 8 values", what);
    if ((c_seq | c_head) & 15) return failf("%s: strides of the cache multiples of 16 bytes", what);
    return 0;
}

int launch_kv8_write(const void* k, const void* v, long long x_seq, long long x_tok, long long x_head, void* k8,
                     void* v8, float* ks, float* vs, long long c_seq, long long c_head, long long s_seq,
                     long long s_head, const int* pos, int batch, int heads, int n, int cap, int block, int kind,
                     cudaStream_t st) {
    if (kv8_check("kv8_write", k, v, k8, v8, ks, vs, x_seq, x_tok, x_head, c_seq, c_head, batch, heads, n, cap, block,
                  kind))
        return -1;
    if (batch == 0 || n == 0) return 0;
    // blocks that n tokens can touch, from any position
    const int most = (cap + block - 1) / block;
    const long touched = pos ? ((long)n + block - 2) / block + 1 : ((long)n + block - 1) / block;
    const int nblk = (int)(touched < most ? touched : most);
    const int per = block <= 32 ? 4 : 128 / block;
    if (!within(std::min(0xffffff00l, 0x7fffffffl * per), {batch, heads, 2, nblk}))
        return fail("kv8_write: more than 2^31 blocks in one call");
    const long items = (long)batch * heads * 2 * nblk, grid = (items + per - 1) / per;
    // two sequences or heads in one place would be written by two blocks at once
    if (!apart((long long)cap * HD, {{batch, c_seq}, {heads, c_head}}) || !apart(most, {{batch, s_seq}, {heads, s_head}}))
        return fail("kv8_write: the cache's sequences and heads overlap");
    if (meet((uint8_t*)v8 - (uint8_t*)k8, (long long)cap * HD, {{batch, c_seq}, {heads, c_head}}) ||
        meet(vs - ks, most, {{batch, s_seq}, {heads, s_head}}))
        return fail("kv8_write: the cache's keys and values overlap");
    DevCtx& dc = dev_ctx();
    if (!dc.ok) return fail(dc.err);
    const Cache c{(uint8_t*)k8, (uint8_t*)v8, ks, vs, (long)c_seq, (long)c_head, (long)s_seq, (long)s_head};
    auto* fn = kind == KV8_INT8 ? kv8_write_kernel<KV8_INT8> : kv8_write_kernel<KV8_E4M3>;
    return check_pdl(launch_pdl(fn, dim3((unsigned)grid), dim3(NT), 0, st, (const h16*)k, (const h16*)v, (long)x_seq,
                                (long)x_tok, (long)x_head, c, pos, heads, n, cap, block, nblk, (unsigned)items),
                     "kv8_write");
}

int launch_kv8_read(const void* k8, const void* v8, const float* ks, const float* vs, long long c_seq, long long c_head,
                    long long s_seq, long long s_head, void* k, void* v, long long y_seq, long long y_tok,
                    long long y_head, const int* pos, const int* lens, int batch, int heads, int n, int cap, int block,
                    int kind, cudaStream_t st) {
    if (kv8_check("kv8_read", k, v, k8, v8, ks, vs, y_seq, y_tok, y_head, c_seq, c_head, batch, heads, n, cap, block,
                  kind))
        return -1;
    if (batch == 0 || n == 0) return 0;
    const long tiles = ((long)n + 127) / 128;
    if (!within(0x7fffffffl, {batch, heads, 2, tiles})) return fail("kv8_read: more than 2^31 blocks in one call");
    const long grid = (long)batch * heads * 2 * tiles;
    if (!apart(HD, {{batch, y_seq}, {n, y_tok}, {heads, y_head}})) return fail("kv8_read: tokens of k and v overlap");
    if (meet((h16*)v - (h16*)k, HD, {{batch, y_seq}, {n, y_tok}, {heads, y_head}})) return fail("kv8_read: k and v overlap");
    DevCtx& dc = dev_ctx();
    if (!dc.ok) return fail(dc.err);
    const Cache c{(uint8_t*)k8, (uint8_t*)v8, (float*)ks, (float*)vs, (long)c_seq, (long)c_head, (long)s_seq, (long)s_head};
    auto* fn = kind == KV8_INT8 ? kv8_read_kernel<KV8_INT8> : kv8_read_kernel<KV8_E4M3>;
    return check_pdl(launch_pdl(fn, dim3((unsigned)grid), dim3(256), 0, st, c, (h16*)k, (h16*)v, (long)y_seq,
                                (long)y_tok, (long)y_head, pos, lens, heads, n, cap, 31 - __builtin_clz(block),
                                (unsigned)tiles),
                     "kv8_read");
}

}  // namespace mmz
