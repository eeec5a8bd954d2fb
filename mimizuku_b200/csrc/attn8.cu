// Attention over the 8-bit key/value cache (kv8.cu), for sm_100a. For sequence b, query row i and query head h, with
// L = min(lens[b], cap) and key head g = h / (q_heads / kv_heads):
//     s_j = scale * ks[b][g][j / block] * (q . k8_j)    for j < limit,  limit = L, or L - rows + i + 1 when causal
//     out = sum_j softmax(s)_j * vs[b][g][j / block] * v8_j      (zeros where limit <= 0)
// and the probabilities of chosen heads as fp16. Products, sums and softmax statistics in fp32; only the outputs are
// rounded.
#include "attn8.h"
#include "fp8_cache.cuh"
#include "launch.h"

namespace mmz {
namespace a8 {
constexpr int NT = 128;
}  // namespace a8

// one CTA to a (sequence, query row, query head); a warp takes every fourth position, two dims to a lane
template <int KIND>
__global__ void __launch_bounds__(a8::NT) attn8_kernel(Attn8 a) {
    __shared__ float red[4][HD + 2];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int h = blockIdx.x % a.q_heads, i = (blockIdx.x / a.q_heads) % a.rows;
    const long b = blockIdx.x / a.q_heads / a.rows;
    const int g = h / (a.q_heads / a.kv_heads);
    griddep_wait();
    const int L = a.lens ? max(0, min(a.lens[b], a.cap)) : a.cap;
    const int limit = a.causal ? max(0, L - a.rows + i + 1) : L;
    const uint8_t* k8 = a.k8 + b * a.c_seq + g * a.c_head;
    const uint8_t* v8 = a.v8 + b * a.c_seq + g * a.c_head;
    const float* ks = a.ks + b * a.s_seq + g * a.s_head;
    const float* vs = a.vs + b * a.s_seq + g * a.s_head;
    const __half2 q2 = reinterpret_cast<const __half2*>(a.q + b * a.q_seq + i * a.q_row + h * a.q_head)[lane];
    const float2 q = __half22float2(q2);
    auto two = [&](const uint8_t* p) {
        const uint32_t w = reinterpret_cast<const uint16_t*>(p)[lane];
        if constexpr (KIND == KV8_E4M3) return h2_to_f2(e4m3x2_to_h2(w));
        return make_float2((float)(int8_t)w, (float)(int8_t)(w >> 8));
    };
    auto score = [&](long j) {
        const float2 k = two(k8 + j * HD);
        float s = q.x * k.x + q.y * k.y;
#pragma unroll
        for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffff, s, o);
        return s * ks[j / a.block] * a.scale;
    };
    float m = -INFINITY, l = 0.f;
    float2 acc = make_float2(0.f, 0.f);
    for (long j = warp; j < limit; j += 4) {
        const float s = score(j), mn = fmaxf(m, s), f = __expf(m - mn), p = __expf(s - mn);
        const float2 v = two(v8 + j * HD);
        const float vsc = p * vs[j / a.block];
        m = mn;
        l = l * f + p;
        acc.x = acc.x * f + vsc * v.x;
        acc.y = acc.y * f + vsc * v.y;
    }
    red[warp][2 * lane] = acc.x;
    red[warp][2 * lane + 1] = acc.y;
    if (lane == 0) red[warp][HD] = m, red[warp][HD + 1] = l;
    __syncthreads();
    float M = -INFINITY, S = 0.f;
    for (int w = 0; w < 4; w++) M = fmaxf(M, red[w][HD]);
    for (int w = 0; w < 4; w++) S += red[w][HD] == -INFINITY ? 0.f : red[w][HD + 1] * __expf(red[w][HD] - M);
    const float inv = S > 0.f ? 1.f / S : 0.f;
    if (threadIdx.x < HD) {
        float o = 0.f;
        for (int w = 0; w < 4; w++)
            o += red[w][HD] == -INFINITY ? 0.f : red[w][threadIdx.x] * __expf(red[w][HD] - M);
        a.out[b * a.o_seq + i * a.o_row + h * a.o_head + threadIdx.x] = __float2half_rn(o * inv);
    }
    const int slot = a.probs ? a.pslot[h] : -1;
    if (slot >= 0 && slot < a.slots) {
        h16* pr = a.probs + ((b * a.slots + slot) * a.rows + i) * (long)a.cap;
        for (long j = warp; j < a.cap; j += 4) {
            const float p = j < limit ? __expf(score(j) - M) * inv : 0.f;
            if (lane == 0) pr[j] = __float2half_rn(p);
        }
    }
}

size_t attn8_scratch_bytes(int, int, int, int, int, int) { return 0; }

int launch_attn8(const Attn8& a, int kind, void*, size_t, cudaStream_t st) {
    if (a.batch < 0 || a.rows < 0 || a.kv_heads < 1 || a.q_heads < 1 || a.cap < 1 || a.slots < 0)
        return fail("attn8: batch >= 0, rows >= 0, heads >= 1, cap >= 1");
    if (a.q_heads % a.kv_heads) return fail("attn8: q_heads a multiple of kv_heads");
    if (!kv8_block_ok(a.block)) return fail("attn8: block is 16, 32, 64 or 128");
    if (kind != KV8_INT8 && kind != KV8_E4M3) return fail("attn8: kind is 0 (int8) or 1 (e4m3)");
    if (a.batch == 0 || a.rows == 0) return 0;
    if (!a.q || !a.k8 || !a.v8 || !a.ks || !a.vs || !a.out) return fail("attn8: null pointer");
    if (a.probs && !a.pslot) return fail("attn8: probs without pslot");
    if (((uintptr_t)a.q | (uintptr_t)a.out | (uintptr_t)a.k8 | (uintptr_t)a.v8 | (uintptr_t)a.probs) & 15)
        return fail("attn8: q, out, probs and the cache 16-byte aligned");
    if ((a.q_seq | a.q_row | a.q_head | a.o_seq | a.o_row | a.o_head) & 7)
        return fail("attn8: strides of q and out multiples of 8 values");
    if ((a.c_seq | a.c_head) & 15) return fail("attn8: strides of the cache multiples of 16 bytes");
    const long grid = (long)a.batch * a.rows * a.q_heads;
    if (grid > 0x7fffffffl) return fail("attn8: more than 2^31 rows and heads in one call");
    DevCtx& dc = dev_ctx();
    if (!dc.ok) return fail(dc.err);
    auto* fn = kind == KV8_INT8 ? attn8_kernel<KV8_INT8> : attn8_kernel<KV8_E4M3>;
    return check_pdl(launch_pdl(fn, dim3((unsigned)grid), dim3(a8::NT), 0, st, a), "attn8");
}

}  // namespace mmz
