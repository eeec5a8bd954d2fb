// Log probabilities from rows of logits, for sm_100a: of a given token, the entropy of the distribution and its
// largest entries. Over the ids whose sup[id] is 0 (argmax_tok's mask, kernels/whisper.cu:451-493):
//     lse = m + log sum e^(x - m),   logp = x_t - lse,   entropy = log sum e^(x - m) - sum e^(x - m) (x - m) / sum e^(x - m)
// and the `top` largest logits, equal ones by the lower id, each with its log probability. Sums in fp32.
#include "launch.h"
#include "logprobs.cuh"

namespace mmz {
namespace lp {
constexpr int NT = 512;
}  // namespace lp

template <typename T>
__global__ void __launch_bounds__(lp::NT) token_logprobs_kernel(const T* x, long ldx, int V,
                                                                const unsigned char* sup, LogpOut o) {
    __shared__ RowStat st[16];
    __shared__ unsigned long long best[16];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const long row = blockIdx.x;
    griddep_wait();
    const T* xr = x + row * ldx;
    const long at = row_at(o, row);
    if (at < 0) return;
    auto logit = [&](int i) { return sup && sup[i] ? -INFINITY : (float)xr[i]; };
    RowStat a = stat_none();
    for (int i = threadIdx.x; i < V; i += lp::NT) stat_add(a, logit(i));
#pragma unroll
    for (int w = 16; w; w >>= 1)
        a = stat_join(a, {__shfl_xor_sync(0xffffffff, a.m, w), __shfl_xor_sync(0xffffffff, a.s, w),
                          __shfl_xor_sync(0xffffffff, a.u, w)});
    if (lane == 0) st[warp] = a;
    __syncthreads();
    a = st[0];
    for (int w = 1; w < lp::NT / 32; w++) a = stat_join(a, st[w]);
    float lse = 0.f;
    if (threadIdx.x == 0) {
        const int t = o.target ? o.target[at] : -1;
        const bool has = t >= 0 && t < V;
        lse = store_row(o, at, a, has, has ? logit(t) : 0.f);
    }
    unsigned long long last = ~0ull;
    for (int k = 0; k < o.top; k++) {
        unsigned long long b = 0;
        for (int i = threadIdx.x; i < V; i += lp::NT) {
            const unsigned long long key = top_key(logit(i), i);
            if (key < last && key > b) b = key;
        }
#pragma unroll
        for (int w = 16; w; w >>= 1) {
            const unsigned long long c = __shfl_xor_sync(0xffffffff, b, w);
            b = c > b ? c : b;
        }
        if (lane == 0) best[warp] = b;
        __syncthreads();
        for (int w = 0; w < lp::NT / 32; w++) b = best[w] > b ? best[w] : b;
        __syncthreads();
        if (threadIdx.x == 0) store_top(o, at, k, b, lse);
        last = b;
    }
}

// what both operators ask of their outputs
int logp_check(const char* what, const LogpOut& o) {
    if (o.top < 0 || o.top > TOP_MAX) return failf("%s: 0 to %d alternatives", what, TOP_MAX);
    if (o.ld < 1) return failf("%s: a stride of at least 1 between the rows' outputs", what);
    if (o.logp && !o.target) return failf("%s: logp without target", what);
    return 0;
}

int launch_token_logprobs(const void* x, long long ldx, int type, int rows, int V, const unsigned char* sup,
                          const LogpOut& o, cudaStream_t st) {
    if (rows < 0 || V < 1 || ldx < V) return fail("token_logprobs: rows >= 0, vocab >= 1, ldx >= vocab");
    if (type != 0 && type != 1) return fail("token_logprobs: type is 0 (fp16) or 1 (fp32)");
    if (logp_check("token_logprobs", o)) return -1;
    if (rows == 0) return 0;
    if (!x || ((uintptr_t)x & (type ? 3 : 1))) return fail("token_logprobs: logits null or not aligned to their type");
    DevCtx& dc = dev_ctx();
    if (!dc.ok) return fail(dc.err);
    return check_pdl(type ? launch_pdl(token_logprobs_kernel<float>, dim3(rows), dim3(lp::NT), 0, st, (const float*)x,
                                       (long)ldx, V, sup, o)
                          : launch_pdl(token_logprobs_kernel<h16>, dim3(rows), dim3(lp::NT), 0, st, (const h16*)x,
                                       (long)ldx, V, sup, o),
                     "token_logprobs");
}

}  // namespace mmz
