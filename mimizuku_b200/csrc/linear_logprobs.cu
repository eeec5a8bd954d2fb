// Log probabilities from hidden states, for sm_100a: token_logprobs (logprobs.cu) of the logits x . emb^T, which keep
// the product's fp32 sums (no rounding between the product and the softmax).
#include "launch.h"
#include "logprobs.cuh"

namespace mmz {
namespace ll {
constexpr int T = 64;  // tile of the product
}  // namespace ll

// y[rows][V] = x . emb^T, 64 x 64 tiles, 4 x 4 sums to a thread
__global__ void __launch_bounds__(256) linear_kernel(const h16* x, long ldx, const h16* emb,
                                                     int rows, int V, int d, float* y) {
    __shared__ float xs[16][ll::T + 1], es[16][ll::T + 1];
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    const long r0 = (long)blockIdx.y * ll::T, v0 = (long)blockIdx.x * ll::T;
    griddep_wait();
    float acc[4][4] = {};
    for (int k0 = 0; k0 < d; k0 += 16) {
        for (int i = threadIdx.x; i < 16 * ll::T; i += 256) {
            const int k = i & 15, r = i >> 4;
            xs[k][r] = r0 + r < rows ? f(x[(r0 + r) * ldx + k0 + k]) : 0.f;
            es[k][r] = v0 + r < V ? f(emb[(v0 + r) * d + k0 + k]) : 0.f;
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < 16; k++)
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
                for (int j = 0; j < 4; j++) acc[i][j] += xs[k][ty + 16 * i] * es[k][tx + 16 * j];
        __syncthreads();
    }
    for (int i = 0; i < 4; i++)
        for (int j = 0; j < 4; j++) {
            const long r = r0 + ty + 16 * i, v = v0 + tx + 16 * j;
            if (r < rows && v < V) y[r * V + v] = acc[i][j];
        }
}

size_t linear_logprobs_scratch_bytes(int rows, int V, int) { return ((size_t)rows * V * 4 + 15) & ~(size_t)15; }

int launch_linear_logprobs(const void* x, long long ldx, const void* emb, int rows, int V, int d,
                           const unsigned char* sup, const LogpOut& o, void* scratch, size_t scratch_bytes,
                           cudaStream_t st) {
    if (rows < 0 || V < 1 || d < 64 || d % 64) return fail("linear_logprobs: rows >= 0, vocab >= 1, width a multiple of 64");
    if (logp_check("linear_logprobs", o)) return -1;
    if (rows == 0) return 0;
    if (!x || !emb || (((uintptr_t)x | (uintptr_t)emb) & 15) || (ldx & 7) || ldx < d)
        return fail("linear_logprobs: x and emb 16-byte aligned, ldx >= width with a 16-byte row pitch");
    const size_t need = linear_logprobs_scratch_bytes(rows, V, d);
    if (need && (!scratch || ((uintptr_t)scratch & 15) || scratch_bytes < need))
        return fail("linear_logprobs: scratch too small or not 16-byte aligned");
    DevCtx& dc = dev_ctx();
    if (!dc.ok) return fail(dc.err);
    const dim3 grid((V + ll::T - 1) / ll::T, (rows + ll::T - 1) / ll::T);
    if (grid.y > 65535) return fail("linear_logprobs: too many rows in one call");
    if (check_pdl(launch_pdl(linear_kernel, grid, dim3(256), 0, st, (const h16*)x, (long)ldx, (const h16*)emb, rows, V, d,
                             (float*)scratch),
                  "linear_logprobs"))
        return -1;
    return launch_token_logprobs(scratch, V, 1, rows, V, sup, o, st);
}

}  // namespace mmz
