// Log probabilities from rows of logits, for sm_100a: of a given token, the entropy of the distribution and its
// largest entries. Over the ids whose sup[id] is 0 (argmax_tok's mask, kernels/whisper.cu:451-493):
//     lse = m + log sum e^(x - m),   logp = x_t - lse,   entropy = log sum e^(x - m) - sum e^(x - m) (x - m) / sum e^(x - m)
// and the `top` largest logits, equal ones by the lower id, each with its log probability. Sums in fp32.
//
// Bound by reading the logits, once: a cluster of 1 to 8 CTAs takes a row, a thread 8 logits at a time (16-byte loads
// from the row's first aligned address on, 64 bytes of a thread in flight), with a running maximum and the two sums in
// packed fp32. The alternatives cost no work per logit: a thread's running maximum is its largest logit, so after the
// pass the top-th largest of the warps' maxima is a bound below which no alternative lies, and only threads whose own
// maximum reaches it (about as many as there are alternatives) have their logits read again, by their whole warp. What
// reaches the bound is ranked by counting. Where more than LIST logits do (rows of equal logits), the alternatives are
// found one after another in `top` passes instead.
#include "launch.h"
#include "logprobs.cuh"

namespace mmz {
namespace lp {
constexpr int NT = 512, NW = NT / 32;
constexpr int LIST = 1024;  // candidates of a CTA
constexpr float LOWEST = -3.402823466e38f, LOG2E = 1.4426950408889634f;

struct Smem {
    unsigned long long list[LIST], best[TOP_MAX], all[8][TOP_MAX];  // all: every CTA's, in the cluster's first
    float wm[NW], ws[NW], wu[NW];
    RowStat stat[8];
    float tau;
    int n;
};

__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

// 8 logits from a 16-byte aligned address
__device__ __forceinline__ void load8(const h16* p, uint4 (&r)[1]) { r[0] = *reinterpret_cast<const uint4*>(p); }
__device__ __forceinline__ void load8(const float* p, uint4 (&r)[2]) {
    r[0] = reinterpret_cast<const uint4*>(p)[0];
    r[1] = reinterpret_cast<const uint4*>(p)[1];
}
__device__ __forceinline__ void floats(const uint4 (&r)[1], float (&x)[8]) {
    const __half2* h = reinterpret_cast<const __half2*>(&r[0]);
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const float2 f = __half22float2(h[i]);
        x[2 * i] = f.x, x[2 * i + 1] = f.y;
    }
}
__device__ __forceinline__ void floats(const uint4 (&r)[2], float (&x)[8]) {
    const float* f = reinterpret_cast<const float*>(&r[0]);
#pragma unroll
    for (int i = 0; i < 8; i++) x[i] = f[i];
}

// the mask bytes of ids i .. i + 7: two aligned words where both lie inside the mask, else byte by byte
__device__ __forceinline__ unsigned long long mask8(const unsigned char* sup, int i, int V) {
    const uintptr_t a = (uintptr_t)(sup + i), w = a & ~(uintptr_t)7;
    const int sh = 8 * (int)(a & 7);
    if (w >= (uintptr_t)sup && w + 16 <= (uintptr_t)(sup + V)) {
        const unsigned long long lo = *(const unsigned long long*)w;
        return sh ? (lo >> sh) | (*(const unsigned long long*)(w + 8) << (64 - sh)) : lo;
    }
    unsigned long long m = 0;
    for (int k = 0; k < 8; k++) m |= (unsigned long long)(sup[i + k] != 0) << (8 * k);
    return m;
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
    __device__ __forceinline__ void add8(const float (&x)[8]) {
        raise(fmax3(fmax3(x[0], x[1], x[2]), fmax3(x[3], x[4], x[5]), fmaxf(x[6], x[7])));
#pragma unroll
        for (int i = 0; i < 8; i += 2) add2(x[i], x[i + 1]);
    }
};
}  // namespace lp
using namespace lp;

template <typename T>
__global__ void __launch_bounds__(NT, 2) token_logprobs_kernel(const T* x, long ldx, int V, const unsigned char* sup,
                                                               LogpOut o, int lg) {
    constexpr int NL = sizeof(T) / 2;        // 16-byte loads of 8 logits
    constexpr int UN = NL == 1 ? 4 : 2;      // vectors of a thread in flight
    __shared__ Smem sm;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, cl = 1 << lg, rank = blockIdx.x & (cl - 1);
    const long row = blockIdx.x >> lg;
    if (threadIdx.x == 0) sm.n = 0;
    griddep_wait();
    griddep_launch_dependents();
    const long at = row_at(o, row);
    if (at < 0) return;  // the whole cluster
    if (cl > 1) cluster_arrive_relaxed();  // the first CTA has started before anything is sent to it
    const T* xr = x + row * ldx;
    // ids before the first aligned address, vectors of 8, ids after the last vector; this CTA's share
    const int head = min(V, (int)((16 - ((uintptr_t)xr & 15)) & 15) / (int)sizeof(T));
    const int nv = (V - head) / 8, tail = head + nv * 8;
    const int v0 = (int)((long)nv * rank >> lg), v1 = (int)((long)nv * (rank + 1) >> lg);
    const int t = o.target ? o.target[at] : -1;
    auto logit = [&](int i) { return sup && sup[i] ? -INFINITY : (float)xr[i]; };
    const bool has = t >= 0 && t < V;
    float tgt = 0.f;
    if (rank == 0 && threadIdx.x == 0 && has) tgt = logit(t);

    auto vec = [&](int v, const uint4 (&r)[NL], float (&f)[8]) {  // vector v's logits, -inf for what is left out
        floats(r, f);
        if (sup) {
            const unsigned long long m = mask8(sup, head + 8 * v, V);
            if (m)
#pragma unroll
                for (int k = 0; k < 8; k++)
                    if (m >> (8 * k) & 0xff) f[k] = -INFINITY;
        }
    };
    // the ids outside the vectors: at most 7 before, with the first CTA, and 7 after, with the last
    const int edge = threadIdx.x < 8 ? (rank == 0 && threadIdx.x < head ? threadIdx.x : -1)
                     : threadIdx.x < 16 && rank == cl - 1 && tail + threadIdx.x - 8 < V ? tail + (int)threadIdx.x - 8 : -1;
    Run run{LOWEST, make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
    if (edge >= 0) {
        const float e = logit(edge);
        run.raise(e);
        run.add2(e, -INFINITY);
    }
    for (int v = v0 + threadIdx.x; v < v1; v += UN * NT) {
        uint4 r[UN][NL];
#pragma unroll
        for (int k = 0; k < UN; k++)
            if (v + k * NT < v1) load8(xr + head + 8l * (v + k * NT), r[k]);
#pragma unroll
        for (int k = 0; k < UN; k++)
            if (v + k * NT < v1) {
                float f[8];
                vec(v + k * NT, r[k], f);
                run.add8(f);
            }
    }
    // ---------------------------------------------------------------- the CTA's statistics
    const float mine = run.m;
    float wm = mine;
#pragma unroll
    for (int w = 16; w; w >>= 1) wm = fmaxf(wm, __shfl_xor_sync(0xffffffff, wm, w));
    if (lane == 0) sm.wm[warp] = wm;
    __syncthreads();
    float M = LOWEST;
#pragma unroll
    for (int w = 0; w < NW; w++) M = fmaxf(M, sm.wm[w]);
    run.raise(M);
    float S = run.s.x + run.s.y, U = run.u.x + run.u.y;
#pragma unroll
    for (int w = 16; w; w >>= 1) {
        S += __shfl_xor_sync(0xffffffff, S, w);
        U += __shfl_xor_sync(0xffffffff, U, w);
    }
    if (lane == 0) sm.ws[warp] = S, sm.wu[warp] = U;
    // ---------------------------------------------------------------- its alternatives
    if (o.top > 0) {
        if (warp == 0 && lane < NW) {  // the top-th largest of the warps' maxima
            const float a = sm.wm[lane];
            int above = 0;
#pragma unroll
            for (int w = 0; w < NW; w++) above += sm.wm[w] > a || (sm.wm[w] == a && w < lane);
            if (above == o.top - 1) sm.tau = a;
        }
        __syncthreads();
        const float tau = sm.tau;
        auto take = [&](float f, int id) {
            const unsigned long long key = f >= tau ? top_key(f, id) : 0ull;
            if (key) {
                const int k = atomicAdd(&sm.n, 1);
                if (k < LIST) sm.list[k] = key;
            }
        };
        if (edge >= 0) take(logit(edge), edge);
        for (unsigned who = __ballot_sync(0xffffffff, mine >= tau); who; who &= who - 1) {
            const int first = v0 + warp * 32 + __ffs(who) - 1;  // the thread's vectors: every NT-th from here
            for (int v = first + lane * NT; v < v1; v += 32 * NT) {
                uint4 r[NL];
                float f[8];
                load8(xr + head + 8l * v, r);
                vec(v, r, f);
#pragma unroll
                for (int k = 0; k < 8; k++) take(f[k], head + 8 * v + k);
            }
        }
        if (threadIdx.x < TOP_MAX) sm.best[threadIdx.x] = 0ull;
        __syncthreads();
        const int n = sm.n;
        if (n <= LIST) {
            for (int i = threadIdx.x; i < n; i += NT) {  // a key's rank is the number of larger ones: no two are equal
                const unsigned long long key = sm.list[i];
                int above = 0;
                for (int k = 0; k < n && above < o.top; k++) above += sm.list[k] > key;
                if (above < o.top) sm.best[above] = key;
            }
        } else {
            unsigned long long last = ~0ull;
            for (int k = 0; k < o.top; k++) {
                unsigned long long b = 0;
                auto see = [&](float f, int id) {
                    const unsigned long long key = top_key(f, id);
                    if (key < last && key > b) b = key;
                };
                if (edge >= 0) see(logit(edge), edge);
                for (int v = v0 + threadIdx.x; v < v1; v += NT) {
                    uint4 r[NL];
                    float f[8];
                    load8(xr + head + 8l * v, r);
                    vec(v, r, f);
#pragma unroll
                    for (int e = 0; e < 8; e++) see(f[e], head + 8 * v + e);
                }
#pragma unroll
                for (int w = 16; w; w >>= 1) {
                    const unsigned long long c = __shfl_xor_sync(0xffffffff, b, w);
                    b = c > b ? c : b;
                }
                if (lane == 0) sm.list[warp] = b;
                __syncthreads();
                for (int w = 0; w < NW; w++) b = sm.list[w] > b ? sm.list[w] : b;
                __syncthreads();
                if (threadIdx.x == 0) sm.best[k] = b;
                last = b;
            }
        }
    }
    __syncthreads();
    if (cl > 1) cluster_wait();
    // ---------------------------------------------------------------- the cluster's CTAs joined in its first
    if (warp == 0) {
        if (lane == 0) {
            S = U = 0.f;
            for (int w = 0; w < NW; w++) S += sm.ws[w], U += sm.wu[w];
            const uint32_t to = dsmem_addr(&sm.stat[rank], 0);
            st_dsmem_f32(to, S == 0.f ? -INFINITY : M);  // nothing above -inf: the empty set
            st_dsmem_f32(to + 4, S);
            st_dsmem_f32(to + 8, U);
        }
        if (lane < TOP_MAX && lane < o.top)
            asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(dsmem_addr(&sm.all[rank][lane], 0)), "l"(sm.best[lane])
                         : "memory");
    }
    if (cl > 1) cluster_sync();
    else __syncthreads();
    if (rank || warp) return;
    RowStat a = sm.stat[0];
    for (int c = 1; c < cl; c++) a = stat_join(a, sm.stat[c]);
    float lse = 0.f;
    if (lane == 0) lse = store_row(o, at, a, has, tgt);
    lse = __shfl_sync(0xffffffff, lse, 0);
    for (int i = lane; i < cl * o.top; i += 32) {
        const unsigned long long key = sm.all[i / o.top][i % o.top];
        int above = 0;
        for (int k = 0; k < cl * o.top; k++) {
            const unsigned long long other = sm.all[k / o.top][k % o.top];
            above += other > key || (other == key && k < i);  // only the empty ones are equal
        }
        if (above < o.top) store_top(o, at, above, key, lse);
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
    if (V > 0x7ffffff0) return fail("token_logprobs: vocab up to 2^31 - 16");
    if (logp_check("token_logprobs", o)) return -1;
    if (rows == 0) return 0;
    if (!x || ((uintptr_t)x & (type ? 3 : 1))) return fail("token_logprobs: logits null or not aligned to their type");
    // CTAs of a row: shares of at most 64 KB, and as many CTAs as fit at once (2 to an SM) while a share is above 8 KB
    const long bytes = (long)V * (type ? 4 : 2);
    int lg = 0;
    while (lg < 3 && (bytes >> lg > 65536 || ((long)rows << lg <= 148 && bytes >> lg > 8192))) lg++;
    const int cl = 1 << lg;
    if ((long)rows * cl > 0x7fffffffl) return fail("token_logprobs: too many rows in one call");
    DevCtx& dc = dev_ctx();
    if (!dc.ok) return fail(dc.err);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(rows * cl));
    cfg.blockDim = dim3(NT);
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = cl;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    return check_pdl(type ? cudaLaunchKernelEx(&cfg, token_logprobs_kernel<float>, (const float*)x, (long)ldx, V, sup, o, lg)
                          : cudaLaunchKernelEx(&cfg, token_logprobs_kernel<h16>, (const h16*)x, (long)ldx, V, sup, o, lg),
                     "token_logprobs");
}

}  // namespace mmz
