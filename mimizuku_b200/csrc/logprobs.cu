// Log probabilities from rows of logits, for sm_100a: of a given token, the entropy of the distribution and its
// largest entries. Over the ids whose sup[id] is 0 (argmax_tok's mask, kernels/whisper.cu:451-493):
//     lse = m + log sum e^(x - m),   logp = x_t - lse,   entropy = log sum e^(x - m) - sum e^(x - m) (x - m) / sum e^(x - m)
// and the `top` largest logits, equal ones by the lower id, each with its log probability. Sums in fp32.
//
// Bound by reading the logits, once: a producer warp streams the row in 16 KB bulk copies through a ring in shared
// memory (96 KB, two CTAs to an SM), so that memory keeps reading while a row is being finished; 8 warps keep a running
// maximum and the two sums in packed fp32, 64 bytes of a thread's logits at a time. CTAs go from row to row; few rows are
// shared by clusters of up to 8 CTAs. The alternatives cost next to no work per logit: a thread keeps the 64 bytes with
// its largest logit, and the largest logit of its others. After the pass the top-th largest of 16 groups' maxima is a
// bound below which no alternative lies: about as many threads as there are alternatives reach it, nearly always with
// the bytes they kept alone; the others' logits are read again, by their whole warp. What reaches the bound is ranked by
// counting. Where more than LIST logits do (rows of equal logits), the alternatives are found one after another in `top`
// passes instead. Measured: 1792 rows of 51865 fp32 logits, 8 alternatives, 86 us = 4.3 TB/s (6.05 rows to a CTA, so 7);
// 32 rows of 51866 fp16 logits, masked, 13 us.
#include "launch.h"
#include "logprobs.cuh"

namespace mmz {
namespace lp {
constexpr int NT = 256, NW = NT / 32, NG = 16;  // threads that sum, their warps, groups of 16 of them
constexpr int NS = 6, CB = 16384;               // stages and bytes of the ring
constexpr int PIECES = CB / 16;                 // 16-byte pieces of a stage: 4 to a thread
constexpr int LIST = 1024;                      // candidates of a CTA

struct Smem {
    uint8_t ring[NS][CB];
    unsigned long long list[LIST], best[TOP_MAX], all[8 * TOP_MAX];  // all: every CTA's, in the cluster's first
    uint64_t full[NS], empty[NS];
    float gm[NG], ws[NW], wu[NW];
    RowStat stat[8];
    float tau;
    int n, abort;
};

__device__ __forceinline__ void sync_sums() { asm volatile("bar.sync 1, %0;" ::"n"(NT) : "memory"); }

// the logits of a 16-byte piece: 8 of fp16, 4 of fp32
template <typename T>
struct Piece;
template <>
struct Piece<h16> {
    static constexpr int N = 8;
    static __device__ __forceinline__ void floats(const uint4& r, float (&x)[N]) {
        const __half2* h = reinterpret_cast<const __half2*>(&r);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float2 f = __half22float2(h[i]);
            x[2 * i] = f.x, x[2 * i + 1] = f.y;
        }
    }
};
template <>
struct Piece<float> {
    static constexpr int N = 4;
    static __device__ __forceinline__ void floats(const uint4& r, float (&x)[N]) {
        x[0] = __uint_as_float(r.x), x[1] = __uint_as_float(r.y), x[2] = __uint_as_float(r.z), x[3] = __uint_as_float(r.w);
    }
};

// the mask bytes of ids i .. i + N - 1: two aligned words where both lie inside the mask, else byte by byte
template <int N>
__device__ __forceinline__ unsigned long long mask_of(const unsigned char* sup, int i, int V) {
    const uintptr_t a = (uintptr_t)(sup + i), w = a & ~(uintptr_t)7;
    const int sh = 8 * (int)(a & 7);
    unsigned long long m = 0;
    if (w >= (uintptr_t)sup && w + 16 <= (uintptr_t)(sup + V)) {
        m = *(const unsigned long long*)w >> sh;
        if (sh > 64 - 8 * N) m |= *(const unsigned long long*)(w + 8) << (64 - sh);
        if (N == 4) m &= 0xffffffffull;
    } else {
        for (int k = 0; k < N; k++) m |= (unsigned long long)(sup[i + k] != 0) << (8 * k);
    }
    return m;
}

}  // namespace lp
using namespace lp;

// grid: rows in turn over gridDim / cl clusters of cl = 2^lg CTAs (cl > 1: one row to a cluster); dynamic shared memory
// sizeof(Smem). BEGIN: `begin` is looked at
template <typename T, bool BEGIN>
__global__ void __launch_bounds__(NT + 32, 2)
    token_logprobs_kernel(const T* x, long ldx, int rows, int V, const unsigned char* sup, LogpOut o, Begin begin,
                          int lg, unsigned* status, unsigned long long limit_ns) {
    constexpr int N = Piece<T>::N;
    extern __shared__ __align__(128) uint8_t smem[];
    Smem& sm = *reinterpret_cast<Smem*>(smem);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, cl = 1 << lg, rank = blockIdx.x & (cl - 1);
    const int row0 = blockIdx.x >> lg, step = gridDim.x >> lg;
    if (threadIdx.x == 0) {
        sm.abort = 0;
        for (int i = 0; i < NS; i++) {
            mbar_init(&sm.full[i], 1);
            mbar_init(&sm.empty[i], NW);
        }
        fence_mbar_init();
    }
    __syncthreads();
    if (cl > 1) cluster_arrive_relaxed();  // the first CTA has started before anything is sent to it
    griddep_wait();
    griddep_launch_dependents();
    const int col = (int)row_at(o, 0);  // the outputs' column, -1: outside them (nothing is read then either)
    // ids before a row's first aligned address, its pieces, ids after the last piece; this CTA's share of the pieces
    struct Row {
        const T* x;
        int head, np, p0, p1;
    };
    auto row_of = [&](int r) {
        Row w;
        w.x = x + r * ldx;
        w.head = min(V, (int)((16 - ((uintptr_t)w.x & 15)) & 15) / (int)sizeof(T));
        w.np = (V - w.head) / N;
        w.p0 = (int)((long)w.np * rank >> lg), w.p1 = (int)((long)w.np * (rank + 1) >> lg);
        return w;
    };
    if (warp == NW) {
        // ---------------------------------------------------------------- producer
        if (lane == 0) {
            unsigned q = 0;
            bool ok = true;
            for (int r = row0; r < rows && col >= 0 && ok; r += step) {
                const Row w = row_of(r);
                for (int p = w.p0; p < w.p1; p += PIECES, q++) {
                    const int st = q % NS;
                    if (q >= NS && !mbar_wait(&sm.empty[st], (q / NS - 1) & 1, &sm.abort, limit_ns, status, K_LOGP, 1)) {
                        ok = false;
                        break;
                    }
                    const uint32_t bytes = (uint32_t)min(PIECES, w.p1 - p) * 16;
                    mbar_expect_tx(&sm.full[st], bytes);
                    bulk_g2s(sm.ring[st], (const uint8_t*)(w.x + w.head) + 16l * p, bytes, &sm.full[st]);
                }
            }
            // the last copies land before the CTA ends, whoever's wait gave up (else the consumers wait for them too)
            for (unsigned i = q > NS ? q - NS : 0; i < q; i++)
                mbar_wait(&sm.full[i % NS], (i / NS) & 1, nullptr, limit_ns, nullptr, 0, 0);
        }
        __syncwarp();
        if (cl > 1) {
            cluster_wait();
            if (col >= 0) cluster_sync();
        }
        return;
    }
    if (cl > 1) cluster_wait();
    if (col < 0) return;
    const bool begins = BEGIN && col == begin.col;
    const int b0 = begins ? begin.id[0] : -1, b1 = begins ? begin.id[1] : -1;
    unsigned q = 0;
    bool ok = true;
    for (int r = row0; r < rows; r += step) {
        const Row w = row_of(r);
        const T* xr = w.x;
        const int head = w.head, tail = head + w.np * N;
        const long at = row_at(o, r);
        const int t = o.target ? o.target[at] : -1;
        auto logit = [&](int i) { return (sup && sup[i]) || (BEGIN && (i == b0 || i == b1)) ? -INFINITY : (float)xr[i]; };
        const bool has = t >= 0 && t < V;
        float tgt = 0.f;
        if (rank == 0 && threadIdx.x == 0 && has) tgt = logit(t);
        auto piece = [&](int p, const uint4& v, float (&f)[N]) {  // piece p's logits, -inf for what is left out
            Piece<T>::floats(v, f);
            if (sup) {
                const unsigned long long m = mask_of<N>(sup, head + N * p, V);
                if (m)
#pragma unroll
                    for (int k = 0; k < N; k++)
                        if (m >> (8 * k) & 0xff) f[k] = -INFINITY;
            }
            if (BEGIN && begins) {
                const int i = head + N * p;
#pragma unroll
                for (int k = 0; k < N; k++)
                    if (i + k == b0 || i + k == b1) f[k] = -INFINITY;
            }
        };
        // the ids outside the pieces: at most 7 before, with the first CTA, and 7 after, with the last
        const int edge = threadIdx.x < 8 ? (rank == 0 && threadIdx.x < head ? (int)threadIdx.x : -1)
                         : threadIdx.x < 16 && rank == cl - 1 && tail + (int)threadIdx.x - 8 < V ? tail + (int)threadIdx.x - 8 : -1;
        Run run{LOWEST, make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
        if (edge >= 0) {
            const float e = logit(edge);
            run.raise(e);
            run.add2(e, -INFINITY);
        }
        uint4 kept[PIECES / NT] = {};            // the stage's pieces with the thread's largest logit,
        int kept_p = -1;                         // the first of them (-1: none),
        float most = LOWEST, others = -INFINITY;  // that logit, and the largest in the thread's other pieces
        for (int p = w.p0; p < w.p1; p += PIECES, q++) {
            const int st = q % NS, n = min(PIECES, w.p1 - p);
            ok = ok && __all_sync(0xffffffff, mbar_wait(&sm.full[st], (q / NS) & 1, &sm.abort, limit_ns, status, K_LOGP, 2));
            if (!ok) continue;
            uint4 v[PIECES / NT];
#pragma unroll
            for (int k = 0; k < PIECES / NT; k++) v[k] = reinterpret_cast<const uint4*>(sm.ring[st])[k * NT + threadIdx.x];
            __syncwarp();
            if (lane == 0) mbar_arrive(&sm.empty[st]);
            float f[PIECES / NT][N];
#pragma unroll
            for (int k = 0; k < PIECES / NT; k++) {
                if (k * NT + (int)threadIdx.x < n) {
                    piece(p + k * NT + threadIdx.x, v[k], f[k]);
                } else {  // past the row's last piece
#pragma unroll
                    for (int e = 0; e < N; e++) f[k][e] = -INFINITY;
                }
            }
            float h = f[0][0];
#pragma unroll
            for (int k = 0; k < PIECES / NT; k++)
#pragma unroll
                for (int i = 0; i < N; i += 2) h = fmax3(h, f[k][i], f[k][i + 1]);
            run.add(f, h);
            if (h > most) {
                others = most, most = h, kept_p = p;
#pragma unroll
                for (int k = 0; k < PIECES / NT; k++) kept[k] = v[k];
            } else {
                others = fmaxf(others, h);
            }
        }
        // ---------------------------------------------------------------- the CTA's statistics
        float gm = run.m;
#pragma unroll
        for (int d = 8; d; d >>= 1) gm = fmaxf(gm, __shfl_xor_sync(0xffffffff, gm, d));
        if ((lane & 15) == 0) sm.gm[threadIdx.x >> 4] = gm;
        if (threadIdx.x == 0) sm.n = 0;
        if (threadIdx.x < TOP_MAX) sm.best[threadIdx.x] = 0ull;
        sync_sums();
        float M = LOWEST;
#pragma unroll
        for (int g = 0; g < NG; g++) M = fmaxf(M, sm.gm[g]);
        run.raise(M);
        float S = run.s.x + run.s.y, U = run.u.x + run.u.y;
#pragma unroll
        for (int d = 16; d; d >>= 1) {
            S += __shfl_xor_sync(0xffffffff, S, d);
            U += __shfl_xor_sync(0xffffffff, U, d);
        }
        if (lane == 0) sm.ws[warp] = S, sm.wu[warp] = U;
        // ---------------------------------------------------------------- its alternatives
        if (o.top > 0) {
            // every warp finds the top-th largest of the groups' maxima
            const float a = sm.gm[lane & 15];
            int above = 0;
#pragma unroll
            for (int g = 0; g < NG; g++) above += sm.gm[g] > a || (sm.gm[g] == a && g < (lane & 15));
            const float tau = __shfl_sync(0xffffffff, a, __ffs(__ballot_sync(0xffffffff, above == o.top - 1)) - 1);
            auto take = [&](float f, int id) {
                const unsigned long long key = f >= tau ? top_key(f, id) : 0ull;
                if (key) {
                    const int k = atomicAdd(&sm.n, 1);
                    if (k < LIST) sm.list[k] = key;
                }
            };
            if (edge >= 0) take(logit(edge), edge);
            if (kept_p >= 0 && most >= tau && !(others >= tau)) {
#pragma unroll
                for (int k = 0; k < PIECES / NT; k++) {
                    const int p = kept_p + k * NT + threadIdx.x;
                    if (p < w.p1) {
                        float f[N];
                        piece(p, kept[k], f);
#pragma unroll
                        for (int e = 0; e < N; e++) take(f[e], head + N * p + e);
                    }
                }
            }
            // two threads' pieces (every NT-th from the thread's first) at a time, two loads of each in flight
            for (unsigned who = __ballot_sync(0xffffffff, others >= tau); who;) {
                int first[2];
                first[0] = first[1] = w.p0 + warp * 32 + __ffs(who) - 1;
                who &= who - 1;
                if (who) first[1] = w.p0 + warp * 32 + __ffs(who) - 1;
                who &= who - 1;
                const int sets = first[1] == first[0] ? 1 : 2;
                for (int d = lane * NT; first[0] + d - lane * NT < w.p1; d += 64 * NT) {
                    uint4 v[4];
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        const int p = first[k >> 1] + d + (k & 1) * 32 * NT;
                        if ((k >> 1) < sets && p < w.p1) v[k] = reinterpret_cast<const uint4*>(xr + head)[p];
                    }
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        const int p = first[k >> 1] + d + (k & 1) * 32 * NT;
                        if ((k >> 1) < sets && p < w.p1) {
                            float f[N];
                            piece(p, v[k], f);
#pragma unroll
                            for (int e = 0; e < N; e++) take(f[e], head + N * p + e);
                        }
                    }
                }
            }
            sync_sums();
            const int n = sm.n;
            if (n <= LIST) {
                for (int i = threadIdx.x; i < n; i += NT) {  // a key's rank is the number of larger ones: no two are equal
                    const unsigned long long key = sm.list[i];
                    int more = 0;
                    for (int k = 0; k < n && more < o.top; k++) more += sm.list[k] > key;
                    if (more < o.top) sm.best[more] = key;
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
                    for (int p = w.p0 + threadIdx.x; p < w.p1; p += NT) {
                        float f[N];
                        piece(p, reinterpret_cast<const uint4*>(xr + head)[p], f);
#pragma unroll
                        for (int e = 0; e < N; e++) see(f[e], head + N * p + e);
                    }
#pragma unroll
                    for (int d = 16; d; d >>= 1) {
                        const unsigned long long c = __shfl_xor_sync(0xffffffff, b, d);
                        b = c > b ? c : b;
                    }
                    sync_sums();
                    if (lane == 0) sm.list[warp] = b;
                    sync_sums();
                    for (int g = 0; g < NW; g++) b = sm.list[g] > b ? sm.list[g] : b;
                    if (threadIdx.x == 0) sm.best[k] = b;
                    last = b;
                }
            }
        }
        sync_sums();
        // ---------------------------------------------------------------- the cluster's CTAs joined in its first
        if (warp == 0) {
            S = lane < NW ? sm.ws[lane] : 0.f, U = lane < NW ? sm.wu[lane] : 0.f;
#pragma unroll
            for (int d = NW / 2; d; d >>= 1) {
                S += __shfl_xor_sync(0xffffffff, S, d);
                U += __shfl_xor_sync(0xffffffff, U, d);
            }
            if (lane == 0) {
                const uint32_t to = dsmem_addr(&sm.stat[rank], 0);
                st_dsmem_f32(to, S == 0.f ? -INFINITY : M);  // nothing above -inf: the empty set
                st_dsmem_f32(to + 4, S);
                st_dsmem_f32(to + 8, U);
            }
            if (lane < TOP_MAX && lane < o.top)
                asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(dsmem_addr(&sm.all[rank * o.top + lane], 0)),
                             "l"(sm.best[lane])
                             : "memory");
            __syncwarp();
        }
        if (cl > 1) cluster_sync();
        if (rank == 0 && warp == 0) {
            const RowStat a = stat_warp(lane < cl ? sm.stat[lane] : stat_none());
            float ls = 0.f;
            if (lane == 0) ls = store_row(o, at, a, has, tgt);
            ls = __shfl_sync(0xffffffff, ls, 0);
            const int n = cl * o.top;
            for (int i = lane; i < n; i += 32) {
                const unsigned long long key = sm.all[i];
                int above = 0;
#pragma unroll 8
                for (int k = 0; k < n; k++) above += sm.all[k] > key || (sm.all[k] == key && k < i);  // only empty ones are equal
                if (above < o.top) store_top(o, at, above, key, a.m, ls);
            }
            __syncwarp();
        }
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
                          const LogpOut& o, cudaStream_t st, const Begin& begin) {
    if (rows < 0 || V < 1 || ldx < V) return fail("token_logprobs: rows >= 0, vocab >= 1, ldx >= vocab");
    if (type != 0 && type != 1) return fail("token_logprobs: type is 0 (fp16) or 1 (fp32)");
    if (type && begin.col >= 0) return fail("token_logprobs: ids left out of one column only of fp16 logits");
    // (a CTA's next row is up to 296 further on)
    if (V > 0x7ffffff0 || rows > 0x7ffffc00) return fail("token_logprobs: vocab up to 2^31 - 16, rows up to 2^31 - 1024");
    if (logp_check("token_logprobs", o)) return -1;
    if (rows == 0) return 0;
    if (!x || ((uintptr_t)x & (type ? 3 : 1))) return fail("token_logprobs: logits null or not aligned to their type");
    // a CTA to a row, two to an SM, each going from row to row; up to 148 rows: clusters, while the CTAs fit at once and a
    // CTA's share is above 8 KB. Rows of 104 KB: 32 of them 13 us in clusters of 8, 18 with a CTA each; 64: 12 in clusters of
    // 4 and less, 19 with a CTA each, 21 in clusters of 8; 120: 15, 19 and 32; 160: a CTA each 21, clusters of 8 43
    const long bytes = (long)V * (type ? 4 : 2);
    int lg = 0;
    while (lg < 3 && (long)rows << lg <= 148 && bytes >> lg > 8192) lg++;
    const int cl = 1 << lg, grid = lg ? rows << lg : rows < 296 ? rows : 296;
    DevCtx& dc = dev_ctx();
    if (!dc.ok) return fail(dc.err);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)grid);
    cfg.blockDim = dim3(NT + 32);
    cfg.dynamicSmemBytes = sizeof(Smem);
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = cl;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    auto run = [&](auto* fn, auto* p) {
        return check_pdl(cudaLaunchKernelEx(&cfg, fn, p, (long)ldx, rows, V, sup, o, begin, lg, dc.status, dc.limit_ns),
                         "token_logprobs");
    };
    if (type) return run(token_logprobs_kernel<float, false>, (const float*)x);
    return run(begin.col < 0 ? token_logprobs_kernel<h16, false> : token_logprobs_kernel<h16, true>, (const h16*)x);
}

void init_logprobs_attrs() {
    auto set = [](auto* fn) { cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, sizeof(Smem)); };
    set(token_logprobs_kernel<float, false>);
    set(token_logprobs_kernel<h16, false>);
    set(token_logprobs_kernel<h16, true>);
}

}  // namespace mmz
