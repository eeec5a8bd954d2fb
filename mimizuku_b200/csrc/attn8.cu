// Attention over the 8-bit key/value cache (kv8.cu), for sm_100a. For sequence b, query row i and query head h, with
// L = min(lens[b], cap) and key head g = h / (q_heads / kv_heads):
//     s_j = scale * ks[b][g][j / block] * (q . k8_j)    for j < limit,  limit = L, or L - rows + i + 1 when causal
//     out = sum_j softmax(s)_j * vs[b][g][j / block] * v8_j      (zeros where limit <= 0)
// and the probabilities of chosen heads as fp16. Sums and softmax statistics in fp32; only the outputs are rounded.
//
// The query heads and rows that share a key head are one block of rows: up to 8 (a decoding step, hypotheses of one
// clip, grouped heads) or tiles of 32 (prompts). A warp takes chunks of 64 positions, keys and values by bulk copies
// into a ring of its own, and works in registers from there:
//   * every code (int8 or e4m3) is a number of fp16, so the products run exactly on the tensor cores (m16n8k16, fp32
//     sums): S^T = K q^T with the 16 positions as M and the 8 rows as N, then O^T = V^T P^T. The contraction indices are
//     dealt so that a lane's K fragment is 16 consecutive bytes of a row and its V fragment 8 consecutive bytes of 4
//     rows; no code is moved between lanes, and P^T is S^T's own layout after one 8 x 8 transpose.
//   * a running maximum and sum per row; p carries a factor 2^10 (it cancels against the sum) and is split into a high
//     and a low fp16 part, each multiplied: what is lost of p is below 2^-21 of it, and below 2^-35 of the row's
//     largest p, so the one rounding that counts stays that of the output.
//   * the scales of a block apply in fp32: ks to the scores, vs to the sums of the positions that share it.
// The 4 warps of a CTA join in shared memory, the CTAs of a cluster (up to 8 along the sequence) through distributed
// shared memory, and where one cluster is too little for a long cache, clusters through scratch and a second kernel.
#include "attn8.h"
#include "fp8_cache.cuh"
#include "launch.h"

namespace mmz {
namespace a8 {

constexpr int WARPS = 4, NT = 32 * WARPS;
constexpr int CH = 64;          // positions per chunk
constexpr int STG = 2;          // chunks in a warp's ring
constexpr int KB = CH * HD;     // bytes of a chunk's keys (and of its values)
constexpr int REC = HD + 2;     // a row's partial result: 64 sums, maximum, sum of p
constexpr float LOG2E = 1.4426950408889634f;
constexpr float PSHIFT = 10.f;  // p <= 2^10

template <int NTL>
struct Smem {
    union {
        uint8_t ring[WARPS][STG][2][KB];
        float part[WARPS][8 * NTL][REC];  // after the last chunk
    };
    float join[8 * NTL][REC];             // this CTA's rows, read by the cluster
    uint64_t full[WARPS][STG];
    int abort;
};

__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
// the low (hi = false) or high two codes of a word as two fp16 numbers
template <int KIND>
__device__ __forceinline__ uint32_t codes2(uint32_t w, bool hi) {
    if constexpr (KIND == KV8_E4M3) return e4m3x2_to_h2(hi ? w >> 16 : w & 0xffff);
    // 0x6400 | u is 1024 + u in fp16; u = code + 128
    const uint32_t u = __byte_perm(w ^ 0x80808080u, 0x64646464u, hi ? 0x4342 : 0x4140);
    const __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&u), __floats2half2_rn(1152.f, 1152.f));
    return *reinterpret_cast<const uint32_t*>(&r);
}
// the position, within a tile of 16, that fragment row r stands for: rows 2t, 2t + 1, 2t + 8, 2t + 9 of lane t of a
// quad are positions t, t + 4, t + 8, t + 12
__device__ __forceinline__ int place(int r) { return (r & 8) | ((r & 1) << 2) | ((r & 6) >> 1); }

// scores of 16 positions (keys at k, 64 bytes a row) against 8 rows per column tile; lane (g, t) receives position
// place(g) (and + 8) for rows 2t and 2t + 1
template <int KIND, int NTL>
__device__ __forceinline__ void scores16(const uint8_t* k, int lane, const uint32_t (&q)[NTL][8], float (&s)[NTL][4]) {
    const uint8_t* p = k + place(lane >> 2) * HD + (lane & 3) * 16;
    const uint4 lo = *reinterpret_cast<const uint4*>(p), hi = *reinterpret_cast<const uint4*>(p + 8 * HD);
    const uint32_t wl[4] = {lo.x, lo.y, lo.z, lo.w}, wh[4] = {hi.x, hi.y, hi.z, hi.w};
#pragma unroll
    for (int n = 0; n < NTL; n++) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const uint32_t a[4] = {codes2<KIND>(wl[j], false), codes2<KIND>(wh[j], false), codes2<KIND>(wl[j], true),
                               codes2<KIND>(wh[j], true)};
#pragma unroll
        for (int n = 0; n < NTL; n++) mma(s[n], a, q[n][2 * j], q[n][2 * j + 1]);
    }
}

// a row's 16 values from dimension 16 t on, as the column fragment of scores16
__device__ __forceinline__ void load_q(const h16* row, int t, uint32_t (&q)[8]) {
    const uint4 x = reinterpret_cast<const uint4*>(row + 16 * t)[0], y = reinterpret_cast<const uint4*>(row + 16 * t)[1];
    q[0] = x.x, q[1] = x.y, q[2] = x.z, q[3] = x.w, q[4] = y.x, q[5] = y.y, q[6] = y.z, q[7] = y.w;
}

__device__ __forceinline__ float weight(float m, float M) { return m == -INFINITY ? 0.f : ex2_approx(m - M); }

__device__ __forceinline__ uint32_t nan_codes(uint32_t w) {  // 0x80 in the bytes of w that hold e4m3's NaN
    return ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
}

}  // namespace a8
using namespace a8;

// grid: cluster rank fastest, then cluster along the sequence, row tile, (sequence, key head); cluster of cs CTAs.
// part null: the cluster's rows go to out (and their statistics to stats, if not null); else to part
template <int KIND, int NTL>
__global__ void __launch_bounds__(NT) attn8_kernel(Attn8 a, int cs, int nclus, int tiles, float* part, float2* stats,
                                                   unsigned* status, unsigned long long limit_ns) {
    constexpr int RT = 8 * NTL;            // rows of a tile
    constexpr int SUB = NTL == 1 ? 64 : 32;  // positions whose scores are in registers at a time
    constexpr int NJ = SUB / 16;
    extern __shared__ __align__(128) uint8_t raw[];
    Smem<NTL>& sm = *reinterpret_cast<Smem<NTL>*>(raw);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int rank = blockIdx.x % cs, clus = (blockIdx.x / cs) % nclus;
    const int tile = (blockIdx.x / cs / nclus) % tiles;
    const long pair = blockIdx.x / cs / nclus / tiles;
    const int hk = (int)(pair % a.kv_heads), group = a.q_heads / a.kv_heads;
    const long b = pair / a.kv_heads;
    const int R = a.rows * group, r0 = tile * RT;
    if (lane == 0)
        for (int i = 0; i < STG; i++) mbar_init(&sm.full[warp][i], 1);
    if (threadIdx.x == 0) sm.abort = 0;
    fence_mbar_init();
    __syncthreads();
    griddep_wait();

    const int L = a.lens ? max(0, min(a.lens[b], a.cap)) : a.cap;
    // what row r of the block sees; the tile's last row sees the most
    auto limit = [&](int r) { return a.causal ? max(0, L - a.rows + r / group + 1) : L; };
    const int most = limit(min(r0 + RT, R) - 1), least = limit(r0);
    const int nch = (most + CH - 1) / CH;
    const int ns = cs * nclus, per = (nch + ns - 1) / ns, split = clus * cs + rank;
    const int c0 = min(split * per, nch), c1 = min(c0 + per, nch);
    const uint8_t* k8 = a.k8 + b * a.c_seq + hk * a.c_head;
    const uint8_t* v8 = a.v8 + b * a.c_seq + hk * a.c_head;
    const float* ks = a.ks + b * a.s_seq + hk * a.s_head;
    const float* vs = a.vs + b * a.s_seq + hk * a.s_head;

    uint64_t* full = sm.full[warp];
    auto issue = [&](int c, int st) {  // lane 0
        const uint32_t bytes = (uint32_t)min(CH, most - c * CH) * HD;
        mbar_expect_tx(&full[st], 2 * bytes);
        bulk_g2s(sm.ring[warp][st][0], k8 + (long)c * KB, bytes, &full[st]);
        bulk_g2s(sm.ring[warp][st][1], v8 + (long)c * KB, bytes, &full[st]);
    };
    // lanes 0-3: the key scales of a chunk's four tiles of 16 positions, lanes 4-7 the value scales
    auto scale_of = [&](int c) {
        if (lane >= 8 || c >= c1) return 0.f;
        const int j = min(c * CH + 16 * (lane & 3), most - 1);
        return lane < 4 ? ks[j / a.block] * (a.scale * LOG2E) : vs[j / a.block];
    };
    int issued = c0 + warp;
    if (lane == 0)
        for (int i = 0; i < STG && c0 + warp + i * WARPS < c1; i++) issue(c0 + warp + i * WARPS, i);
    float sc_next = scale_of(c0 + warp);

    uint32_t q[NTL][8];
    int lim[NTL][2];
#pragma unroll
    for (int n = 0; n < NTL; n++) {
        const int r = r0 + 8 * n + g;
        if (r < R) load_q(a.q + b * a.q_seq + (r / group) * a.q_row + (hk * group + r % group) * a.q_head, t, q[n]);
        else
            for (int i = 0; i < 8; i++) q[n][i] = 0;
        lim[n][0] = limit(min(r0 + 8 * n + 2 * t, R - 1));
        lim[n][1] = limit(min(r0 + 8 * n + 2 * t + 1, R - 1));
    }
    float m[NTL][2], l[NTL][2], o[4][NTL][4];
#pragma unroll
    for (int n = 0; n < NTL; n++) {
        m[n][0] = m[n][1] = -INFINITY;
        l[n][0] = l[n][1] = 0.f;
#pragma unroll
        for (int i = 0; i < 4; i++) o[i][n][0] = o[i][n][1] = o[i][n][2] = o[i][n][3] = 0.f;
    }

    const int same = min(a.block, SUB) / 16 - 1;  // tiles of 16 that share a scale, less one: 0, 1 or 3
    bool ok = true;
    int it = 0;
    for (int c = c0 + warp; c < c1; c += WARPS, it++) {
        const int st = it % STG;
        ok = __all_sync(0xffffffff, mbar_wait(&full[st], (it / STG) & 1, &sm.abort, limit_ns, status, K_ATTN8, 1));
        if (!ok) break;
        const float sc = sc_next;
        sc_next = scale_of(c + WARPS);
        const uint8_t* ck = sm.ring[warp][st][0];
        uint8_t* cv = sm.ring[warp][st][1];
        const int base = c * CH;
        // the sequence's last chunk: the rows that were not copied hold what the ring held (nothing follows this chunk
        // in the warp's ring). Their weights are 0, but a NaN times 0 would not be
        if (base + CH > most) {
            for (int i = (most - base) * HD + lane * 16; i < KB; i += 512)
                *reinterpret_cast<uint4*>(cv + i) = make_uint4(0, 0, 0, 0);
            __syncwarp();
        }
        const bool whole = base + CH <= least;  // every row sees the whole chunk
#pragma unroll
        for (int sub = 0; sub < CH / SUB; sub++) {
            const int sb = base + sub * SUB;
            if (sub && sb >= most) break;
            float s[NJ][NTL][4];
#pragma unroll
            for (int j = 0; j < NJ; j++) {
                scores16<KIND, NTL>(ck + (sub * SUB + 16 * j) * HD, lane, q, s[j]);
                const float f = __shfl_sync(0xffffffff, sc, sub * NJ + j);
#pragma unroll
                for (int n = 0; n < NTL; n++)
#pragma unroll
                    for (int e = 0; e < 4; e++) s[j][n][e] *= f;
            }
            if (!whole) {
#pragma unroll
                for (int j = 0; j < NJ; j++) {
                    const int p = sb + 16 * j + place(g);
#pragma unroll
                    for (int n = 0; n < NTL; n++)
#pragma unroll
                        for (int e = 0; e < 4; e++)
                            if (p + (e >> 1) * 8 >= lim[n][e & 1]) s[j][n][e] = -INFINITY;
                }
            }
            // running maximum, p and its sum
            uint32_t ph[NJ][NTL][2], pl[NJ][NTL][2];
            float alpha[NTL][2];
#pragma unroll
            for (int n = 0; n < NTL; n++) {
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    float mx = m[n][e];
#pragma unroll
                    for (int j = 0; j < NJ; j++) mx = fmaxf(mx, fmaxf(s[j][n][e], s[j][n][e + 2]));
                    mx = fmaxf(mx, __shfl_xor_sync(0xffffffff, mx, 4));
                    mx = fmaxf(mx, __shfl_xor_sync(0xffffffff, mx, 8));
                    mx = fmaxf(mx, __shfl_xor_sync(0xffffffff, mx, 16));
                    alpha[n][e] = weight(m[n][e], mx);
                    m[n][e] = mx;
                    const float off = (mx == -INFINITY ? 0.f : mx) - PSHIFT;
                    float sum = 0.f;
#pragma unroll
                    for (int j = 0; j < NJ; j++) {
                        s[j][n][e] = ex2_approx(s[j][n][e] - off);
                        s[j][n][e + 2] = ex2_approx(s[j][n][e + 2] - off);
                        sum += s[j][n][e] + s[j][n][e + 2];
                    }
                    l[n][e] = l[n][e] * alpha[n][e] + sum;
                }
#pragma unroll
                for (int j = 0; j < NJ; j++)
#pragma unroll
                    for (int u = 0; u < 2; u++) {
                        const float x = s[j][n][2 * u], y = s[j][n][2 * u + 1];
                        const __half2 hi = __floats2half2_rn(x, y);
                        const float2 back = __half22float2(hi);
                        const __half2 lo = __floats2half2_rn(x - back.x, y - back.y);
                        ph[j][n][u] = transpose8(*reinterpret_cast<const uint32_t*>(&hi));
                        pl[j][n][u] = transpose8(*reinterpret_cast<const uint32_t*>(&lo));
                    }
            }
            // values: lane (g, t) has dimensions 8 g .. 8 g + 7 of positions t, t + 4, t + 8, t + 12 of each tile
            uint2 w[NJ][4];
            uint32_t nan = 0;
#pragma unroll
            for (int j = 0; j < NJ; j++)
#pragma unroll
                for (int u = 0; u < 4; u++) {
                    w[j][u] = *reinterpret_cast<const uint2*>(cv + (sub * SUB + 16 * j + t + 4 * u) * HD + 8 * g);
                    if (KIND == KV8_E4M3 && !whole) nan |= nan_codes(w[j][u].x) | nan_codes(w[j][u].y);
                }
            // a NaN that some of the rows do not see: taken out of the products, and put into the sums of the rows
            // that do see it (nanpos: the first position with one, for each of the lane's dimensions)
            const bool nans = KIND == KV8_E4M3 && !whole && __any_sync(0xffffffff, nan != 0);
            int nanpos[8];
            if (nans) {
#pragma unroll
                for (int d = 0; d < 8; d++) nanpos[d] = 0x7fffffff;
#pragma unroll
                for (int j = NJ - 1; j >= 0; j--)
#pragma unroll
                    for (int u = 3; u >= 0; u--) {
                        uint32_t* x = &w[j][u].x;
#pragma unroll
                        for (int d = 0; d < 8; d++)
                            if (nan_codes(x[d >> 2]) >> (8 * (d & 3) + 7) & 1) {
                                nanpos[d] = sb + 16 * j + t + 4 * u;
                                x[d >> 2] &= ~(0xffu << (8 * (d & 3)));
                            }
                    }
#pragma unroll
                for (int d = 0; d < 8; d++) {
                    nanpos[d] = min(nanpos[d], __shfl_xor_sync(0xffffffff, nanpos[d], 1));
                    nanpos[d] = min(nanpos[d], __shfl_xor_sync(0xffffffff, nanpos[d], 2));
                }
            }
#pragma unroll
            for (int i = 0; i < 4; i++) {  // dimensions 8 g + 2 i and 8 g + 2 i + 1
#pragma unroll
                for (int n = 0; n < NTL; n++)
#pragma unroll
                    for (int e = 0; e < 4; e++) o[i][n][e] *= alpha[n][e & 1];
                float acc[NTL][4];
#pragma unroll
                for (int j = 0; j < NJ; j++) {
                    if ((j & same) == 0)
#pragma unroll
                        for (int n = 0; n < NTL; n++) acc[n][0] = acc[n][1] = acc[n][2] = acc[n][3] = 0.f;
                    const uint32_t sel = i & 1 ? 0x7362 : 0x5140;
                    const uint32_t x = i < 2 ? __byte_perm(w[j][0].x, w[j][1].x, sel) : __byte_perm(w[j][0].y, w[j][1].y, sel);
                    const uint32_t y = i < 2 ? __byte_perm(w[j][2].x, w[j][3].x, sel) : __byte_perm(w[j][2].y, w[j][3].y, sel);
                    const uint32_t f[4] = {codes2<KIND>(x, false), codes2<KIND>(x, true), codes2<KIND>(y, false),
                                           codes2<KIND>(y, true)};
#pragma unroll
                    for (int n = 0; n < NTL; n++) {
                        mma(acc[n], f, ph[j][n][0], ph[j][n][1]);
                        mma(acc[n], f, pl[j][n][0], pl[j][n][1]);
                    }
                    if (((j + 1) & same) == 0) {
                        const float vsc = __shfl_sync(0xffffffff, sc, 4 + sub * NJ + j);
#pragma unroll
                        for (int n = 0; n < NTL; n++)
#pragma unroll
                            for (int e = 0; e < 4; e++) o[i][n][e] += vsc * acc[n][e];
                    }
                }
                if (nans) {
#pragma unroll
                    for (int n = 0; n < NTL; n++)
#pragma unroll
                        for (int e = 0; e < 4; e++)
                            if (nanpos[2 * i + (e >> 1)] < lim[n][e & 1]) o[i][n][e] = NAN;
                }
            }
        }
        __syncwarp();
        if (lane == 0 && c + STG * WARPS < c1) issue(c + STG * WARPS, st);
        issued = c + WARPS;
    }
    if (!ok && lane == 0) {  // let the copies in flight land before the shared memory is used for something else
        for (int i = 0; i < STG; i++, it++)
            if (issued + i * WARPS < c1)
                mbar_wait(&full[it % STG], (it / STG) & 1, nullptr, limit_ns, nullptr, 0, 0);
    }

    // ---------------------------------------------------------------- the warps' rows joined
    __syncthreads();
#pragma unroll
    for (int n = 0; n < NTL; n++)
#pragma unroll
        for (int e = 0; e < 2; e++) {
            float x = l[n][e];
            x += __shfl_xor_sync(0xffffffff, x, 4);
            x += __shfl_xor_sync(0xffffffff, x, 8);
            x += __shfl_xor_sync(0xffffffff, x, 16);
            float* rec = sm.part[warp][8 * n + 2 * t + e];
            if (g == 0) rec[HD] = m[n][e], rec[HD + 1] = x;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                rec[8 * g + 2 * i] = o[i][n][e];
                rec[8 * g + 2 * i + 1] = o[i][n][e + 2];
            }
        }
    __syncthreads();
    for (int i = threadIdx.x; i < RT * HD; i += NT) {
        const int r = i / HD, d = i % HD;
        float M = -INFINITY, S = 0.f, O = 0.f;
        for (int w = 0; w < WARPS; w++) M = fmaxf(M, sm.part[w][r][HD]);
        for (int w = 0; w < WARPS; w++) {
            const float f = weight(sm.part[w][r][HD], M);
            S += f * sm.part[w][r][HD + 1];
            O += f * sm.part[w][r][d];
        }
        sm.join[r][d] = O;
        if (d == 0) sm.join[r][HD] = M, sm.join[r][HD + 1] = S;
    }
    if (cs > 1) cluster_sync();
    else __syncthreads();
    // ---------------------------------------------------------------- and the cluster's CTAs', each for its share
    for (int i = rank * NT + threadIdx.x; i < RT * (HD / 2); i += cs * NT) {
        const int r = i / (HD / 2), d = 2 * (i % (HD / 2));
        if (r0 + r >= R) break;
        float M = -INFINITY, S = 0.f;
        float2 O = make_float2(0.f, 0.f);
        for (int w = 0; w < cs; w++) M = fmaxf(M, ld_dsmem_f32(dsmem_addr(&sm.join[r][HD], w)));
        for (int w = 0; w < cs; w++) {
            const float2 ms = ld_dsmem_f32x2(dsmem_addr(&sm.join[r][HD], w)), x = ld_dsmem_f32x2(dsmem_addr(&sm.join[r][d], w));
            const float f = weight(ms.x, M);
            S += f * ms.y;
            O.x += f * x.x;
            O.y += f * x.y;
        }
        const long row = (pair * tiles + tile) * RT + r;
        if (nclus > 1) {
            float* rec = part + (((pair * tiles + tile) * nclus + clus) * RT + r) * REC;
            *reinterpret_cast<float2*>(rec + d) = O;
            if (d == 0) *reinterpret_cast<float2*>(rec + HD) = make_float2(M, S);
        } else {
            const float inv = S > 0.f ? 1.f / S : (S == S ? 0.f : S);
            const int qi = (r0 + r) / group, h = hk * group + (r0 + r) % group;
            *reinterpret_cast<__half2*>(a.out + b * a.o_seq + qi * a.o_row + h * a.o_head + d) =
                __floats2half2_rn(O.x * inv, O.y * inv);
            if (stats && d == 0) stats[row] = make_float2(M, inv);
        }
    }
    if (cs > 1) cluster_sync();  // the others may still read this CTA's rows
}

// the clusters' partial rows joined: one CTA of 128 threads to a row tile
template <int NTL>
__global__ void __launch_bounds__(NT) attn8_join_kernel(Attn8 a, int nclus, int tiles, const float* __restrict__ part,
                                                        float2* stats) {
    constexpr int RT = 8 * NTL;
    const int tile = blockIdx.x % tiles;
    const long pair = blockIdx.x / tiles, b = pair / a.kv_heads;
    const int hk = (int)(pair % a.kv_heads), group = a.q_heads / a.kv_heads, R = a.rows * group, r0 = tile * RT;
    griddep_wait();
    for (int i = threadIdx.x; i < RT * (HD / 2); i += NT) {
        const int r = i / (HD / 2), d = 2 * (i % (HD / 2));
        if (r0 + r >= R) break;
        const float* rec = part + ((pair * tiles + tile) * nclus * RT + r) * (long)REC;
        float M = -INFINITY, S = 0.f;
        float2 O = make_float2(0.f, 0.f);
        for (int w = 0; w < nclus; w++) M = fmaxf(M, rec[(long)w * RT * REC + HD]);
        for (int w = 0; w < nclus; w++) {
            const float* x = rec + (long)w * RT * REC;
            const float f = weight(x[HD], M);
            S += f * x[HD + 1];
            O.x += f * x[d];
            O.y += f * x[d + 1];
        }
        const float inv = S > 0.f ? 1.f / S : (S == S ? 0.f : S);
        const int qi = (r0 + r) / group, h = hk * group + (r0 + r) % group;
        *reinterpret_cast<__half2*>(a.out + b * a.o_seq + qi * a.o_row + h * a.o_head + d) =
            __floats2half2_rn(O.x * inv, O.y * inv);
        if (stats && d == 0) stats[(pair * tiles + tile) * RT + r] = make_float2(M, inv);
    }
}

// The probabilities of the chosen heads, from the rows' statistics: the scores again (the same products in the same
// order), p = 2^(s - M) / S. grid: (256 positions, 8 rows) tiles of each (sequence, slot); a warp takes 64 positions
template <int KIND>
__global__ void __launch_bounds__(NT) attn8_probs_kernel(Attn8 a, int tiles, int rt, const float2* __restrict__ stats) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int pt = (a.cap + 255) / 256, nrt = (a.rows + 7) / 8;
    const int pblk = blockIdx.x % pt, rtile = (blockIdx.x / pt) % nrt, slot = (blockIdx.x / pt / nrt) % a.slots;
    const long b = blockIdx.x / pt / nrt / a.slots;
    griddep_wait();
    int h = -1;
    for (int i = lane; i < a.q_heads; i += 32)
        if (h < 0 && a.pslot[i] == slot) h = i;
    h = __reduce_min_sync(0xffffffff, h < 0 ? 0x7fffffff : h);
    if (h >= a.q_heads) return;
    const int group = a.q_heads / a.kv_heads, hk = h / group;
    const int L = a.lens ? max(0, min(a.lens[b], a.cap)) : a.cap;
    const uint8_t* k8 = a.k8 + b * a.c_seq + hk * a.c_head;
    const float* ks = a.ks + b * a.s_seq + hk * a.s_head;
    uint32_t q[1][8];
    const int r0 = rtile * 8;
    if (r0 + g < a.rows) load_q(a.q + b * a.q_seq + (r0 + g) * a.q_row + h * a.q_head, t, q[0]);
    else
        for (int i = 0; i < 8; i++) q[0][i] = 0;
    float2 ms[2];
    int lim[2];
    for (int e = 0; e < 2; e++) {
        const int i = min(r0 + 2 * t + e, a.rows - 1), r = i * group + h % group;
        ms[e] = stats[((b * a.kv_heads + hk) * tiles + r / rt) * (long)rt + r % rt];
        lim[e] = a.causal ? max(0, L - a.rows + i + 1) : L;
    }
    const int last = a.causal ? max(0, L - a.rows + min(r0 + 8, a.rows)) : L;  // positions that some row sees
    for (int j = 0; j < 4; j++) {
        const int base = pblk * 256 + warp * 64 + j * 16;
        if (base >= a.cap) break;
        float s[1][4] = {};
        if (base + 16 <= last) {
            scores16<KIND, 1>(k8 + (long)base * HD, lane, q, s);
        } else if (base < last) {  // rows past the cache's end are not read: the last visible one instead
            const int p0 = min(base + place(g), last - 1), p1 = min(base + place(g) + 8, last - 1);
            const uint4 lo = *reinterpret_cast<const uint4*>(k8 + (long)p0 * HD + 16 * t);
            const uint4 hi = *reinterpret_cast<const uint4*>(k8 + (long)p1 * HD + 16 * t);
            const uint32_t wl[4] = {lo.x, lo.y, lo.z, lo.w}, wh[4] = {hi.x, hi.y, hi.z, hi.w};
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const uint32_t f[4] = {codes2<KIND>(wl[e], false), codes2<KIND>(wh[e], false), codes2<KIND>(wl[e], true),
                                       codes2<KIND>(wh[e], true)};
                mma(s[0], f, q[0][2 * e], q[0][2 * e + 1]);
            }
        }
        const float f = base < last ? ks[base / a.block] * (a.scale * LOG2E) : 0.f;
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const int p = base + place(g) + 8 * (e >> 1), i = r0 + 2 * t + (e & 1);
            if (p >= a.cap || i >= a.rows) continue;
            const float x =
                p < lim[e & 1] ? ex2_approx(s[0][e] * f - (ms[e & 1].x - PSHIFT)) * ms[e & 1].y : 0.f;
            a.probs[((b * a.slots + slot) * a.rows + i) * (long)a.cap + p] = __float2half_rn(x);
        }
    }
}

// How a call is laid out, from its sizes alone (lens is on the device): rows of a tile, tiles, CTAs of a cluster and
// clusters along the sequence, and the scratch.
namespace {
struct Plan {
    int ntl, tiles, cs, nclus;
    size_t part, stats;
};
Plan plan(int batch, int rows, int q_heads, int kv_heads, int cap, int slots) {
    Plan p;
    const long R = (long)rows * (q_heads / kv_heads);
    p.ntl = R <= 8 ? 1 : 4;
    p.tiles = (int)((R + 8 * p.ntl - 1) / (8 * p.ntl));
    const long units = (long)batch * kv_heads * p.tiles, chunks = ((long)cap + CH - 1) / CH;
    // CTAs for every SM several times over (148 SMs x 3 resident x 2), and a chunk at least to each warp
    long s = (888 + units - 1) / units;
    const long top = (chunks + WARPS - 1) / WARPS;
    if (s > top) s = top;
    p.cs = s <= 1 ? 1 : s <= 2 ? 2 : s <= 4 ? 4 : 8;
    p.nclus = (int)((s + p.cs - 1) / p.cs);
    const size_t rr = (size_t)units * 8 * p.ntl;
    p.part = p.nclus > 1 ? ((rr * p.nclus * REC * 4 + 15) & ~(size_t)15) : 0;
    p.stats = slots > 0 ? rr * 8 : 0;
    return p;
}

template <int KIND, int NTL>
int launch_main(const Attn8& a, const Plan& p, float* part, float2* stats, DevCtx& dc, cudaStream_t st) {
    const size_t smem = sizeof(Smem<NTL>);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)((long)a.batch * a.kv_heads * p.tiles * p.nclus * p.cs));
    cfg.blockDim = dim3(NT);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = p.cs;
    at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 2;
    if (check_pdl(cudaLaunchKernelEx(&cfg, attn8_kernel<KIND, NTL>, a, p.cs, p.nclus, p.tiles, part, stats, dc.status,
                                     dc.limit_ns),
                  "attn8"))
        return -1;
    if (p.nclus == 1) return 0;
    return check_pdl(launch_pdl(attn8_join_kernel<NTL>, dim3((unsigned)((long)a.batch * a.kv_heads * p.tiles)), dim3(NT),
                                0, st, a, p.nclus, p.tiles, (const float*)part, stats),
                     "attn8");
}
}  // namespace

size_t attn8_scratch_bytes(int batch, int rows, int q_heads, int kv_heads, int cap, int slots) {
    const Plan p = plan(batch, rows, q_heads, kv_heads, cap, slots);
    return p.part + p.stats;
}

int launch_attn8(const Attn8& a, int kind, void* scratch, size_t scratch_bytes, cudaStream_t st) {
    if (a.batch < 0 || a.rows < 0 || a.kv_heads < 1 || a.q_heads < 1 || a.cap < 1 || a.slots < 0)
        return fail("attn8: batch >= 0, rows >= 0, heads >= 1, cap >= 1");
    if (a.cap > 0x7fff0000) return fail("attn8: cap up to 2^31 - 65536");
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
    const int slots = a.probs ? a.slots : 0;
    if ((long)a.rows * (a.q_heads / a.kv_heads) > 0x7fffff00l) return fail("attn8: too many rows in one call");
    const Plan p = plan(a.batch, a.rows, a.q_heads, a.kv_heads, a.cap, slots);
    const long grid = (long)a.batch * a.kv_heads * p.tiles * p.nclus * p.cs;
    const long pgrid = (long)a.batch * slots * ((a.rows + 7) / 8) * ((a.cap + 255) / 256);
    if (grid > 0x7fffffffl || pgrid > 0x7fffffffl) return fail("attn8: more than 2^31 blocks in one call");
    if (p.part + p.stats && (!scratch || ((uintptr_t)scratch & 15) || scratch_bytes < p.part + p.stats))
        return fail("attn8: scratch too small or not 16-byte aligned");
    DevCtx& dc = dev_ctx();
    if (!dc.ok) return fail(dc.err);
    float* part = (float*)scratch;
    float2* stats = slots ? (float2*)((char*)scratch + p.part) : nullptr;
    int r;
    if (kind == KV8_INT8)
        r = p.ntl == 1 ? launch_main<KV8_INT8, 1>(a, p, part, stats, dc, st) : launch_main<KV8_INT8, 4>(a, p, part, stats, dc, st);
    else
        r = p.ntl == 1 ? launch_main<KV8_E4M3, 1>(a, p, part, stats, dc, st) : launch_main<KV8_E4M3, 4>(a, p, part, stats, dc, st);
    if (r || !slots) return r;
    auto* fn = kind == KV8_INT8 ? attn8_probs_kernel<KV8_INT8> : attn8_probs_kernel<KV8_E4M3>;
    return check_pdl(launch_pdl(fn, dim3((unsigned)pgrid), dim3(NT), 0, st, a, p.tiles, 8 * p.ntl, (const float2*)stats),
                     "attn8");
}

void init_attn8_attrs() {
    cudaFuncSetAttribute(attn8_kernel<KV8_INT8, 1>, cudaFuncAttributeMaxDynamicSharedMemorySize, sizeof(Smem<1>));
    cudaFuncSetAttribute(attn8_kernel<KV8_E4M3, 1>, cudaFuncAttributeMaxDynamicSharedMemorySize, sizeof(Smem<1>));
    cudaFuncSetAttribute(attn8_kernel<KV8_INT8, 4>, cudaFuncAttributeMaxDynamicSharedMemorySize, sizeof(Smem<4>));
    cudaFuncSetAttribute(attn8_kernel<KV8_E4M3, 4>, cudaFuncAttributeMaxDynamicSharedMemorySize, sizeof(Smem<4>));
}

}  // namespace mmz
