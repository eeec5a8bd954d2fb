// Attention over the 8-bit key/value cache (kv8.cu), for sm_100a. For sequence b, query row i and query head h, with
// L = min(lens[b], cap) and key head g = h / (q_heads / kv_heads):
//     s_j = scale * ks[b][g][j / block] * (q . k8_j)    for j < limit,  limit = L, or L - rows + i + 1 when causal
//     out = sum_j softmax(s)_j * vs[b][g][j / block] * v8_j      (zeros where limit <= 0)
// and the probabilities of chosen heads as fp16. Sums and softmax statistics in fp32; only the outputs are rounded.
//
// The query heads and rows that share a key head are one block of rows: up to 8 (a decoding step, hypotheses of one
// clip, grouped heads) or tiles of 16 (prompts). A warp takes chunks of 64 positions, keys and values by bulk copies
// into a ring of its own, and works in registers from there:
//   * every code (int8 or e4m3) is a number of fp16, so the products run exactly on the tensor cores (m16n8k16, fp32
//     sums): S^T = K q^T with the 16 positions as M and the 8 rows as N, then O^T = V^T P^T. The contraction indices are
//     dealt so that a lane's K fragment is 16 consecutive bytes of a row and its V fragment 8 consecutive bytes of 4
//     rows; no code is moved between lanes, and P^T is S^T's own layout after one 8 x 8 transpose.
//   * a running maximum and sum per row; p carries a factor 2^10 (it cancels against the sum) and is split into a high
//     and a low fp16 part, each multiplied: what is lost of p is below 2^-21 of it, and below 2^-35 of the row's
//     largest p, so the one rounding that counts stays that of the output. Up to 4 rows the two parts are columns
//     r and r + 4 of one product (the lanes of columns 4-7 hold the same scores and keep the low part).
//   * the scales of a block apply in fp32: ks to the scores, vs to the sums of the positions that share it.
// Three ways through the cache (plan() chooses):
//   cluster  a CTA to a (pair, row block), its warps along the positions; CTAs of a cluster split the sequence and join
//            through distributed shared memory, and where one cluster is too little (and more than 8 rows), clusters
//            through scratch and a second kernel
//   rows     more than 16 rows, enough of them to fill the GPU (prompts): a CTA of one warp to 16 rows, which takes all they see
//   flat     up to 8 rows and too few pairs for a cluster each to fill the GPU (long caches): a fixed number of warps,
//            each with an equal share of all sequences' and heads' chunks in a row, whatever the lengths; a pair's parts on
//            several warps join in a second kernel
// Measured (calls in a CUDA graph): 32 sequences x 20 heads x 1500 positions, int8, 29 us = 4.3 TB/s, with 6 heads recorded
// 32; 3 sequences of up to 131072 positions and 5 key heads x 4, e4m3, 33 us = 3.8 TB/s; one sequence of 20 heads 5.3 us.
// What bounds the first two is not the bytes (DRAM 48 and 52 %): a chunk is 870 to 920 instructions of a warp, and 2 to 3
// warps to a scheduler cover half of their latencies (46 to 51 % of the issue slots used).
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

struct Smem {
    uint8_t ring[WARPS][STG][2][KB];
    uint64_t full[WARPS][STG];
    int abort, pad[3];
    // cluster: followed by what the cluster's warps send this CTA for each of the block's rows: statistics float2
    // [row][source], then sums float [row][source][64 / cs] of the dimensions that this CTA joins
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

// scores of 16 positions against 8 rows per column tile, from 16 bytes of the keys place(g) and place(g) + 8 (those from
// byte 16 t on); lane (g, t) receives these positions for rows 2t and 2t + 1
template <int KIND, int NTL>
__device__ __forceinline__ void scores16(const uint4& lo, const uint4& hi, const uint32_t (&q)[NTL][8], float (&s)[NTL][4]) {
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

__device__ __forceinline__ void st_dsmem_f32x4(uint32_t addr, float x, float y, float z, float w) {
    asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "f"(x), "f"(y), "f"(z), "f"(w) : "memory");
}

__device__ __forceinline__ int seq_len(const Attn8& a, long b) {
    if (a.done && a.done[b]) return 0;
    return a.lens ? max(0, min(a.lens[b], a.cap)) : a.cap;
}
__device__ __forceinline__ float weight(float m, float M) { return m == -INFINITY ? 0.f : ex2_approx(m - M); }

// 1 / the sum of a row's p: 0 for a row that saw nothing, NaN kept
__device__ __forceinline__ float inverse(float l) { return l > 0.f ? 1.f / l : (l == l ? 0.f : l); }

__device__ __forceinline__ uint32_t nan_codes(uint32_t w) {  // 0x80 in the bytes of w that hold e4m3's NaN
    return ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
}

// A warp's rows and their running results. MODE 0: up to 4 rows, columns 4-7 repeat columns 0-3; 1: up to 8; 2: up to 16.
// Lane (g, t) of the warp (g = lane / 4, t = lane % 4) holds columns 8 n + 2 t + e of dimensions 8 g .. 8 g + 7.
template <int KIND, int MODE>
struct Rows {
    static constexpr int NTL = MODE == 2 ? 2 : 1;        // column tiles of 8
    static constexpr int SUB = NTL == 1 ? 64 : 32;       // positions whose scores are in registers at a time
    static constexpr int NJ = SUB / 16;
    uint32_t q[NTL][8];
    float m[NTL][2], l[NTL][2], o[4][NTL][4];  // o[i][n][e + 2 k]: dimension 8 g + 2 i + k, column 8 n + 2 t + e
    float* raw[NTL][2];                        // where the scores of the lane's columns go, null: nowhere
    bool any;                                  // some lane of the warp has a raw
    int badpos;                                // the first position whose value scale is not finite (odd_scales)

    // the row of column c of tile n
    static __device__ __forceinline__ int row(int n, int c) { return MODE == 0 ? c & 3 : 8 * n + c; }
    // rows r0 .. R - 1 of a pair (heads hk * group ..), query row r / group, head r % group
    __device__ __forceinline__ void queries(const Attn8& a, long b, int hk, int group, int r0, int R, int lane) {
#pragma unroll
        for (int n = 0; n < NTL; n++) {
            const int r = r0 + row(n, lane >> 2);
            if (r < R) load_q(a.q + b * a.q_seq + (r / group) * a.q_row + (hk * group + r % group) * a.q_head, lane & 3, q[n]);
            else
                for (int i = 0; i < 8; i++) q[n][i] = 0;
        }
    }
    // the rows' places in raw scores [batch][slots][rows][cap]
    __device__ __forceinline__ void record(const Attn8& a, float* to, long b, int hk, int group, int r0, int R, int lane) {
        bool have_one = false;
#pragma unroll
        for (int n = 0; n < NTL; n++)
#pragma unroll
            for (int e = 0; e < 2; e++) {
                const int r = r0 + 8 * n + 2 * (lane & 3) + e;
                raw[n][e] = nullptr;
                if (!to || r >= R || !have(lane & 3)) continue;
                const int slot = a.pslot[hk * group + r % group];
                if (slot < 0 || slot >= a.slots) continue;
                raw[n][e] = to + ((b * a.slots + slot) * a.rows + r / group) * (long)a.cap;
                have_one = true;
            }
        any = to && __any_sync(0xffffffff, have_one);
    }
    __device__ __forceinline__ void clear() {
        badpos = 0x7fffffff;
#pragma unroll
        for (int n = 0; n < NTL; n++) {
            m[n][0] = m[n][1] = -INFINITY;
            l[n][0] = l[n][1] = 0.f;
#pragma unroll
            for (int i = 0; i < 4; i++) o[i][n][0] = o[i][n][1] = o[i][n][2] = o[i][n][3] = 0.f;
        }
    }
    // O = O alpha + (the values' products with P). ONE: the SUB positions share one scale; else tiles of 16 that do are
    // `same` + 1 in number (1 or 2)
    template <bool ONE>
    __device__ __forceinline__ void values(const uint2 (&w)[NJ][4], const uint32_t (&ph)[NJ][NTL][2],
                                           const uint32_t (&pl)[NJ][NTL][2], const float (&alpha)[NTL][2], float sc,
                                           int from, int same) {
        const float v0 = __shfl_sync(0xffffffff, sc, from);
#pragma unroll
        for (int i = 0; i < 4; i++) {  // dimensions 8 g + 2 i and 8 g + 2 i + 1
#pragma unroll
            for (int n = 0; n < NTL; n++)
#pragma unroll
                for (int e = 0; e < 4; e++) o[i][n][e] *= alpha[n][e & 1];
            float acc[NTL][4];
#pragma unroll
            for (int j = 0; j < NJ; j++) {
                if (j == 0 || (!ONE && (j & same) == 0))
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
                    if (MODE != 0) mma(acc[n], f, pl[j][n][0], pl[j][n][1]);
                }
                if (ONE ? j == NJ - 1 : ((j + 1) & same) == 0) {
                    const float vsc = ONE ? v0 : __shfl_sync(0xffffffff, sc, from + j);
#pragma unroll
                    for (int n = 0; n < NTL; n++)
#pragma unroll
                        for (int e = 0; e < 4; e++) o[i][n][e] += vsc * acc[n][e];
                }
            }
        }
    }
    // A value scale (chunk_scale's lanes 4-7) that is not finite, in a chunk that some rows see only a part of: left out of
    // the sums (a weight of 0 times it would not be 0), and the rows that do see its positions are NaN in the end
    __device__ __forceinline__ void odd_scales(float& sc, int base, int lane) {
        const bool odd = lane >= 4 && !(fabsf(sc) <= 3.402823466e38f);
        const unsigned tiles = __ballot_sync(0xffffffff, odd) >> 4;
        if (tiles) {
            badpos = min(badpos, base + 16 * (__ffs(tiles) - 1));
            if (odd) sc = 0.f;
        }
    }
    // One chunk: codes at ck, cv (shared memory), positions base .. base + 63 of which those below `most` exist. sc:
    // chunk_scale's; scale: the scores' factor. lim: what the lane's columns see; whole: every row sees the whole chunk.
    __device__ __forceinline__ void chunk(const uint8_t* ck, uint8_t* cv, int base, int most, bool whole, float sc,
                                          float scale, const int (&lim)[NTL][2], int block, int lane) {
        const int g = lane >> 2, t = lane & 3;
        if (lane < 4) sc *= scale * LOG2E;
        // the sequence's last chunk: the rows that were not copied hold what the ring held. Their weights are 0, but a
        // NaN times 0 would not be
        if (base + CH > most) {
            for (int i = (most - base) * HD + lane * 16; i < KB; i += 512)
                *reinterpret_cast<uint4*>(cv + i) = make_uint4(0, 0, 0, 0);
            __syncwarp();
        }
#pragma unroll
        for (int sub = 0; sub < CH / SUB; sub++) {
            const int sb = base + sub * SUB;
            if (sub && sb >= most) break;
            float s[NJ][NTL][4];
#pragma unroll
            for (int j = 0; j < NJ; j++) {
                const uint8_t* k = ck + (sub * SUB + 16 * j + place(g)) * HD + 16 * t;
                scores16<KIND, NTL>(*reinterpret_cast<const uint4*>(k), *reinterpret_cast<const uint4*>(k + 8 * HD), q, s[j]);
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
            if (any) {
#pragma unroll
                for (int j = 0; j < NJ; j++)
#pragma unroll
                    for (int n = 0; n < NTL; n++)
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            const int p = sb + 16 * j + place(g) + 8 * (e >> 1);
                            if (raw[n][e & 1] && p < lim[n][e & 1]) raw[n][e & 1][p] = s[j][n][e];
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
                    for (int j = 0; j < NJ; j++) mx = fmax3(mx, s[j][n][e], s[j][n][e + 2]);
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
                        const uint32_t h = *reinterpret_cast<const uint32_t*>(&hi), z = *reinterpret_cast<const uint32_t*>(&lo);
                        if (MODE == 0) {
                            ph[j][n][u] = transpose8(t < 2 ? h : z);
                        } else {
                            ph[j][n][u] = transpose8(h);
                            pl[j][n][u] = transpose8(z);
                        }
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
            if (block >= SUB) values<true>(w, ph, pl, alpha, sc, 4 + sub * NJ, 0);
            else values<false>(w, ph, pl, alpha, sc, 4 + sub * NJ, block / 16 - 1);
            if (nans) {
#pragma unroll
                for (int i = 0; i < 4; i++)
#pragma unroll
                    for (int n = 0; n < NTL; n++)
#pragma unroll
                        for (int e = 0; e < 4; e++)
                            if (nanpos[2 * i + (e >> 1)] < lim[n][e & 1]) o[i][n][e] = NAN;
            }
        }
    }
    // after the last chunk: the lanes' sums of p added up, and the two parts of MODE 0. Columns with have(t) are valid
    __device__ __forceinline__ void finish(const int (&lim)[NTL][2]) {
#pragma unroll
        for (int n = 0; n < NTL; n++)
#pragma unroll
            for (int e = 0; e < 2; e++) {
                if (badpos < lim[n][e])
#pragma unroll
                    for (int i = 0; i < 4; i++) o[i][n][e] = o[i][n][e + 2] = NAN;
                l[n][e] += __shfl_xor_sync(0xffffffff, l[n][e], 4);
                l[n][e] += __shfl_xor_sync(0xffffffff, l[n][e], 8);
                l[n][e] += __shfl_xor_sync(0xffffffff, l[n][e], 16);
            }
        if (MODE == 0)
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
                for (int e = 0; e < 4; e++) o[i][0][e] += __shfl_xor_sync(0xffffffff, o[i][0][e], 2);
    }
    static __device__ __forceinline__ bool have(int t) { return MODE != 0 || t < 2; }
    // the finished rows, divided by their sums, to out (and their statistics)
    __device__ __forceinline__ void store(const Attn8& a, long b, int hk, int group, int r0, int R, float2* stats, int lane) {
        const int g = lane >> 2, t = lane & 3;
#pragma unroll
        for (int n = 0; n < NTL; n++)
#pragma unroll
            for (int e = 0; e < 2; e++) {
                const int r = r0 + 8 * n + 2 * t + e;
                if (!have(t) || r >= R) continue;
                const float inv = inverse(l[n][e]);
                uint4 x;
                __half2* h = reinterpret_cast<__half2*>(&x);
#pragma unroll
                for (int i = 0; i < 4; i++) h[i] = __floats2half2_rn(o[i][n][e] * inv, o[i][n][e + 2] * inv);
                *reinterpret_cast<uint4*>(a.out + b * a.o_seq + (r / group) * a.o_row + (hk * group + r % group) * a.o_head +
                                          8 * g) = x;
                if (stats && g == 0) stats[(b * a.kv_heads + hk) * R + r] = make_float2(m[n][e], inv);
            }
    }
};

// lanes 0-3: the key scales of a chunk's four tiles of 16 positions, lanes 4-7 the value scales. A load whose result is
// first used with the chunk, so that it is never waited for on the way there
__device__ __forceinline__ float chunk_scale(const float* ks, const float* vs, int c, int most, int shift, int lane) {
    if (lane >= 8) return 0.f;
    const int j = min(c * CH + 16 * (lane & 3), most - 1) >> shift;
    return lane < 4 ? ks[j] : vs[j];
}

// How a cluster call is laid out along its CTAs (plan() below).
struct Lay {
    int cs, nclus;  // CTAs of a cluster, clusters along the sequence
    int block;      // rows of a CTA that exist at most (what its shared memory holds)
    int tiles;      // CTAs along the rows
    int inside;     // the parts are exchanged where the ring was
};

}  // namespace a8
using namespace a8;

// grid: cluster rank fastest, then cluster along the sequence, (sequence, key head), row block; cluster of cs CTAs.
// nclus 1: the cluster's rows go to out (and their statistics to stats, if not null); else to part
template <int KIND, int MODE>
__global__ void __launch_bounds__(NT, 3) attn8_kernel(Attn8 a, Lay lay, float* part, float2* stats, float* raws, unsigned* status,
                                                   unsigned long long limit_ns) {
    constexpr int NTL = Rows<KIND, MODE>::NTL, RT = 8 * NTL;
    extern __shared__ __align__(128) uint8_t smem[];
    Smem& sm = *reinterpret_cast<Smem*>(smem);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int cs = lay.cs;
    unsigned x = blockIdx.x;
    const int rank = x % cs;
    x /= cs;
    const int clus = x % lay.nclus;
    x /= lay.nclus;
    // every pair's last rows first: with causal they have the most to do, and the first rows' blocks fill up the end
    const unsigned pairs = (unsigned)a.batch * a.kv_heads, pair = x % pairs;
    const int tile = lay.tiles - 1 - (int)(x / pairs);
    const int hk = (int)(pair % a.kv_heads), group = a.q_heads / a.kv_heads;
    const long b = pair / a.kv_heads;
    const int R = a.rows * group;
    const int r0 = tile * RT;  // first row
    if (lane == 0)
        for (int i = 0; i < STG; i++) mbar_init(&sm.full[warp][i], 1);
    if (threadIdx.x == 0) sm.abort = 0;
    fence_mbar_init();
    __syncthreads();
    if (cs > 1) cluster_arrive_relaxed();  // the cluster's CTAs have started before anything is sent to them
    griddep_wait();
    griddep_launch_dependents();

    Rows<KIND, MODE> w;
    w.queries(a, b, hk, group, r0, R, lane);
    w.record(a, raws, b, hk, group, r0, R, lane);
    w.clear();
    const int L = seq_len(a, b);
    // what row r sees; the warp's last row sees the most
    auto limit = [&](int r) { return a.causal ? max(0, L - a.rows + r / group + 1) : L; };
    const int most = r0 < R ? limit(min(r0 + RT, R) - 1) : 0, least = r0 < R ? limit(r0) : 0;
    const int nch = (most + CH - 1) / CH;
    const int ns = cs * lay.nclus, per = (nch + ns - 1) / ns, split = clus * cs + rank;
    const int c0 = min(split * per, nch), c1 = min(c0 + per, nch);
    const int cw = c0 + warp;  // the warp's first chunk; then every WARPS-th
    const uint8_t* k8 = a.k8 + b * a.c_seq + hk * a.c_head;
    const uint8_t* v8 = a.v8 + b * a.c_seq + hk * a.c_head;
    const float* ks = a.ks + b * a.s_seq + hk * a.s_head;
    const float* vs = a.vs + b * a.s_seq + hk * a.s_head;
    const int shift = 31 - __clz(a.block);

    uint64_t* full = sm.full[warp];
    auto issue = [&](int c, int st) {  // lane 0
        const uint32_t bytes = (uint32_t)min(CH, most - c * CH) * HD;
        mbar_expect_tx(&full[st], 2 * bytes);
        bulk_g2s(sm.ring[warp][st][0], k8 + (long)c * KB, bytes, &full[st]);
        bulk_g2s(sm.ring[warp][st][1], v8 + (long)c * KB, bytes, &full[st]);
    };
    auto scale_of = [&](int c) { return c < c1 ? chunk_scale(ks, vs, c, most, shift, lane) : 0.f; };
    int at = cw;
    if (lane == 0)
        for (int i = 0; i < STG && cw + i * WARPS < c1; i++) issue(cw + i * WARPS, i);
    float sc_next = scale_of(cw);
    int lim[NTL][2];
#pragma unroll
    for (int n = 0; n < NTL; n++)
#pragma unroll
        for (int e = 0; e < 2; e++) lim[n][e] = limit(min(r0 + w.row(n, 2 * t + e), R - 1));

    bool ok = true;
    int it = 0;
    for (int c = cw; c < c1; c += WARPS, it++) {
        const int st = it % STG;
        ok = __all_sync(0xffffffff, mbar_wait(&full[st], (it / STG) & 1, &sm.abort, limit_ns, status, K_ATTN8, 1));
        if (!ok) break;
        float sc = sc_next;
        if (least < most && c * CH + CH > least) w.odd_scales(sc, c * CH, lane);
        sc_next = scale_of(c + WARPS);
        w.chunk(sm.ring[warp][st][0], sm.ring[warp][st][1], c * CH, most, c * CH + CH <= least, sc, a.scale, lim,
                a.block, lane);
        __syncwarp();
        if (lane == 0 && c + STG * WARPS < c1) issue(c + STG * WARPS, st);
        at = c + WARPS;
    }
    if (!ok && lane == 0) {  // a wait gave up: let the copies in flight land before the CTA ends
        for (int i = 0; i < STG; i++, it++)
            if (at + i * WARPS < c1) mbar_wait(&full[it % STG], (it / STG) & 1, nullptr, limit_ns, nullptr, 0, 0);
    }
    w.finish(lim);

    // ---------------------------------------------------------------- the parts of a row joined
    // Each warp sends its rows' statistics to every CTA of the cluster and its sums to the CTA that joins those
    // dimensions (the lane's 8 have one owner): stores, and one barrier, instead of loads that are waited for.
    const int nsrc = cs * WARPS, src = rank * WARPS + warp, share = HD / cs;
    if (MODE == 2 && lay.inside) __syncthreads();
    float2* ms = reinterpret_cast<float2*>(smem + (MODE == 2 && lay.inside ? 0 : sizeof(Smem)));
    float* sums = reinterpret_cast<float*>(ms + lay.block * nsrc + (lay.block * nsrc & 1));
    if (cs > 1) cluster_wait();
#pragma unroll
    for (int n = 0; n < NTL; n++)
#pragma unroll
        for (int e = 0; e < 2; e++) {
            const int r = 8 * n + 2 * t + e;  // row of the block
            if (!w.have(t) || r >= lay.block) continue;
            if (g < cs) st_dsmem_f32x2(dsmem_addr(&ms[r * nsrc + src], g), make_float2(w.m[n][e], w.l[n][e]));
            const uint32_t to = dsmem_addr(&sums[(r * nsrc + src) * share + 8 * g % share], 8 * g / share);
            st_dsmem_f32x4(to, w.o[0][n][e], w.o[0][n][e + 2], w.o[1][n][e], w.o[1][n][e + 2]);
            st_dsmem_f32x4(to + 16, w.o[2][n][e], w.o[2][n][e + 2], w.o[3][n][e], w.o[3][n][e + 2]);
        }
    if (cs > 1) cluster_sync();
    else __syncthreads();
    for (int i = threadIdx.x; i < lay.block * (share / 2); i += NT) {
        const int r = i / (share / 2), dl = 2 * (i % (share / 2)), d = rank * share + dl;
        if (r0 + r >= R) break;
        float M = -INFINITY, S = 0.f;
        float2 O = make_float2(0.f, 0.f);
#pragma unroll 4
        for (int w = 0; w < nsrc; w++) M = fmaxf(M, ms[r * nsrc + w].x);
#pragma unroll 4
        for (int w = 0; w < nsrc; w++) {
            const float2 y = ms[r * nsrc + w], x = *reinterpret_cast<const float2*>(&sums[(r * nsrc + w) * share + dl]);
            const float f = weight(y.x, M);
            S += f * y.y;
            O.x += f * x.x;
            O.y += f * x.y;
        }
        const long row = (long)pair * R + r0 + r;
        if (lay.nclus > 1) {
            float* rec = part + (row * lay.nclus + clus) * REC;
            *reinterpret_cast<float2*>(rec + d) = O;
            if (d == 0) *reinterpret_cast<float2*>(rec + HD) = make_float2(M, S);
        } else {
            const float inv = inverse(S);
            const int qi = (r0 + r) / group, h = hk * group + (r0 + r) % group;
            *reinterpret_cast<__half2*>(a.out + b * a.o_seq + qi * a.o_row + h * a.o_head + d) =
                __floats2half2_rn(O.x * inv, O.y * inv);
            if (stats && d == 0) stats[row] = make_float2(M, inv);
        }
    }
}

// ---------------------------------------------------------------- rows of a warp's own
namespace a8 {
// A CTA of one warp: the last ones of a grid fill the GPU evenly, whatever the lengths (223 causal rows on 160 pairs of 150 to
// 448 positions: 30 us, with four such warps to a CTA 37)
struct RowsSmem {
    uint8_t ring[STG][2][KB];
    uint64_t full[STG];
};
}  // namespace a8

// grid: (sequence, key head) fastest, then tile of 16 rows, the last tile first (with causal it has the most to do).
// Static shared memory above 16 KB of ring: 12 CTAs to an SM
template <int KIND>
__global__ void __launch_bounds__(32, 12) attn8_rows_kernel(Attn8 a, int tiles, float2* stats, float* raws, unsigned* status,
                                                            unsigned long long limit_ns) {
    constexpr int NTL = Rows<KIND, 2>::NTL, RT = 8 * NTL;
    __shared__ __align__(128) RowsSmem sm;
    const int lane = threadIdx.x & 31, t = lane & 3;
    const unsigned pairs = (unsigned)a.batch * a.kv_heads, pair = blockIdx.x % pairs;
    const int hk = (int)(pair % a.kv_heads), group = a.q_heads / a.kv_heads;
    const long b = pair / a.kv_heads;
    const int R = a.rows * group, r0 = (tiles - 1 - (int)(blockIdx.x / pairs)) * RT;
    if (lane == 0)
        for (int i = 0; i < STG; i++) mbar_init(&sm.full[i], 1);
    fence_mbar_init();
    __syncwarp();
    griddep_wait();
    griddep_launch_dependents();

    Rows<KIND, 2> w;
    w.queries(a, b, hk, group, r0, R, lane);
    w.record(a, raws, b, hk, group, r0, R, lane);
    w.clear();
    const int L = seq_len(a, b);
    auto limit = [&](int r) { return a.causal ? max(0, L - a.rows + r / group + 1) : L; };
    const int most = limit(min(r0 + RT, R) - 1), least = limit(r0), nch = (most + CH - 1) / CH;
    const uint8_t* k8 = a.k8 + b * a.c_seq + hk * a.c_head;
    const uint8_t* v8 = a.v8 + b * a.c_seq + hk * a.c_head;
    const float* ks = a.ks + b * a.s_seq + hk * a.s_head;
    const float* vs = a.vs + b * a.s_seq + hk * a.s_head;
    const int shift = 31 - __clz(a.block);
    auto issue = [&](int c) {  // lane 0
        const uint32_t bytes = (uint32_t)min(CH, most - c * CH) * HD;
        uint64_t* full = &sm.full[c % STG];
        mbar_expect_tx(full, 2 * bytes);
        bulk_g2s(sm.ring[c % STG][0], k8 + (long)c * KB, bytes, full);
        bulk_g2s(sm.ring[c % STG][1], v8 + (long)c * KB, bytes, full);
    };
    auto scale_of = [&](int c) { return c < nch ? chunk_scale(ks, vs, c, most, shift, lane) : 0.f; };
    if (lane == 0)
        for (int c = 0; c < STG && c < nch; c++) issue(c);
    float sc_next = scale_of(0);
    int lim[NTL][2];
#pragma unroll
    for (int n = 0; n < NTL; n++)
#pragma unroll
        for (int e = 0; e < 2; e++) lim[n][e] = limit(min(r0 + w.row(n, 2 * t + e), R - 1));

    int c = 0;
    for (; c < nch; c++) {
        const int st = c % STG;
        if (!__all_sync(0xffffffff, mbar_wait(&sm.full[st], (c / STG) & 1, nullptr, limit_ns, status, K_ATTN8, 3))) break;
        float sc = sc_next;
        if (least < most && c * CH + CH > least) w.odd_scales(sc, c * CH, lane);
        sc_next = scale_of(c + 1);
        w.chunk(sm.ring[st][0], sm.ring[st][1], c * CH, most, c * CH + CH <= least, sc, a.scale, lim, a.block, lane);
        __syncwarp();
        if (lane == 0 && c + STG < nch) issue(c + STG);
    }
    if (lane == 0)  // after a wait that gave up: let the copies in flight land before the CTA ends
        for (int i = c; i < min(c + STG, nch); i++) mbar_wait(&sm.full[i % STG], (i / STG) & 1, nullptr, limit_ns, nullptr, 0, 0);
    w.finish(lim);
    w.store(a, b, hk, group, r0, R, stats, lane);
}

// ---------------------------------------------------------------- flat
// All chunks of all (sequence, key head) pairs in one row, pairs in order, chunks in order. Of its T chunks each of the W
// warps has T / W, the first T % W one more. Where a pair lies on several warps, the warp with its first chunk leaves its
// part in record 2 w + 1, the others in 2 w. (T below 2^31: 32-bit divisions, the 64-bit ones cost microseconds here.)
namespace a8 {
constexpr int RECF = 8 * HD + 16;  // a record: [8 rows][64] sums, [8][2] statistics

struct Share {
    unsigned T, W, per, more;
    __device__ __forceinline__ Share(unsigned T, unsigned W) : T(T), W(W), per(T / W), more(T % W) {}
    __device__ __forceinline__ unsigned first(unsigned w) const { return w * per + min(w, more); }
    __device__ __forceinline__ unsigned count(unsigned w) const { return per + (w < more ? 1 : 0); }
    __device__ __forceinline__ unsigned owner(unsigned f) const {  // the warp that has chunk f
        const unsigned big = more * (per + 1);
        return f < big ? f / (per + 1) : more + (f - big) / per;
    }
};
struct Flat {
    const Attn8& a;
    const int cap, batch, kv_heads;
    const bool all_alike;  // every sequence has cap positions
    __device__ __forceinline__ Flat(const Attn8& a)
        : a(a), cap(a.cap), batch(a.batch), kv_heads(a.kv_heads), all_alike(!a.lens && !a.done) {}
    __device__ __forceinline__ int len(int b) const { return seq_len(a, b); }
    __device__ __forceinline__ unsigned chunks(int b) const { return b < batch ? (unsigned)(len(b) + CH - 1) / CH : 0; }
    // whole warp: the chunks of the sequences before b, and of all of them
    __device__ __forceinline__ void before(int b, int lane, unsigned& upto, unsigned& all) const {
        upto = all = 0;
        if (all_alike) {
            upto = (unsigned)b * chunks(0) * kv_heads;
            all = (unsigned)batch * chunks(0) * kv_heads;
            return;
        }
        for (int i = lane; i < batch; i += 32) {
            const unsigned n = chunks(i);
            all += n;
            if (i < b) upto += n;
        }
        all = __reduce_add_sync(0xffffffff, all) * kv_heads;
        upto = __reduce_add_sync(0xffffffff, upto) * kv_heads;
    }
    // whole warp: the chunks that warp w of W has, and where they start: sequence b, and f its place among that
    // sequence's. One load per lane for up to 32 sequences
    __device__ __forceinline__ unsigned find(unsigned w, unsigned W, int lane, int& b, int& len, unsigned& f) const {
        unsigned upto, all, n;
        if (all_alike) {
            before(0, lane, upto, all);
            const Share share(all, W);
            const unsigned per = chunks(0) * kv_heads;
            f = share.first(w);
            b = f / per, len = cap;
            f -= b * per;
            return share.count(w);
        }
        all = 0;
        if (batch > 32) before(0, lane, upto, all);
        for (int i = 0;; i += 32) {
            const int l = i + lane < batch ? this->len(i + lane) : 0;
            const unsigned mine = (unsigned)(l + CH - 1) / CH * kv_heads;
            unsigned up = mine;  // through this lane's sequence
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const unsigned x = __shfl_up_sync(0xffffffff, up, o);
                if (lane >= o) up += x;
            }
            if (i == 0) {
                if (batch <= 32) all = __shfl_sync(0xffffffff, up, 31);
                const Share share(all, W);
                n = share.count(w);
                if (n == 0) return 0;
                f = share.first(w);
            }
            const unsigned hit = __ballot_sync(0xffffffff, up > f);
            if (hit) {
                const int k = __ffs(hit) - 1;
                f -= __shfl_sync(0xffffffff, up - mine, k);
                b = i + k, len = __shfl_sync(0xffffffff, l, k);
                return n;
            }
            f -= __shfl_sync(0xffffffff, up, 31);
            if (i + 32 >= batch) return 0;  // not reached: f is below the total
        }
    }
};
// where a warp stands in the row of chunks
struct Place {
    int b, hk, c, len, nch;
    __device__ __forceinline__ void next(const Flat& f) {
        if (++c < nch) return;
        c = 0;
        if (++hk < f.kv_heads) return;
        hk = 0;
        do b++;
        while (b < f.batch && (nch = ((len = f.len(b)) + CH - 1) / CH) == 0);
    }
};
}  // namespace a8

// (at most 128 registers, so that the next kernel's blocks find room beside three CTAs)
template <int KIND, int MODE>
__global__ void __launch_bounds__(NT, 4) attn8_flat_kernel(Attn8 a, float* rec, float2* stats, float* raws, unsigned* status,
                                                        unsigned long long limit_ns) {
    extern __shared__ __align__(128) uint8_t smem[];
    Smem& sm = *reinterpret_cast<Smem*>(smem);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int group = a.q_heads / a.kv_heads, R = a.rows * group;
    const Flat flat(a);
    uint64_t* full = sm.full[warp];
    if (lane == 0)
        for (int i = 0; i < STG; i++) mbar_init(&full[i], 1);
    if (threadIdx.x == 0) sm.abort = 0;
    fence_mbar_init();
    __syncthreads();  // the last barrier of the CTA: from here on the warps are on their own
    griddep_wait();
    griddep_launch_dependents();
    const unsigned me = blockIdx.x * WARPS + warp;
    Place cur;
    unsigned f;
    const unsigned n = flat.find(me, gridDim.x * WARPS, lane, cur.b, cur.len, f);
    if (n == 0) return;
    cur.nch = (cur.len + CH - 1) / CH;
    cur.hk = f / (unsigned)cur.nch;
    cur.c = f % (unsigned)cur.nch;
    Place ahead = cur;
    const int shift = 31 - __clz(a.block);
    float sc[STG];  // the scales of the chunks in the ring, the next one first
    unsigned sent = 0;
    auto issue = [&](int st) {  // the chunk at `ahead` into stage st; returns its scales
        const long at = (long)ahead.b * a.c_seq + ahead.hk * a.c_head + (long)ahead.c * KB;
        if (lane == 0) {
            const uint32_t bytes = (uint32_t)min(CH, ahead.len - ahead.c * CH) * HD;
            mbar_expect_tx(&full[st], 2 * bytes);
            bulk_g2s(sm.ring[warp][st][0], a.k8 + at, bytes, &full[st]);
            bulk_g2s(sm.ring[warp][st][1], a.v8 + at, bytes, &full[st]);
        }
        const long sat = (long)ahead.b * a.s_seq + ahead.hk * a.s_head;
        const float x = chunk_scale(a.ks + sat, a.vs + sat, ahead.c, ahead.len, shift, lane);
        sent++;
        if (sent < n) ahead.next(flat);
        return x;
    };
#pragma unroll
    for (int i = 0; i < STG; i++) sc[i] = sent < n ? issue(i) : 0.f;

    Rows<KIND, MODE> w;
    int lim[1][2], from = cur.c;  // the segment's first chunk
    auto begin = [&]() {
        w.queries(a, cur.b, cur.hk, group, 0, R, lane);
        w.record(a, raws, cur.b, cur.hk, group, 0, R, lane);
        w.clear();
#pragma unroll
        for (int e = 0; e < 2; e++) {
            const int i = min(w.row(0, 2 * t + e), R - 1) / group;
            lim[0][e] = a.causal ? max(0, cur.len - a.rows + i + 1) : cur.len;
        }
        from = cur.c;
    };
    begin();
    bool ok = true;
    unsigned it = 0;
    for (; it < n; it++) {
        const int st = it % STG;
        ok = __all_sync(0xffffffff, mbar_wait(&full[st], (it / STG) & 1, &sm.abort, limit_ns, status, K_ATTN8, 2));
        if (!ok) break;
        const int base = cur.c * CH, least = a.causal ? max(0, cur.len - a.rows + 1) : cur.len;
        if (least < cur.len && base + CH > least) w.odd_scales(sc[0], base, lane);
        w.chunk(sm.ring[warp][st][0], sm.ring[warp][st][1], base, cur.len, base + CH <= least, sc[0], a.scale, lim,
                a.block, lane);
        if (base + CH > cur.len) fence_proxy_async_smem();  // zeros written behind the end, before the next copy
        __syncwarp();
#pragma unroll
        for (int i = 0; i + 1 < STG; i++) sc[i] = sc[i + 1];
        if (sent < n) sc[STG - 1] = issue(st);
        const bool last = cur.c + 1 == cur.nch;
        if (last || it + 1 == n) {
            w.finish(lim);
            if (last && from == 0) {
                w.store(a, cur.b, cur.hk, group, 0, R, stats, lane);
            } else {
                float* to = rec + (2 * me + (from == 0 ? 1 : 0)) * (long)RECF;
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    const int r = 2 * t + e;
                    if (!w.have(t) || r >= R) continue;
                    float4* x = reinterpret_cast<float4*>(to + r * HD + 8 * g);
                    x[0] = make_float4(w.o[0][0][e], w.o[0][0][e + 2], w.o[1][0][e], w.o[1][0][e + 2]);
                    x[1] = make_float4(w.o[2][0][e], w.o[2][0][e + 2], w.o[3][0][e], w.o[3][0][e + 2]);
                    if (g == 0) *reinterpret_cast<float2*>(to + 8 * HD + 2 * r) = make_float2(w.m[0][e], w.l[0][e]);
                }
            }
            if (it + 1 < n) {
                cur.next(flat);
                begin();
            }
        } else {
            cur.c++;
        }
    }
    if (!ok && lane == 0)  // a wait gave up: let the copies in flight land before the CTA ends
        for (unsigned i = it; i < sent; i++) mbar_wait(&full[i % STG], (i / STG) & 1, nullptr, limit_ns, nullptr, 0, 0);
}

// ---------------------------------------------------------------- after the main kernel: parts joined, probabilities
namespace a8 {

// Where a row's parts lie: the k-th at (k ? more + k * step : one), its statistics `st` and its sums `so` floats in
struct Parts {
    const float *one, *more;
    int step, n, st, so;  // n 0: one warp or cluster had the row, which is written; -1: an empty sequence, zeros
    unsigned w0, none;    // flat: warps from `none` on have no chunks (fewer chunks than warps); the first is w0
    __device__ __forceinline__ const float* at(int k) const { return k ? more + (long)k * step : one; }
    __device__ __forceinline__ bool some(int k) const { return w0 + k < none; }
};
// (b, hk, r): the row's sequence, key head and place among the pair's R rows
__device__ __forceinline__ Parts parts_of(const Attn8& a, const float* part, int nclus, unsigned W, int b, int hk, int r,
                                          int R, int lane) {
    Parts p;
    p.w0 = 0, p.none = 0xffffffffu;
    if (W == 0) {
        p.one = p.more = part + (((long)b * a.kv_heads + hk) * R + r) * nclus * REC;
        p.step = REC, p.n = nclus > 1 ? nclus : 0, p.st = HD, p.so = 0;
        return p;
    }
    const Flat flat(a);
    unsigned upto, all;
    flat.before(b, lane, upto, all);
    const unsigned nch = flat.chunks(b);
    p.st = 8 * HD + 2 * r, p.so = r * HD, p.n = -1;
    if (nch == 0) return p;
    const Share share(all, W);
    const unsigned f0 = upto + hk * nch;
    p.w0 = share.owner(f0);
    p.n = (int)(share.owner(f0 + nch - 1) - p.w0 + 1);
    if (p.n == 1) p.n = 0;
    if (share.per == 0) p.none = share.more;
    p.one = part + (2 * p.w0 + 1) * (long)RECF;
    p.more = part + 2 * p.w0 * (long)RECF;
    p.step = 2 * RECF;
    return p;
}
// whole warp: the parts from first, first + stride.. on, 32 each, of a row joined into (M, S) and, SUMS, the lane's two
// dimensions
template <bool SUMS>
__device__ __forceinline__ void join_parts(const Parts& p, int first, int stride, int lane, float& M, float& S, float2& O) {
    M = -INFINITY, S = 0.f, O = make_float2(0.f, 0.f);
    for (int k0 = first; k0 < p.n; k0 += stride) {
        const int k = k0 + lane;
        float2 y = make_float2(-INFINITY, 0.f);
        if (k < p.n && p.some(k)) y = *reinterpret_cast<const float2*>(p.at(k) + p.st);
        float m = fmaxf(M, y.x);
#pragma unroll
        for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffff, m, o));
        const float f = weight(M, m), g = weight(y.x, m);
        M = m;
        float s = g * y.y;  // (0 where a part saw nothing; a NaN stays)
#pragma unroll
        for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffff, s, o);
        S = S * f + s;
        if constexpr (SUMS) {
            O.x *= f, O.y *= f;
            const unsigned have = __ballot_sync(0xffffffff, y.x != -INFINITY);  // a part whose row saw something
            const int n = min(32, p.n - k0);
            for (int j0 = 0; j0 < n; j0 += 16) {  // 16 loads at once
                float2 x[16];
#pragma unroll
                for (int j = 0; j < 16; j++) {
                    x[j] = make_float2(0.f, 0.f);
                    if (have >> (j0 + j) & 1) x[j] = *reinterpret_cast<const float2*>(p.at(k0 + j0 + j) + p.so + 2 * lane);
                }
#pragma unroll
                for (int j = 0; j < 16; j++) {
                    const float gj = __shfl_sync(0xffffffff, g, j0 + j);
                    O.x += gj * x[j].x;
                    O.y += gj * x[j].y;
                }
            }
        }
    }
}
}  // namespace a8

// Blocks 0 .. jblocks - 1: rows whose parts are joined and written, one to a block (jrows 1: the warps share its parts)
// or one to a warp (where a row has a few parts). The others: the probabilities of a (sequence, slot, row),
// p = 2^(s - M) / S from the scores that the main kernel left. This kernel starts once the main one has waited for what
// came before, and finds out where the parts lie meanwhile. (The probabilities at the end of the main kernel's CTAs instead:
// 5 rows on 120 pairs 17 us, this way 12; 32 sequences of one row 33 and 32.)
__global__ void __launch_bounds__(512) attn8_post_kernel(Attn8 a, unsigned jblocks, int jrows, int nclus, unsigned W,
                                                         const float* part, const float2* stats, const float* raws) {
    __shared__ float red[16][REC];
    __shared__ float2 rowms;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, nw = blockDim.x >> 5;
    const int group = a.q_heads / a.kv_heads, R = a.rows * group;
    Parts p;
    p.n = 0;
    if (blockIdx.x < jblocks) {
        const unsigned row = jrows == 1 ? blockIdx.x : blockIdx.x * nw + warp, pair = row / R;
        const int r = row % R, hk = pair % a.kv_heads, b = pair / a.kv_heads;
        if (b < a.batch) p = parts_of(a, part, nclus, W, b, hk, r, R, lane);
        griddep_wait();
        griddep_launch_dependents();
        if (p.n == 0) return;
        float M, S;
        float2 O;
        join_parts<true>(p, jrows == 1 ? 32 * warp : 0, jrows == 1 ? 32 * nw : 32, lane, M, S, O);
        if (jrows == 1) {
            red[warp][2 * lane] = O.x;
            red[warp][2 * lane + 1] = O.y;
            if (lane == 0) red[warp][HD] = M, red[warp][HD + 1] = S;
            __syncthreads();
            if (warp) return;
            float m = M;
            for (int w = 1; w < nw; w++) m = fmaxf(m, red[w][HD]);
            S = 0.f, O = make_float2(0.f, 0.f);
            for (int w = 0; w < nw; w++) {
                const float f = weight(red[w][HD], m);
                S += f * red[w][HD + 1];
                O.x += f * red[w][2 * lane];
                O.y += f * red[w][2 * lane + 1];
            }
        }
        const float inv = inverse(S);
        const int h = hk * group + r % group;
        *reinterpret_cast<__half2*>(a.out + (long)b * a.o_seq + (r / group) * a.o_row + h * a.o_head + 2 * lane) =
            __floats2half2_rn(O.x * inv, O.y * inv);
        return;
    }
    unsigned x = blockIdx.x - jblocks;
    const int i = x % a.rows;
    x /= a.rows;
    const int slot = x % a.slots, b = x / a.slots;
    int h = 0x7fffffff;
    for (int k = lane; k < a.q_heads; k += 32)
        if (h == 0x7fffffff && a.pslot[k] == slot) h = k;
    h = __reduce_min_sync(0xffffffff, h);
    const bool live = h < a.q_heads;  // a slot that no head has is left as it is
    const int hk = live ? h / group : 0, r = i * group + (live ? h % group : 0);
    if (live && warp == 0) p = parts_of(a, part, nclus, W, b, hk, r, R, lane);
    const int L = seq_len(a, b), lim = a.causal ? max(0, L - a.rows + i + 1) : L;
    griddep_wait();
    griddep_launch_dependents();
    if (!live || (a.done && a.done[b])) return;
    if (warp == 0) {
        float M = 0.f, S = 0.f;
        float2 O;
        if (p.n > 0) join_parts<false>(p, 0, 32, lane, M, S, O);
        if (lane == 0)
            rowms = p.n == 0 ? stats[((long)b * a.kv_heads + hk) * R + r] : make_float2(M, inverse(S));
    }
    __syncthreads();
    const float off = rowms.x - PSHIFT, inv = rowms.y;
    const long at = (((long)b * a.slots + slot) * a.rows + i) * a.cap;
    h16* to = a.probs + b * a.p_seq + (a.pctr ? *a.pctr * a.p_step : 0) + ((long)slot * a.rows + i) * a.cap;
    for (int j0 = threadIdx.x; j0 < a.cap; j0 += 8 * blockDim.x) {  // 8 loads at once
        float v[8];
#pragma unroll
        for (int k = 0; k < 8; k++) {
            const int j = j0 + k * blockDim.x;
            v[k] = j < lim ? raws[at + j] : -INFINITY;
        }
#pragma unroll
        for (int k = 0; k < 8; k++) {
            const int j = j0 + k * blockDim.x;
            if (j < a.cap) to[j] = __float2half_rn(j < lim ? ex2_approx(v[k] - off) * inv : 0.f);
        }
    }
}

// The layout of a call, from its sizes alone (lens is on the device), and its scratch.
namespace {
constexpr long SLOTS = 148 * 3;   // CTAs that a B200 holds at once (shared memory: 3 to an SM)
constexpr long PAIRED = 148 * 2;  // the same at two to an SM
constexpr size_t ALONE3 = 78 << 10;  // shared memory of which an SM has two, not three
struct Plan {
    int mode;   // Rows' MODE
    bool rows, flat;
    Lay lay;
    size_t smem, part, stats, raws;
};
// sizes that the products below can take; a call's blocks and scratch are fewer
bool sizes_ok(int batch, int rows, int q_heads, int kv_heads, int cap, int slots) {
    return within(0x7fffff00l, {rows, q_heads / kv_heads}) && within(1l << 40, {batch, rows, q_heads}) &&
           within(1l << 46, {batch, rows, slots, cap});
}
Plan plan(int batch, int rows, int q_heads, int kv_heads, int cap, int slots) {
    Plan p;
    const long R = (long)rows * (q_heads / kv_heads), pairs = (long)batch * kv_heads, chunks = ((long)cap + CH - 1) / CH;
    const long rt = R <= 8 ? 8 : 16;
    p.mode = R <= 4 ? 0 : R <= 8 ? 1 : 2;
    p.stats = slots > 0 ? ((size_t)pairs * R * 8 + 15) & ~(size_t)15 : 0;
    p.raws = (size_t)batch * slots * rows * cap * 4;
    // Warps take rows of their own where their tiles fill the GPU well enough: with few, four warps to a tile finish sooner,
    // and the longer the cache the less their join weighs. 7 chunks: 640 tiles 20.0 us, positions split 22.7; 320 tiles 16.9
    // and 13.5. 24 chunks: 640 tiles 61 and 46, 1280 tiles 82 and 76. 223 causal rows on 160 pairs of 150 to 448: 30 and 61
    p.rows = R > 16 && pairs * ((R + rt - 1) / rt) >= 64 * (chunks < 28 ? chunks : 28);
    p.lay.block = (int)(R < rt ? R : rt);
    p.lay.tiles = (int)((R + rt - 1) / rt);
    if (p.rows) {
        p.flat = false, p.smem = 0, p.part = 0;
        p.lay.cs = p.lay.nclus = 1;
        return p;
    }
    // Splits of the sequence: no more CTAs than the GPU holds at once (5 rows on 120 pairs: 2 CTAs a pair 16 us, 4 in more
    // than one wave 23), and a chunk at least to each warp
    const long units = pairs * p.lay.tiles, top = (chunks + WARPS - 1) / WARPS;
    long s = (p.mode == 2 ? PAIRED : SLOTS) / units;  // (16 rows in a cluster: two CTAs to an SM)
    s = s < 1 ? 1 : s > top ? top : s;
    const int cs = s < 2 ? 1 : s < 4 ? 2 : s < 8 ? 4 : 8;
    p.lay.cs = cs;
    p.lay.nclus = (int)(s / cs);
    // Where one cluster is too little the parts join in a second kernel in any case, and equal shares of all chunks are
    // better (15 pairs of 0 to 131072 positions: 32 us, clusters 47). With one cluster a pair they are not: 640 pairs of 1500
    // positions 29 us flat, 28 in clusters, 320 pairs 18.7 and 17.6, 20 pairs 7.5 and 5.5.
    p.flat = R <= 8 && p.lay.nclus > 1 && pairs * chunks < 0x7fffffffl;
    if (p.flat) {
        p.lay = {1, 1, 0, 1, 0};
        p.smem = sizeof(Smem);
        p.part = (size_t)SLOTS * WARPS * 2 * RECF * 4;
        return p;
    }
    const size_t n = (size_t)p.lay.block * cs * WARPS;  // (row, source) pairs
    // 16 rows' exchange beside the ring leaves room for two CTAs to an SM. More CTAs than that exchange inside the ring, behind
    // a barrier more (320 tiles of 7 chunks 13.5 us, beside it 20)
    p.lay.inside = p.mode == 2 && cs == 1 && units > PAIRED;
    p.smem = sizeof(Smem) + (p.lay.inside ? 0 : (n + (n & 1)) * 8 + n * (HD / cs) * 4);
    // Up to two CTAs to an SM: shared memory that no third one fits into, or the first SMs get three and others one (240 CTAs
    // of 12 chunks 13.9 us, without 16.4)
    if (units * cs * p.lay.nclus <= PAIRED) p.smem = p.smem > ALONE3 ? p.smem : ALONE3;
    p.part = p.lay.nclus > 1 ? ((size_t)pairs * R * p.lay.nclus * REC * 4 + 15) & ~(size_t)15 : 0;
    return p;
}

template <int KIND, int MODE>
int launch_main(const Attn8& a, const Plan& p, float* part, float2* stats, float* raws, DevCtx& dc, cudaStream_t st) {
    if constexpr (MODE != 2) {
        if (p.flat)
            return check_pdl(launch_pdl(attn8_flat_kernel<KIND, MODE>, dim3(SLOTS), dim3(NT), p.smem, st, a, part, stats, raws,
                                        dc.status, dc.limit_ns),
                             "attn8");
    } else if (p.rows) {
        return check_pdl(launch_pdl(attn8_rows_kernel<KIND>, dim3((unsigned)((long)a.batch * a.kv_heads * p.lay.tiles)),
                                    dim3(32), 0, st, a, p.lay.tiles, stats, raws, dc.status, dc.limit_ns),
                         "attn8");
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)((long)a.batch * a.kv_heads * p.lay.tiles * p.lay.nclus * p.lay.cs));
    cfg.blockDim = dim3(NT);
    cfg.dynamicSmemBytes = p.smem;
    cfg.stream = st;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = p.lay.cs;
    at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 2;
    return check_pdl(cudaLaunchKernelEx(&cfg, attn8_kernel<KIND, MODE>, a, p.lay, part, stats, raws, dc.status, dc.limit_ns),
                     "attn8");
}

template <int KIND>
int launch_mode(const Attn8& a, const Plan& p, float* part, float2* stats, float* raws, DevCtx& dc, cudaStream_t st) {
    return p.mode == 0   ? launch_main<KIND, 0>(a, p, part, stats, raws, dc, st)
           : p.mode == 1 ? launch_main<KIND, 1>(a, p, part, stats, raws, dc, st)
                         : launch_main<KIND, 2>(a, p, part, stats, raws, dc, st);
}
}  // namespace

size_t attn8_scratch_bytes(int batch, int rows, int q_heads, int kv_heads, int cap, int slots) {
    if (!sizes_ok(batch, rows, q_heads, kv_heads, cap, slots)) return 0;
    const Plan p = plan(batch, rows, q_heads, kv_heads, cap, slots);
    return p.part + p.stats + p.raws;
}

int attn8_launches(int batch, int rows, int q_heads, int kv_heads, int cap, int slots) {
    const Plan p = plan(batch, rows, q_heads, kv_heads, cap, slots);
    return p.flat || p.lay.nclus > 1 || slots ? 2 : 1;
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
    if (!sizes_ok(a.batch, a.rows, a.q_heads, a.kv_heads, a.cap, slots)) return fail("attn8: too many rows in one call");
    const Plan p = plan(a.batch, a.rows, a.q_heads, a.kv_heads, a.cap, slots);
    const long grid = (long)a.batch * a.kv_heads * p.lay.tiles * p.lay.nclus * p.lay.cs;
    // rows with parts: one to a warp, or where a row has more than 32 parts or so one to a block
    const long jall = p.flat || p.lay.nclus > 1 ? (long)a.batch * a.rows * a.q_heads : 0;
    const int jrows = (p.flat ? SLOTS * WARPS / ((long)a.batch * a.kv_heads) : p.lay.nclus) > 32 ? 1 : 8;
    const long jblocks = (jall + jrows - 1) / jrows;
    const long post = jblocks + (long)a.batch * slots * a.rows;
    if (grid > 0x7fffffffl || post > 0x7fffffffl) return fail("attn8: more than 2^31 blocks in one call");
    if (!apart(HD, {{a.batch, a.o_seq}, {a.rows, a.o_row}, {a.q_heads, a.o_head}})) return fail("attn8: rows of out overlap");
    const size_t need = p.part + p.stats + p.raws;
    if (need && (!scratch || ((uintptr_t)scratch & 15) || scratch_bytes < need))
        return fail("attn8: scratch too small or not 16-byte aligned");
    // A block of rows reads all of its q before it writes any of its out, and no q but its own: out may be q itself. Rows
    // of out over other rows of q would be read after they were written
    const bool alike = (a.batch < 2 || a.q_seq == a.o_seq) && (a.rows < 2 || a.q_row == a.o_row) && (a.q_heads < 2 || a.q_head == a.o_head);
    auto span = [&](const __half* p, long seq, long row, long head) {  // first and last value
        std::pair<__int128, __int128> x((intptr_t)p / 2, (intptr_t)p / 2 + HD - 1);
        for (const std::pair<int, long>& d : {std::pair<int, long>(a.batch, seq), {a.rows, row}, {a.q_heads, head}})
            (d.second < 0 ? x.first : x.second) += (__int128)d.second * (d.first - 1);
        return x;
    };
    const auto in = span(a.q, a.q_seq, a.q_row, a.q_head), to = span(a.out, a.o_seq, a.o_row, a.o_head);
    if (in.first <= to.second && to.first <= in.second && !(alike && a.q == a.out) &&
        !(alike && !meet(a.out - a.q, HD, {{a.batch, a.o_seq}, {a.rows, a.o_row}, {a.q_heads, a.o_head}})))
        return fail("attn8: out over q, and not q itself");
    DevCtx& dc = dev_ctx();
    if (!dc.ok) return fail(dc.err);
    float* part = (float*)scratch;
    float2* stats = slots ? (float2*)((char*)scratch + p.part) : nullptr;
    float* raws = slots ? (float*)((char*)scratch + p.part + p.stats) : nullptr;
    const int r = kind == KV8_INT8 ? launch_mode<KV8_INT8>(a, p, part, stats, raws, dc, st)
                                   : launch_mode<KV8_E4M3>(a, p, part, stats, raws, dc, st);
    if (r || !post) return r;
    return check_pdl(launch_pdl(attn8_post_kernel, dim3((unsigned)post), dim3(jrows == 1 ? 512 : 256), 0, st, a,
                                (unsigned)jblocks, jrows, p.lay.nclus, p.flat ? (unsigned)(SLOTS * WARPS) : 0u,
                                (const float*)part, (const float2*)stats, (const float*)raws),
                     "attn8");
}

void init_attn8_attrs() {
    const int most = (int)(sizeof(Smem) + WARPS * 16 * (8 * 8 + HD * 4));  // any layout's shared memory (above ALONE3)
    // every kernel asks for the largest shared memory of an SM: the split from the L1 cache changes only on an idle SM,
    // and a CTA of the main kernel that finds too little beside the last call's blocks starts when the others end
    auto carve = [&](auto* fn) {
        cudaFuncSetAttribute(fn, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
    };
    auto set = [&](auto* fn) {
        cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, most);
        carve(fn);
    };
    carve(attn8_post_kernel);
    carve(attn8_rows_kernel<KV8_INT8>);
    carve(attn8_rows_kernel<KV8_E4M3>);
    set(attn8_kernel<KV8_INT8, 0>);
    set(attn8_kernel<KV8_INT8, 1>);
    set(attn8_kernel<KV8_INT8, 2>);
    set(attn8_kernel<KV8_E4M3, 0>);
    set(attn8_kernel<KV8_E4M3, 1>);
    set(attn8_kernel<KV8_E4M3, 2>);
    set(attn8_flat_kernel<KV8_INT8, 0>);
    set(attn8_flat_kernel<KV8_INT8, 1>);
    set(attn8_flat_kernel<KV8_E4M3, 0>);
    set(attn8_flat_kernel<KV8_E4M3, 1>);
}

}  // namespace mmz
