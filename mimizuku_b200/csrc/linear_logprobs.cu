// Log probabilities from hidden states, for sm_100a: token_logprobs (logprobs.cu) of the logits x . emb^T, without the
// logits in memory. A product on the 5th-generation tensor cores whose epilogue, instead of storing a tile, takes it into
// its rows' running maximum, sums and alternatives; the fp32 sums are used as they are.
//
// D[rows][vocabulary ids], so that a thread of the epilogue has a row: one TMEM lane, 32 ids at a time. Per id it does
// what token_logprobs does (packed fp32, one exponential); where a chunk of 32 has a logit above the row's last
// alternative, or the target, the warp puts the chunk into shared memory and each lane picks its own out. Each CTA (or
// pair) has an equal share of the (row tile, vocabulary) sequence, vocabulary innermost, and leaves one record per row
// tile it worked on; a second kernel joins the records of a row.
//   up to 32 rows    linear_one_kernel<true>: 128 rows (32 loaded, the rest of the product is not looked at) x up to 128
//                    ids, a CTA to an SM, shares in units of 32 ids. One warp can read the 32 rows' TMEM lanes: it
//                    hands the chunks to the four warps of the epilogue through shared memory
//   up to 128        linear_one_kernel<false>: the same, each of the four warps with its 32 rows
//                    Both are bound by reading the embedding once
//   more             linear_pair_kernel: tiles of 256 x 256 on pairs of CTAs (cta_group::2). Bound by the tensor cores
//                    (at a width of 1280 a tile's products take about five times its epilogue)
// Measured, 51866 ids: 32 rows of width 1280 33 us (in the form for 128 rows 35; one row of width 384 17 and 22), 128 rows
// 35 us (in pairs 43), 256 rows 44, 7168 rows 700 us = 1350 TFLOP/s in a burst, 800 = 1190 back to back under the power cap.
// All: a TMA producer and an MMA issuer (one warp each) feed two TMEM accumulators in turn, the epilogue works on one
// while the other fills. Every wait is bounded; a CTA that gives up lets its copies land, waits for its MMAs and frees its
// TMEM.
#include "launch.h"
#include "logprobs.cuh"

namespace mmz {
namespace ll {

constexpr int BK = 64;              // K per stage (one 128-byte swizzle atom)
constexpr int FIELDS = 4 + 2 * TOP_MAX;  // a record: m, s, u, the target's logit, (logit, id) of the alternatives
constexpr int PAIRS = 74;           // pairs of SMs of a B200

// equal contiguous shares of T tiles for W workers, the first T % W have one more
struct Share {
    int T, W, per, more;
    __host__ __device__ Share(int T, int W) : T(T), W(W), per(T / W), more(T % W) {}
    __host__ __device__ int first(int w) const { return w * per + (w < more ? w : more); }
    __host__ __device__ int count(int w) const { return per + (w < more ? 1 : 0); }
    __host__ __device__ int owner(int f) const {
        const int big = more * (per + 1);
        return f < big ? f / (per + 1) : more + (f - big) / per;
    }
};

// One row's running state in a thread of the epilogue.
struct RowState {
    Run run;
    float v[TOP_MAX], tgt, kth;
    int id[TOP_MAX];
    __device__ __forceinline__ void clear(bool live) {  // a row that does not exist takes no alternatives
        run = {LOWEST, make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
        tgt = -INFINITY, kth = live ? -INFINITY : INFINITY;
#pragma unroll
        for (int i = 0; i < TOP_MAX; i++) v[i] = -INFINITY, id[i] = -1;
    }
    // x among the largest, behind equal ones (ids come in order)
    __device__ __forceinline__ void insert(float x, int n, int top) {
#pragma unroll
        for (int i = TOP_MAX - 1; i >= 0; i--) {
            const bool here = x > v[i], up = i > 0 && x > v[i > 0 ? i - 1 : 0];
            v[i] = up ? v[i > 0 ? i - 1 : 0] : here ? x : v[i];
            id[i] = up ? id[i > 0 ? i - 1 : 0] : here ? n : id[i];
        }
        kth = v[0];
#pragma unroll
        for (int i = 1; i < TOP_MAX; i++)
            if (i < top) kth = v[i];
    }
    // 32 logits of ids c0 .. c0 + 31, those with a bit in `out` left out; box: [32 ids][32 lanes] floats of the warp, which
    // hold the logits already where STORED
    template <bool STORED>
    __device__ __forceinline__ void take(float (&x)[1][32], int c0, uint32_t out, int target, int top, float* box, int lane) {
        if (out) {
#pragma unroll
            for (int i = 0; i < 32; i++)
                if (out >> i & 1) x[0][i] = -INFINITY;
        }
        float g[8];  // the largest of each four
#pragma unroll
        for (int i = 0; i < 8; i++) g[i] = fmaxf(fmax3(x[0][4 * i], x[0][4 * i + 1], x[0][4 * i + 2]), x[0][4 * i + 3]);
        const float h = fmaxf(fmax3(fmax3(g[0], g[1], g[2]), g[3], g[4]), fmax3(g[5], g[6], g[7]));
        run.add(x, h);
        const bool mine = target >= c0 && target < c0 + 32, more = top > 0 && h > kth;
        if (!__any_sync(0xffffffff, mine || more)) return;
        // an empty list: only what reaches the top-th largest of the fours' maxima can end up in it
        float least = -INFINITY;
        if (__any_sync(0xffffffff, more && kth == -INFINITY)) {
#pragma unroll
            for (int i = 0; i < 8; i++) {
                int above = 0;
#pragma unroll
                for (int j = 0; j < 8; j++)
                    if (j != i) above += g[j] > g[i] || (j < i && g[j] == g[i]);
                if (above == top - 1 && g[i] == g[i]) least = g[i];
            }
        }
        uint32_t cand = 0;
#pragma unroll
        for (int i = 0; i < 32; i++) {
            if (!STORED) box[i * 32 + lane] = x[0][i];  // read by the same lane only
            if (x[0][i] > kth && x[0][i] >= least) cand |= 1u << i;
        }
        if (mine) tgt = out >> (target - c0) & 1 ? -INFINITY : box[(target - c0) * 32 + lane];
        if (top == 0) return;
        for (; cand; cand &= cand - 1) {
            const int i = __ffs(cand) - 1;
            const float f = box[i * 32 + lane];
            if (f > kth) insert(f, c0 + i, top);
        }
    }
    __device__ __forceinline__ RowStat stat() const {  // nothing above -inf: the empty set
        const float s = run.s.x + run.s.y;
        return {s == 0.f ? -INFINITY : run.m, s, run.u.x + run.u.y};
    }
    __device__ __forceinline__ void store(float* rec, int top) const {
        const RowStat a = stat();
        float4* to = reinterpret_cast<float4*>(rec);
        to[0] = make_float4(a.m, a.s, a.u, tgt);
#pragma unroll
        for (int i = 0; i < TOP_MAX; i += 2)
            if (i < top) to[1 + i / 2] = make_float4(v[i], __int_as_float(id[i]), v[i + 1], __int_as_float(id[i + 1]));
    }
};

// the ids c0 .. c0 + 31 that are left out: suppressed, or past the vocabulary
__device__ __forceinline__ uint32_t left_out(const unsigned char* sup, int c0, int V, int lane) {
    const int id = c0 + lane;
    return __ballot_sync(0xffffffff, id >= V || (sup && sup[id]));
}

namespace one {
constexpr int BM = 128, NTHREADS = 192;   // warps 0-3 epilogue, 4 TMA, 5 MMA
constexpr int UNIT = 32, UB = UNIT * BK * 2;  // ids and bytes (4 KB) of a unit; up to 4 units to a tile
template <bool NARROW>
struct Smem {
    static constexpr int NS = NARROW ? 8 : 6, AT = NARROW ? 32 * BK * 2 : BM * BK * 2;
    uint8_t a[NS][AT];  // NARROW: the product reads 128 rows from a stage's 32 on, what they hold is not looked at
    uint8_t b[NS][4 * UB];
    float box[NARROW ? 2 : 1][4][32 * 32];
    uint64_t full[NS], empty[NS], accf[2], acce[2], fin;
    uint32_t tmem;
    int abort;
};
}  // namespace one

namespace pair {
constexpr int BMC = 128, BN = 256, NS = 5, EPW = 8, NTHREADS = 64 + 32 * EPW;  // warp 0 TMA, 1 MMA, 2-9 epilogue
constexpr int AT = BMC * BK * 2, BT = BN / 2 * BK * 2;                         // 16 KB each, in each CTA
constexpr uint32_t IDESC = idesc_f16_f32(2 * BMC, BN, false);
struct Smem {
    uint8_t a[NS][AT], b[NS][BT];
    float box[EPW][32 * 32];
    uint64_t full[NS], empty[NS], accf[2], acce[2], fin;
    uint32_t tmem;
    int abort;
};
}  // namespace pair
}  // namespace ll
using namespace ll;

// grid min(SMs, units of 32 ids), block NTHREADS, dynamic shared memory sizeof(Smem) + 1024 (alignment slack). xbox: rows
// that a load of x brings (a multiple of 8); emap: a box of 32 ids. rec [CTAs][128][FIELDS], NARROW
// [CTAs][4 warps][32][FIELDS]
template <bool NARROW>
__global__ void __launch_bounds__(one::NTHREADS, 1)
    linear_one_kernel(const __grid_constant__ CUtensorMap xmap, const __grid_constant__ CUtensorMap emap, int rows, int V,
                      int d, int xbox, const unsigned char* sup, LogpOut o, float* rec, unsigned* status,
                      unsigned long long limit_ns) {
    using namespace one;
    using SM = Smem<NARROW>;
    constexpr int NS = SM::NS;
    extern __shared__ uint8_t smem_raw[];
    SM& s = *reinterpret_cast<SM*>(smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023));
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, cta = blockIdx.x;
    const Share share((V + UNIT - 1) / UNIT, gridDim.x);
    const int u0 = share.first(cta), units = share.count(cta), my = (units + 3) / 4, nch = d / BK;
    volatile int* abort = &s.abort;
    if (warp == 4 && lane == 0) {
        s.abort = 0;
        for (int i = 0; i < NS; i++) {
            mbar_init(&s.full[i], 1);
            mbar_init(&s.empty[i], 1);
        }
        for (int a = 0; a < 2; a++) {
            mbar_init(&s.accf[a], 1);
            mbar_init(&s.acce[a], NARROW ? 1 : 4);
        }
        mbar_init(&s.fin, 1);
        fence_mbar_init();
        prefetch_tmap(&xmap);
        prefetch_tmap(&emap);
    }
    if (warp == 5) {
        tmem_alloc(&s.tmem, 256);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    griddep_wait();
    griddep_launch_dependents();
    const uint32_t tb = s.tmem;
    if (warp == 4) {
        // ---------------------------------------------------------------- producer
        if (lane == 0) {
            int issued = 0, st = 0, ph = 0;  // ring slot and its use count
            bool ok = true;
            for (int i = 0; ok && i < my; i++) {
                const int n = min(4, units - 4 * i), id0 = (u0 + 4 * i) * UNIT;
                for (int kc = 0; kc < nch; kc++) {
                    if (issued >= NS && !mbar_wait_spin(&s.empty[st], (ph - 1) & 1, abort, limit_ns, status, K_LOGP, 3)) {
                        ok = false;
                        break;
                    }
                    mbar_expect_tx(&s.full[st], n * UB + xbox * BK * 2);
                    for (int u = 0; u < n; u++) tma_load_2d(s.b[st] + u * UB, &emap, kc * BK, id0 + u * UNIT, &s.full[st]);
                    tma_load_2d(s.a[st], &xmap, kc * BK, 0, &s.full[st]);
                    issued++;
                    if (++st == NS) st = 0, ph++;
                }
            }
            // the last copies land before the shared memory is released, whoever's wait gave up (else the issuer waits for
            // them too)
            for (int q = issued > NS ? issued - NS : 0; q < issued; q++)
                mbar_wait(&s.full[q % NS], (q / NS) & 1, nullptr, limit_ns, nullptr, 0, 0);
        }
    } else if (warp == 5) {
        // ---------------------------------------------------------------- MMA issuer
        if (lane == 0) {
            const uint64_t ad0 = sdesc_sw128(smem_u32(s.a[0]), 16, 1024), bd0 = sdesc_sw128(smem_u32(s.b[0]), 16, 1024);
            constexpr uint64_t ASTAGE = SM::AT >> 4, BSTAGE = 4 * UB >> 4, KSTEP = 32 >> 4;
            bool ok = true;
            int st = 0, ph = 0;
            for (int i = 0; ok && i < my; i++) {
                const int a = i & 1;
                const uint32_t idesc = idesc_f16_f32(BM, UNIT * min(4, units - 4 * i), false);
                if (i >= 2 && !mbar_wait_spin(&s.acce[a], ((i >> 1) - 1) & 1, abort, limit_ns, status, K_LOGP, 4)) break;
                tc_fence_after();
                for (int kc = 0; kc < nch; kc++) {
                    if (!mbar_wait_spin(&s.full[st], ph & 1, abort, limit_ns, status, K_LOGP, 5)) {
                        ok = false;
                        break;
                    }
                    tc_fence_after();
#pragma unroll
                    for (int kk = 0; kk < BK / 16; kk++)
                        umma_f16_ss(tb + a * 128, ad0 + st * ASTAGE + kk * KSTEP, bd0 + st * BSTAGE + kk * KSTEP, idesc,
                                    (kc > 0 || kk > 0) ? 1u : 0u);
                    umma_commit(&s.empty[st]);
                    if (++st == NS) st = 0, ph++;
                }
                if (ok) umma_commit(&s.accf[a]);
            }
            umma_commit(&s.fin);  // completes once every MMA issued above has finished
        }
    } else {
        // ---------------------------------------------------------------- epilogue: thread = row
        const int row = NARROW ? lane : warp * 32 + lane, col = (int)row_at(o, 0);
        const bool live = (NARROW || warp * 32 < rows) && col >= 0;
        const int target = live && row < rows && o.target ? o.target[row_at(o, row)] : -1;
        const uint32_t tl = tb + ((uint32_t)(NARROW ? 0 : warp * 32) << 16);
        RowState r;
        r.clear(row < rows);
        for (int i = 0; i < my; i++) {
            const int a = i & 1, n = min(4, units - 4 * i), id0 = (u0 + 4 * i) * UNIT;
            if (NARROW) {
                // warp 0 hands the tile's chunks round, one to a warp; every warp reaches the barrier of every tile
                float(*box)[32 * 32] = s.box[a];
                if (warp == 0) {
                    const bool ok = __all_sync(
                        0xffffffff, mbar_wait_spin(&s.accf[a], (i >> 1) & 1, abort, limit_ns, status, K_LOGP, 6));
                    if (ok) {
                        tc_fence_after();
                        uint32_t acc[128];  // (columns past the tile's ids hold an earlier tile's and go nowhere)
                        tmem_ld128(tl + a * 128, acc);
#pragma unroll
                        for (int u = 0; u < 4; u++)
                            if (u < n)
#pragma unroll
                                for (int k = 0; k < 32; k++) box[u][k * 32 + lane] = __uint_as_float(acc[32 * u + k]);
                        tc_fence_before();
                    }
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&s.acce[a]);
                }
                asm volatile("bar.sync 1, 128;" ::: "memory");  // the boxes of two tiles: written again after the next one's
                if (live && warp < n) {
                    const uint32_t out = left_out(sup, id0 + UNIT * warp, V, lane);
                    float x[1][32];
#pragma unroll
                    for (int k = 0; k < 32; k++) x[0][k] = box[warp][k * 32 + lane];
                    if (out != 0xffffffffu) r.take<true>(x, id0 + UNIT * warp, out, target, o.top, box[warp], lane);
                }
            } else {
                const bool ok =
                    __all_sync(0xffffffff, mbar_wait_spin(&s.accf[a], (i >> 1) & 1, abort, limit_ns, status, K_LOGP, 6));
                if (ok && live) {
                    tc_fence_after();
#pragma unroll 1
                    for (int u = 0; u < n; u++) {
                        const uint32_t out = left_out(sup, id0 + UNIT * u, V, lane);
                        uint32_t acc[32];
                        __syncwarp();
                        tmem_ld32(tl + a * 128 + 32 * u, acc);
                        float x[1][32];
#pragma unroll
                        for (int k = 0; k < 32; k++) x[0][k] = __uint_as_float(acc[k]);
                        if (out != 0xffffffffu) r.take<false>(x, id0 + UNIT * u, out, target, o.top, s.box[0][warp], lane);
                    }
                    tc_fence_before();
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(&s.acce[a]);
            }
        }
        if (live && row < rows) r.store(rec + (NARROW ? ((long)cta * 4 + warp) * 32 + row : (long)cta * BM + row) * FIELDS, o.top);
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 5) {  // the MMA pipe must drain before the TMEM is released
        mbar_wait(&s.fin, 0, nullptr, limit_ns, status, K_LOGP, 7);
        __syncwarp();
        tc_fence_after();
        tmem_dealloc(tb, 256);
    }
}

// grid 2 x pairs, cluster (2, 1, 1), block NTHREADS, dynamic shared memory sizeof(Smem) + 1024. emap: a box of 128 ids
// (half of a tile's). rec [row tiles][parts][2 halves of a tile's ids][256][FIELDS]
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(pair::NTHREADS, 1)
    linear_pair_kernel(const __grid_constant__ CUtensorMap xmap, const __grid_constant__ CUtensorMap emap, int rows, int V,
                       int d, int parts, const unsigned char* sup, LogpOut o, float* rec, unsigned* status,
                       unsigned long long limit_ns) {
    using namespace pair;
    extern __shared__ uint8_t smem_raw[];
    Smem& s = *reinterpret_cast<Smem*>(smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023));
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = cluster_rank();  // 0: the CTA that issues the MMAs
    const bool lead = rank == 0;
    const int pid = blockIdx.x / 2, nt = (V + BN - 1) / BN, mt = (rows + 2 * BMC - 1) / (2 * BMC);
    const Share share(mt * nt, gridDim.x / 2);
    const int t0 = share.first(pid), my = share.count(pid), nch = d / BK;
    volatile int* abort = &s.abort;
    if (warp == 0 && lane == 0) {
        s.abort = 0;
        for (int i = 0; i < NS; i++) {
            mbar_init(&s.full[i], 1);  // the even CTA's producer (expected bytes of both CTAs)
            mbar_init(&s.empty[i], 1);
        }
        for (int a = 0; a < 2; a++) {
            mbar_init(&s.accf[a], 1);
            mbar_init(&s.acce[a], 2 * EPW);  // both CTAs' epilogue warps (used in the even CTA)
        }
        mbar_init(&s.fin, 1);
        fence_mbar_init();
        prefetch_tmap(&xmap);
        prefetch_tmap(&emap);
    }
    if (warp == 1) {
        tmem_alloc_pair(&s.tmem, 2 * BN);
        tmem_relinquish_pair();
    }
    tc_fence_before();
    cluster_sync();  // both CTAs' barriers initialised and TMEM allocated before either touches the other's
    tc_fence_after();
    griddep_wait();
    griddep_launch_dependents();
    const uint32_t tb = s.tmem;
    if (warp == 0) {
        // ---------------------------------------------------------------- producer (each CTA, its own halves)
        if (lane == 0) {
            const uint32_t full0 = dsmem_addr(&s.full[0], 0);
            int issued = 0, st = 0, ph = 0;  // ring slot and its use count
            for (int i = 0; i < my; i++) {
                const int arow = (t0 + i) / nt * 2 * BMC + (int)rank * BMC, brow = (t0 + i) % nt * BN + (int)rank * (BN / 2);
                bool ok = true;
                for (int kc = 0; kc < nch; kc++) {
                    if (issued >= NS && !mbar_wait_spin(&s.empty[st], (ph - 1) & 1, abort, limit_ns, status, K_LOGP, 8)) {
                        ok = false;
                        break;
                    }
                    if (lead) mbar_expect_tx(&s.full[st], 2 * (AT + BT));
                    tma_load_2d_pair(s.b[st], &emap, kc * BK, brow, full0 + 8 * st);
                    tma_load_2d_pair(s.a[st], &xmap, kc * BK, arow, full0 + 8 * st);
                    issued++;
                    if (++st == NS) st = 0, ph++;
                }
                if (!ok) break;
            }
            // the last copies land before shared memory is released, whoever's wait gave up: both CTAs' are counted on the
            // even CTA's barriers, and the pair leaves together
            if (lead)
                for (int q = issued > NS ? issued - NS : 0; q < issued; q++)
                    mbar_wait(&s.full[q % NS], (q / NS) & 1, nullptr, limit_ns, nullptr, 0, 0);
        }
    } else if (warp == 1) {
        // ---------------------------------------------------------------- MMA issuer (even CTA)
        if (lead && lane == 0) {
            const uint64_t ad0 = sdesc_sw128(smem_u32(s.a[0]), 16, 1024), bd0 = sdesc_sw128(smem_u32(s.b[0]), 16, 1024);
            constexpr uint64_t ASTAGE = AT >> 4, BSTAGE = BT >> 4, KSTEP = 32 >> 4;
            const uint32_t empty0[2] = {dsmem_addr(&s.empty[0], 0), dsmem_addr(&s.empty[0], 1)};
            const uint32_t accf0[2] = {dsmem_addr(&s.accf[0], 0), dsmem_addr(&s.accf[0], 1)};
            bool ok = true;
            int st = 0, ph = 0;
            for (int i = 0; ok && i < my; i++) {
                const int a = i & 1;
                if (i >= 2 && !mbar_wait_cluster(&s.acce[a], ((i >> 1) - 1) & 1, abort, limit_ns, status, K_LOGP, 9)) break;
                tc_fence_after();
                for (int kc = 0; kc < nch; kc++) {
                    if (!mbar_wait_spin(&s.full[st], ph & 1, abort, limit_ns, status, K_LOGP, 10)) {
                        ok = false;
                        break;
                    }
                    tc_fence_after();
                    const uint64_t ad = ad0 + st * ASTAGE, bd = bd0 + st * BSTAGE;
#pragma unroll
                    for (int kk = 0; kk < BK / 16; kk++)
                        umma_f16_ss_pair(tb + a * BN, ad + kk * KSTEP, bd + kk * KSTEP, IDESC, (kc > 0 || kk > 0) ? 1u : 0u);
                    umma_commit_pair(empty0[0] + 8 * st);
                    umma_commit_pair(empty0[1] + 8 * st);
                    if (++st == NS) st = 0, ph++;
                }
                if (ok) {
                    umma_commit_pair(accf0[0] + 8 * a);
                    umma_commit_pair(accf0[1] + 8 * a);
                }
            }
            umma_commit_pair(dsmem_addr(&s.fin, 0));  // both CTAs: every MMA issued above has finished
            umma_commit_pair(dsmem_addr(&s.fin, 1));
        }
    } else {
        // ---------------------------------------------------------------- epilogue: thread = row, half of a tile's ids
        const int qd = warp & 3, half = (warp - 2) >> 2;  // the TMEM lane quarter this warp may read
        const int col = (int)row_at(o, 0), lrow = (int)rank * BMC + qd * 32 + lane;  // row of the tile
        const uint32_t tl = tb + ((uint32_t)(qd * 32) << 16) + half * (BN / 2);
        const uint32_t acce0 = dsmem_addr(&s.acce[0], 0);
        RowState r;
        r.clear(false);
        int m = -1, target = -1;  // row tile
        auto finish = [&]() {
            if (m < 0 || m * 2 * BMC + lrow >= rows || col < 0) return;
            const int k = pid - share.owner(m * nt);  // this pair's part of the row tile
            r.store(rec + ((((long)m * parts + k) * 2 + half) * 2 * BMC + lrow) * FIELDS, o.top);
        };
        for (int i = 0; i < my; i++) {
            const int a = i & 1, n0 = (t0 + i) % nt * BN + half * (BN / 2);
            if ((t0 + i) / nt != m) {
                finish();
                m = (t0 + i) / nt;
                const int row = m * 2 * BMC + lrow;
                r.clear(row < rows);
                target = row < rows && o.target && col >= 0 ? o.target[row_at(o, row)] : -1;
            }
            const bool ok =
                __all_sync(0xffffffff, mbar_wait_spin(&s.accf[a], (i >> 1) & 1, abort, limit_ns, status, K_LOGP, 11));
            if (ok && m * 2 * BMC + (int)rank * BMC + qd * 32 < rows) {
                tc_fence_after();
#pragma unroll 1
                for (int c = 0; c < BN / 64; c++) {
                    const uint32_t out = left_out(sup, n0 + 32 * c, V, lane);
                    uint32_t acc[32];
                    __syncwarp();
                    tmem_ld32(tl + a * BN + 32 * c, acc);
                    float x[1][32];
#pragma unroll
                    for (int k = 0; k < 32; k++) x[0][k] = __uint_as_float(acc[k]);
                    if (out != 0xffffffffu) r.take<false>(x, n0 + 32 * c, out, target, o.top, s.box[warp - 2], lane);
                }
                tc_fence_before();
            }
            __syncwarp();
            if (lane == 0) {
                if (lead) mbar_arrive(&s.acce[a]);
                else mbar_arrive_remote(acce0 + 8 * a);
            }
        }
        finish();
    }
    // teardown: every MMA into either CTA's TMEM has finished before the pair releases it, and neither CTA leaves while
    // the other may still signal its barriers
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        mbar_wait(&s.fin, 0, nullptr, limit_ns, status, K_LOGP, 12);
        __syncwarp();
    }
    tc_fence_before();
    cluster_sync();
    tc_fence_after();
    if (warp == 1) tmem_dealloc_pair(tb, 2 * BN);
}

// A block to a row, its records joined (a record to a thread) and the outputs written. `tr` rows to a tile, `bn` ids to a
// unit of work, `halves` records to a worker and row tile: of the halves of each unit (pairs), or of every fourth unit
// from the worker's first on (quarters 1)
__global__ void __launch_bounds__(1024) linear_join_kernel(const float* rec, int rows, int V, int tr, int bn, int halves,
                                                           int quarters, int workers, int parts, LogpOut o) {
    __shared__ RowStat st[32];
    __shared__ unsigned long long tops[32][TOP_MAX];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, nw = blockDim.x >> 5;
    // rows of few records go to the warps of a block of 128, one each
    const bool small = parts * halves <= 32;
    const int row = small ? blockIdx.x * 4 + warp : blockIdx.x, first = small ? lane : threadIdx.x;
    const int mt = (rows + tr - 1) / tr, nt = (V + bn - 1) / bn, m = row / tr;
    const Share share(mt * nt, workers);
    const int w0 = share.owner(m * nt), n = row < rows ? (share.owner((m + 1) * nt - 1) - w0 + 1) * halves : 0;
    const float* base = rec + ((long)m * parts * halves * tr + row % tr) * FIELDS;
    griddep_wait();
    griddep_launch_dependents();
    const long at = row_at(o, row);
    if (at < 0 || row >= rows) return;  // the whole block, or the whole warp of a small one
    int t = -1;
    if (first == 0 && o.target) t = o.target[at];
    RowStat a = stat_none();
    unsigned long long key[TOP_MAX] = {};
    if (first < n) {
        const float4* f = reinterpret_cast<const float4*>(base + (long)first * tr * FIELDS);
        const float4 y = f[0];
        float4 z[TOP_MAX / 2];
#pragma unroll
        for (int i = 0; i < TOP_MAX / 2; i++)
            if (2 * i < o.top) z[i] = f[1 + i];
        a = {y.x, y.y, y.z};
#pragma unroll
        for (int i = 0; i < TOP_MAX; i++)
            if (i < o.top) {
                const float4 q = z[i / 2];
                key[i] = i & 1 ? top_key(q.z, __float_as_int(q.w)) : top_key(q.x, __float_as_int(q.y));
            }
    }
    const bool has = t >= 0 && t < V;  // (only the first thread looks)
    float tgt = 0.f;
    if (has) {
        const int unit = m * nt + t / bn, w = share.owner(unit);
        const int k = (w - w0) * halves + (quarters ? (unit - share.first(w)) & 3 : t % bn / (bn / halves));
        tgt = base[(long)k * tr * FIELDS + 3];
    }
    // the lanes' lists, each in order, popped in turn: the i-th largest ends up with lane i
    auto pop = [&]() {
        unsigned long long mine = 0;
        for (int i = 0; i < o.top; i++) {
            const unsigned hi = __reduce_max_sync(0xffffffff, (unsigned)(key[0] >> 32));
            const unsigned lo = __reduce_max_sync(0xffffffff, (unsigned)(key[0] >> 32) == hi ? (unsigned)key[0] : 0u);
            const unsigned long long x = (unsigned long long)hi << 32 | lo;
            if (lane == i) mine = x;
            if (key[0] == x && x) {
#pragma unroll
                for (int j = 0; j + 1 < TOP_MAX; j++) key[j] = key[j + 1];
                key[TOP_MAX - 1] = 0ull;
            }
        }
        return mine;
    };
    unsigned long long mine = pop();
    a = stat_warp(a);
    if (!small) {
        if (lane == 0) st[warp] = a;
        if (lane < TOP_MAX) tops[warp][lane] = lane < o.top ? mine : 0ull;
        __syncthreads();
        if (warp) return;
        a = lane < nw ? st[lane] : stat_none();
#pragma unroll
        for (int i = 0; i < TOP_MAX; i++) key[i] = lane < nw ? tops[lane][i] : 0ull;
        mine = pop();
        a = stat_warp(a);
    }
    float ls = 0.f;
    if (lane == 0) ls = store_row(o, at, a, has, tgt);
    ls = __shfl_sync(0xffffffff, ls, 0);
    if (lane < o.top) store_top(o, at, lane, mine, a.m, ls);
}

// the layout of a call, from its sizes
namespace {
struct Plan {
    bool pairs;
    int tr, bn, halves, quarters, workers, parts;  // as linear_join_kernel has them
    size_t bytes;
};
Plan plan(int rows, int V) {
    Plan p;
    p.pairs = rows > 128;
    p.quarters = rows <= 32;
    p.tr = p.pairs ? 256 : p.quarters ? 32 : 128;
    p.bn = p.pairs ? pair::BN : one::UNIT;
    p.halves = p.pairs ? 2 : p.quarters ? 4 : 1;
    const long mt = ((long)rows + p.tr - 1) / p.tr, nt = ((long)V + p.bn - 1) / p.bn, most = p.pairs ? PAIRS : 2 * PAIRS;
    const long T = mt * nt;
    p.workers = (int)(T < most ? T : most);
    const long per = T / p.workers;
    p.parts = (int)((nt + per - 1) / per) + 1;  // workers that a row tile's vocabulary can lie on
    if (p.parts > p.workers) p.parts = p.workers;
    p.bytes = (size_t)mt * p.parts * p.halves * FIELDS * p.tr * 4;
    return p;
}
}  // namespace

size_t linear_logprobs_scratch_bytes(int rows, int V, int) { return plan(rows, V).bytes; }

int launch_linear_logprobs(const void* x, long long ldx, const void* emb, int rows, int V, int d,
                           const unsigned char* sup, const LogpOut& o, void* scratch, size_t scratch_bytes,
                           cudaStream_t st) {
    if (rows < 0 || V < 1 || d < 64 || d % 64) return fail("linear_logprobs: rows >= 0, vocab >= 1, width a multiple of 64");
    if (V > 0x7ffffc00 || rows > 0x7ffffc00) return fail("linear_logprobs: vocab and rows up to 2^31 - 1024");
    if (logp_check("linear_logprobs", o)) return -1;
    if (rows == 0) return 0;
    if (!x || !emb || (((uintptr_t)x | (uintptr_t)emb) & 15) || (ldx & 7) || ldx < d)
        return fail("linear_logprobs: x and emb 16-byte aligned, ldx >= width with a 16-byte row pitch");
    const long tiles = ((long)rows + 127) / 128 * (((long)V + 127) / 128);
    if (tiles > 0x7fffffffl) return fail("linear_logprobs: more than 2^31 tiles in one call");
    const Plan p = plan(rows, V);
    if (!scratch || ((uintptr_t)scratch & 15) || scratch_bytes < p.bytes)
        return fail("linear_logprobs: scratch too small or not 16-byte aligned");
    DevCtx& dc = dev_ctx();
    if (!dc.ok) return fail(dc.err);
    CUtensorMap xm, em;
    const int xbox = p.pairs ? 128 : rows <= 32 ? 32 : (rows + 7) / 8 * 8;
    const uint64_t xd[2] = {(uint64_t)d, (uint64_t)rows}, xs[1] = {(uint64_t)ldx * 2};
    const uint32_t xb[2] = {BK, (uint32_t)xbox};
    const uint64_t ed[2] = {(uint64_t)d, (uint64_t)V}, es[1] = {(uint64_t)d * 2};
    const uint32_t eb[2] = {BK, p.pairs ? 128u : (uint32_t)one::UNIT};
    if (make_tmap_2d(&xm, x, xd, xs, xb, 128) || make_tmap_2d(&em, emb, ed, es, eb, 128))
        return fail("linear_logprobs: cuTensorMapEncodeTiled failed");
    float* rec = (float*)scratch;
    int e;
    if (p.pairs)
        e = check_pdl(launch_pdl(linear_pair_kernel, dim3(2 * p.workers), dim3(pair::NTHREADS), sizeof(pair::Smem) + 1024, st,
                                 xm, em, rows, V, d, p.parts, sup, o, rec, dc.status, dc.limit_ns),
                      "linear_logprobs");
    else if (rows <= 32)
        e = check_pdl(launch_pdl(linear_one_kernel<true>, dim3(p.workers), dim3(one::NTHREADS),
                                 sizeof(one::Smem<true>) + 1024, st, xm, em, rows, V, d, xbox, sup, o, rec, dc.status,
                                 dc.limit_ns),
                      "linear_logprobs");
    else
        e = check_pdl(launch_pdl(linear_one_kernel<false>, dim3(p.workers), dim3(one::NTHREADS),
                                 sizeof(one::Smem<false>) + 1024, st, xm, em, rows, V, d, xbox, sup, o, rec, dc.status,
                                 dc.limit_ns),
                      "linear_logprobs");
    if (e) return e;
    const int n = p.parts * p.halves;  // at most 4 x 148
    return check_pdl(launch_pdl(linear_join_kernel, dim3(n <= 32 ? (rows + 3) / 4 : rows), dim3(n <= 32 ? 128 : (n + 31) & ~31),
                                0, st, (const float*)rec, rows, V, p.tr, p.bn, p.halves, p.quarters, p.workers, p.parts, o),
                     "linear_logprobs");
}

void init_linear_logprobs_attrs() {
    auto set = [](auto* fn, size_t bytes) {
        cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes + 1024);
    };
    set(linear_one_kernel<true>, sizeof(one::Smem<true>));
    set(linear_one_kernel<false>, sizeof(one::Smem<false>));
    set(linear_pair_kernel, sizeof(pair::Smem));
}

}  // namespace mmz
