// k_gmm.cu -- dense and grouped products of e4m3 rows with block scales, and of bf16 / f16 rows, on the 5th-generation
// tensor cores (tcgen05.mma kind::f8f6f4 / kind::f16), sm_100a (inzg_matmul_q8, inzg_grouped_matmul).
//
//   out[i][j] = scale_i * sum_b as[i][b] ws[j / 128][b] * (sum_{k in block b} a[i][k] w[g][j][k])
//
// The tensor core sums one block of 128 k in fp32 (TMEM); the block's two scales enter in the fold, which keeps the running
// sum in fp32 registers: f = fma(dot_b, as * ws, f). bf16 / f16 have no scales and stay in TMEM over the whole k.
//
// Work item: 128 rows of w (the MMA's M, one TMEM lane each) x up to 128 entries of one group (its N, rounded up to
// 16). The weights are the M side because a decoding call has a row or two per expert: the MMA, the copies and the
// fold then shrink with the entries, while a weight tile is streamed once whatever their number. A tile of 128 rows
// of w has one weight scale per k block, so as * ws is formed once per entry and block and kept in shared memory.
//   warp 0      TMA producer: per 128-byte step of k a box of 128 weight rows and the entries' rows, in boxes of 16 or 128
//               rows, or four at a time by index (tile::gather4), 128-byte swizzle, into a 6-stage ring
//   warp 1      allocates all 512 TMEM columns (four 128-column accumulators), one lane issues 4 MMAs per stage
//   warps 2-9   fold and write: thread = (row of w, every other 32 entries)
// Persistent: one CTA per SM walks the items; the offsets are turned into tile numbers by every CTA for itself, which
// costs a read of off and a scan instead of a launch. Every mbarrier wait is bounded; on expiry the CTA records an
// error, drains what it issued, frees its TMEM and returns.
#include <cuda.h>
#include <cudaTypedefs.h>

#include <algorithm>

#include "inzg_internal.h"
#include "k_async.cuh"
#include "k_launch.h"
#include "k_q8.cuh"

namespace inzg {

constexpr int GM = 128, GT = 128, GB = 128, GSTAGES = 6;  // weight rows, entries, bytes of k per stage
constexpr int kGmmEpiWarps = 8, kGmmEpi = kGmmEpiWarps * 32, kGmmThreads = 64 + kGmmEpi;
constexpr int kGmmStage = (GM + GT) * GB;
constexpr int kGmmKc = 8;  // k blocks whose scales are staged at once

struct GmmArgs {
    int groups, n, nrb, steps, entries, a_rows, out_rows_n, out_type;
    const int32_t *off, *in_rows, *out_rows;  // off null: one group of all entries
    const float *out_scale, *as, *ws;
    int64_t ldas, ldo;
    void *out;
    uint32_t idesc;  // without N
    int32_t *err;
};

struct GmmShared {
    uint64_t full[GSTAGES], empty[GSTAGES], acc_full[4], acc_empty[4], drain;
    uint32_t tmem_base;
    int abort, never, bad;
    int wsum[kGmmThreads / 32];
    alignas(16) float p[2][kGmmKc][GT];  // as * ws of the staged blocks
    int orow[2][GT];                     // row of out of each entry (-1: not written), per item parity
    float ow[2][GT];
    int tstart[INZG_MAX_GROUPS + 1];     // first tile of each group
    int off[INZG_MAX_GROUPS + 1];
};

__device__ __forceinline__ uint64_t gmm_desc(const void *smem) {  // K-major, 128-byte swizzle, 8-row atoms of 1024 bytes
    const uint64_t a = smem_u32(smem);
    return ((a & 0x3FFFFull) >> 4) | (1ull << 16) | (64ull << 32) | (1ull << 46) | (2ull << 61);
}

template <bool F8>
__device__ __forceinline__ void gmm_mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    if (F8)
        asm volatile(
            "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, {%5, %5, %5, %5}, p;\n\t}" ::"r"(d),
            "l"(a), "l"(b), "r"(idesc), "r"(acc), "r"(0));
    else
        asm volatile(
            "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, {%5, %5, %5, %5}, p;\n\t}" ::"r"(d),
            "l"(a), "l"(b), "r"(idesc), "r"(acc), "r"(0));
}

__device__ __forceinline__ void gmm_commit(uint64_t *bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar))
                 : "memory");
}

__device__ __forceinline__ void gmm_ld32(uint32_t taddr, float (&v)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]), "=f"(v[8]),
          "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15]), "=f"(v[16]),
          "=f"(v[17]), "=f"(v[18]), "=f"(v[19]), "=f"(v[20]), "=f"(v[21]), "=f"(v[22]), "=f"(v[23]), "=f"(v[24]),
          "=f"(v[25]), "=f"(v[26]), "=f"(v[27]), "=f"(v[28]), "=f"(v[29]), "=f"(v[30]), "=f"(v[31])
        : "r"(taddr));
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}

// four rows of the map (box one row high) by index, 512 bytes
__device__ __forceinline__ void tma_gather4(void *dst, const CUtensorMap *map, int x, int r0, int r1, int r2, int r3,
                                            uint64_t *bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.tile::gather4.mbarrier::complete_tx::bytes "
        "[%0], [%1, {%2, %3, %4, %5, %6}], [%7];" ::"r"(smem_u32(dst)),
        "l"(map), "r"(x), "r"(r0), "r"(r1), "r"(r2), "r"(r3), "r"(smem_u32(bar))
        : "memory");
}

__device__ __forceinline__ void store_out(void *out, int type, int64_t at, float v) {
    if (type == INZG_T_F32) static_cast<float *>(out)[at] = v;
    else if (type == INZG_T_BF16) static_cast<__nv_bfloat16 *>(out)[at] = __float2bfloat16_rn(v);
    else static_cast<__half *>(out)[at] = __float2half_rn(v);
}

// an item of the walk: entries [base, base + nt) of group g against rows [rb * 128, rb * 128 + 128) of its weights
struct GmmItem {
    int g, base, nt, rb;
};

__device__ __forceinline__ GmmItem gmm_item(const GmmShared &S, int groups, int nrb, int item) {
    const int tile = item / nrb;
    int lo = 0, hi = groups;  // the last group whose first tile is not past `tile`; empty groups share a first tile
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (S.tstart[mid] <= tile) lo = mid;
        else hi = mid;
    }
    GmmItem I;
    I.g = lo;
    I.base = S.off[lo] + (tile - S.tstart[lo]) * GT;
    I.nt = min(GT, S.off[lo + 1] - I.base);
    I.rb = item - tile * nrb;
    return I;
}

// map_w: [groups * n][k] in 128-row boxes; map_a16 / map_a128: the rows of a in boxes of 16 / 128 rows; map_a1: of one row
template <bool F8>
__global__ void __launch_bounds__(kGmmThreads, 1)
gmm_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_a,
           const __grid_constant__ CUtensorMap map_a128, const __grid_constant__ GmmArgs A) {
    extern __shared__ __align__(1024) uint8_t gmm_dyn[];
    uint8_t *ring = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(gmm_dyn) + 1023) & ~uintptr_t(1023));
    GmmShared &S = *reinterpret_cast<GmmShared *>(ring + GSTAGES * kGmmStage);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    volatile int *abort = &S.abort;
    volatile int *never = &S.never;
    constexpr int kElem = F8 ? 1 : 2;

    if (threadIdx.x == 0) {
        for (int s = 0; s < GSTAGES; s++) {
            mbar_init(&S.full[s], 1);
            mbar_init(&S.empty[s], 1);
        }
        for (int b = 0; b < 4; b++) {
            mbar_init(&S.acc_full[b], 1);
            mbar_init(&S.acc_empty[b], kGmmEpiWarps);
        }
        mbar_init(&S.drain, 1);
        S.abort = 0;
        S.never = 0;
        S.bad = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&S.tmem_base)));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = S.tmem_base;

    // tile numbers: a thread counts the tiles of `per` neighbouring groups, then a scan over the block
    const int per = (A.groups + kGmmThreads - 1) / kGmmThreads, g0 = threadIdx.x * per;
    int mine = 0;
    for (int g = g0; g < min(g0 + per, A.groups); g++) {
        const int o0 = A.off ? A.off[g] : 0, o1 = A.off ? A.off[g + 1] : A.entries;
        if (o0 < 0 || o1 < o0 || o1 > A.entries) S.bad = 1;
        else mine += (o1 - o0 + GT - 1) / GT;
        S.off[g] = o0;
        if (g == A.groups - 1) S.off[g + 1] = o1;
    }
    int scan = mine;
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
        const int v = __shfl_up_sync(0xffffffffu, scan, d);
        if (lane >= d) scan += v;
    }
    if (lane == 31) S.wsum[warp] = scan;
    __syncthreads();
    int first = scan - mine;
    for (int k = 0; k < warp; k++) first += S.wsum[k];
    if (!S.bad)
        for (int g = g0; g < min(g0 + per, A.groups); g++) {
            S.tstart[g] = first;
            first += (S.off[g + 1 <= A.groups ? g + 1 : g] - S.off[g] + GT - 1) / GT;
            if (g == A.groups - 1) S.tstart[g + 1] = first;
        }
    __syncthreads();
    const int nitems = S.bad ? 0 : S.tstart[A.groups] * A.nrb;
    if (S.bad && threadIdx.x == 0) atomicCAS(A.err, kErrNone, kErrOverflow);
    const int steps = A.steps;

    if (warp == 0) {
        // ---------------- TMA producer ----------------
        int kg = 0;  // stages issued by this CTA
        bool ok = true;
        for (int item = blockIdx.x; item < nitems && ok; item += gridDim.x) {
            const GmmItem I = gmm_item(S, A.groups, A.nrb, item);
            const int nt16 = (I.nt + 15) & ~15;
            const bool whole = !A.in_rows && I.nt > 64;
            int r[4] = {0, 0, 0, 0};
            if (A.in_rows)
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const int v = A.in_rows[I.base + min(lane * 4 + j, I.nt - 1)];
                    r[j] = (unsigned)v < (unsigned)A.a_rows ? v : 0;  // such an entry is not written and reported below
                }
            for (int k = 0; k < steps && ok; k++, kg++) {
                const int s = kg % GSTAGES, x = k * (GB / kElem);
                if (kg >= GSTAGES) ok = mbar_wait(&S.empty[s], ((kg / GSTAGES) - 1) & 1, abort);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                uint8_t *stage = ring + s * kGmmStage;
                if (lane == 0) {
                    mbar_expect_tx(&S.full[s], (GM + (whole ? GT : nt16)) * GB);
                    tma_load_2d(stage, &map_w, x, I.g * A.n + I.rb * GM, &S.full[s]);
                    if (whole) tma_load_2d(stage + GM * GB, &map_a128, x, I.base, &S.full[s]);
                }
                __syncwarp();
                if (A.in_rows) {
                    if (lane * 4 < nt16)
                        tma_gather4(stage + GM * GB + lane * 4 * GB, &map_a, x, r[0], r[1], r[2], r[3], &S.full[s]);
                } else if (!whole && lane * 16 < nt16) {
                    tma_load_2d(stage + GM * GB + lane * 16 * GB, &map_a, x, I.base + lane * 16, &S.full[s]);
                }
            }
        }
        if (!ok) S.abort = 1;
        // every issued copy has landed before the CTA may leave (bounded; each slot's latest phase)
        for (int k = max(0, kg - GSTAGES); k < kg; k++) mbar_wait(&S.full[k % GSTAGES], (k / GSTAGES) & 1, never);
    } else if (warp == 1) {
        // ---------------- MMA issuer ----------------
        if (lane == 0) {
            bool ok = true;
            int kg = 0, bg = 0;  // stages consumed, accumulators handed over by this CTA
            for (int item = blockIdx.x; item < nitems && ok; item += gridDim.x) {
                const GmmItem I = gmm_item(S, A.groups, A.nrb, item);
                const uint32_t idesc = A.idesc | (uint32_t)(((I.nt + 15) & ~15) >> 3) << 17;
                for (int k = 0; k < steps; k++, kg++) {
                    const int s = kg % GSTAGES, buf = bg & 3;
                    const bool open = F8 || k == 0, close = F8 || k == steps - 1;
                    if (open && bg >= 4 && !mbar_wait(&S.acc_empty[buf], ((bg / 4) - 1) & 1, abort)) { ok = false; break; }
                    if (!mbar_wait(&S.full[s], (kg / GSTAGES) & 1, abort)) { ok = false; break; }
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    const uint8_t *stage = ring + s * kGmmStage;
                    const uint64_t da = gmm_desc(stage), db = gmm_desc(stage + GM * GB);
#pragma unroll
                    for (int j = 0; j < GB / 32; j++)  // 32 bytes of k per MMA
                        gmm_mma<F8>(tmem + buf * GT, da + (uint64_t)(j * 2), db + (uint64_t)(j * 2), idesc, !(open && j == 0));
                    gmm_commit(&S.empty[s]);
                    if (close) {
                        gmm_commit(&S.acc_full[buf]);
                        bg++;
                    }
                }
            }
            if (!ok) S.abort = 1;
            // every MMA issued by this CTA has completed before TMEM and shared memory are released (bounded)
            gmm_commit(&S.drain);
            mbar_wait(&S.drain, 0, never);
        }
        __syncwarp();
    } else {
        // ---------------- fold and write ----------------
        // TMEM lane quadrant = warp % 4; of a tile's 32-entry chunks warps 2-5 take the even, warps 6-9 the odd ones
        const int sub = warp & 3, half = (warp - 2) >> 2, et = threadIdx.x - 64;
        const int r = sub * 32 + lane;
        bool ok = true;  // a thread whose wait ran out goes on without waiting or writing: the block barriers stay matched
        int bg = 0, it = 0;
        const int nkc = F8 ? (steps + kGmmKc - 1) / kGmmKc : 1;
        // scales of blocks [kc * 8, kc * 8 + 8) times the weights' block scales: thread = (entry, 4 blocks)
        float pre[4] = {0, 0, 0, 0};
        int pre_row = 0;  // row of a of this thread's entry (of the item whose scales are loaded next)
        const int pe = et >> 1, pk = (et & 1) * 4;
        auto entry_row = [&](const GmmItem &I) {
            const int i = I.base + min(pe, I.nt - 1);
            const int v = A.in_rows ? A.in_rows[i] : i;
            return (unsigned)v < (unsigned)A.a_rows ? v : 0;
        };
        auto load_scales = [&](const GmmItem &I, int kc) {
            const float *as = A.as + (int64_t)pre_row * A.ldas;
            const float *ws = A.ws + ((int64_t)I.g * A.nrb + I.rb) * steps;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const int b = kc * kGmmKc + pk + j;
                pre[j] = b < steps && pe < I.nt ? __ldg(as + b) * __ldg(ws + b) : 0.0f;
            }
        };
        GmmItem I{0, 0, 0, 0}, N{0, 0, 0, 0};
        if ((int)blockIdx.x < nitems) {
            N = gmm_item(S, A.groups, A.nrb, blockIdx.x);
            if (F8) {
                pre_row = entry_row(N);
                load_scales(N, 0);
            }
        }
        int cbuf = 0;  // chunks of scales staged so far
        for (int item = blockIdx.x; item < nitems; item += gridDim.x, it++) {
            I = N;
            const bool more = item + (int)gridDim.x < nitems;
            if (more) N = gmm_item(S, A.groups, A.nrb, item + gridDim.x);
            int(&orow)[GT] = S.orow[it & 1];
            float(&ow)[GT] = S.ow[it & 1];
            if (et < GT && et < I.nt) {
                const int i = I.base + et;
                int o = A.out_rows ? A.out_rows[i] : i;
                if ((unsigned)o >= (unsigned)A.out_rows_n) o = -1;
                if (A.in_rows && (unsigned)A.in_rows[i] >= (unsigned)A.a_rows) o = -1;
                if (o < 0) atomicCAS(A.err, kErrNone, kErrBadSlot);
                orow[et] = o;
                ow[et] = A.out_scale ? A.out_scale[i] : 1.0f;
            }
            float2 f[32];
#pragma unroll
            for (int j = 0; j < 32; j++) f[j] = make_float2(0.0f, 0.0f);
            for (int kc = 0; kc < nkc; kc++, cbuf++) {
                float(&p)[kGmmKc][GT] = S.p[cbuf & 1];
                if (F8)
#pragma unroll
                    for (int j = 0; j < 4; j++) p[pk + j][pe] = pre[j];
                asm volatile("bar.sync 1, %0;" ::"n"(kGmmEpi) : "memory");
                if (F8) {  // the next chunk's scales are in flight during this chunk's fold
                    if (kc + 1 < nkc) {
                        load_scales(I, kc + 1);
                    } else if (more) {
                        pre_row = entry_row(N);
                        load_scales(N, 0);
                    }
                }
                const int nb = F8 ? min(kGmmKc, steps - kc * kGmmKc) : 1;
                for (int b = 0; b < nb; b++, bg++) {
                    const int buf = bg & 3;
                    if (ok && !mbar_wait(&S.acc_full[buf], (bg / 4) & 1, abort)) ok = false;
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    ok = __all_sync(0xffffffffu, ok);
                    if (ok) {
#pragma unroll
                        for (int c = 0; c < 2; c++) {
                            const int c0 = (half + 2 * c) * 32;
                            if (c0 >= I.nt) continue;
                            float v[32];
                            gmm_ld32(tmem + ((uint32_t)(sub * 32) << 16) + buf * GT + c0, v);
#pragma unroll
                            for (int j = 0; j < 8; j++) {
                                const int o = c * 16 + j * 2;
                                if (F8) {
                                    const float4 s4 = *reinterpret_cast<const float4 *>(&p[b][c0 + j * 4]);
                                    f[o] = __ffma2_rn(make_float2(v[j * 4], v[j * 4 + 1]), make_float2(s4.x, s4.y), f[o]);
                                    f[o + 1] = __ffma2_rn(make_float2(v[j * 4 + 2], v[j * 4 + 3]), make_float2(s4.z, s4.w), f[o + 1]);
                                } else {
                                    f[o] = make_float2(v[j * 4], v[j * 4 + 1]);
                                    f[o + 1] = make_float2(v[j * 4 + 2], v[j * 4 + 3]);
                                }
                            }
                        }
                    }
                    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&S.acc_empty[buf]);
                }
            }
            const int col = I.rb * GM + r;
            if (ok && col < A.n) {
#pragma unroll
                for (int j = 0; j < 64; j++) {
                    const int t = (half + 2 * (j >> 5)) * 32 + (j & 31);
                    const float fj = (j & 1) ? f[j >> 1].y : f[j >> 1].x;
                    if (t < I.nt && orow[t] >= 0) store_out(A.out, A.out_type, (int64_t)orow[t] * A.ldo + col, fj * ow[t]);
                }
            }
        }
        if (!ok) S.abort = 1;
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (S.abort && threadIdx.x == 0) atomicCAS(A.err, kErrNone, kErrTimeout);
    if (warp == 1) {
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem));
    }
}

// ---------------------------------------------------------------------------------------------------------------------

static PFN_cuTensorMapEncodeTiled_v12000 gmm_encode_fn() {
    static PFN_cuTensorMapEncodeTiled_v12000 fn = [] {
        cudaDriverEntryPointQueryResult q;
        void *p = nullptr;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess ||
            q != cudaDriverEntryPointSuccess)
            p = nullptr;
        return reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
    }();
    return fn;
}

// 2-D map over [rows][k] with a row pitch of ld elements, boxes of box_rows x 128 bytes, 128-byte swizzle; what lies
// outside reads as zeros
static bool gmm_map(CUtensorMap *m, const void *base, int elem, int64_t rows, int64_t k, int64_t ld, int box_rows) {
    auto fn = gmm_encode_fn();
    if (!fn) return false;
    const cuuint64_t dims[2] = {(cuuint64_t)k, (cuuint64_t)rows};
    const cuuint64_t strides[1] = {(cuuint64_t)(ld * elem)};
    const cuuint32_t box[2] = {(cuuint32_t)(GB / elem), (cuuint32_t)box_rows};
    const cuuint32_t estr[2] = {1, 1};
    return fn(m, elem == 1 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_UINT16, 2, const_cast<void *>(base),
              dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
              CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

constexpr size_t kGmmSmem = (size_t)GSTAGES * kGmmStage + sizeof(GmmShared) + 1024;
static_assert(kGmmSmem <= 227 * 1024, "shared memory of one CTA");

void gmm_set_attributes() {
    cudaFuncSetAttribute(gmm_kernel<true>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kGmmSmem);
    cudaFuncSetAttribute(gmm_kernel<false>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kGmmSmem);
}

int launch_grouped_matmul(const inzg_grouped_matmul_args &G, int num_sms, int32_t *err, cudaStream_t st) {
    const bool f8 = G.type == INZG_T_E4M3;
    const int elem = f8 ? 1 : 2;
    const int64_t lda = G.lda ? G.lda : G.k, ldw = G.ldw ? G.ldw : G.k;
    CUtensorMap map_w, map_a, map_a128;
    if (!gmm_map(&map_w, G.w, elem, (int64_t)G.groups * G.n, G.k, ldw, GM) ||
        !gmm_map(&map_a, G.a, elem, G.a_rows, G.k, lda, G.in_rows ? 1 : 16) ||
        !gmm_map(&map_a128, G.a, elem, G.a_rows, G.k, lda, GT))
        return -1;
    GmmArgs A{};
    A.groups = G.groups;
    A.n = G.n;
    A.nrb = (G.n + GM - 1) / GM;
    A.steps = (int)(((int64_t)G.k * elem + GB - 1) / GB);
    A.entries = G.entries;
    A.a_rows = G.a_rows;
    A.out_rows_n = G.out_rows_n;
    A.out_type = G.out_type;
    A.off = G.off;
    A.in_rows = G.in_rows;
    A.out_rows = G.out_rows;
    A.out_scale = G.out_scale;
    A.as = G.a_scale;
    A.ldas = G.lda_scale ? G.lda_scale : A.steps;
    A.ws = G.w_scale;
    A.out = G.out;
    A.ldo = G.ldo ? G.ldo : G.n;
    A.err = err;
    // fp32 accumulators; e4m3 (0), bf16 (1) or f16 (0) operands, both K-major; M = 128
    const uint32_t fmt = G.type == INZG_T_BF16 ? 1u : 0u;
    A.idesc = (1u << 4) | (fmt << 7) | (fmt << 10) | ((uint32_t)(GM >> 4) << 24);
    const int64_t tiles = std::min<int64_t>(G.entries, G.entries / GT + G.groups);  // at most so many
    const int grid = (int)std::min<int64_t>(num_sms, tiles * A.nrb);
    if (f8) gmm_kernel<true><<<grid, kGmmThreads, kGmmSmem, st>>>(map_w, map_a, map_a128, A);
    else gmm_kernel<false><<<grid, kGmmThreads, kGmmSmem, st>>>(map_w, map_a, map_a128, A);
    return 1;
}

}  // namespace inzg
