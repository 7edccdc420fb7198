// k_gmm_large.cu -- the grouped product of e4m3 rows for many entries per group (k_gmm.cu has the mathematics and the other
// kernel), sm_100a: the entries are the MMA's M, one TMEM lane each, 256 rows of w its N.
//
// With the entries on the M side a thread of the fold owns one entry and 128 columns, all in one block of w's scales: the
// block's factor as * ws is one number per thread and the fold 64 packed multiply-adds per 128 columns without a read of
// shared memory (344 cycles for all 256 columns, measured alone, beside 512 cycles of MMA per 128 k). Two 256-column
// accumulators alternate by k block.
//   warp 0      TMA producer: per 128-byte step of k the CTA's rows of w and, unless they are gathered, its rows of a
//   warp 1      allocates all 512 TMEM columns, one lane issues 4 MMAs per stage
//   warps 2-3   stage as * ws and where each entry's result goes, ahead of the fold
//   warps 4-7   the entries' rows by index
//   warps 8-15  fold and write: thread = (entry, 128 of the 256 columns); the others hand registers over to these
// Persistent, one CTA per SM; every mbarrier wait is bounded (k_gmm.cu).
// Measured on B200, back to back in CUDA graphs: 4000 x 10240 x 2560 in 121 us at best (1730 TFLOP/s), 126 to 134 in the median; 4096 tokens'
// down products (512 experts, 2048 x 640, fp32 slots) in 224 us at best, 245 to 257 in the median (1.03 GB); their gate|up (1280 x 2048,
// gathered, bf16) in 342 us at best, 407 in the median, 294 and 343 to 370 with rows in order. Eager calls take 142 and 258 us.
// What bounds a step of 128 k is open: 830 cycles in the kernel, 572 for MMA, fold and hand-over measured alone, 862 for its 48 KB at the
// 57 bytes a cycle that an SM alone got from L2 (k_gmm.cu), while a pair of CTAs that shares its copies gained 1 %. An item's
// results take some 4000 cycles more, a fifth of a dense item, half of one with five steps, and are not overlapped with the next one's.
#include <algorithm>

#include "k_gmm.cuh"
#include "k_launch.h"

namespace inzg {

constexpr int kLargeThreads = 512, kLargeGatherWarps = 4;
constexpr int kLargeKc = 4;  // k blocks whose scales are staged at once
constexpr int LM = 128, LN = 256, LACC = 2;  // entries per CTA, rows of w per item, accumulators

constexpr int LSTAGES = 3, kLargeStage = (LM + LN) * kGmmBytes;

struct LargeShared {
    uint64_t full[LSTAGES], empty[LSTAGES], acc_full[LACC], acc_empty[LACC], drain;
    uint32_t tmem_base;
    int abort, never;
    alignas(16) uint4 out[8][32 * 9];  // per warp of the fold: 128 bytes of 32 rows on their way out
    GmmStaged<LM, 1, 2, kLargeKc> staged;
    GmmWalk walk;
};

// The warp's results to their rows: lane l has 128 neighbouring results f of entry l, for columns from col0 on of the row dst
// (null: not written). 128 bytes of each row at a time pass through shared memory (`stage`: 32 rows of 9 x 16 bytes, so that
// both the writes by row and the reads by piece meet no bank twice), and leave as whole lines: 8 lanes per row. Straight from the
// registers, 32 bytes of 32 rows per instruction, an item's results took some 6000 of its 26000 cycles.
template <class T>
__device__ __forceinline__ void write_rows(uint4 *stage, char *dst, int col0, int n, float w, const float2 (&f)[64], bool wide) {
    constexpr int COLS = 128 / sizeof(T), E16 = 16 / sizeof(T);  // columns of a pass, elements of a piece
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int p = 0; p < 128 / COLS; p++) {
        const int c0 = col0 + p * COLS;
        if (c0 >= n) break;
#pragma unroll
        for (int q = 0; q < 8; q++) {
            T v[E16];
#pragma unroll
            for (int e = 0; e < E16; e++) {
                const float2 x = f[(p * COLS + q * E16 + e) >> 1];
                from_f32(((e & 1) ? x.y : x.x) * w, v[e]);
            }
            uint4 o;
            memcpy(&o, v, 16);
            stage[lane * 9 + q] = o;
        }
        __syncwarp();
        if (wide) {
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const int r = i * 4 + (lane >> 3), piece = lane & 7, c = c0 + piece * E16;
                char *row = reinterpret_cast<char *>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(dst), r));
                const uint4 o = stage[r * 9 + piece];
                if (row && c + E16 <= n) {
                    store_global(reinterpret_cast<uint4 *>(row + (int64_t)c * sizeof(T)), o);
                } else if (row) {
                    T v[E16];
                    memcpy(v, &o, 16);
#pragma unroll
                    for (int e = 0; e < E16; e++)
                        if (c + e < n) store_global(reinterpret_cast<T *>(row) + c + e, v[e]);
                }
            }
        } else {
#pragma unroll 4
            for (int r = 0; r < 32; r++) {
                T *row = reinterpret_cast<T *>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(dst), r));
                const T *from = reinterpret_cast<const T *>(stage + r * 9);
#pragma unroll
                for (int e = lane; e < COLS; e += 32)
                    if (row && c0 + e < n) store_global(row + c0 + e, from[e]);
            }
        }
        __syncwarp();
    }
}

// map_w: [groups * n][k] in 256-row boxes; map_a: the rows of a in 128-row boxes
__global__ void __launch_bounds__(kLargeThreads, 1)
gmm_large_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_a,
                 const __grid_constant__ GmmArgs A) {
    extern __shared__ __align__(1024) uint8_t gmm_dyn[];
    // an offset, not a rounded address: the compiler has to see shared memory, or every access becomes a generic one
    uint8_t *ring = gmm_dyn + (-smem_u32(gmm_dyn) & 1023u);
    LargeShared &S = *reinterpret_cast<LargeShared *>(ring + LSTAGES * kLargeStage);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    volatile int *abort = &S.abort;
    volatile int *never = &S.never;

    const GmmOffsets<kLargeThreads> offsets(A);  // on their way while barriers and TMEM are set up
    if (threadIdx.x == 0) {
        for (int s = 0; s < LSTAGES; s++) {
            mbar_init(&S.full[s], A.in_rows ? 1 + kLargeGatherWarps : 1);
            mbar_init(&S.empty[s], 1);
        }
        for (int b = 0; b < LACC; b++) {
            mbar_init(&S.acc_full[b], 1);
            mbar_init(&S.acc_empty[b], 8);
        }
        mbar_init(&S.drain, 1);
        gmm_staged_init(S.staged);
        S.abort = 0;
        S.never = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) gmm_tmem_alloc(&S.tmem_base);
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();  // TMEM's address is read here: read after the walk it is not kept in a register (4096 tokens, down: 226 -> 235 us)
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = S.tmem_base;
    const int nitems = gmm_walk_init<LM, kLargeThreads>(S.walk, A, offsets, blockIdx.x, gridDim.x);
    const int steps = A.steps;

    // registers: 128 per thread at launch, 16 warps; 8 * 80 + 8 * 176 = 16 * 128
    if (warp < 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 80;");
        if (warp == 0) {
            // ---------------- TMA producer ----------------
            if (gmm_elect()) {
                int issued = 0;  // stages, counted up to the ring's size
                bool ok = true;
                GmmSlot<LSTAGES> slot;
                const uint32_t bytes = (LN + (A.in_rows ? 0 : LM)) * kGmmBytes;
                for (int item = blockIdx.x, n = 0; item < nitems && ok; item += gridDim.x, n++) {
                    const GmmItem I = gmm_item<LM>(S.walk, A, item, n);
                    const int wrow = I.g * A.n + I.rb * LN;
                    for (int k = 0, x = 0; k < steps; k++, x += kGmmBytes) {
                        if (issued == LSTAGES) {
                            if (!(ok = mbar_wait(&S.empty[slot.i], slot.parity ^ 1, abort))) break;
                        } else {
                            issued++;
                        }
                        uint8_t *stage = ring + slot.i * kLargeStage;
                        uint64_t *full = &S.full[slot.i];
                        mbar_expect_tx(full, bytes);
                        tma_load_2d(stage + LM * kGmmBytes, &map_w, x, wrow, full);
                        if (!A.in_rows) tma_load_2d(stage, &map_a, x, I.base, full);
                        slot.next();
                    }
                }
                if (!ok) S.abort = 1;
                // every issued copy has landed before the CTA may leave (bounded): the last round of each slot in use
                for (int k = 0; k < issued; k++) {
                    if (issued == LSTAGES) mbar_wait(&S.full[slot.i], slot.parity ^ 1, never);
                    else mbar_wait(&S.full[k], 0, never);
                    slot.next();
                }
            }
            __syncwarp();
        } else if (warp == 1) {
            // ---------------- MMA issuer ----------------
            if (gmm_elect()) {
                bool ok = true;
                GmmSlot<LSTAGES> slot;
                GmmSlot<LACC> at;
                int given = 0;  // accumulators handed over, counted up to LACC
                const uint64_t desc0 = gmm_desc(ring);
                for (int item = blockIdx.x; item < nitems && ok; item += gridDim.x) {
                    const uint32_t n16 = (uint32_t)min(LN, (A.n - item % A.nrb * LN + 15) & ~15);
                    const uint32_t idesc = A.idesc | (n16 >> 3) << 17;
                    for (int k = 0; k < steps; k++) {
                        if (given == LACC) ok = mbar_wait(&S.acc_empty[at.i], at.parity ^ 1, abort);
                        else given++;
                        if (!ok || !(ok = mbar_wait(&S.full[slot.i], slot.parity, abort))) break;
                        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                        const uint64_t da = desc0 + (uint64_t)(slot.i * (kLargeStage >> 4));
                        gmm_mma_stage<true>(tmem + at.i * LN, da, da + (LM * kGmmBytes >> 4), idesc, true);
                        gmm_commit(&S.acc_full[at.i]);
                        at.next();
                        gmm_commit(&S.empty[slot.i]);
                        slot.next();
                    }
                }
                if (!ok) S.abort = 1;
                // every MMA issued by this CTA has completed before TMEM and shared memory are released (bounded)
                gmm_commit(&S.drain);
                mbar_wait(&S.drain, 0, never);
            }
            __syncwarp();
        } else if (warp == 2 || warp == 3) {
            if (!gmm_stage_walk<true, LM>(S.staged, S.walk, A, nitems, abort)) S.abort = 1;
        } else if (warp >= 4 && A.in_rows) {
            if (!gmm_gather<LM, LSTAGES, 1, kLargeGatherWarps>(S.walk, A, threadIdx.x - 128, nitems, ring, kLargeStage, 0, S.full, S.empty,
                                                            abort))
                S.abort = 1;
        }
    } else {
        // ---------------- fold and write: thread = (entry = TMEM lane, 128 of the 256 columns) ----------------
        asm volatile("setmaxnreg.inc.sync.aligned.u32 176;");
        const int sub = warp & 3, half = (warp - 8) >> 2, r = sub * 32 + lane;
        bool ok = true;
        GmmSlot<LACC> acc;
        GmmSlot<kGmmRing> ps, ts;
        const uint32_t lanes = tmem + ((uint32_t)(sub * 32) << 16) + half * 128;
        for (int item = blockIdx.x, n = 0; item < nitems && ok; item += gridDim.x, n++) {
            const GmmItem I = gmm_item<LM>(S.walk, A, item, n);
            const int col0 = I.rb * LN + half * 128;
            const bool mine = col0 < A.n && sub * 32 < I.nt;  // the warp has columns and entries
            float2 f[64];
#pragma unroll
            for (int j = 0; j < 64; j++) f[j] = make_float2(0.0f, 0.0f);
            for (int b0 = 0; b0 < steps; b0 += kLargeKc) {
                ok = mbar_wait(&S.staged.p_full[0][ps.i], ps.parity, abort);
                const int nb = min(kLargeKc, steps - b0);
                for (int b = 0; b < nb; b++) {
                    const float s = S.staged.p[0][ps.i][half][b][r];
                    const float2 s2 = make_float2(s, s);
                    if (ok) ok = mbar_wait(&S.acc_full[acc.i], acc.parity, abort);
                    ok = __all_sync(0xffffffffu, ok);
                    if (!ok) break;
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    if (mine) {
#pragma unroll
                        for (int c = 0; c < 4; c++) {
                            float v[32];
                            gmm_ld(lanes + acc.i * LN + c * 32, v);
#pragma unroll
                            for (int j = 0; j < 16; j++)
                                f[c * 16 + j] = __ffma2_rn(make_float2(v[2 * j], v[2 * j + 1]), s2, f[c * 16 + j]);
                        }
                    }
                    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&S.acc_empty[acc.i]);
                    acc.next();
                }
                if (!ok) break;
                __syncwarp();
                if (lane == 0) mbar_arrive(&S.staged.p_empty[0][ps.i]);
                ps.next();
            }
            if (ok) ok = mbar_wait(&S.staged.to_full[0][ts.i], ts.parity, abort);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            const GmmTo to = S.staged.to[0][ts.i][r];
            __syncwarp();
            if (lane == 0) mbar_arrive(&S.staged.to_empty[0][ts.i]);
            ts.next();
            if (mine) {
                uint4 *stage = S.out[warp - 8];
                if (A.out_type == INZG_T_F32) write_rows<float>(stage, to.row, col0, A.n, to.w, f, A.wide_out);
                else if (A.out_type == INZG_T_BF16) write_rows<__nv_bfloat16>(stage, to.row, col0, A.n, to.w, f, A.wide_out);
                else write_rows<__half>(stage, to.row, col0, A.n, to.w, f, A.wide_out);
            }
        }
        if (!ok) S.abort = 1;
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (S.abort && threadIdx.x == 0) atomicCAS(A.err, kErrNone, kErrTimeout);
    if (warp == 1) gmm_tmem_free(tmem);
}

// ---------------------------------------------------------------------------------------------------------------------

constexpr size_t kLargeSmem = (size_t)LSTAGES * kLargeStage + sizeof(LargeShared) + 1024;
// more than half of an SM's shared memory, so that a CTA is alone on its SM with all of TMEM
static_assert(kLargeSmem <= 227 * 1024 && kLargeSmem > 116 * 1024, "one CTA per SM");

bool gmm_large_set_attributes() {
    return cudaFuncSetAttribute(gmm_large_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kLargeSmem) == cudaSuccess &&
           gmm_split_holds(gmm_large_kernel);
}

int gmm_large_launch(const inzg_grouped_matmul_args &G, GmmArgs A, int num_sms, cudaStream_t st) {
    CUtensorMap map_w, map_a;
    if (!gmm_map(&map_w, G.w, 1, (int64_t)G.groups * G.n, G.k, G.ldw ? G.ldw : G.k, LN) ||
        !gmm_map(&map_a, G.a, 1, G.a_rows, G.k, G.lda ? G.lda : G.k, LM))
        return -1;
    A.nrb = (G.n + LN - 1) / LN;
    const int esize = G.out_type == INZG_T_F32 ? 4 : 2;
    A.wide_out = !(reinterpret_cast<uintptr_t>(G.out) % 16) && !(A.ldo * esize % 16);
    const int64_t tiles = std::min<int64_t>(G.entries, G.entries / LM + G.groups);  // at most so many
    const int grid = (int)std::min<int64_t>(num_sms, tiles * A.nrb);
    gmm_large_kernel<<<grid, kLargeThreads, kLargeSmem, st>>>(map_w, map_a, A);
    return 1;
}

}  // namespace inzg
