// k_gmm_large.cu -- the grouped product for many entries per group (k_gmm.cu has the mathematics and the other kernel):
// work items of 128 entries (the MMA's M, one TMEM lane each) x 256 rows of w (its N), sm_100a.
//
// With the entries on the M side a thread of the fold owns one entry and 128 columns, all in one block of w's scales: the
// block's factor as * ws is one number per thread and the fold is 64 packed multiply-adds per 128 columns, with no reads of
// shared memory, beside 512 cycles of MMA per 128 k. Two 256-column accumulators alternate by k block (e4m3) or by item.
//   warp 0      TMA producer: per 128-byte step of k a box of 256 rows of w and, unless they are gathered, 128 rows of a
//   warp 1      allocates all 512 TMEM columns, one lane issues 4 MMAs per stage
//   warps 2-3   the entries' rows by index
//   warps 4-11  fold and write: thread = (entry, 128 of the 256 columns); the first warpgroup hands registers over to these
// Persistent, one CTA per SM; every mbarrier wait is bounded (k_gmm.cu).
#include <algorithm>

#include "k_gmm.cuh"
#include "k_launch.h"

namespace inzg {

constexpr int LM = 128, LN = 256, LSTAGES = 4, LACC = 2;
constexpr int kLargeStage = (LM + LN) * kGmmBytes;

struct LargeShared {
    uint64_t full[LSTAGES], empty[LSTAGES], acc_full[LACC], acc_empty[LACC], drain;
    uint32_t tmem_base;
    int abort, never;
    GmmWalk walk;
};

// 32 bytes of one row
__device__ __forceinline__ void store_32b(void *p, const uint32_t (&w)[8]) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]),
                 "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
                 : "memory");
}

template <class T>
__device__ __forceinline__ uint32_t pack2(float a, float b) {  // two 16-bit results, the first in the low half
    T v[2];
    from_f32(a, v[0]);
    from_f32(b, v[1]);
    uint32_t o;
    memcpy(&o, v, sizeof(o));
    return o;
}

// 32 neighbouring results of one entry to its row (from column `col` on, `left` columns of the row remain)
template <class T>
__device__ __forceinline__ void put32(char *row, int64_t col, int left, float w, const float2 *f, bool wide) {
    T *o = reinterpret_cast<T *>(row) + col;
    if (wide && left >= 32) {
#pragma unroll
        for (int q = 0; q < (int)sizeof(T); q++) {  // 32 bytes each
            uint32_t v[8];
#pragma unroll
            for (int i = 0; i < 8; i++) {
                if constexpr (sizeof(T) == 4) {
                    const float2 x = f[q * 4 + (i >> 1)];
                    v[i] = __float_as_uint(((i & 1) ? x.y : x.x) * w);
                } else {
                    const float2 x = f[q * 8 + i];
                    v[i] = pack2<T>(x.x * w, x.y * w);
                }
            }
            store_32b(o + q * (32 / sizeof(T)), v);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 32; i++) {
            T v;
            from_f32(((i & 1) ? f[i >> 1].y : f[i >> 1].x) * w, v);
            if (i < left) o[i] = v;
        }
    }
}
__device__ __forceinline__ void put32_any(int type, char *row, int64_t col, int left, float w, const float2 *f, bool wide) {
    if (type == INZG_T_F32) put32<float>(row, col, left, w, f, wide);
    else if (type == INZG_T_BF16) put32<__nv_bfloat16>(row, col, left, w, f, wide);
    else put32<__half>(row, col, left, w, f, wide);
}

// map_w: [groups * n][k] in 256-row boxes; map_a: the rows of a in 128-row boxes
template <bool F8>
__global__ void __launch_bounds__(kGmmThreads, 1)
gmm_large_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_a,
                 const __grid_constant__ GmmArgs A) {
    extern __shared__ __align__(1024) uint8_t gmm_dyn[];
    uint8_t *ring = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(gmm_dyn) + 1023) & ~uintptr_t(1023));
    LargeShared &S = *reinterpret_cast<LargeShared *>(ring + LSTAGES * kLargeStage);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    volatile int *abort = &S.abort;
    volatile int *never = &S.never;
    constexpr int kElem = F8 ? 1 : 2;

    if (threadIdx.x == 0) {
        for (int s = 0; s < LSTAGES; s++) {
            mbar_init(&S.full[s], A.in_rows ? 1 + kGmmGatherWarps : 1);
            mbar_init(&S.empty[s], 1);
        }
        for (int b = 0; b < LACC; b++) {
            mbar_init(&S.acc_full[b], 1);
            mbar_init(&S.acc_empty[b], 8);
        }
        mbar_init(&S.drain, 1);
        S.abort = 0;
        S.never = 0;
        S.walk.bad = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) gmm_tmem_alloc(&S.tmem_base);
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = S.tmem_base;
    gmm_walk_init<LM>(S.walk, A);
    const int nitems = S.walk.bad ? 0 : S.walk.tstart[A.groups] * A.nrb;
    if (S.walk.bad && threadIdx.x == 0) atomicCAS(A.err, kErrNone, kErrOverflow);
    const int steps = A.steps;

    // registers: 168 per thread at launch, 12 warps; 4 * 88 + 8 * 208 = 12 * 168
    if (warp < 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
        if (warp == 0) {
            // ---------------- TMA producer ----------------
            if (lane == 0) {
                int kg = 0;  // stages issued by this CTA
                bool ok = true;
                for (int item = blockIdx.x; item < nitems && ok; item += gridDim.x) {
                    const GmmItem I = gmm_item<LM>(S.walk, A.groups, A.nrb, item);
                    for (int k = 0; k < steps; k++, kg++) {
                        const int s = kg % LSTAGES, x = k * (kGmmBytes / kElem);
                        if (kg >= LSTAGES && !mbar_wait(&S.empty[s], ((kg / LSTAGES) - 1) & 1, abort)) {
                            ok = false;
                            break;
                        }
                        uint8_t *stage = ring + s * kLargeStage;
                        mbar_expect_tx(&S.full[s], (LN + (A.in_rows ? 0 : LM)) * kGmmBytes);
                        tma_load_2d(stage + LM * kGmmBytes, &map_w, x, I.g * A.n + I.rb * LN, &S.full[s]);
                        if (!A.in_rows) tma_load_2d(stage, &map_a, x, I.base, &S.full[s]);
                    }
                }
                if (!ok) S.abort = 1;
                // every issued copy has landed before the CTA may leave (bounded; each slot's latest phase)
                for (int k = max(0, kg - LSTAGES); k < kg; k++) mbar_wait(&S.full[k % LSTAGES], (k / LSTAGES) & 1, never);
            }
            __syncwarp();
        } else if (warp == 1) {
            // ---------------- MMA issuer ----------------
            if (lane == 0) {
                bool ok = true;
                int kg = 0, bg = 0;  // stages consumed, accumulators handed over by this CTA
                for (int item = blockIdx.x; item < nitems && ok; item += gridDim.x) {
                    const int rb = item % A.nrb;
                    const uint32_t n16 = (uint32_t)min(LN, (A.n - rb * LN + 15) & ~15);
                    const uint32_t idesc = A.idesc | (n16 >> 3) << 17;
                    for (int k = 0; k < steps; k++, kg++) {
                        const int s = kg % LSTAGES, buf = bg % LACC;
                        const bool open = F8 || k == 0, close = F8 || k == steps - 1;
                        if (open && bg >= LACC && !mbar_wait(&S.acc_empty[buf], ((bg / LACC) - 1) & 1, abort)) { ok = false; break; }
                        if (!mbar_wait(&S.full[s], (kg / LSTAGES) & 1, abort)) { ok = false; break; }
                        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                        const uint8_t *stage = ring + s * kLargeStage;
                        const uint64_t da = gmm_desc(stage), db = gmm_desc(stage + LM * kGmmBytes);
#pragma unroll
                        for (int j = 0; j < kGmmBytes / 32; j++)  // 32 bytes of k per MMA
                            gmm_mma<F8>(tmem + buf * LN, da + (uint64_t)(j * 2), db + (uint64_t)(j * 2), idesc, !(open && j == 0));
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
        } else if (A.in_rows) {
            if (!gmm_gather<LM, LSTAGES>(S.walk, A, nitems, ring, kLargeStage, 0, S.full, S.empty, abort)) S.abort = 1;
        }
    } else {
        // ---------------- fold and write: thread = (entry = TMEM lane, 128 of the 256 columns) ----------------
        asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
        const int sub = warp & 3, half = (warp - 4) >> 2;
        const int r = sub * 32 + lane;
        const int esize = A.out_type == INZG_T_F32 ? 4 : 2;
        bool ok = true;
        int bg = 0;
        for (int item = blockIdx.x; item < nitems && ok; item += gridDim.x) {
            const GmmItem I = gmm_item<LM>(S.walk, A.groups, A.nrb, item);
            // this thread's entry: its row of a (for the scales), its row of out, its weight
            const int i = I.base + min(r, I.nt - 1);
            int row = A.in_rows ? A.in_rows[i] : i;
            int o = A.out_rows ? A.out_rows[i] : i;
            const bool bad = (unsigned)row >= (unsigned)A.a_rows || (unsigned)o >= (unsigned)A.out_rows_n;
            if (bad) atomicCAS(A.err, kErrNone, kErrBadSlot);
            if ((unsigned)row >= (unsigned)A.a_rows) row = 0;
            const float w = A.out_scale ? A.out_scale[i] : 1.0f;
            char *dst = r < I.nt && !bad ? static_cast<char *>(A.out) + (int64_t)o * A.ldo * esize : nullptr;
            const int col0 = I.rb * LN + half * 128;
            const bool mine = col0 < A.n;  // the warp's columns exist
            const uint32_t taddr = tmem + ((uint32_t)(sub * 32) << 16) + half * 128;
            if (F8) {
                float2 f[64];
#pragma unroll
                for (int j = 0; j < 64; j++) f[j] = make_float2(0.0f, 0.0f);
                const float *as = A.as + (int64_t)row * A.ldas;
                const float *ws = A.ws + ((int64_t)I.g * A.nrb128 + I.rb * 2 + (mine ? half : 0)) * steps;
                float next = __ldg(as) * __ldg(ws);
                for (int b = 0; b < steps; b++, bg++) {
                    const int buf = bg % LACC;
                    const float2 s2 = make_float2(next, next);
                    if (b + 1 < steps) next = __ldg(as + b + 1) * __ldg(ws + b + 1);
                    if (ok && !mbar_wait(&S.acc_full[buf], (bg / LACC) & 1, abort)) ok = false;
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    ok = __all_sync(0xffffffffu, ok);
                    if (!ok) break;
                    if (mine) {
#pragma unroll
                        for (int c = 0; c < 4; c++) {
                            float v[32];
                            gmm_ld32(taddr + buf * LN + c * 32, v);
#pragma unroll
                            for (int j = 0; j < 16; j++)
                                f[c * 16 + j] = __ffma2_rn(make_float2(v[2 * j], v[2 * j + 1]), s2, f[c * 16 + j]);
                        }
                    }
                    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&S.acc_empty[buf]);
                }
                if (ok && mine && dst)
#pragma unroll
                    for (int c = 0; c < 4; c++)
                        if (col0 + c * 32 < A.n)
                            put32_any(A.out_type, dst, col0 + c * 32, A.n - col0 - c * 32, w, f + c * 16, A.wide_out);
            } else {
                const int buf = bg % LACC;
                if (!mbar_wait(&S.acc_full[buf], (bg / LACC) & 1, abort)) ok = false;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                bg++;
                if (mine) {
#pragma unroll
                    for (int c = 0; c < 4; c++) {
                        float v[32];
                        gmm_ld32(taddr + buf * LN + c * 32, v);
                        float2 f[16];
#pragma unroll
                        for (int j = 0; j < 16; j++) f[j] = make_float2(v[2 * j], v[2 * j + 1]);
                        if (dst && col0 + c * 32 < A.n)
                            put32_any(A.out_type, dst, col0 + c * 32, A.n - col0 - c * 32, w, f, A.wide_out);
                        __syncwarp();
                    }
                }
                asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                __syncwarp();
                if (lane == 0) mbar_arrive(&S.acc_empty[buf]);
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
static_assert(kLargeSmem <= 227 * 1024, "shared memory of one CTA");

void gmm_large_set_attributes() {
    cudaFuncSetAttribute(gmm_large_kernel<true>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kLargeSmem);
    cudaFuncSetAttribute(gmm_large_kernel<false>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kLargeSmem);
}

int gmm_large_launch(const inzg_grouped_matmul_args &G, GmmArgs A, int num_sms, cudaStream_t st) {
    const bool f8 = G.type == INZG_T_E4M3;
    const int elem = f8 ? 1 : 2;
    CUtensorMap map_w, map_a;
    if (!gmm_map(&map_w, G.w, elem, (int64_t)G.groups * G.n, G.k, G.ldw ? G.ldw : G.k, LN) ||
        !gmm_map(&map_a, G.a, elem, G.a_rows, G.k, G.lda ? G.lda : G.k, LM))
        return -1;
    A.nrb = (G.n + LN - 1) / LN;
    const int esize = G.out_type == INZG_T_F32 ? 4 : 2;
    A.wide_out = !(reinterpret_cast<uintptr_t>(G.out) % 32) && !(A.ldo * esize % 32);
    const int64_t tiles = std::min<int64_t>(G.entries, G.entries / LM + G.groups);  // at most so many
    const int grid = (int)std::min<int64_t>(num_sms, tiles * A.nrb);
    if (f8) gmm_large_kernel<true><<<grid, kGmmThreads, kLargeSmem, st>>>(map_w, map_a, A);
    else gmm_large_kernel<false><<<grid, kGmmThreads, kLargeSmem, st>>>(map_w, map_a, A);
    return 1;
}

}  // namespace inzg
