// k_gmm.cu -- dense and grouped products of e4m3 rows with block scales, and of bf16 / f16 rows, on the 5th-generation
// tensor cores (tcgen05.mma kind::f8f6f4 / kind::f16), sm_100a (inzg_matmul_q8, inzg_grouped_matmul): the kernel for few
// entries per group, and the launch of it or the one for many (k_gmm_large.cu).
//
//   out[i][j] = scale_i * sum_b as[i][b] ws[j / 128][b] * (sum_{k in block b} a[i][k] w[g][j][k])
//
// The tensor core sums one block of 128 k in fp32 (TMEM); the block's two scales enter in the fold, which keeps the running
// sum in fp32 registers: f = fma(dot_b, as * ws, f). bf16 / f16 have no scales, but each MMA truncates the sum that it leaves in
// TMEM (16 k: some 0.4 * 2^-24 of it, always towards zero), so that a long k would drift: they leave TMEM every 256 k (kFold
// steps) and are added up in fp32 registers, rounded to nearest. Error against 64 bits, fp32 results of random rows: 2.7e-6 at k = 2560
// and 1.1e-5 at 10240 with the whole k in TMEM, 2.4e-7 and 2.6e-7 as it is (f16 3.5e-7). It costs 1 to 4 %: gate|up of 64 experts, 1280 x
// 2560 bf16, one token 17.3 -> 18.0 us, 333 tokens 81.8 -> 82.5, 2000 tokens 222 -> 230.
//
// Work item: 128 rows of w (the MMA's M, one TMEM lane each) x up to TN entries of one group (its N, rounded up to
// 16). The weights are the M side because a decoding call has a row or two per expert: the MMA, the copies and the
// fold then shrink with the entries, while a weight tile is streamed once whatever their number. A tile of 128 rows
// of w has one weight scale per k block, so as * ws is formed once per entry and block and kept in shared memory.
//   warp 0      TMA producer: per 128-byte step of k a box of 128 weight rows and, unless they are gathered, the entries'
//               rows in boxes of 16 or TN rows, 128-byte swizzle
//   warp 1      allocates all 512 TMEM columns, one lane issues 4 MMAs per step
//   warps 2-3   stage as * ws and where each entry's result goes, ahead of the fold
//   warps 4-7   the entries' rows by index
//   warps 8-15  fold and write, thread = a row of w. TN = 128 (bf16 / f16): all eight warps share an item, every other 32
//               entries; TN = 32: the two warpgroups take the items in turn, so one writes while the other folds
// Measured on B200, back to back in CUDA graphs, top-10 of 512 experts, gate|up 1280 x 2048 e4m3: 32 tokens 73 to 85 us (6 TB/s from
// DRAM), one token 10.5 us; bf16 64 experts 1280 x 2560, 333 tokens 82.5 us (430 MB, 5.2 TB/s), 2000 tokens 230 us.
// Persistent: one CTA per SM walks the items; the offsets are turned into tile numbers by every CTA for itself, which
// costs a read of off and a scan instead of a launch. Every mbarrier wait is bounded; on expiry the CTA records an
// error, drains what it issued, frees its TMEM and returns.
#include <cudaTypedefs.h>

#include <algorithm>
#include <type_traits>

#include "host/op_check.h"
#include "k_gmm.cuh"
#include "k_launch.h"

namespace inzg {

constexpr int kGmmThreads = 512;  // sixteen warps, as above
constexpr int kGmmGatherWarps = 4;
constexpr int GM = 128;    // weight rows of an item
constexpr int kGmmKc = 8;  // k blocks whose scales are staged at once

template <int TN>
struct GmmCfg {
    static constexpr int kTeams = TN <= 32 ? 2 : 1, kTeamWarps = 8 / kTeams;
    // A stage has kSub steps of k behind one pair of barriers; of e4m3 they are handed to the fold together (a slot of kSub
    // accumulators) and slots go back in groups of kGroup: a wait on a completed barrier takes some 90 cycles, and a step of few
    // entries, some 470 cycles, had four of them. Measured against one step and one accumulator at a time, us: a dense row of
    // 10240 x 2560 9.7 -> 9.0, top-10 of 512 e4m3, 2 tokens 17.9 -> 16.5, 64 experts bf16, 2 tokens 32.2 -> 28.0. A step of one
    // item alone now takes some 320 cycles in both types, 18 KB at 57 bytes a cycle: what one SM gets from L2.
    static constexpr int kSub = TN <= 32 ? 2 : 1, kSubBytes = (GM + TN) * kGmmBytes;
    static constexpr int kStages = TN <= 32 ? 5 : 6, kStage = kSub * kSubBytes;
    static constexpr int kFold = 4;                             // bf16 / f16: steps of k that stay in TMEM
    static constexpr int kSlot = kSub * TN;                     // TMEM columns of a slot
    static constexpr int kAcc = 512 / kSlot / kTeams, kGroup = kAcc / 2;  // slots per team: a team waits for its own alone, so it
                                                                // is never two phases ahead
    static constexpr int kChunks = TN / 32 / (2 / kTeams);      // 32-entry chunks per thread
};

template <int TN>
struct GmmShared {
    using C = GmmCfg<TN>;
    uint64_t full[C::kStages], empty[C::kStages], acc_full[C::kTeams][C::kAcc], acc_empty[C::kTeams][2], drain;
    uint32_t tmem_base;
    int abort, never;
    GmmStaged<TN, C::kTeams, 1, kGmmKc> staged;
    GmmWalk walk;
};

template <class T>
__device__ __forceinline__ void gmm_put(const GmmTo &t, int64_t col, float v) {
    T o;
    from_f32(v * t.w, o);
    if (t.row) store_global(reinterpret_cast<T *>(t.row) + col, o);
}

// map_w: [groups * n][k] in 128-row boxes; map_a16 / map_a: the rows of a in boxes of 16 / TN rows
template <bool F8, int TN>
__global__ void __launch_bounds__(kGmmThreads, 1)
gmm_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_a16,
           const __grid_constant__ CUtensorMap map_a, const __grid_constant__ GmmArgs A) {
    using C = GmmCfg<TN>;
    constexpr int ST = C::kStages, NA = C::kAcc;
    extern __shared__ __align__(1024) uint8_t gmm_dyn[];
    // an offset, not a rounded address: the compiler has to see shared memory, or every access becomes a generic one
    uint8_t *ring = gmm_dyn + (-smem_u32(gmm_dyn) & 1023u);
    GmmShared<TN> &S = *reinterpret_cast<GmmShared<TN> *>(ring + ST * C::kStage);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    volatile int *abort = &S.abort;
    volatile int *never = &S.never;
    constexpr int kElem = F8 ? 1 : 2;

    const GmmOffsets<kGmmThreads> offsets(A);  // on their way while barriers and TMEM are set up
    if (threadIdx.x == 0) {
        for (int s = 0; s < ST; s++) {
            mbar_init(&S.full[s], A.in_rows ? 1 + kGmmGatherWarps : 1);
            mbar_init(&S.empty[s], 1);
        }
        for (int t = 0; t < C::kTeams; t++) {
            for (int b = 0; b < NA; b++) mbar_init(&S.acc_full[t][b], 1);
            for (int b = 0; b < 2; b++) mbar_init(&S.acc_empty[t][b], C::kTeamWarps);
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
    const int nitems = gmm_walk_init<TN, kGmmThreads>(S.walk, A, offsets, blockIdx.x, gridDim.x);
    const int steps = A.steps;

    // registers: 128 per thread at launch, 16 warps; 8 * 88 + 8 * 168 = 16 * 128
    if (warp < 8) {
        if (TN > 32) asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
        if (warp == 0) {
            // ---------------- TMA producer ----------------
            if (gmm_elect()) {
                int issued = 0;  // stages, counted up to the ring's size
                bool ok = true;
                GmmSlot<ST> slot;
                for (int item = blockIdx.x, n = 0; item < nitems && ok; item += gridDim.x, n++) {
                    const GmmItem I = gmm_item<TN>(S.walk, A, item, n);
                    const bool whole = I.nt > 16;
                    const uint32_t bytes = (GM + (A.in_rows ? 0 : whole ? TN : 16)) * kGmmBytes;
                    const int wrow = I.g * A.n + I.rb * GM;
                    for (int k = 0; k < steps; k += C::kSub) {
                        if (issued == ST) {
                            if (!(ok = mbar_wait(&S.empty[slot.i], slot.parity ^ 1, abort))) break;
                        } else {
                            issued++;
                        }
                        uint64_t *full = &S.full[slot.i];
                        const int subs = C::kSub == 1 ? 1 : min(C::kSub, steps - k);
                        mbar_expect_tx(full, subs * bytes);
                        for (int j = 0; j < subs; j++) {
                            uint8_t *stage = ring + slot.i * C::kStage + j * C::kSubBytes;
                            const int x = (k + j) * (kGmmBytes / kElem);
                            tma_load_2d(stage, &map_w, x, wrow, full);
                            if (!A.in_rows) {
                                if (whole) tma_load_2d(stage + GM * kGmmBytes, &map_a, x, I.base, full);
                                else tma_load_2d(stage + GM * kGmmBytes, &map_a16, x, I.base, full);
                            }
                        }
                        slot.next();
                    }
                }
                if (!ok) S.abort = 1;
                // every issued copy has landed before the CTA may leave (bounded): the last round of each slot in use
                for (int k = 0; k < issued; k++) {
                    if (issued == ST) mbar_wait(&S.full[slot.i], slot.parity ^ 1, never);
                    else mbar_wait(&S.full[k], 0, never);
                    slot.next();
                }
            }
            __syncwarp();
        } else if (warp == 1) {
            // ---------------- MMA issuer ----------------
            if (gmm_elect()) {
                bool ok = true;
                GmmSlot<ST> slot;
                struct Accs {  // one team's accumulators
                    GmmSlot<NA> at;
                    int given = 0;  // groups handed over, counted up to 2
                };
                Accs mine, other;  // of the current item's team and (two teams) of the next item's: they change places
                const uint64_t desc0 = gmm_desc(ring);
                for (int item = blockIdx.x, team = 0, n = 0; item < nitems && ok; item += gridDim.x, team = (team + 1) % C::kTeams, n++) {
                    const GmmItem I = gmm_item<TN>(S.walk, A, item, n);
                    const uint32_t idesc = A.idesc | (uint32_t)(((I.nt + 15) & ~15) >> 3) << 17;
                    for (int k0 = 0; k0 < steps; k0 += C::kSub) {
                        if (!(ok = mbar_wait(&S.full[slot.i], slot.parity, abort))) break;
                        const int subs = C::kSub == 1 ? 1 : min(C::kSub, steps - k0);
                        const int in = F8 ? 0 : k0 % C::kFold;  // steps of the slot's sum before this one
                        const bool open = in == 0, close = F8 || in + C::kSub == C::kFold || k0 + C::kSub >= steps;
                        if (open && mine.at.i % C::kGroup == 0) {
                            if (mine.given == 2) ok = mbar_wait(&S.acc_empty[team][mine.at.i / C::kGroup], mine.at.parity ^ 1, abort);
                            else mine.given++;
                            if (!ok) break;
                        }
                        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                        for (int j = 0; j < subs; j++) {
                            const uint64_t da = desc0 + (uint64_t)((slot.i * C::kStage + j * C::kSubBytes) >> 4);
                            gmm_mma_stage<F8>(tmem + (team * NA + mine.at.i) * C::kSlot + (F8 ? j * TN : 0), da,
                                              da + (GM * kGmmBytes >> 4), idesc, F8 || in + j == 0);
                        }
                        if (close) {
                            gmm_commit(&S.acc_full[team][mine.at.i]);
                            mine.at.next();
                        }
                        gmm_commit(&S.empty[slot.i]);
                        slot.next();
                    }
                    if constexpr (C::kTeams == 2) {
                        const Accs t = mine;
                        mine = other;
                        other = t;
                    }
                }
                if (!ok) S.abort = 1;
                // every MMA issued by this CTA has completed before TMEM and shared memory are released (bounded)
                gmm_commit(&S.drain);
                mbar_wait(&S.drain, 0, never);
            }
            __syncwarp();
        } else if (warp < 4) {
            if (!gmm_stage_walk<F8, TN>(S.staged, S.walk, A, nitems, abort)) S.abort = 1;
        } else if (warp >= 4) {
            if (A.in_rows && !gmm_gather<TN, ST, C::kSub, kGmmGatherWarps>(S.walk, A, threadIdx.x - 128, nitems, ring, C::kSubBytes,
                                                                           GM * kGmmBytes, S.full, S.empty, abort))
                S.abort = 1;
        }
    } else {
        // ---------------- fold and write ----------------
        if (TN > 32) asm volatile("setmaxnreg.inc.sync.aligned.u32 168;");
        // TMEM lane quadrant = warp % 4. One team: warps 8-11 take the even 32-entry chunks of every item, warps 12-15 the
        // odd ones; two teams: each takes every other item whole.
        const int sub = warp & 3, upper = (warp - 8) >> 2;
        const int team = C::kTeams == 2 ? upper : 0, c_first = C::kTeams == 2 ? 0 : upper, c_step = C::kTeams == 2 ? 1 : 2;
        bool ok = true;
        GmmSlot<NA> acc;
        GmmSlot<kGmmRing> ps, ts;
        const uint32_t lanes = tmem + ((uint32_t)(sub * 32) << 16) + team * NA * C::kSlot + c_first * 32;
        for (int item = blockIdx.x + team * gridDim.x, n = team; item < nitems && ok; item += C::kTeams * gridDim.x, n += C::kTeams) {
            const GmmItem I = gmm_item<TN>(S.walk, A, item, n);
            float2 f[C::kChunks * 16];
#pragma unroll
            for (int j = 0; j < C::kChunks * 16; j++) f[j] = make_float2(0.0f, 0.0f);
            // W: columns of an accumulator that are read and factors that are fetched ahead of it. All 32 against as many as the
            // item has, 20 steps of a dense product, us: 8 entries 10.2 -> 9.7, 24 entries as before; top-10 of 512, 4 tokens: 23.4 -> 23.2
            auto fold = [&](auto width) {
                constexpr int W = decltype(width)::value;
                const int sums = F8 ? steps : (steps + C::kFold - 1) / C::kFold;
                for (int b0 = 0; b0 < sums; b0 += kGmmKc) {
                    if (F8) ok = mbar_wait(&S.staged.p_full[team][ps.i], ps.parity, abort);
                    const float(&p)[kGmmKc][TN] = S.staged.p[team][ps.i][0];
                    const int nb = min(kGmmKc, sums - b0);
                    for (int b = 0; b < nb; b += F8 ? C::kSub : 1) {
                        const uint32_t from = lanes + acc.i * C::kSlot;
                        const bool two = F8 && b + 1 < nb;
                        float4 s4[2][W < 32 ? W / 4 : 1];
                        if constexpr (W < 32) {
#pragma unroll
                            for (int q = 0; q < 2; q++)
#pragma unroll
                                for (int j = 0; j < W / 4; j++)
                                    s4[q][j] = q == 0 || two ? *reinterpret_cast<const float4 *>(&p[b + q][j * 4]) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                        }
                        if (ok) ok = mbar_wait(&S.acc_full[team][acc.i], acc.parity, abort);
                        ok = __all_sync(0xffffffffu, ok);
                        if (!ok) break;
                        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                        auto add = [&](float2 *to, const float *v, const float4 &s) {
                            to[0] = __ffma2_rn(make_float2(v[0], v[1]), make_float2(s.x, s.y), to[0]);
                            to[1] = __ffma2_rn(make_float2(v[2], v[3]), make_float2(s.z, s.w), to[1]);
                        };
                        if constexpr (W < 32) {
                            float v[2][W];
                            gmm_ld(from, two ? from + TN : from, v);
#pragma unroll
                            for (int q = 0; q < 2; q++)
                                if (q == 0 || two) {
#pragma unroll
                                    for (int j = 0; j < W / 4; j++) add(&f[j * 2], &v[q][j * 4], s4[q][j]);
                                }
                        } else {
#pragma unroll
                            for (int c = 0; c < C::kChunks; c++) {
                                const int c0 = (c_first + c_step * c) * 32;
                                if (c0 >= I.nt) continue;
#pragma unroll
                                for (int q = 0; q < (F8 ? C::kSub : 1); q++) {
                                    if (q && !two) break;
                                    float v[32];
                                    gmm_ld(from + q * TN + c_step * c * 32, v);
#pragma unroll
                                    for (int j = 0; j < 8; j++) {
                                        float2 *to = &f[c * 16 + j * 2];
                                        if (F8) {
                                            add(to, &v[j * 4], *reinterpret_cast<const float4 *>(&p[b + q][c0 + j * 4]));
                                        } else {
                                            to[0] = __fadd2_rn(make_float2(v[j * 4], v[j * 4 + 1]), to[0]);
                                            to[1] = __fadd2_rn(make_float2(v[j * 4 + 2], v[j * 4 + 3]), to[1]);
                                        }
                                    }
                                }
                            }
                        }
                        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                        __syncwarp();
                        if (acc.i % C::kGroup == C::kGroup - 1 && lane == 0) mbar_arrive(&S.acc_empty[team][acc.i / C::kGroup]);
                        acc.next();
                    }
                    if (!ok) break;
                    if (F8) {
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&S.staged.p_empty[team][ps.i]);
                        ps.next();
                    }
                }
            };
            if (F8 && TN <= 32 && I.nt <= 8) fold(std::integral_constant<int, 8>());
            else if (F8 && TN <= 32 && I.nt <= 16) fold(std::integral_constant<int, 16>());
            else fold(std::integral_constant<int, 32>());
            if (ok) ok = mbar_wait(&S.staged.to_full[team][ts.i], ts.parity, abort);
            ok = __all_sync(0xffffffffu, ok);
            const GmmTo(&tos)[TN] = S.staged.to[team][ts.i];
            const int col = I.rb * GM + sub * 32 + lane;
            if (ok && col < A.n) {
                auto write = [&](auto zero) {
                    using T = decltype(zero);
#pragma unroll
                    for (int j8 = 0; j8 < C::kChunks * 4; j8++) {
                        const int t = (c_first + c_step * (j8 >> 2)) * 32 + (j8 & 3) * 8;
                        if (t >= I.nt) continue;
                        asm volatile("" ::: "memory");  // eight targets at a time, or they take the registers of all
#pragma unroll
                        for (int j = 0; j < 8; j++) gmm_put<T>(tos[t + j], col, (j & 1) ? f[j8 * 4 + (j >> 1)].y : f[j8 * 4 + (j >> 1)].x);
                    }
                };
                if (A.out_type == INZG_T_F32) write(0.0f);
                else if (A.out_type == INZG_T_BF16) write(__nv_bfloat16());
                else write(__half());
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&S.staged.to_empty[team][ts.i]);
            ts.next();
        }
        if (!ok) S.abort = 1;
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (S.abort && threadIdx.x == 0) atomicCAS(A.err, kErrNone, kErrTimeout);
    if (warp == 1) gmm_tmem_free(tmem);
}

// ---------------------------------------------------------------------------------------------------------------------

bool gmm_map(CUtensorMap *m, const void *base, int elem, int64_t rows, int64_t k, int64_t ld, int box_rows) {
    static const auto fn = [] {
        cudaDriverEntryPointQueryResult q;
        void *p = nullptr;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess ||
            q != cudaDriverEntryPointSuccess)
            p = nullptr;
        return reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
    }();
    if (!fn) return false;
    const cuuint64_t dims[2] = {(cuuint64_t)k, (cuuint64_t)rows};
    const cuuint64_t strides[1] = {(cuuint64_t)(ld * elem)};
    const cuuint32_t box[2] = {(cuuint32_t)(kGmmBytes / elem), (cuuint32_t)box_rows};
    const cuuint32_t estr[2] = {1, 1};
    return fn(m, elem == 1 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_UINT16, 2, const_cast<void *>(base),
              dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
              CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int TN>
constexpr size_t gmm_smem() {
    return (size_t)GmmCfg<TN>::kStages * GmmCfg<TN>::kStage + sizeof(GmmShared<TN>) + 1024;
}
// more than half of an SM's shared memory, so that a CTA is alone on its SM with all of TMEM
static_assert(gmm_smem<32>() <= 227 * 1024 && gmm_smem<32>() > 116 * 1024, "one CTA per SM");
static_assert(gmm_smem<128>() <= 227 * 1024 && gmm_smem<128>() > 116 * 1024, "one CTA per SM");
static bool g_wide_ok = false, g_large_ok = false;  // the kernels with a register split may be launched

void gmm_set_attributes() {
    cudaFuncSetAttribute(gmm_kernel<true, 32>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)gmm_smem<32>());
    cudaFuncSetAttribute(gmm_kernel<false, 32>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)gmm_smem<32>());
    g_wide_ok = cudaFuncSetAttribute(gmm_kernel<false, 128>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)gmm_smem<128>()) ==
                    cudaSuccess &&
                gmm_split_holds(gmm_kernel<false, 128>);
    g_large_ok = gmm_large_set_attributes();
}

template <bool F8, int TN>
static int gmm_launch(const inzg_grouped_matmul_args &G, const GmmArgs &A, int num_sms, cudaStream_t st) {
    constexpr int elem = F8 ? 1 : 2;
    const int64_t lda = G.lda ? G.lda : G.k, ldw = G.ldw ? G.ldw : G.k;
    CUtensorMap map_w, map_a16, map_a;
    if (!gmm_map(&map_w, G.w, elem, (int64_t)G.groups * G.n, G.k, ldw, GM) ||
        !gmm_map(&map_a16, G.a, elem, G.a_rows, G.k, lda, 16) || !gmm_map(&map_a, G.a, elem, G.a_rows, G.k, lda, TN))
        return -1;
    const int64_t tiles = std::min<int64_t>(G.entries, G.entries / TN + G.groups);  // at most so many
    const int grid = (int)std::min<int64_t>(num_sms, tiles * A.nrb);
    gmm_kernel<F8, TN><<<grid, kGmmThreads, gmm_smem<TN>(), st>>>(map_w, map_a16, map_a, A);
    return 1;
}

int launch_grouped_matmul(const inzg_grouped_matmul_args &G, int num_sms, int32_t *err, cudaStream_t st) {
    const int elem = G.type == INZG_T_E4M3 ? 1 : 2;
    GmmArgs A{};
    A.groups = G.groups;
    A.n = G.n;
    A.nrb = A.nrb128 = (G.n + GM - 1) / GM;
    A.steps = (int)(((int64_t)G.k * elem + kGmmBytes - 1) / kGmmBytes);
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
    A.a = static_cast<const uint8_t *>(G.a);
    A.lda_bytes = (G.lda ? G.lda : G.k) * elem;
    A.k_bytes = (int64_t)G.k * elem;
    A.out = G.out;
    A.ldo = G.ldo ? G.ldo : G.n;
    A.err = err;
    // fp32 accumulators; e4m3 (0), bf16 (1) or f16 (0) operands, both K-major; M = 128
    const uint32_t fmt = G.type == INZG_T_BF16 ? 1u : 0u;
    A.idesc = (1u << 4) | (fmt << 7) | (fmt << 10) | ((uint32_t)(GM >> 4) << 24);
    const bool small = inzg__grouped_matmul_tile(G.type, G.groups, G.entries, G.n, num_sms) == 32;
    if (G.type != INZG_T_E4M3) {
        if (small || !g_wide_ok) return gmm_launch<false, 32>(G, A, num_sms, st);
        return gmm_launch<false, 128>(G, A, num_sms, st);
    }
    if (small || !g_large_ok) return gmm_launch<true, 32>(G, A, num_sms, st);
    return gmm_large_launch(G, A, num_sms, st);
}

}  // namespace inzg
