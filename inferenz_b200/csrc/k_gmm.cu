// k_gmm.cu -- dense and grouped products of e4m3 rows with block scales, and of bf16 / f16 rows, on the 5th-generation
// tensor cores (tcgen05.mma kind::f8f6f4 / kind::f16), sm_100a (inzg_matmul_q8, inzg_grouped_matmul): the kernel for few
// entries per group, and the choice between it and the one for many (k_gmm_large.cu).
//
//   out[i][j] = scale_i * sum_b as[i][b] ws[j / 128][b] * (sum_{k in block b} a[i][k] w[g][j][k])
//
// The tensor core sums one block of 128 k in fp32 (TMEM); the block's two scales enter in the fold, which keeps the running
// sum in fp32 registers: f = fma(dot_b, as * ws, f). bf16 / f16 have no scales and stay in TMEM over the whole k.
//
// Work item: 128 rows of w (the MMA's M, one TMEM lane each) x up to TN entries of one group (its N, rounded up to
// 16). The weights are the M side because a decoding call has a row or two per expert: the MMA, the copies and the
// fold then shrink with the entries, while a weight tile is streamed once whatever their number. A tile of 128 rows
// of w has one weight scale per k block, so as * ws is formed once per entry and block and kept in shared memory.
//   warp 0      TMA producer: per 128-byte step of k a box of 128 weight rows and, unless they are gathered, the entries'
//               rows in boxes of 16 or TN rows, 128-byte swizzle
//   warp 1      allocates all 512 TMEM columns (4 accumulators per team), one lane issues 4 MMAs per stage
//   warps 2-3   the entries' rows by index
//   warps 4-11  fold and write, thread = a row of w. TN = 128: all eight warps share an item, every other 32 entries;
//               TN = 32: the two warpgroups take the items in turn, so one writes while the other folds
// Persistent: one CTA per SM walks the items; the offsets are turned into tile numbers by every CTA for itself, which
// costs a read of off and a scan instead of a launch. Every mbarrier wait is bounded; on expiry the CTA records an
// error, drains what it issued, frees its TMEM and returns.
#include <cudaTypedefs.h>

#include <algorithm>

#include "k_gmm.cuh"
#include "k_launch.h"

namespace inzg {

constexpr int GM = 128;      // weight rows of an item
constexpr int kGmmKc = 8;    // k blocks whose scales are staged at once

template <int TN>
struct GmmCfg {
    static constexpr int kTeams = TN <= 32 ? 2 : 1, kTeamWarps = 8 / kTeams, kTeamThreads = kTeamWarps * 32;
    static constexpr int kStages = TN <= 32 ? 10 : 6, kStage = (GM + TN) * kGmmBytes;
    static constexpr int kAcc = 4;                              // accumulators of TN columns, per team: a team waits for its
                                                                // own alone, so it is never two phases of one ahead
    static constexpr int kChunks = TN / 32 / (2 / kTeams);      // 32-entry chunks per thread
    static constexpr int kPre = kGmmKc * TN / kTeamThreads;     // staged scales per thread
    static constexpr int kParts = kGmmKc / kPre;                // threads per entry in the staging
};

// where an entry's result goes: its row of out (null: not written) and its weight
struct alignas(16) GmmTo {
    char *row;
    float w;
};

template <int TN>
struct GmmShared {
    using C = GmmCfg<TN>;
    uint64_t full[C::kStages], empty[C::kStages], acc_full[C::kTeams][C::kAcc], acc_empty[C::kTeams][C::kAcc], drain;
    uint32_t tmem_base;
    int abort, never;
    alignas(16) float p[C::kTeams][2][kGmmKc][TN];  // as * ws of the staged blocks
    GmmTo to[C::kTeams][2][TN];
    GmmWalk walk;
};

template <class T>
__device__ __forceinline__ void gmm_put(const GmmTo &t, int64_t col, float v) {
    T o;
    from_f32(v * t.w, o);
    if (t.row) reinterpret_cast<T *>(t.row)[col] = o;
}

// map_w: [groups * n][k] in 128-row boxes; map_a16 / map_a: the rows of a in boxes of 16 / TN rows
template <bool F8, int TN>
__global__ void __launch_bounds__(kGmmThreads, 1)
gmm_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_a16,
           const __grid_constant__ CUtensorMap map_a, const __grid_constant__ GmmArgs A) {
    using C = GmmCfg<TN>;
    constexpr int ST = C::kStages, NA = C::kAcc;
    extern __shared__ __align__(1024) uint8_t gmm_dyn[];
    uint8_t *ring = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(gmm_dyn) + 1023) & ~uintptr_t(1023));
    GmmShared<TN> &S = *reinterpret_cast<GmmShared<TN> *>(ring + ST * C::kStage);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    volatile int *abort = &S.abort;
    volatile int *never = &S.never;
    constexpr int kElem = F8 ? 1 : 2;

    if (threadIdx.x == 0) {
        for (int s = 0; s < ST; s++) {
            mbar_init(&S.full[s], A.in_rows ? 1 + kGmmGatherWarps : 1);
            mbar_init(&S.empty[s], 1);
        }
        for (int t = 0; t < C::kTeams; t++)
            for (int b = 0; b < NA; b++) {
                mbar_init(&S.acc_full[t][b], 1);
                mbar_init(&S.acc_empty[t][b], C::kTeamWarps);
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
    gmm_walk_init<TN>(S.walk, A);
    const int nitems = S.walk.bad ? 0 : S.walk.tstart[A.groups] * A.nrb;
    if (S.walk.bad && threadIdx.x == 0) atomicCAS(A.err, kErrNone, kErrOverflow);
    const int steps = A.steps;

    if (warp == 0) {
        // ---------------- TMA producer ----------------
        int kg = 0;  // stages issued by this CTA
        bool ok = true;
        for (int item = blockIdx.x; item < nitems && ok; item += gridDim.x) {
            const GmmItem I = gmm_item<TN>(S.walk, A.groups, A.nrb, item);
            const int n16 = (I.nt + 15) & ~15;
            const bool whole = I.nt > TN / 2;
            const uint32_t bytes = (GM + (A.in_rows ? 0 : whole ? TN : n16)) * kGmmBytes;
            for (int k = 0; k < steps; k++, kg++) {
                const int s = kg % ST, x = k * (kGmmBytes / kElem);
                if (kg >= ST) ok = mbar_wait(&S.empty[s], ((kg / ST) - 1) & 1, abort);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                uint8_t *stage = ring + s * C::kStage;
                if (lane == 0) {
                    mbar_expect_tx(&S.full[s], bytes);
                    tma_load_2d(stage, &map_w, x, I.g * A.n + I.rb * GM, &S.full[s]);
                    if (!A.in_rows && whole) tma_load_2d(stage + GM * kGmmBytes, &map_a, x, I.base, &S.full[s]);
                }
                __syncwarp();
                if (!A.in_rows && !whole && lane * 16 < n16)
                    tma_load_2d(stage + (GM + lane * 16) * kGmmBytes, &map_a16, x, I.base + lane * 16, &S.full[s]);
            }
        }
        if (!ok) S.abort = 1;
        // every issued copy has landed before the CTA may leave (bounded; each slot's latest phase)
        for (int k = max(0, kg - ST); k < kg; k++) mbar_wait(&S.full[k % ST], (k / ST) & 1, never);
    } else if (warp == 1) {
        // ---------------- MMA issuer ----------------
        if (lane == 0) {
            bool ok = true;
            int kg = 0, it = 0;  // stages consumed, items begun by this CTA
            for (int item = blockIdx.x; item < nitems && ok; item += gridDim.x, it++) {
                const int team = it % C::kTeams;
                int bg = it / C::kTeams * (F8 ? steps : 1);  // accumulators handed to this team so far
                const GmmItem I = gmm_item<TN>(S.walk, A.groups, A.nrb, item);
                const uint32_t idesc = A.idesc | (uint32_t)(((I.nt + 15) & ~15) >> 3) << 17;
                for (int k = 0; k < steps; k++, kg++) {
                    const int s = kg % ST, buf = bg % NA;
                    const bool open = F8 || k == 0, close = F8 || k == steps - 1;
                    if (open && bg >= NA && !mbar_wait(&S.acc_empty[team][buf], ((bg / NA) - 1) & 1, abort)) { ok = false; break; }
                    if (!mbar_wait(&S.full[s], (kg / ST) & 1, abort)) { ok = false; break; }
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    const uint8_t *stage = ring + s * C::kStage;
                    const uint64_t da = gmm_desc(stage), db = gmm_desc(stage + GM * kGmmBytes);
#pragma unroll
                    for (int j = 0; j < kGmmBytes / 32; j++)  // 32 bytes of k per MMA
                        gmm_mma<F8>(tmem + (team * NA + buf) * TN, da + (uint64_t)(j * 2), db + (uint64_t)(j * 2), idesc, !(open && j == 0));
                    gmm_commit(&S.empty[s]);
                    if (close) {
                        gmm_commit(&S.acc_full[team][buf]);
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
    } else if (warp < 4) {
        if (A.in_rows && !gmm_gather<TN, ST>(S.walk, A, nitems, ring, C::kStage, GM * kGmmBytes, S.full, S.empty, abort))
            S.abort = 1;
    } else {
        // ---------------- fold and write ----------------
        // TMEM lane quadrant = warp % 4. One team: warps 4-7 take the even 32-entry chunks of every item, warps 8-11 the
        // odd ones; two teams: each takes every other item whole.
        const int sub = warp & 3, upper = (warp - 4) >> 2;
        const int team = C::kTeams == 2 ? upper : 0, c_first = C::kTeams == 2 ? 0 : upper, c_step = C::kTeams == 2 ? 1 : 2;
        const int et = (threadIdx.x - 128) % C::kTeamThreads;
        const int esize = A.out_type == INZG_T_F32 ? 4 : 2;
        bool ok = true;  // a thread whose wait ran out goes on without waiting or writing: the team's barriers stay matched
        const int nkc = F8 ? (steps + kGmmKc - 1) / kGmmKc : 1, accs = F8 ? steps : 1;
        const int pe = et / C::kParts, pk = (et % C::kParts) * C::kPre;  // staging: entry, first of its blocks
        float pre[C::kPre];
        // what the next item needs is loaded while the current one folds: the rows behind its entries first, the scales of its
        // first blocks once those are there
        int row = 0;
        GmmTo to{nullptr, 0.0f};
        bool bad_row = false;
        auto load_entry = [&](const GmmItem &I) {
            if (F8) {
                const int i = I.base + min(pe, I.nt - 1);
                const int v = A.in_rows ? A.in_rows[i] : i;
                row = (unsigned)v < (unsigned)A.a_rows ? v : 0;
            }
            to.row = nullptr;
            if (et < I.nt) {
                const int i = I.base + et;
                const int o = A.out_rows ? A.out_rows[i] : i;
                bad_row = (unsigned)o >= (unsigned)A.out_rows_n || (A.in_rows && (unsigned)A.in_rows[i] >= (unsigned)A.a_rows);
                if (!bad_row) to.row = static_cast<char *>(A.out) + (int64_t)o * A.ldo * esize;
                to.w = A.out_scale ? A.out_scale[i] : 1.0f;
            }
        };
        auto load_scales = [&](const GmmItem &I, int kc) {
            const float *as = A.as + (int64_t)row * A.ldas;
            const float *ws = A.ws + ((int64_t)I.g * A.nrb128 + I.rb) * steps;
#pragma unroll
            for (int j = 0; j < C::kPre; j++) {
                const int b = kc * kGmmKc + pk + j;
                pre[j] = b < steps && pe < I.nt ? __ldg(as + b) * __ldg(ws + b) : 0.0f;
            }
        };
        const int first = blockIdx.x + team * gridDim.x, stride = C::kTeams * gridDim.x;
        GmmItem I{0, 0, 0, 0}, N{0, 0, 0, 0};
        if (first < nitems) {
            N = gmm_item<TN>(S.walk, A.groups, A.nrb, first);
            load_entry(N);
            if (F8) load_scales(N, 0);
        }
        int it = 0, cbuf = 0;  // items of this team, chunks of scales staged so far
        for (int item = first; item < nitems; item += stride, it++) {
            I = N;
            const bool more = item + stride < nitems;
            GmmTo(&tos)[TN] = S.to[team][it & 1];
            if (et < TN) tos[et] = to;
            if (bad_row) atomicCAS(A.err, kErrNone, kErrBadSlot);
            bad_row = false;
            const int bg0 = it * accs;  // accumulators of this team before this item
            float2 f[C::kChunks * 16];
#pragma unroll
            for (int j = 0; j < C::kChunks * 16; j++) f[j] = make_float2(0.0f, 0.0f);
            for (int kc = 0; kc < nkc; kc++, cbuf++) {
                float(&p)[kGmmKc][TN] = S.p[team][cbuf & 1];
                if (F8)
#pragma unroll
                    for (int j = 0; j < C::kPre; j++) p[pk + j][pe] = pre[j];
                asm volatile("bar.sync %0, %1;" ::"r"(1 + team), "n"(C::kTeamThreads) : "memory");
                if (F8 && kc + 1 < nkc) load_scales(I, kc + 1);
                if (more && kc + 1 == nkc) {  // before that `row` still serves this item's later chunks
                    N = gmm_item<TN>(S.walk, A.groups, A.nrb, item + stride);
                    load_entry(N);
                }
                const int nb = F8 ? min(kGmmKc, steps - kc * kGmmKc) : 1;
                for (int b = 0; b < nb; b++) {
                    const int bg = bg0 + kc * kGmmKc + b, buf = bg % NA;
                    if (ok && !mbar_wait(&S.acc_full[team][buf], (bg / NA) & 1, abort)) ok = false;
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    ok = __all_sync(0xffffffffu, ok);
                    if (ok) {
#pragma unroll
                        for (int c = 0; c < C::kChunks; c++) {
                            const int c0 = (c_first + c_step * c) * 32;
                            if (c0 >= I.nt) continue;
                            float v[32];
                            gmm_ld32(tmem + ((uint32_t)(sub * 32) << 16) + (team * NA + buf) * TN + c0, v);
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
                    if (lane == 0) mbar_arrive(&S.acc_empty[team][buf]);
                }
                if (F8 && more && kc + 1 == nkc) load_scales(N, 0);
            }
            const int col = I.rb * GM + sub * 32 + lane;
            if (ok && col < A.n) {
                auto write = [&](auto zero) {
                    using T = decltype(zero);
#pragma unroll
                    for (int j8 = 0; j8 < C::kChunks * 4; j8++) {
                        const int t = (c_first + c_step * (j8 >> 2)) * 32 + (j8 & 3) * 8;
                        if (t >= I.nt) continue;
#pragma unroll
                        for (int j = 0; j < 8; j++) gmm_put<T>(tos[t + j], col, (j & 1) ? f[j8 * 4 + (j >> 1)].y : f[j8 * 4 + (j >> 1)].x);
                    }
                };
                if (A.out_type == INZG_T_F32) write(0.0f);
                else if (A.out_type == INZG_T_BF16) write(__nv_bfloat16());
                else write(__half());
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
static_assert(gmm_smem<32>() <= 227 * 1024 && gmm_smem<128>() <= 227 * 1024, "shared memory of one CTA");

void gmm_set_attributes() {
    cudaFuncSetAttribute(gmm_kernel<true, 32>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)gmm_smem<32>());
    cudaFuncSetAttribute(gmm_kernel<false, 32>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)gmm_smem<32>());
    cudaFuncSetAttribute(gmm_kernel<true, 128>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)gmm_smem<128>());
    cudaFuncSetAttribute(gmm_kernel<false, 128>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)gmm_smem<128>());
    gmm_large_set_attributes();
}

template <int TN>
static int gmm_launch(const inzg_grouped_matmul_args &G, const GmmArgs &A, int num_sms, cudaStream_t st) {
    const bool f8 = G.type == INZG_T_E4M3;
    const int elem = f8 ? 1 : 2;
    const int64_t lda = G.lda ? G.lda : G.k, ldw = G.ldw ? G.ldw : G.k;
    CUtensorMap map_w, map_a16, map_a;
    if (!gmm_map(&map_w, G.w, elem, (int64_t)G.groups * G.n, G.k, ldw, GM) ||
        !gmm_map(&map_a16, G.a, elem, G.a_rows, G.k, lda, 16) || !gmm_map(&map_a, G.a, elem, G.a_rows, G.k, lda, TN))
        return -1;
    const int64_t tiles = std::min<int64_t>(G.entries, G.entries / TN + G.groups);  // at most so many
    const int grid = (int)std::min<int64_t>(num_sms, tiles * A.nrb);
    if (f8) gmm_kernel<true, TN><<<grid, kGmmThreads, gmm_smem<TN>(), st>>>(map_w, map_a16, map_a, A);
    else gmm_kernel<false, TN><<<grid, kGmmThreads, gmm_smem<TN>(), st>>>(map_w, map_a16, map_a, A);
    return 1;
}

// Many entries per group: the product is bound by the tensor pipe and the fold, and the kernel with 128 x 256 tiles is
// the faster one.
static bool gmm_use_large(const inzg_grouped_matmul_args &G) { return G.entries >= 256 * (int64_t)G.groups; }

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
    if (gmm_use_large(G)) return gmm_large_launch(G, A, num_sms, st);
    if (G.entries <= 16 * (int64_t)G.groups) return gmm_launch<32>(G, A, num_sms, st);
    return gmm_launch<128>(G, A, num_sms, st);
}

}  // namespace inzg
