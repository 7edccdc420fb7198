// k_gmm.cuh -- what the grouped product's kernels share: arguments, tcgen05 primitives, the walk over tiles, the gathering
// producer, sm_100a.
#pragma once

#include <cuda.h>

#include "inzg_internal.h"
#include "k_async.cuh"
#include "k_q8.cuh"

namespace inzg {

constexpr int kGmmBytes = 128;    // bytes of k per ring stage: one swizzle row, one scale block of e4m3
constexpr int kGmmThreads = 384;  // warp 0 TMA, warp 1 MMA, warps 2-3 gather, warps 4-11 fold and write
constexpr int kGmmGatherWarps = 2;

struct GmmArgs {
    int groups, n, nrb, nrb128, steps, entries, a_rows, out_rows_n, out_type, wide_out;
    const int32_t *off, *in_rows, *out_rows;  // off null: one group of all entries
    const float *out_scale, *as, *ws;
    const uint8_t *a;  // read directly where rows are gathered
    int64_t lda_bytes, k_bytes, ldas, ldo;
    void *out;
    uint32_t idesc;  // without N
    int32_t *err;
};

// the offsets and each group's first tile, in every CTA's shared memory
struct GmmWalk {
    int bad;
    int wsum[kGmmThreads / 32];
    int tstart[INZG_MAX_GROUPS + 1];
    int off[INZG_MAX_GROUPS + 1];
};

// an item of the walk: entries [base, base + nt) of group g against row block rb of its weights
struct GmmItem {
    int g, base, nt, rb;
};

// Tile numbers from the offsets, by the whole block (bad set to 0 and a barrier passed before): a thread counts the tiles of
// `per` neighbouring groups, then a scan over the block. Ends with a barrier.
template <int TILE>
__device__ __forceinline__ void gmm_walk_init(GmmWalk &W, const GmmArgs &A) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int per = (A.groups + kGmmThreads - 1) / kGmmThreads, g0 = threadIdx.x * per, g1 = min(g0 + per, A.groups);
    int mine = 0;
    for (int g = g0; g < g1; g++) {
        const int o0 = A.off ? A.off[g] : 0, o1 = A.off ? A.off[g + 1] : A.entries;
        if (o0 < 0 || o1 < o0 || o1 > A.entries) W.bad = 1;
        else mine += (o1 - o0 + TILE - 1) / TILE;
        W.off[g] = o0;
        if (g == A.groups - 1) W.off[g + 1] = o1;
    }
    int scan = mine;
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
        const int v = __shfl_up_sync(0xffffffffu, scan, d);
        if (lane >= d) scan += v;
    }
    if (lane == 31) W.wsum[warp] = scan;
    __syncthreads();
    int first = scan - mine;
    for (int k = 0; k < warp; k++) first += W.wsum[k];
    if (!W.bad)
        for (int g = g0; g < g1; g++) {
            W.tstart[g] = first;
            first += (W.off[g + 1] - W.off[g] + TILE - 1) / TILE;
            if (g == A.groups - 1) W.tstart[g + 1] = first;
        }
    __syncthreads();
}

template <int TILE>
__device__ __forceinline__ GmmItem gmm_item(const GmmWalk &W, int groups, int nrb, int item) {
    const int tile = item / nrb;
    int lo = 0, hi = groups;  // the last group whose first tile is not past `tile`; empty groups share a first tile
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (W.tstart[mid] <= tile) lo = mid;
        else hi = mid;
    }
    GmmItem I;
    I.g = lo;
    I.base = W.off[lo] + (tile - W.tstart[lo]) * TILE;
    I.nt = min(TILE, W.off[lo + 1] - I.base);
    I.rb = item - tile * nrb;
    return I;
}

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

// TMEM of the CTA (all 512 columns) by one warp; the address lands in *base
__device__ __forceinline__ void gmm_tmem_alloc(uint32_t *base) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(base)));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
}
__device__ __forceinline__ void gmm_tmem_free(uint32_t tmem) {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem));
}

// The entries' rows by index: warps 2-3 copy 16 bytes per thread and step (cp.async, zeros behind k) into the places that a
// tiled copy with 128-byte swizzle would fill, and arrive on the stage's barrier (one arrival per warp) once the copies of
// LAG stages earlier have landed and are fenced for the tensor core's reads. tile::gather4 would need no warps, but moved
// only four rows in some 70 ns: 225 us at 333 bf16 tokens (52 rows a tile) against 90 us with neighbouring rows.
// Returns false when a wait ran out. ROWS: rows of a tile; b_off: the rows' place in a stage.
template <int ROWS, int STAGES>
__device__ __forceinline__ bool gmm_gather(const GmmWalk &W, const GmmArgs &A, int nitems, uint8_t *ring, int stage_bytes,
                                           int b_off, uint64_t *full, uint64_t *empty, volatile int *abort) {
    constexpr int LAG = 2, PER = ROWS * 8 / (kGmmGatherWarps * 32);  // 16-byte pieces of a stage per thread
    static_assert(LAG < STAGES && PER >= 1, "gather pipeline");
    const int tid = threadIdx.x - 64, lane = threadIdx.x & 31;
    const int piece = tid & 7, row0 = tid >> 3;  // this thread: piece `piece` of rows row0, row0 + 8, ...
    int kg = 0;
    bool ok = true;
    for (int item = blockIdx.x; item < nitems && ok; item += gridDim.x) {
        const GmmItem I = gmm_item<ROWS>(W, A.groups, A.nrb, item);
        const int n16 = (I.nt + 15) & ~15;
        const uint8_t *src[PER];
#pragma unroll
        for (int j = 0; j < PER; j++) {
            const int v = A.in_rows[I.base + min(row0 + j * 8, I.nt - 1)];
            // a bad index reads row 0; the fold neither writes that entry nor stays silent about it
            src[j] = A.a + ((unsigned)v < (unsigned)A.a_rows ? v : 0) * A.lda_bytes + piece * 16;
        }
        for (int k = 0; k < A.steps; k++, kg++) {
            const int s = kg % STAGES;
            if (kg >= STAGES) ok = mbar_wait(&empty[s], ((kg / STAGES) - 1) & 1, abort);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            const int64_t at = (int64_t)k * kGmmBytes;
            const int64_t left = A.k_bytes - at - piece * 16;
            const int size = left >= 16 ? 16 : left > 0 ? (int)left : 0;
            const int64_t from = size ? at : -(int64_t)piece * 16;  // nothing is read then: stay inside the row
            const uint32_t dst = smem_u32(ring + s * stage_bytes + b_off);
#pragma unroll
            for (int j = 0; j < PER; j++) {
                const int row = row0 + j * 8;
                if (row < n16)
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst + row * 128 + ((piece ^ (row & 7)) << 4)),
                                 "l"(src[j] + from), "r"(size)
                                 : "memory");
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
            if (kg >= LAG) {
                asm volatile("cp.async.wait_group %0;" ::"n"(LAG) : "memory");
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(&full[(kg - LAG) % STAGES]);
            }
        }
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0)
        for (int k = max(0, kg - LAG); k < kg; k++) mbar_arrive(&full[k % STAGES]);
    return ok;
}

// 2-D tensor map over [rows][k] with a row pitch of ld elements, boxes of box_rows x 128 bytes, 128-byte swizzle; what lies
// outside reads as zeros. False when the driver refuses it.
bool gmm_map(CUtensorMap *m, const void *base, int elem, int64_t rows, int64_t k, int64_t ld, int box_rows);

// The two kernels' launchers (k_gmm.cu, k_gmm_large.cu): A holds everything but nrb and the tile-dependent bits
void gmm_large_set_attributes();
int gmm_large_launch(const inzg_grouped_matmul_args &G, GmmArgs A, int num_sms, cudaStream_t st);

}  // namespace inzg
