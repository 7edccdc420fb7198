// k_gmm.cuh -- what the grouped product's kernels share: arguments, tcgen05 primitives, the walk over tiles, the gathering
// producer, sm_100a.
#pragma once

#include <cuda.h>

#include "inzg_internal.h"
#include "k_async.cuh"
#include "k_q8.cuh"

namespace inzg {

constexpr int kGmmBytes = 128;    // bytes of k per ring stage: one swizzle row, one scale block of e4m3
constexpr int kGmmRing = 2;              // staged chunks of scales, and staged items, per team

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

// an item of the walk: entries [base, base + nt) of group g against row block rb of its weights
struct alignas(16) GmmItem {
    int g, base, nt, rb;
};

// each group's first tile and the CTA's first items, in every CTA's shared memory
constexpr int kGmmList = 512;
struct GmmWalk {
    int wsum[16];
    int tstart[INZG_MAX_GROUPS + 1];
    GmmItem list[kGmmList];
};

template <int TILE>
__device__ __forceinline__ GmmItem gmm_search(const GmmWalk &W, const GmmArgs &A, int item) {
    const int tile = item / A.nrb;
    int lo = 0, hi = A.groups;  // the last group whose first tile is not past `tile`; empty groups share a first tile
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (W.tstart[mid] <= tile) lo = mid;
        else hi = mid;
    }
    GmmItem I;
    I.g = lo;
    I.base = (A.off ? A.off[lo] : 0) + (tile - W.tstart[lo]) * TILE;
    I.nt = min(TILE, (A.off ? A.off[lo + 1] : A.entries) - I.base);
    I.rb = item - tile * A.nrb;
    return I;
}

// the CTA's n-th item, `item` of all (n counts from 0). The search takes some 1100 cycles, an item of a short k 5000: the first
// items are listed at the start, later ones (a CTA seldom has that many) searched for by each role for itself.
template <int TILE>
__device__ __forceinline__ GmmItem gmm_item(const GmmWalk &W, const GmmArgs &A, int item, int n) {
    if (n < kGmmList) return W.list[n];
    return gmm_search<TILE>(W, A, item);
}

// What a thread needs of the offsets: its groups are g0, g0 + 1, ..., their first entries o[0], o[1], ...
template <int THREADS>
struct GmmOffsets {
    static constexpr int kMost = (INZG_MAX_GROUPS + THREADS - 1) / THREADS;
    int g0, count, o[kMost + 1];
    __device__ __forceinline__ explicit GmmOffsets(const GmmArgs &A) {
        const int per = (A.groups + THREADS - 1) / THREADS;
        g0 = threadIdx.x * per;
        count = max(0, min(per, A.groups - g0));
        o[0] = 0;
#pragma unroll
        for (int j = 0; j <= kMost; j++)
            if (j <= count && count) o[j] = A.off ? __ldg(A.off + g0 + j) : j ? A.entries : 0;
    }
};

// Tile numbers from the offsets, by the whole block: a thread counts the tiles of its groups, a scan over the block numbers them,
// and the thread enters those of its items that are the CTA's (first, first + stride, ...) in the CTA's list. Returns the number of
// items of all CTAs, 0 when the offsets are bad. Against a search for each of the CTA's items after the scan, and with the offsets
// on their way during the setup, 1 token of top-10 of 512 takes 11.5 us instead of 12.2. What the block's threads wrote to shared memory before is seen by all afterwards.
template <int TILE, int THREADS>
__device__ __forceinline__ int gmm_walk_init(GmmWalk &W, const GmmArgs &A, const GmmOffsets<THREADS> &O, int first, int stride) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    auto tiles_of = [&](int j) { return (O.o[j + 1] - O.o[j] + TILE - 1) / TILE; };
    bool bad = false;
    int mine = 0;
#pragma unroll
    for (int j = 0; j < O.kMost; j++)
        if (j < O.count) {
            if (O.o[j] < 0 || O.o[j + 1] < O.o[j] || O.o[j + 1] > A.entries) bad = true;
            else mine += tiles_of(j);
        }
    int scan = mine;
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
        const int v = __shfl_up_sync(0xffffffffu, scan, d);
        if (lane >= d) scan += v;
    }
    if (lane == 31) W.wsum[warp] = scan;
    if (__syncthreads_or(bad)) {
        if (threadIdx.x == 0) atomicCAS(A.err, kErrNone, kErrOverflow);
        return 0;
    }
    int at = scan - mine, all = 0;
#pragma unroll
    for (int k = 0; k < THREADS / 32; k++) {
        const int v = W.wsum[k];
        if (k < warp) at += v;
        all += v;
    }
    if (threadIdx.x == 0) W.tstart[A.groups] = all;
    const int dt = stride / A.nrb, dr = stride - dt * A.nrb;
#pragma unroll
    for (int j = 0; j < O.kMost; j++)
        if (j < O.count) {
            const int tiles = tiles_of(j), lo = at * A.nrb;
            W.tstart[O.g0 + j] = at;
            if (tiles) {
                int n = lo > first ? (lo - first + stride - 1) / stride : 0;
                const int skip = first + n * stride - lo;
                int t = skip / A.nrb, rb = skip - t * A.nrb;
                for (; t < tiles && n < kGmmList; n++, t += dt, rb += dr) {
                    if (rb >= A.nrb) {
                        rb -= A.nrb;
                        if (++t >= tiles) break;
                    }
                    GmmItem I;
                    I.g = O.g0 + j;
                    I.base = O.o[j] + t * TILE;
                    I.nt = min(TILE, O.o[j + 1] - I.base);
                    I.rb = rb;
                    W.list[n] = I;
                }
            }
            at += tiles;
        }
    __syncthreads();
    return all * A.nrb;
}

// One lane of a converged warp. The producer and the MMA warp run their whole loops under this predicate: the compiler then
// knows that one thread is active and keeps the operands in uniform registers. Four MMAs of N = 16 and two commits take
// 156 cycles that way, 240 with an election per stage, 271 under `lane == 0` (measured alone; 512 at N = 256 either way).
__device__ __forceinline__ bool gmm_elect() {
    uint32_t p;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
    return p != 0;
}

// a position in a ring of N barriers: slot and the parity of its current round
template <int N>
struct GmmSlot {
    int i = 0;
    uint32_t parity = 0;
    __device__ __forceinline__ void next() {
        if (++i == N) {
            i = 0;
            parity ^= 1;
        }
    }
};

// the four 32-byte steps of one 128-byte stage; `fresh`: the accumulator's first
template <bool F8>
__device__ __forceinline__ void gmm_mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc);
template <bool F8>
__device__ __forceinline__ void gmm_mma_stage(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool fresh) {
#pragma unroll
    for (int j = 0; j < kGmmBytes / 32; j++) gmm_mma<F8>(d, a + (uint64_t)(j * 2), b + (uint64_t)(j * 2), idesc, !(fresh && j == 0));
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

// as many columns of the warp's 32 TMEM lanes as v has places
__device__ __forceinline__ void gmm_ld(uint32_t taddr, float (&v)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]), "=f"(v[8]),
          "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15]), "=f"(v[16]),
          "=f"(v[17]), "=f"(v[18]), "=f"(v[19]), "=f"(v[20]), "=f"(v[21]), "=f"(v[22]), "=f"(v[23]), "=f"(v[24]),
          "=f"(v[25]), "=f"(v[26]), "=f"(v[27]), "=f"(v[28]), "=f"(v[29]), "=f"(v[30]), "=f"(v[31])
        : "r"(taddr)
        : "memory");
}

// the first columns of two accumulators
__device__ __forceinline__ void gmm_ld(uint32_t first, uint32_t second, float (&v)[2][8]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%16];\n\t"
        "tcgen05.ld.sync.aligned.32x32b.x8.b32 {%8,%9,%10,%11,%12,%13,%14,%15}, [%17];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : "=f"(v[0][0]), "=f"(v[0][1]), "=f"(v[0][2]), "=f"(v[0][3]), "=f"(v[0][4]), "=f"(v[0][5]), "=f"(v[0][6]), "=f"(v[0][7]),
          "=f"(v[1][0]), "=f"(v[1][1]), "=f"(v[1][2]), "=f"(v[1][3]), "=f"(v[1][4]), "=f"(v[1][5]), "=f"(v[1][6]), "=f"(v[1][7])
        : "r"(first), "r"(second)
        : "memory");
}

__device__ __forceinline__ void gmm_ld(uint32_t first, uint32_t second, float (&v)[2][16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%32];\n\t"
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%33];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : "=f"(v[0][0]), "=f"(v[0][1]), "=f"(v[0][2]), "=f"(v[0][3]), "=f"(v[0][4]), "=f"(v[0][5]), "=f"(v[0][6]), "=f"(v[0][7]), "=f"(v[0][8]), "=f"(v[0][9]), "=f"(v[0][10]), "=f"(v[0][11]), "=f"(v[0][12]), "=f"(v[0][13]), "=f"(v[0][14]), "=f"(v[0][15]),
          "=f"(v[1][0]), "=f"(v[1][1]), "=f"(v[1][2]), "=f"(v[1][3]), "=f"(v[1][4]), "=f"(v[1][5]), "=f"(v[1][6]), "=f"(v[1][7]), "=f"(v[1][8]), "=f"(v[1][9]), "=f"(v[1][10]), "=f"(v[1][11]), "=f"(v[1][12]), "=f"(v[1][13]), "=f"(v[1][14]), "=f"(v[1][15])
        : "r"(first), "r"(second)
        : "memory");
}

// where an entry's result goes: its row of out (null: not written) and its weight
struct alignas(16) GmmTo {
    char *row;
    float w;
};

// What the fold needs beside the accumulators, staged ahead by two warps: per chunk of KC k blocks the factors as * ws of
// every entry (PLANES: one per 128 rows of w in the item), per item where the entries' results go. A ring per team; a team
// waits for its own slots alone and is never two phases of one ahead.
template <int TN, int TEAMS, int PLANES, int KC>
struct GmmStaged {
    uint64_t p_full[TEAMS][kGmmRing], p_empty[TEAMS][kGmmRing], to_full[TEAMS][kGmmRing], to_empty[TEAMS][kGmmRing];
    alignas(16) float p[TEAMS][kGmmRing][PLANES][KC][TN];
    GmmTo to[TEAMS][kGmmRing][TN];
};

template <int TN>
constexpr int gmm_stagers() {  // staging warps: each has half of the entries
    return TN > 32 ? 2 : 1;
}

template <int TN, int TEAMS, int PLANES, int KC>
__device__ __forceinline__ void gmm_staged_init(GmmStaged<TN, TEAMS, PLANES, KC> &T) {  // by one thread
    for (int t = 0; t < TEAMS; t++)
        for (int i = 0; i < kGmmRing; i++) {
            mbar_init(&T.p_full[t][i], gmm_stagers<TN>());
            mbar_init(&T.p_empty[t][i], 8 / TEAMS);
            mbar_init(&T.to_full[t][i], gmm_stagers<TN>());
            mbar_init(&T.to_empty[t][i], 8 / TEAMS);
        }
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

// The entries' rows by index: WARPS warps copy 16 bytes per thread and step (cp.async, zeros behind k) into the places that a
// tiled copy with 128-byte swizzle would fill, and arrive on the stage's barrier (one arrival per warp) once the copies of
// LAG stages earlier have landed and are fenced for the tensor core's reads. tile::gather4 would need no warps, but moved
// only four rows in some 70 ns: 225 us at 333 bf16 tokens (52 rows a tile) against 90 us with neighbouring rows.
// Returns false when a wait ran out. tid: the thread among the gathering ones; a stage has SUB steps of sub_bytes each, b_off is the
// rows' place in one.
template <int TILE, int STAGES, int SUB, int WARPS>
__device__ __forceinline__ bool gmm_gather(const GmmWalk &W, const GmmArgs &A, int tid, int nitems, uint8_t *ring, int sub_bytes,
                                           int b_off, uint64_t *full, uint64_t *empty, volatile int *abort) {
    constexpr int LAG = 2, PER = (TILE * 8 + WARPS * 32 - 1) / (WARPS * 32);  // 16-byte pieces of a stage per thread
    static_assert(LAG < STAGES && PER >= 1, "gather pipeline");
    const int lane = threadIdx.x & 31;
    const int piece = tid & 7, row0 = tid >> 3;  // this thread: piece `piece` of rows row0, row0 + APART, ...
    constexpr int APART = WARPS * 4;
    int kg = 0;
    bool ok = true;
    for (int item = blockIdx.x, n = 0; item < nitems && ok; item += gridDim.x, n++) {
        const GmmItem I = gmm_item<TILE>(W, A, item, n);
        const int n16 = (I.nt + 15) & ~15;
        const uint8_t *src[PER];
#pragma unroll
        for (int j = 0; j < PER; j++) {
            const int v = A.in_rows[I.base + min(row0 + j * APART, I.nt - 1)];
            // a bad index reads row 0; the fold neither writes that entry nor stays silent about it
            src[j] = A.a + ((unsigned)v < (unsigned)A.a_rows ? v : 0) * A.lda_bytes + piece * 16;
        }
        for (int k = 0; k < A.steps; k += SUB, kg++) {
            const int s = kg % STAGES;
            if (kg >= STAGES) ok = mbar_wait(&empty[s], ((kg / STAGES) - 1) & 1, abort);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
#pragma unroll
            for (int u = 0; u < SUB; u++) {
                if (SUB > 1 && k + u >= A.steps) break;
                const int64_t at = (int64_t)(k + u) * kGmmBytes;
                const int64_t left = A.k_bytes - at - piece * 16;
                const int size = left >= 16 ? 16 : left > 0 ? (int)left : 0;
                const int64_t from = size ? at : -(int64_t)piece * 16;  // nothing is read then: stay inside the row
                const uint32_t dst = smem_u32(ring + (s * SUB + u) * sub_bytes + b_off);
#pragma unroll
                for (int j = 0; j < PER; j++) {
                    const int row = row0 + j * APART;
                    if (row < n16)
                        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst + row * 128 + ((piece ^ (row & 7)) << 4)),
                                     "l"(src[j] + from), "r"(size)
                                     : "memory");
                }
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

// The staging warps' walk; an item has PLANES blocks of 128 rows of w. The loads of the next chunk, and the indexes of the next
// item, are in flight while the current chunk waits for its place. Returns false when a wait
// ran out.
template <bool F8, int TILE, int TEAMS, int PLANES, int KC>
__device__ __forceinline__ bool gmm_stage_walk(GmmStaged<TILE, TEAMS, PLANES, KC> &T, const GmmWalk &W, const GmmArgs &A, int nitems,
                                               volatile int *abort) {
    constexpr int NW = gmm_stagers<TILE>(), PER = TILE / 32 / NW;  // entries per lane
    const int first = blockIdx.x, stride = gridDim.x;
    const int lane = threadIdx.x & 31, t0 = (threadIdx.x >> 5) - 2 == 0 ? lane : lane + PER * 32;
    if (NW == 1 && t0 != lane) return true;
    const int esize = A.out_type == INZG_T_F32 ? 4 : 2;
    const bool vec = F8 && A.ldas % 4 == 0 && !(reinterpret_cast<uintptr_t>(A.as) & 15);
    struct Ring {  // one team's places
        GmmSlot<kGmmRing> p, t;
        int chunks = 0, items = 0;  // staged so far, counted up to the ring's size
    };
    Ring mine, other;  // of the current item's team and (TEAMS = 2) of the next item's: they change places
    bool ok = true;
    struct Entry {
        int row, o;
        float w;
    };
    Entry cur[PER], nxt[PER];
    float v[PER][KC], u[PLANES];  // the chunk in flight: a's scales of this lane's entries; lane b: w's scale of block b
    auto load_entries = [&](const GmmItem &I, Entry(&e)[PER]) {
#pragma unroll
        for (int j = 0; j < PER; j++) {
            const int i = I.base + min(t0 + 32 * j, I.nt - 1);
            e[j].row = A.in_rows ? A.in_rows[i] : i;
            e[j].o = A.out_rows ? A.out_rows[i] : i;
            e[j].w = A.out_scale ? A.out_scale[i] : 1.0f;
        }
    };
    auto load_chunk = [&](const GmmItem &I, const Entry(&e)[PER], int b0) {
        const int nb = min(KC, A.steps - b0);
#pragma unroll
        for (int j = 0; j < PER; j++) {
            const int row = (unsigned)e[j].row < (unsigned)A.a_rows ? e[j].row : 0;
            const float *as = A.as + (int64_t)row * A.ldas + b0;
#pragma unroll
            for (int b = 0; b < KC; b += 4) {
                if (vec && b + 4 <= nb) {
                    const float4 x = __ldg(reinterpret_cast<const float4 *>(as + b));
                    v[j][b] = x.x;
                    v[j][b + 1] = x.y;
                    v[j][b + 2] = x.z;
                    v[j][b + 3] = x.w;
                } else {
#pragma unroll
                    for (int k = b; k < b + 4; k++) v[j][k] = k < nb ? __ldg(as + k) : 0.0f;
                }
            }
        }
#pragma unroll
        for (int q = 0; q < PLANES; q++)
            u[q] = lane < nb && I.rb * PLANES + q < A.nrb128
                       ? __ldg(A.ws + ((int64_t)I.g * A.nrb128 + I.rb * PLANES + q) * A.steps + b0 + lane)
                       : 0.0f;
    };
    if (first >= nitems) return true;
    GmmItem I = gmm_item<TILE>(W, A, first, 0);
    load_entries(I, cur);
    if constexpr (F8) load_chunk(I, cur, 0);
    for (int item = first, team = 0, n = 0; item < nitems; item += stride, team = (team + 1) % TEAMS, n++) {
        const bool more = item + stride < nitems;
        GmmItem N = I;
        if (more) {
            N = gmm_item<TILE>(W, A, item + stride, n + 1);
            load_entries(N, nxt);
        }
        if (mine.items == kGmmRing) ok = mbar_wait(&T.to_empty[team][mine.t.i], mine.t.parity ^ 1, abort);
        else mine.items++;
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
#pragma unroll
        for (int j = 0; j < PER; j++) {
            const int t = t0 + 32 * j;
            const bool bad = (unsigned)cur[j].row >= (unsigned)A.a_rows || (unsigned)cur[j].o >= (unsigned)A.out_rows_n;
            if (bad) atomicCAS(A.err, kErrNone, kErrBadSlot);
            GmmTo to;
            to.row = t < I.nt && !bad ? static_cast<char *>(A.out) + (int64_t)cur[j].o * A.ldo * esize : nullptr;
            to.w = cur[j].w;
            T.to[team][mine.t.i][t] = to;
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&T.to_full[team][mine.t.i]);
        mine.t.next();
        if constexpr (F8) {
            for (int b0 = 0; b0 < A.steps; b0 += KC) {
                float x[PER][KC], y[PLANES];
#pragma unroll
                for (int j = 0; j < PER; j++)
#pragma unroll
                    for (int b = 0; b < KC; b++) x[j][b] = v[j][b];
#pragma unroll
                for (int q = 0; q < PLANES; q++) y[q] = u[q];
                if (b0 + KC < A.steps) load_chunk(I, cur, b0 + KC);
                else if (more) load_chunk(N, nxt, 0);
                if (mine.chunks == kGmmRing) ok = mbar_wait(&T.p_empty[team][mine.p.i], mine.p.parity ^ 1, abort);
                else mine.chunks++;
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
#pragma unroll
                for (int q = 0; q < PLANES; q++)
#pragma unroll
                    for (int b = 0; b < KC; b++) {
                        const float s = __shfl_sync(0xffffffffu, y[q], b);
#pragma unroll
                        for (int j = 0; j < PER; j++) T.p[team][mine.p.i][q][b][t0 + 32 * j] = x[j][b] * s;
                    }
                __syncwarp();
                if (lane == 0) mbar_arrive(&T.p_full[team][mine.p.i]);
                mine.p.next();
            }
            if (!ok) break;
        }
        I = N;
#pragma unroll
        for (int j = 0; j < PER; j++) cur[j] = nxt[j];
        if constexpr (TEAMS == 2) {
            const Ring t = mine;
            mine = other;
            other = t;
        }
    }
    return ok;
}

// 2-D tensor map over [rows][k] with a row pitch of ld elements, boxes of box_rows x 128 bytes, 128-byte swizzle; what lies
// outside reads as zeros. False when the driver refuses it.
bool gmm_map(CUtensorMap *m, const void *base, int elem, int64_t rows, int64_t k, int64_t ld, int box_rows);

// Kernels that hand registers from some warps to others (setmaxnreg) need the 128 per thread at launch that their split adds up
// to, or the receiving warps wait for ever: whether `kernel` was built with them.
template <class F>
inline bool gmm_split_holds(F kernel) {
    cudaFuncAttributes at{};
    return cudaFuncGetAttributes(&at, kernel) == cudaSuccess && at.numRegs == 128;
}

// The kernel for many entries (k_gmm_large.cu): A holds everything but nrb and the tile-dependent bits. The attributes' call returns
// false when the kernel may not be launched.
bool gmm_large_set_attributes();
int gmm_large_launch(const inzg_grouped_matmul_args &G, GmmArgs A, int num_sms, cudaStream_t st);

}  // namespace inzg
