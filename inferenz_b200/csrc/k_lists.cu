// k_lists.cu -- the entries of the router's selections in order of expert, on sm_100a (inzg_expert_lists): a stable counting sort
// without scratch in global memory; its shared-memory atomics only count and set bits, so the order is fixed.
//
// One block, or for more than 2048 entries a cluster of sixteen (past the portable eight, which took 14.1 us
// where this takes 11.7: the scattered results leave through twice the SMs). Sixteen blocks of up to 208 KB of shared memory want as many
// SMs of one GPC: where a device cannot hold them (lists_most_cluster) it is eight, or one. A warp owns a contiguous run of the entries, a row of
// counters in shared memory, one per expert, and a row of lane masks: within a step of 32 entries the lanes set their bits in
// their experts' masks (match.any, which does the same, goes through the distinct values one by one and was slower), so that
//   place = (entries of smaller experts) + (own expert: earlier blocks, earlier warps, earlier steps, lower lanes)
// The blocks of the cluster read one another's totals through distributed shared memory. Each entry is read twice; what bounds it
// is the chain of two passes, a scan over the experts and two cluster barriers. A block per expert (or per four) that counted
// every entry for itself took 20 to 26 us at 4096 tokens, top-10; this takes 11.7 us, and 3.6 us at 32 tokens.
#include <algorithm>

#include "inzg_internal.h"
#include "k_async.cuh"
#include "k_launch.h"

namespace inzg {

constexpr int kListThreads = 1024, kListCounters = 24576;  // counters of all warps, and as many masks: 192 KB

__device__ __forceinline__ void lists_cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ int lists_remote(const int *p, int rank) {  // *p of block `rank` of the cluster
    uint32_t a;
    int v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(p)), "r"(rank));
    asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(a));  // volatile: stays between the cluster's barriers
    return v;
}

// shared: counters [warps][E], masks [warps][E], then this block's totals [E] and the first place of each expert's entries of this
// block [E]
template <int CLUSTER>
__global__ void __launch_bounds__(kListThreads)
expert_lists_kernel(const int32_t *__restrict__ sel, const float *__restrict__ w, int entries, int topk, int E, int32_t *__restrict__ off,
                    int32_t *__restrict__ rows, int32_t *__restrict__ slots, float *__restrict__ w_out, int32_t *err) {
    extern __shared__ __align__(16) int lists_dyn[];
    __shared__ int s_scan[32];
    const int nw = blockDim.x >> 5, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, rank = CLUSTER > 1 ? blockIdx.x : 0;
    int *count = lists_dyn + warp * E, *total = lists_dyn + 2 * nw * E, *place = total + E;
    uint32_t *mask = reinterpret_cast<uint32_t *>(count + nw * E);
    const int steps = (int)(((int64_t)entries + CLUSTER * nw * 32 - 1) / (CLUSTER * nw * 32));
    const int64_t first = (int64_t)(rank * nw + warp) * steps * 32 + lane;
    int next = steps && first < entries ? sel[first] : -1;
    for (int i = threadIdx.x; i < (2 * nw * E + 3) / 4; i += blockDim.x) reinterpret_cast<int4 *>(lists_dyn)[i] = make_int4(0, 0, 0, 0);
    __syncthreads();
    const uint32_t below = (1u << lane) - 1;
    // first pass: entries per expert of this warp's run
    bool bad = false;
    for (int j = 0; j < steps; j++) {
        const int e = next;
        const int64_t i = first + (j + 1) * 32;
        if (j + 1 < steps) next = i < entries ? sel[i] : -1;
        bad |= e >= E;
        if ((uint32_t)e < (uint32_t)E) atomicAdd(&count[e], 1);
    }
    if (bad) atomicCAS(err, kErrNone, kErrBadExpert);
    __syncthreads();
    // per expert: the warps' counts become what the warps before have; a thread has `per` neighbouring experts
    const int per = (E + blockDim.x - 1) / blockDim.x, e0 = threadIdx.x * per, e1 = min(e0 + per, E);
    for (int e = e0; e < e1; e++) {
        int run = 0;
        for (int k = 0; k < nw; k += 8) {  // eight loads at a time
            int t[8];
#pragma unroll
            for (int j = 0; j < 8; j++) t[j] = k + j < nw ? lists_dyn[(k + j) * E + e] : 0;
#pragma unroll
            for (int j = 0; j < 8; j++) {
                if (k + j < nw) lists_dyn[(k + j) * E + e] = run;
                run += t[j];
            }
        }
        total[e] = run;
    }
    if (CLUSTER > 1) lists_cluster_sync();
    // the cluster's entries per expert, and a scan over the experts
    int mine = 0;
    for (int e = e0; e < e1; e++) {
        int before = 0, all = 0, t[CLUSTER];
#pragma unroll
        for (int q = 0; q < CLUSTER; q++) t[q] = CLUSTER > 1 ? lists_remote(total + e, q) : total[e];
#pragma unroll
        for (int q = 0; q < CLUSTER; q++) {
            if (q < rank) before += t[q];
            all += t[q];
        }
        place[e] = mine + before;  // within this thread's experts so far
        if (rank == 0) off[e] = mine;
        mine += all;
    }
    int scan = mine;
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
        const int t = __shfl_up_sync(0xffffffffu, scan, d);
        if (lane >= d) scan += t;
    }
    if (lane == 31) s_scan[warp] = scan;
    __syncthreads();
    int start = scan - mine;
    for (int k = 0; k < warp; k++) start += s_scan[k];
    for (int e = e0; e < e1; e++) {
        place[e] += start;
        if (rank == 0) off[e] += start;
    }
    if (rank == 0 && e0 < E && e1 == E) off[E] = start + mine;
    __syncthreads();
    // second pass: every entry to its place
    next = steps && first < entries ? sel[first] : -1;
    float w_next = w && steps && first < entries ? w[first] : 0.0f;
    for (int j = 0; j < steps; j++) {
        const int e = next;
        const float we = w_next;
        const int64_t i = first + j * 32;
        if (j + 1 < steps) {
            next = i + 32 < entries ? sel[i + 32] : -1;
            if (w) w_next = i + 32 < entries ? w[i + 32] : 0.0f;
        }
        const bool own = (uint32_t)e < (uint32_t)E;
        if (own) atomicOr(&mask[e], 1u << lane);
        __syncwarp();
        uint32_t same = 0;
        if (own) {
            same = mask[e];
            const int at = place[e] + count[e] + __popc(same & below);
            slots[at] = (int)i;
            rows[at] = (int)i / topk;
            if (w_out) w_out[at] = we;
        }
        __syncwarp();
        if (own && !(same & below)) {
            count[e] += __popc(same);
            mask[e] = 0;
        }
        __syncwarp();
    }
    if (CLUSTER > 1) lists_cluster_sync();  // no block leaves while another may still read its totals
}

constexpr int kListSmem = (2 * kListCounters + 2 * INZG_MAX_GROUPS) * (int)sizeof(int);  // of the longest lists

static void lists_config(cudaLaunchConfig_t &cfg, cudaLaunchAttribute &at, int cluster, int threads, size_t smem, cudaStream_t st) {
    cfg.gridDim = dim3(cluster);
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    at.id = cudaLaunchAttributeClusterDimension;
    at.val.clusterDim.x = cluster;
    at.val.clusterDim.y = at.val.clusterDim.z = 1;
    cfg.attrs = &at;
    cfg.numAttrs = 1;
}

// whether the device holds a cluster of so many blocks at their largest
template <int CLUSTER>
static bool lists_holds() {
    const auto kernel = expert_lists_kernel<CLUSTER>;
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kListSmem) != cudaSuccess) return false;
    if (CLUSTER > 8 && cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess) return false;
    cudaLaunchConfig_t cfg{};
    cudaLaunchAttribute at{};
    lists_config(cfg, at, CLUSTER, kListThreads, kListSmem, nullptr);
    int clusters = 0;
    return cudaOccupancyMaxActiveClusters(&clusters, kernel, &cfg) == cudaSuccess && clusters >= 1;
}

int lists_most_cluster(bool sixteen, bool eight) { return sixteen ? 16 : eight ? 8 : 1; }

int lists_set_attributes() {
    cudaFuncSetAttribute(expert_lists_kernel<1>, cudaFuncAttributeMaxDynamicSharedMemorySize, kListSmem);
    const bool sixteen = lists_holds<16>(), eight = lists_holds<8>();
    cudaGetLastError();  // a size that the device refuses is no error of the caller's
    return lists_most_cluster(sixteen, eight);
}

int launch_expert_lists(int n, int topk, int E, const int32_t *sel, const float *w, int32_t *off, int32_t *rows,
                        int32_t *slots, float *w_out, int most_cluster, int32_t *err, cudaStream_t st) {
    const int entries = n * topk;
    const int cluster = entries > 2048 ? most_cluster : 1;
    const int warps = std::max(1, std::min({kListThreads / 32, kListCounters / E, (entries + cluster * 32 - 1) / (cluster * 32)}));
    const size_t smem = sizeof(int) * (2 * (size_t)warps * E + 2 * (size_t)E);
    if (cluster == 1) {
        expert_lists_kernel<1><<<1, warps * 32, smem, st>>>(sel, w, entries, topk, E, off, rows, slots, w_out, err);
        return 1;
    }
    cudaLaunchConfig_t cfg{};
    cudaLaunchAttribute at{};
    lists_config(cfg, at, cluster, warps * 32, smem, st);
    cudaLaunchKernelEx(&cfg, cluster == 16 ? expert_lists_kernel<16> : expert_lists_kernel<8>, sel, w, entries, topk, E, off, rows, slots,
                       w_out, err);
    return 1;
}

}  // namespace inzg
