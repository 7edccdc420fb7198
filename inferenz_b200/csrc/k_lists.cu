// k_lists.cu -- the entries of the router's selections in order of expert, on sm_100a (inzg_expert_lists).
//
// One block per expert, no scratch and no atomics: the block reads every selection, counts those of smaller experts (its
// list's offset) and its own, and writes its own in slot order. A warp owns a contiguous run of the entries, so an
// entry's place is off + (own entries of earlier warps) + (own entries of this warp so far) + its rank in the warp's
// ballot: the order is fixed. Work is n_expert * n * topk compares, each entry read by every block from L2.
#include <algorithm>

#include "inzg_internal.h"
#include "k_launch.h"

namespace inzg {

constexpr int kListWarps = 16;

template <bool VEC>
__global__ void __launch_bounds__(kListWarps * 32) expert_lists_kernel(const int32_t *__restrict__ sel, const float *__restrict__ w,
                                                                       int entries, int topk, int E, int32_t *__restrict__ off,
                                                                       int32_t *__restrict__ rows, int32_t *__restrict__ slots,
                                                                       float *__restrict__ w_out, int32_t *err) {
    __shared__ int s_less[kListWarps], s_own[kListWarps];
    const int e = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, nw = blockDim.x >> 5;
    // whole 128-entry steps per warp
    const int steps = (entries + nw * 128 - 1) / (nw * 128);
    const int first = warp * steps * 128;
    auto load = [&](int i) {  // entries i .. i + 3; -1 behind the last
        int4 v = make_int4(-1, -1, -1, -1);
        if (VEC && i + 3 < entries) {
            v = *reinterpret_cast<const int4 *>(sel + i);
        } else {
            if (i < entries) v.x = sel[i];
            if (i + 1 < entries) v.y = sel[i + 1];
            if (i + 2 < entries) v.z = sel[i + 2];
            if (i + 3 < entries) v.w = sel[i + 3];
        }
        return v;
    };
    int less = 0, own = 0;
    bool bad = false;
    for (int j = 0; j < steps; j++) {
        const int i = first + j * 128 + lane * 4;
        const int4 v = load(i);
        const int a[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int c = 0; c < 4; c++) {
            less += a[c] >= 0 && a[c] < e;
            own += a[c] == e;
            bad |= a[c] >= E;
        }
    }
    if (bad && e == 0) atomicCAS(err, kErrNone, kErrBadExpert);
    less = __reduce_add_sync(0xffffffffu, less);
    own = __reduce_add_sync(0xffffffffu, own);
    if (lane == 0) {
        s_less[warp] = less;
        s_own[warp] = own;
    }
    __syncthreads();
    int base = 0, total = 0;
    for (int k = 0; k < nw; k++) {
        base += s_less[k] + (k < warp ? s_own[k] : 0);
        total += s_less[k] + s_own[k];
    }
    if (threadIdx.x == 0) {
        off[e] = total - [&] { int t = 0; for (int k = 0; k < nw; k++) t += s_own[k]; return t; }();
        if (e == E - 1) off[E] = total;
    }
    if (own == 0) return;
    for (int j = 0; j < steps; j++) {
        const int i = first + j * 128 + lane * 4;
        const int4 v = load(i);
        const int a[4] = {v.x, v.y, v.z, v.w};
        const uint32_t below = (1u << lane) - 1;
        int at = base, mine = 0;
#pragma unroll
        for (int c = 0; c < 4; c++) {
            const uint32_t m = __ballot_sync(0xffffffffu, a[c] == e);
            at += __popc(m & below);
            mine += __popc(m);
        }
#pragma unroll
        for (int c = 0; c < 4; c++) {
            if (a[c] != e) continue;
            slots[at] = i + c;
            rows[at] = (i + c) / topk;
            if (w_out) w_out[at] = w[i + c];
            at++;
        }
        base += mine;
    }
}

int launch_expert_lists(int n, int topk, int E, const int32_t *sel, const float *w, int32_t *off, int32_t *rows,
                        int32_t *slots, float *w_out, int32_t *err, cudaStream_t st) {
    const int entries = n * topk;
    const int warps = std::max(1, std::min(kListWarps, (entries + 127) / 128));
    if (reinterpret_cast<uintptr_t>(sel) & 15)
        expert_lists_kernel<false><<<E, warps * 32, 0, st>>>(sel, w, entries, topk, E, off, rows, slots, w_out, err);
    else
        expert_lists_kernel<true><<<E, warps * 32, 0, st>>>(sel, w, entries, topk, E, off, rows, slots, w_out, err);
    return 1;
}

}  // namespace inzg
