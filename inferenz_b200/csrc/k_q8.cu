// k_q8.cu -- the row operators of the 8-bit floating point path on sm_100a: the RMS norm with the residual's addition
// and SiLU(gate) * up, each with an e4m3 output and one fp32 scale per 128 columns.
//
//   norm: h = x + res, r = 1 / sqrt(sum(h^2) / cols + eps), v = (h * r) * w
//   silu: v = g / (1 + exp(-g)) * u
//
// Both read each input once and write each output once: the row stays in registers (fp32) between the sum of squares
// and the outputs, the block's largest value is a shuffle over 16 lanes, nothing passes through memory in between.
#include "k_launch.h"
#include "k_q8.cuh"

namespace inzg {

// One row per block; thread t holds chunks t, t + blockDim, ... (NCH of them, 8 columns each).
template <class T, int NCH, bool VEC>
__global__ void __launch_bounds__(1024) rmsnorm_q8_kernel(const inzg_rmsnorm_q8_args A) {
    __shared__ float part[32];
    const int64_t row = blockIdx.x;
    const int cols = A.cols, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const T *x = static_cast<const T *>(A.x) + row * A.ldx;
    const T *res = A.res ? static_cast<const T *>(A.res) + row * A.ldres : nullptr;
    T *sum = A.sum ? static_cast<T *>(A.sum) + row * A.ldsum : nullptr;
    float h[NCH][8];
    float ss = 0.0f;
#pragma unroll
    for (int j = 0; j < NCH; j++) {
        const int c = (threadIdx.x + j * blockDim.x) * 8, left = cols - c;
        if (left > 0) load_chunk<T, VEC>(x + c, left, h[j]);
        else
#pragma unroll
            for (int i = 0; i < 8; i++) h[j][i] = 0.0f;
    }
    if (res) {
#pragma unroll
        for (int j = 0; j < NCH; j++) {
            const int c = (threadIdx.x + j * blockDim.x) * 8, left = cols - c;
            if (left <= 0) continue;
            float r[8];
            load_chunk<T, VEC>(res + c, left, r);
#pragma unroll
            for (int i = 0; i < 8; i++) h[j][i] += r[i];
        }
    }
#pragma unroll
    for (int j = 0; j < NCH; j++) {
        const int c = (threadIdx.x + j * blockDim.x) * 8, left = cols - c;
        if (sum && left > 0) store_chunk<T, VEC>(sum + c, left, h[j]);
#pragma unroll
        for (int i = 0; i < 8; i++) ss = fmaf(h[j][i], h[j][i], ss);
    }
#pragma unroll
    for (int d = 16; d; d >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, d);
    if (lane == 0) part[warp] = ss;
    __syncthreads();
    ss = lane < (int)(blockDim.x >> 5) ? part[lane] : 0.0f;
#pragma unroll
    for (int d = 16; d; d >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, d);
    const float r = __frcp_rn(__fsqrt_rn(__fdiv_rn(ss, (float)cols) + A.eps));
#pragma unroll
    for (int j = 0; j < NCH; j++) {
        const int chunk = threadIdx.x + j * blockDim.x, c = chunk * 8, left = cols - c;
        float v[8];
        if (left > 0) load_chunk<float, VEC>(A.w + c, left, v);
        else
#pragma unroll
            for (int i = 0; i < 8; i++) v[i] = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = left > i ? h[j][i] * r * v[i] : 0.0f;
        if (A.y && left > 0) store_chunk<T, VEC>(static_cast<T *>(A.y) + row * A.ldy + c, left, v);
        if (A.q) {
            float s;
            const uint2 q = quantize_chunk(v, s);
            if (left > 0) {
                store_q<VEC>(static_cast<uint8_t *>(A.q) + row * A.ldq + c, left, q);
                if ((chunk & 15) == 0) A.s[row * A.lds + (chunk >> 4)] = s;
            }
        }
    }
}

// exp(x) for x in fp32: 2^(x log2 e) with the product's rounding error carried to first order, so that the relative error
// stays at a few 2^-24 for large |x| too, where the hardware's 2^t on the rounded product alone loses |x| * 2^-24.
__device__ __forceinline__ float exp_carried(float x) {
    const float t = x * 1.4426950408889634f;
    const float lo = fmaf(x, 1.4426950408889634f, -t) + x * 1.925963033500938e-8f;  // log2 e = hi + 1.926e-8
    float e;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(t));
    return fabsf(t) < 160.0f ? fmaf(e, lo * 0.6931471805599453f, e) : e;  // past that e is 0, inf or NaN already
}

// A thread's slot: one chunk of one row; slots per row are rounded up to whole blocks of 128 columns.
template <class T, bool VEC>
__global__ void __launch_bounds__(256) silu_mul_q8_kernel(const inzg_silu_mul_q8_args A, uint32_t slots, uint32_t per_row) {
    const int cols = A.cols;
    // whole warps stay in the loop: the quantizer shuffles
    for (uint32_t i = blockIdx.x * blockDim.x + threadIdx.x; i - threadIdx.x % 32 < slots; i += gridDim.x * blockDim.x) {
        const uint32_t row = i / per_row, chunk = i % per_row;
        const int c = (int)chunk * 8, left = i < slots ? cols - c : 0;
        float g[8], u[8];
        if (left > 0) {
            const T *x = static_cast<const T *>(A.x) + (int64_t)row * A.ldx;
            load_chunk<T, VEC>(x + c, left, g);
            load_chunk<T, VEC>(x + cols + c, left, u);
        } else {
#pragma unroll
            for (int j = 0; j < 8; j++) g[j] = u[j] = 0.0f;
        }
#pragma unroll
        for (int j = 0; j < 8; j++) u[j] *= __fdividef(g[j], 1.0f + exp_carried(-g[j]));
        if (A.y && left > 0) store_chunk<T, VEC>(static_cast<T *>(A.y) + (int64_t)row * A.ldy + c, left, u);
        if (A.q) {
            float s;
            const uint2 q = quantize_chunk(u, s);
            if (left > 0) {
                store_q<VEC>(static_cast<uint8_t *>(A.q) + (int64_t)row * A.ldq + c, left, q);
                if ((chunk & 15) == 0) A.s[(int64_t)row * A.lds + (chunk >> 4)] = s;
            }
        }
    }
}

// ---------------------------------------------------------------------------------------------------------------------

static bool aligned(const void *p, int64_t ld_bytes, int to) {
    return !p || !((reinterpret_cast<uintptr_t>(p) | (uintptr_t)ld_bytes) & (uintptr_t)(to - 1));
}

template <class T>
static int norm_typed(const inzg_rmsnorm_q8_args &A, int num_sms, cudaStream_t st) {
    const int64_t b = sizeof(T);
    const bool vec = aligned(A.x, A.ldx * b, 16) && aligned(A.res, A.ldres * b, 16) && aligned(A.sum, A.ldsum * b, 16) &&
                     aligned(A.y, A.ldy * b, 16) && aligned(A.q, A.ldq, 8) && aligned(A.w, 0, 16);
    const int chunks = (A.cols + 7) / 8;
    // few rows: one chunk per thread, the shortest chain; many: two, so that a block holds fewer warps and more rows are
    // in flight; wide rows as many as 1024 threads need
    int nch = A.n <= num_sms ? 1 : 2;
    while (nch < 4 && chunks > nch * 1024) nch *= 2;
    const int threads = ((chunks + nch - 1) / nch + 31) / 32 * 32;
#define INZG_NORM(NCH)                                                                                        \
    do {                                                                                                      \
        if (vec) rmsnorm_q8_kernel<T, NCH, true><<<A.n, threads, 0, st>>>(A);                                 \
        else rmsnorm_q8_kernel<T, NCH, false><<<A.n, threads, 0, st>>>(A);                                    \
    } while (0)
    if (nch == 1) INZG_NORM(1);
    else if (nch == 2) INZG_NORM(2);
    else INZG_NORM(4);
#undef INZG_NORM
    return 1;
}

int launch_rmsnorm_q8(const inzg_rmsnorm_q8_args &args, int num_sms, cudaStream_t st) {
    inzg_rmsnorm_q8_args A = args;
    if (!A.ldx) A.ldx = A.cols;
    if (!A.ldres) A.ldres = A.cols;
    if (!A.ldsum) A.ldsum = A.cols;
    if (!A.ldy) A.ldy = A.cols;
    if (!A.ldq) A.ldq = A.cols;
    if (!A.lds) A.lds = (A.cols + kQB - 1) / kQB;
    if (A.type == INZG_T_F32) return norm_typed<float>(A, num_sms, st);
    if (A.type == INZG_T_F16) return norm_typed<__half>(A, num_sms, st);
    return norm_typed<__nv_bfloat16>(A, num_sms, st);
}

template <class T>
static int silu_typed(inzg_silu_mul_q8_args A, int num_sms, cudaStream_t st) {
    const int64_t b = sizeof(T);
    const bool vec = aligned(A.x, A.ldx * b, 16) && aligned(A.x, A.cols * b, 16) && aligned(A.y, A.ldy * b, 16) &&
                     aligned(A.q, A.ldq, 8);
    const uint32_t per_row = (uint32_t)(A.cols + kQB - 1) / kQB * 16;
    const int rows_max = (int)(0x40000000u / per_row);  // slots are counted in 32 bits: more rows take more launches
    int launches = 0;
    for (int64_t done = 0; done < A.n; done += rows_max) {
        inzg_silu_mul_q8_args P = A;
        P.n = (int)((A.n - done) < rows_max ? A.n - done : rows_max);
        P.x = static_cast<const T *>(A.x) + done * A.ldx;
        if (A.y) P.y = static_cast<T *>(A.y) + done * A.ldy;
        if (A.q) P.q = static_cast<uint8_t *>(A.q) + done * A.ldq;
        if (A.s) P.s = A.s + done * A.lds;
        const uint32_t slots = (uint32_t)P.n * per_row;
        const uint32_t want = (slots + 255) / 256, most = (uint32_t)num_sms * 8;
        const uint32_t grid = want < most ? want : most;
        if (vec) silu_mul_q8_kernel<T, true><<<grid, 256, 0, st>>>(P, slots, per_row);
        else silu_mul_q8_kernel<T, false><<<grid, 256, 0, st>>>(P, slots, per_row);
        launches++;
    }
    return launches;
}

int launch_silu_mul_q8(const inzg_silu_mul_q8_args &args, int num_sms, cudaStream_t st) {
    inzg_silu_mul_q8_args A = args;
    if (!A.ldx) A.ldx = 2 * (int64_t)A.cols;
    if (!A.ldy) A.ldy = A.cols;
    if (!A.ldq) A.ldq = A.cols;
    if (!A.lds) A.lds = (A.cols + kQB - 1) / kQB;
    if (A.type == INZG_T_F32) return silu_typed<float>(A, num_sms, st);
    if (A.type == INZG_T_F16) return silu_typed<__half>(A, num_sms, st);
    return silu_typed<__nv_bfloat16>(A, num_sms, st);
}

}  // namespace inzg
