// k_q8.cu -- the row operators of the 8-bit floating point path on sm_100a: the RMS norm with the residual's addition
// and SiLU(gate) * up, each with an e4m3 output and one fp32 scale per 128 columns.
//
//   norm: h = x + res, r = 1 / sqrt(sum(h^2) / cols + eps), v = (h * r) * w
//   silu: v = g / (1 + exp(-g)) * u
//
// Both read each input once and write each output once: the row stays in registers (fp32) between the sum of squares
// and the outputs, the block's largest value is a shuffle over 16 lanes, nothing passes through memory in between.
// Measured on B200, back to back in CUDA graphs: norm of 4096 x 2560 bf16 with residual, y and e4m3 19.5 us (94.7 MB, 4.85 TB/s; the
// next row's loads in flight took it from 24.7 to 21.3 us when they came, one chunk per thread to 18.7), one row 2.2 us; SiLU of
// 40960 x 640 bf16 28.0 us (131.9 MB, 4.7 TB/s). Eager calls from Python take 21.0 and 29.7 us. Rows that are not whole aligned chunks
// go element by element: the norm with a pitch of 2563 49 to 72 us from one GPU to the next, SiLU of 40960 x 636 47 to 63 us.
#include <algorithm>

#include "k_launch.h"
#include "k_q8.cuh"

namespace inzg {

constexpr float kMeanLeast = 8.077935669463161e-28f;  // 2^-90: squares lost below the normal range are some 2^-60 of it

// y, q and s of a thread's chunk of a row; rs: the row's factor. (The kernel's own rows have it written out: by this function
// 4096 x 2560 bf16 took 20.0 us instead of 19.5.)
template <class T, bool VEC>
__device__ __forceinline__ void norm_out(const inzg_rmsnorm_q8_args &A, int64_t row, int chunk, const float (&h)[8], float rs,
                                         const float (&w)[8]) {
    const int c = chunk * 8, left = A.cols - c;
    float v[8], z[8];  // z: v without the row's factor
#pragma unroll
    for (int i = 0; i < 8; i++) v[i] = left > i ? h[i] * rs * w[i] : 0.0f;
#pragma unroll
    for (int i = 0; i < 8; i++) z[i] = left > i ? h[i] * w[i] : 0.0f;
    if (A.y && left > 0) store_chunk<T, VEC>(static_cast<T *>(A.y) + row * A.ldy + c, left, v);
    if (A.q) {
        float s;
        const uint2 q = quantize_scaled(z, v, rs, s);
        if (left > 0) {
            store_q<VEC>(static_cast<uint8_t *>(A.q) + row * A.ldq + c, left, q);
            if ((chunk & 15) == 0) A.s[row * A.lds + (chunk >> 4)] = s;
        }
    }
}

__device__ __forceinline__ bool norm_is_far(float ms) { return !(ms >= kMeanLeast && ms < __int_as_float(0x7F800000)); }

// Those of the block's rows whose squares left fp32's range, or may have: h (and eps) are multiplied by a power of two that brings the
// row's largest value, or the root of eps, to 1 to 4. After the other rows and from memory once more, over what was written for these
// rows, so that the others do not wait for the decision: with h multiplied in their way 8192 columns took 64.7 us instead of
// 56.5 and 10240 109 instead of 86. `mark`: a bit for each of the block's rows; what x and res of the others hold by now may be sums.
constexpr int kNormRows = 8192;  // rows of a block that can be marked; more take more launches
template <class T, bool VEC>
__device__ __forceinline__ void norm_far_rows(const inzg_rmsnorm_q8_args &A, float (&part)[32], const uint32_t *mark) {
    const int cols = A.cols, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
    const int nch = (cols + 8 * blockDim.x - 1) / (8 * blockDim.x);  // every thread goes round as often: the quantizer shuffles
    auto reduce = [&](float v, auto op) {                            // over the block, in every thread
#pragma unroll
        for (int d = 16; d; d >>= 1) v = op(v, __shfl_xor_sync(0xffffffffu, v, d));
        if (warps == 1) return v;
        __syncthreads();
        if (lane == 0) part[warp] = v;
        __syncthreads();
        v = lane < warps ? part[lane] : 0.0f;  // none is negative
#pragma unroll
        for (int d = 16; d; d >>= 1) v = op(v, __shfl_xor_sync(0xffffffffu, v, d));
        return v;
    };
    auto load = [&](int64_t row, int chunk, float(&h)[8]) {
        const int c = chunk * 8, left = cols - c;
        Chunk<T> x;
        load_raw<T, VEC>(static_cast<const T *>(A.x) + row * A.ldx + c, left, x);
#pragma unroll
        for (int i = 0; i < 8; i++) h[i] = to_f32(x.v[i]);
        if (!A.res) return;
        load_raw<T, VEC>(static_cast<const T *>(A.res) + row * A.ldres + c, left, x);
#pragma unroll
        for (int i = 0; i < 8; i++) h[i] += to_f32(x.v[i]);
    };
    auto mean = [&](int64_t row, float f) {  // of the squares of h f
        float ss = 0.0f;
#pragma unroll 1
        for (int j = 0; j < nch; j++) {
            float h[8];
            load(row, threadIdx.x + j * blockDim.x, h);
#pragma unroll
            for (int i = 0; i < 8; i++) ss = fmaf(h[i] * f, h[i] * f, ss);
        }
        return __fdiv_rn(reduce(ss, [](float a, float b) { return a + b; }), (float)cols);
    };
    __syncthreads();  // all marks are set
    int at = -1;
#pragma unroll 1
    for (int64_t row = blockIdx.x; row < A.n; row += gridDim.x) {
        at++;
        if (!(mark[at >> 5] >> (at & 31) & 1)) continue;
        float ms = mean(row, 1.0f) + A.eps;
        float most = __fsqrt_rn(A.eps), f = 1.0f;
#pragma unroll 1
        for (int j = 0; j < nch; j++) {
            float h[8];
            load(row, threadIdx.x + j * blockDim.x, h);
#pragma unroll
            for (int i = 0; i < 8; i++) most = fmaxf(most, fabsf(h[i]));
        }
        most = reduce(most, [](float a, float b) { return fmaxf(a, b); });
        if (most > 0.0f && most < __int_as_float(0x7F800000)) {
            f = __int_as_float(max(254 - (__float_as_int(most) >> 23), 1) << 23);
            ms = mean(row, f) + A.eps * f * f;
        }
        const float rs = __frcp_rn(__fsqrt_rn(ms));
#pragma unroll 1
        for (int j = 0; j < nch; j++) {
            const int chunk = threadIdx.x + j * blockDim.x, c = chunk * 8, left = cols - c;
            float h[8], w[8];
            load(row, chunk, h);
            load_chunk<float, VEC>(A.w + c, left, w);
            if (A.sum && left > 0) store_chunk<T, VEC>(static_cast<T *>(A.sum) + row * A.ldsum + c, left, h);
#pragma unroll
            for (int i = 0; i < 8; i++) h[i] *= f;
            norm_out<T, VEC>(A, row, chunk, h, rs, w);
        }
    }
}

// A block walks rows blockIdx.x, blockIdx.x + gridDim.x, ...; thread t holds chunks t, t + blockDim, ... of a row (NCH of them, 8
// columns each). Up to 8192 columns it keeps their weights, and the next row's x and res are in flight while the current one is
// reduced and written; wider rows (NCH = 4, up to 1024 threads of 64 registers) load both when they are due. LATE: sum lies over x or
// res and is written only when it is known that the row is not needed once more.
template <class T, int NCH, bool VEC, bool LATE>
__global__ void __launch_bounds__(NCH > 2 ? 1024 : 512) rmsnorm_q8_kernel(const inzg_rmsnorm_q8_args A) {
    constexpr bool AHEAD = NCH <= 2;
    __shared__ float part[2][32];
    __shared__ uint32_t mark[kNormRows / 32];
    const int cols = A.cols, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
    Chunk<T> x[AHEAD ? NCH : 1], r[AHEAD ? NCH : 1];
    auto load_part = [&](int64_t row, int j, int to) {
        const int c = (threadIdx.x + j * blockDim.x) * 8, left = cols - c;
        load_raw<T, VEC>(static_cast<const T *>(A.x) + row * A.ldx + c, left, x[to]);
        if (A.res) load_raw<T, VEC>(static_cast<const T *>(A.res) + row * A.ldres + c, left, r[to]);
    };
    auto load_row = [&](int64_t row) {
#pragma unroll
        for (int j = 0; j < NCH; j++) load_part(row, j, AHEAD ? j : 0);
    };
    if (AHEAD) load_row(blockIdx.x);
    float w[AHEAD ? NCH : 1][8];
    auto load_w = [&](int j, float(&o)[8]) {
        const int c = (threadIdx.x + j * blockDim.x) * 8;
        load_chunk<float, VEC>(A.w + c, cols - c, o);
    };
    if (AHEAD)
#pragma unroll
        for (int j = 0; j < NCH; j++) load_w(j, w[AHEAD ? j : 0]);
    const int rows = (A.n - 1 - (int)blockIdx.x) / (int)gridDim.x + 1;  // of the block
    for (int i = threadIdx.x; i < (rows + 31) / 32; i += blockDim.x) mark[i] = 0;
    __syncwarp();  // several warps pass a barrier before the first mark
    int flip = 0;
    bool far = false;  // whether one of the block's rows is
    for (int64_t row = blockIdx.x; row < A.n; row += gridDim.x, flip ^= 1) {
        float h[NCH][8], ss = 0.0f;
#pragma unroll
        for (int j = 0; j < NCH; j++) {
            const int jj = AHEAD ? j : 0;
            if (!AHEAD) load_part(row, j, jj);
#pragma unroll
            for (int i = 0; i < 8; i++) {
                h[j][i] = to_f32(x[jj].v[i]);
                if (A.res) h[j][i] += to_f32(r[jj].v[i]);
                ss = fmaf(h[j][i], h[j][i], ss);
            }
        }
        if (AHEAD && row + gridDim.x < A.n) load_row(row + gridDim.x);
        auto store_sum = [&] {
#pragma unroll
            for (int j = 0; j < NCH; j++) {
                const int c = (threadIdx.x + j * blockDim.x) * 8, left = cols - c;
                if (left > 0) store_chunk<T, VEC>(static_cast<T *>(A.sum) + row * A.ldsum + c, left, h[j]);
            }
        };
        if (!LATE && A.sum) store_sum();
#pragma unroll
        for (int d = 16; d; d >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, d);
        if (warps > 1) {
            if (lane == 0) part[flip][warp] = ss;
            __syncthreads();  // the other half of `part` is free: its readers have passed this barrier
            ss = lane < warps ? part[flip][lane] : 0.0f;
#pragma unroll
            for (int d = 16; d; d >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, d);
        }
        const float ms = __fdiv_rn(ss, (float)cols) + A.eps;
        const bool far_row = norm_is_far(ms);  // the same for all threads of the block
        far |= far_row;
        if (far_row && threadIdx.x == 0) {
            const int at = (int)((row - blockIdx.x) / gridDim.x);
            mark[at >> 5] |= 1u << (at & 31);
        }
        if (LATE && !far_row) store_sum();
        const float rs = __frcp_rn(__fsqrt_rn(ms));
#pragma unroll
        for (int j = 0; j < NCH; j++) {
            const int chunk = threadIdx.x + j * blockDim.x, c = chunk * 8, left = cols - c;
            float v[8], (&wj)[8] = w[AHEAD ? j : 0];
            if (!AHEAD) load_w(j, wj);
#pragma unroll
            for (int i = 0; i < 8; i++) v[i] = left > i ? h[j][i] * rs * wj[i] : 0.0f;
            float z[8];  // v without the row's factor
#pragma unroll
            for (int i = 0; i < 8; i++) z[i] = left > i ? h[j][i] * wj[i] : 0.0f;
            if (A.y && left > 0) store_chunk<T, VEC>(static_cast<T *>(A.y) + row * A.ldy + c, left, v);
            if (A.q) {
                float s;
                const uint2 q = quantize_scaled(z, v, rs, s);
                if (left > 0) {
                    store_q<VEC>(static_cast<uint8_t *>(A.q) + row * A.ldq + c, left, q);
                    if ((chunk & 15) == 0) A.s[row * A.lds + (chunk >> 4)] = s;
                }
            }
        }
    }
    if (far) norm_far_rows<T, VEC>(A, part[0], mark);
}

// g / (1 + exp(-g)) of two values, in packed arithmetic. With x = g clamped to 88 and t = x log2 e rounded, exp(-x) =
// 2^-t exp(t ln 2 - x); the last factor is within 2^-17 of 1, so 1 + (t ln 2 - x) stands for it and the relative error stays at a few
// 2^-24 for large |x| too, where 2^-t alone loses |x| * 2^-24. Below -87.3 the divisor passes 2^126 and its estimated reciprocal
// is 0: silu_far is for gates below -87. A NaN passes through the last product.
__device__ __forceinline__ float2 silu2(float2 g) {
    const float2 x = make_float2(fminf(fmaxf(g.x, -88.0f), 88.0f), fminf(fmaxf(g.y, -88.0f), 88.0f));
    const float2 t = __fmul2_rn(x, make_float2(1.4426950408889634f, 1.4426950408889634f));
    const float hi = 0.69314718246459961f, lo = -1.9046542999848e-9f;  // ln 2 = hi + lo
    const float2 r = __ffma2_rn(t, make_float2(-hi, -hi), x);          // x - t hi
    const float2 c = __ffma2_rn(t, make_float2(lo, lo), make_float2(1.0f, 1.0f));
    const float2 m = __ffma2_rn(r, make_float2(-1.0f, -1.0f), c);  // 1 + t ln 2 - x
    float2 e;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e.x) : "f"(-t.x));
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e.y) : "f"(-t.y));
    const float2 d = __ffma2_rn(e, m, make_float2(1.0f, 1.0f));
    return __fmul2_rn(g, make_float2(rcp_approx(d.x), rcp_approx(d.y)));
}

// g exp(g) u, which is g / (1 + exp(-g)) * u to within exp(-87) below -87: two factors take half of the exponential each, which alone
// leaves fp32's normal range there while the product need not (u may be as large as 2^127), and what is below -160 comes last, when the
// product is that small itself. Three exponentials (2 * 2^-24 each), four products.
__device__ __noinline__ float silu_far(float g, float u) {
    const float h = fmaxf(g, -160.0f), e = expf(0.5f * h);
    return (g * e) * (u * e) * expf(g - h);
}

// the least of a chunk, NaN apart
__device__ __forceinline__ float least_of(const Chunk<float> &c) {
    float m = c.v[0];
#pragma unroll
    for (int i = 1; i < 8; i++) m = fminf(m, c.v[i]);
    return m;
}
__device__ __forceinline__ float least_of(const Chunk<__nv_bfloat16> &c) {
    const __nv_bfloat162 *p = reinterpret_cast<const __nv_bfloat162 *>(c.v);
    const __nv_bfloat162 m = __hmin2(__hmin2(p[0], p[1]), __hmin2(p[2], p[3]));
    return __bfloat162float(__hmin(m.x, m.y));
}
__device__ __forceinline__ float least_of(const Chunk<__half> &c) {
    const __half2 *p = reinterpret_cast<const __half2 *>(c.v);
    const __half2 m = __hmin2(__hmin2(p[0], p[1]), __hmin2(p[2], p[3]));
    return __half2float(__hmin(m.x, m.y));
}

// A thread's slot: one chunk of one row; slots per row are rounded up to whole blocks of 128 columns. A thread goes on by
// `step_rows` rows and `step_chunks` chunks, the grid's size in slots, and has the next slot's loads in flight. Four blocks per SM
// (64 registers): 40960 x 640 bf16 26.1 us; 2 blocks 35.9, 3 28.8, 5 27.4, 6 28.0, 8 27.8; four with two slots ahead 29.1. (28.0
// since: 1.3 us for the exact quotient, 0.8 to look for gates below -87.)
constexpr int kSiluBlocks = 4;
constexpr float kSiluFar = -87.0f;
template <class T, bool VEC>
__global__ void __launch_bounds__(256, kSiluBlocks) silu_mul_q8_kernel(const inzg_silu_mul_q8_args A, uint32_t slots, uint32_t per_row,
                                                          uint32_t step_rows, uint32_t step_chunks) {
    const int cols = A.cols;
    uint32_t i = blockIdx.x * blockDim.x + threadIdx.x, row = i / per_row, chunk = i % per_row;
    Chunk<T> g, u;
    auto load = [&] {
        const int c = (int)chunk * 8, left = i < slots ? cols - c : 0;
        const T *x = static_cast<const T *>(A.x) + (int64_t)row * A.ldx + c;
        load_raw<T, VEC>(x, left, g);
        load_raw<T, VEC>(x + cols, left, u);
    };
    load();
    // whole warps stay in the loop: the quantizer shuffles
    while (i - threadIdx.x % 32 < slots) {
        const int c = (int)chunk * 8, left = i < slots ? cols - c : 0;
        const bool first = (chunk & 15) == 0;
        const int64_t r = row, block = chunk >> 4;
        float v[8], gate[8];
#pragma unroll
        for (int j = 0; j < 8; j++) {
            gate[j] = to_f32(g.v[j]);
            v[j] = to_f32(u.v[j]);
        }
        const bool far = least_of(g) < kSiluFar;
        i += gridDim.x * blockDim.x;
        row += step_rows;
        chunk += step_chunks;
        if (chunk >= per_row) {
            chunk -= per_row;
            row++;
        }
        load();
#pragma unroll
        for (int j = 0; j < 8; j += 2) {
            const float2 o = __fmul2_rn(silu2(make_float2(gate[j], gate[j + 1])), make_float2(v[j], v[j + 1]));
            v[j] = o.x;
            v[j + 1] = o.y;
        }
        if (__any_sync(0xffffffffu, far)) {  // seldom: once more from memory
            const T *x = static_cast<const T *>(A.x) + r * A.ldx + c;
#pragma unroll
            for (int j = 0; j < 8; j++)
                if (j < left && to_f32(x[j]) < kSiluFar) v[j] = silu_far(to_f32(x[j]), to_f32(x[cols + j]));
        }
        if (A.y && left > 0) store_chunk<T, VEC>(static_cast<T *>(A.y) + r * A.ldy + c, left, v);
        if (A.q) {
            float s;
            const uint2 q = quantize_chunk<true>(v, s);
            if (left > 0) {
                store_q<VEC>(static_cast<uint8_t *>(A.q) + r * A.ldq + c, left, q);
                if (first) A.s[r * A.lds + block] = s;
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
    const bool vec = A.cols % 8 == 0 && aligned(A.x, A.ldx * b, 16) && aligned(A.res, A.ldres * b, 16) && aligned(A.sum, A.ldsum * b, 16) &&
                     aligned(A.y, A.ldy * b, 16) && aligned(A.q, A.ldq, 8) && aligned(A.w, 0, 16);
    const int chunks = (A.cols + 7) / 8;
    const int nch = chunks <= 512 ? 1 : chunks <= 1024 ? 2 : 4;  // chunks per thread
    const int threads = ((chunks + nch - 1) / nch + 31) / 32 * 32;
    // Blocks per SM: as many as its registers hold with one chunk per thread (up to 64 registers). With two (91 to 112 registers) an SM holds
    // one block of the one to three, and the others come after it.
    const int per_sm = threads > 512 ? 1 : 1024 / threads;
    const int64_t most = (int64_t)num_sms * per_sm * kNormRows;  // rows of a launch
    const bool late = A.sum && A.res && (A.sum == A.x || A.sum == A.res);
#define INZG_NORM(NCH)                                                                                        \
    do {                                                                                                      \
        if (vec && late) rmsnorm_q8_kernel<T, NCH, true, true><<<grid, threads, 0, st>>>(P);                  \
        else if (vec) rmsnorm_q8_kernel<T, NCH, true, false><<<grid, threads, 0, st>>>(P);                    \
        else if (late) rmsnorm_q8_kernel<T, NCH, false, true><<<grid, threads, 0, st>>>(P);                   \
        else rmsnorm_q8_kernel<T, NCH, false, false><<<grid, threads, 0, st>>>(P);                            \
    } while (0)
    int launches = 0;
    for (int64_t done = 0; done < A.n; done += most, launches++) {
        inzg_rmsnorm_q8_args P = A;
        P.n = (int)std::min(A.n - done, most);
        P.x = static_cast<const T *>(A.x) + done * A.ldx;
        if (A.res) P.res = static_cast<const T *>(A.res) + done * A.ldres;
        if (A.sum) P.sum = static_cast<T *>(A.sum) + done * A.ldsum;
        if (A.y) P.y = static_cast<T *>(A.y) + done * A.ldy;
        if (A.q) P.q = static_cast<uint8_t *>(A.q) + done * A.ldq;
        if (A.s) P.s = A.s + done * A.lds;
        const int grid = std::min(P.n, num_sms * per_sm);
        if (nch == 1) INZG_NORM(1);
        else if (nch == 2) INZG_NORM(2);
        else INZG_NORM(4);
    }
#undef INZG_NORM
    return launches;
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
    const bool vec = A.cols % 8 == 0 && aligned(A.x, A.ldx * b, 16) && aligned(A.y, A.ldy * b, 16) &&
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
        const uint32_t want = (slots + 255) / 256, most = (uint32_t)num_sms * kSiluBlocks;
        const uint32_t grid = want < most ? want : most, step = grid * 256;
        if (vec) silu_mul_q8_kernel<T, true><<<grid, 256, 0, st>>>(P, slots, per_row, step / per_row, step % per_row);
        else silu_mul_q8_kernel<T, false><<<grid, 256, 0, st>>>(P, slots, per_row, step / per_row, step % per_row);
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
