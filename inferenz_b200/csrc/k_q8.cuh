// k_q8.cuh -- element access and the block-of-128 e4m3 quantizer shared by the 8-bit floating point operators, sm_100a.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include "../../include/inzg.h"

namespace inzg {

constexpr int kQB = INZG_Q8_BLOCK;  // columns per scale
constexpr float kE4m3Max = 448.0f;
constexpr float kAmaxFloor = 7.888609052210118e-31f;  // 2^-100: keeps the scale and its reciprocal normal numbers

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ void from_f32(float v, float &o) { o = v; }
__device__ __forceinline__ void from_f32(float v, __half &o) { o = __float2half_rn(v); }
__device__ __forceinline__ void from_f32(float v, __nv_bfloat16 &o) { o = __float2bfloat16_rn(v); }

// plain stores that are said to be to global memory (a pointer that passed through shared memory is not known to be); under an
// `if` they become predicated instructions
__device__ __forceinline__ void store_global(float *p, float v) { asm volatile("st.global.f32 [%0], %1;" ::"l"(p), "f"(v) : "memory"); }
__device__ __forceinline__ void store_global(__half *p, __half v) {
    asm volatile("st.global.b16 [%0], %1;" ::"l"(p), "h"(__half_as_ushort(v)) : "memory");
}
__device__ __forceinline__ void store_global(__nv_bfloat16 *p, __nv_bfloat16 v) {
    asm volatile("st.global.b16 [%0], %1;" ::"l"(p), "h"(__bfloat16_as_ushort(v)) : "memory");
}
__device__ __forceinline__ void store_global(uint4 *p, uint4 v) {
    asm volatile("st.global.v4.b32 [%0], {%1, %2, %3, %4};" ::"l"(p), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}

// A thread's chunk: 8 neighbouring elements (16 or 32 bytes), so that a block of 128 columns is 16 lanes of one warp.
template <class T>
struct alignas(16) Chunk {
    T v[8];
};

// the chunk at p as fp32. `left`: elements of the row from p on (what lies behind reads 0). VEC: p is 16-byte aligned and a row a
// multiple of 8 elements, so a chunk lies inside or behind it
template <class T, bool VEC>
__device__ __forceinline__ void load_chunk(const T *p, int left, float (&o)[8]) {
    if (VEC && left >= 8) {
        Chunk<T> c;
#pragma unroll
        for (int i = 0; i < (int)sizeof(c) / 16; i++)
            reinterpret_cast<uint4 *>(&c)[i] = reinterpret_cast<const uint4 *>(p)[i];
#pragma unroll
        for (int i = 0; i < 8; i++) o[i] = to_f32(c.v[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) o[i] = !VEC && i < left ? to_f32(p[i]) : 0.0f;
    }
}

// the same as it lies in memory (behind the row: zeros)
template <class T, bool VEC>
__device__ __forceinline__ void load_raw(const T *p, int left, Chunk<T> &o) {
    if (VEC && left >= 8) {
#pragma unroll
        for (int i = 0; i < (int)sizeof(o) / 16; i++) reinterpret_cast<uint4 *>(&o)[i] = reinterpret_cast<const uint4 *>(p)[i];
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) {
            if (!VEC && i < left) o.v[i] = p[i];
            else from_f32(0.0f, o.v[i]);
        }
    }
}

template <class T, bool VEC>
__device__ __forceinline__ void store_chunk(T *p, int left, const float (&v)[8]) {
    Chunk<T> c;
#pragma unroll
    for (int i = 0; i < 8; i++) from_f32(v[i], c.v[i]);
    if (VEC && left >= 8) {
#pragma unroll
        for (int i = 0; i < (int)sizeof(c) / 16; i++)
            reinterpret_cast<uint4 *>(p)[i] = reinterpret_cast<const uint4 *>(&c)[i];
    } else if (!VEC) {
#pragma unroll
        for (int i = 0; i < 8; i++)
            if (i < left) p[i] = c.v[i];
    }
}

// two fp32 -> two e4m3 (nearest, ties to even, saturating; NaN stays NaN), the first in the low byte
__device__ __forceinline__ uint32_t cvt_e4m3x2(float lo, float hi) {
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
    return r;
}

// max of `least` and |v| over the 16 lanes of a block (every lane of the warp calls it; NaN is dropped)
__device__ __forceinline__ float block_amax(const float (&v)[8], float least) {
    float a = least;
#pragma unroll
    for (int i = 0; i < 8; i++) a = fmaxf(a, fabsf(v[i]));
#pragma unroll
    for (int d = 8; d; d >>= 1) a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, d));
    return a;
}

// a / 448, rounded to nearest: the product with 1 / 448 and one correction by its remainder (an infinity has none)
__device__ __forceinline__ float scale_of(float a) {
    const float t = a * (1.0f / kE4m3Max);
    const float s = fmaf(fmaf(-kE4m3Max, t, a), 1.0f / kE4m3Max, t);
    return s < __int_as_float(0x7F800000) ? s : a;
}

__device__ __forceinline__ float rcp_approx(float x) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

// 8 values as e4m3
__device__ __forceinline__ uint2 e4m3_of(const float (&v)[8]) {
    uint32_t h[4];
#pragma unroll
    for (int i = 0; i < 4; i++) h[i] = cvt_e4m3x2(v[2 * i], v[2 * i + 1]);
    return make_uint2(h[0] | h[1] << 16, h[2] | h[3] << 16);
}

// s = max(max |v|, 2^-100) / 448 over the 16 lanes of a block (every lane of the warp calls it), q = e4m3(v / s) of this lane's 8. EXACT: the
// quotient is the one that a division in fp32 gives: 1 / s is held as a sum of two numbers, good to 2^-45, and v times it is rounded
// once. (For blocks above 2^112 the smaller one is subnormal: within 2^-7 of a step from the middle of two fp32 numbers the quotient may
// be the other one.) 3 of 12.8 million random values had another q with v * (1 / s), 1.3 us
// less in the SiLU of 40960 x 640 bf16 (25.7 us); without EXACT it is that, within 2^-23 of the quotient. fmaxf drops NaN, so the others keep a scale; an infinity makes s
// infinite and every value of the block NaN.
template <bool EXACT>
__device__ __forceinline__ uint2 quantize_chunk(const float (&v)[8], float &s) {
    s = scale_of(block_amax(v, kAmaxFloor));
    // 1 / s: the hardware's estimate and one Newton step (s is a normal number with a normal reciprocal, or infinite)
    float inv = rcp_approx(s), more = 0.0f;
    inv = fmaf(fmaf(-s, inv, 1.0f), inv, inv);
    if (EXACT) {
        inv = __int_as_float(__float_as_int(inv) - 1);  // a step below it, so that `more` is not negative and -0 stays -0
        more = fmaf(-s, inv, 1.0f) * inv;
    }
    float t[8];
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
        const float2 x = make_float2(v[i], v[i + 1]), f = make_float2(inv, inv);
        const float2 o = EXACT ? __ffma2_rn(x, f, __fmul2_rn(x, make_float2(more, more))) : __fmul2_rn(x, f);
        t[i] = o.x;
        t[i + 1] = o.y;
    }
    return e4m3_of(t);
}

// The same for v = z * r with one r > 0 for the row, without r's error in the quotients: v / s = z * (448 / max |z|), the
// factor rounded once. Where that leaves the normal range (and for blocks at the floor) v itself is quantized.
__device__ __forceinline__ uint2 quantize_scaled(const float (&z)[8], const float (&v)[8], float r, float &s) {
    const float a = block_amax(z, 0.0f);
    const bool plain = a > 8.077935669463161e-28f && a < 8.507059173023462e37f && a * r > kAmaxFloor;  // 2^-90, 2^126
    uint2 q = make_uint2(0, 0);
    if (!__all_sync(0xffffffffu, plain)) q = quantize_chunk<false>(v, s);
    if (plain) {
        s = scale_of(a * r);
        const float e = rcp_approx(a), f0 = kE4m3Max * e, f = fmaf(fmaf(-f0, a, kE4m3Max), e, f0);
        float t[8];
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
            const float2 o = __fmul2_rn(make_float2(z[i], z[i + 1]), make_float2(f, f));
            t[i] = o.x;
            t[i + 1] = o.y;
        }
        q = e4m3_of(t);
    }
    return q;
}

template <bool VEC>
__device__ __forceinline__ void store_q(uint8_t *p, int left, uint2 q) {
    if (VEC && left >= 8) {
        *reinterpret_cast<uint2 *>(p) = q;
    } else if (!VEC) {
#pragma unroll
        for (int i = 0; i < 8; i++)
            if (i < left) p[i] = (uint8_t)((i < 4 ? q.x : q.y) >> (8 * (i & 3)));
    }
}

}  // namespace inzg
