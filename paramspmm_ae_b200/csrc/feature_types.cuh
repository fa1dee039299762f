// Element types, vectors and the 8-bit form shared by the operators around the layers
// (rms_norm.cu, rows8.cu, rows8_mm.cu, embedding.cu).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "pspmm_common.cuh"

namespace feat {

typedef __nv_bfloat16 bf16;
typedef __half f16;

constexpr int EIGHT_BLOCK = 128;             // columns that share a scale
constexpr float EIGHT_TINY = 0x1p-119f;      // a / 127 is a normal number and 127 / a is finite from here on

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(bf16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_float(f16 v) { return __half2float(v); }
template <typename T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ float from_float<float>(float v) { return v; }
template <> __device__ __forceinline__ bf16 from_float<bf16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ f16 from_float<f16>(float v) { return __float2half_rn(v); }

// VW neighbouring values, moved by one instruction.
template <typename T, int VW> struct alignas(sizeof(T) * VW) Vec { T v[VW]; };

template <typename T, int VW> __device__ __forceinline__ void load_vec(float (&f)[VW], const T *p)
{
    const Vec<T, VW> u = *reinterpret_cast<const Vec<T, VW> *>(p);
#pragma unroll
    for (int i = 0; i < VW; ++i)
        f[i] = to_float(u.v[i]);
}
template <typename T, int VW> __device__ __forceinline__ void store_vec(T *p, const float (&f)[VW])
{
    Vec<T, VW> u;
#pragma unroll
    for (int i = 0; i < VW; ++i)
        u.v[i] = from_float<T>(f[i]);
    *reinterpret_cast<Vec<T, VW> *>(p) = u;
}

// Two floats side by side in 64 bits, for the packed instructions.
typedef unsigned long long pair_t;
__device__ __forceinline__ pair_t make_pair(float x0, float x1)
{
    pair_t p;
    asm("mov.b64 %0, {%1, %2};" : "=l"(p) : "f"(x0), "f"(x1));
    return p;
}
__device__ __forceinline__ void get_pair(pair_t p, float &x0, float &x1) { asm("mov.b64 {%0, %1}, %2;" : "=f"(x0), "=f"(x1) : "l"(p)); }
__device__ __forceinline__ pair_t add_pair(pair_t a, pair_t b)
{
    pair_t p;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(p) : "l"(a), "l"(b));
    return p;
}
__device__ __forceinline__ pair_t mul_pair(pair_t a, pair_t b)
{
    pair_t p;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(p) : "l"(a), "l"(b));
    return p;
}
__device__ __forceinline__ pair_t sub_pair(pair_t a, pair_t b)
{
    pair_t p;
    asm("sub.rn.f32x2 %0, %1, %2;" : "=l"(p) : "l"(a), "l"(b));
    return p;
}
__device__ __forceinline__ pair_t fma_pair(pair_t a, pair_t b, pair_t c)
{
    pair_t p;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(p) : "l"(a), "l"(b), "l"(c));
    return p;
}

// The larger one; NaN where either is.
__device__ __forceinline__ float max_nan(float a, float b)
{
    float d;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
    return d;
}

// Scale of a block and the factor that takes its values to whole numbers, from the bits of its largest magnitude.  (As bits
// a NaN is larger than an infinity is larger than any number, so one maximum of integers finds all three.)
__device__ __forceinline__ void eight_scale(uint32_t top, float &scale, float &up)
{
    const float a = __uint_as_float(top);
    scale = a / 127.f;
    up = 127.f / a;
    if (a < EIGHT_TINY)
        scale = up = 0.f;
    if (top >= 0x7f800000u) {  // the whole block is returned as NaN
        scale = __int_as_float(0x7fc00000);
        up = 0.f;
    }
}

// The low byte is rint(x * up), ties to even: one rounding, that of the multiply-add.  |x * up| < 128.
__device__ __forceinline__ uint32_t eight_round(float x, float up) { return __float_as_uint(fmaf(x, up, 12582912.f)); }
__device__ __forceinline__ uint32_t eight_round(double x, double up)
{
    return (uint32_t)__double2loint(fma(x, up, 6755399441055744.0));
}
// rint(x * up) from the rounded product, and how far that is from it: what a second number adds to x, 2^-24 of it at most, and the
// product's rounding matter within NEAR_HALF of a half (127 2^-24 and 2^-18 together are a quarter of that).
constexpr float NEAR_HALF = 0x1p-15f;
__device__ __forceinline__ uint32_t eight_round(float x, float up, float &off)
{
    const float z = x * up, m = z + 12582912.f;
    off = fabsf(z - (m - 12582912.f));
    return __float_as_uint(m);
}
// The same for x + low, low what x's rounding left of it.
__device__ __forceinline__ uint32_t eight_round_low(float x, float low, float up)
{
    const float z = x * up, ez = fmaf(low, up, fmaf(x, up, -z));
    const float m = z + 12582912.f;
    const float d = z - (m - 12582912.f);  // from the whole number that z is nearest to; exact, as 1/2 - d is where it matters
    return __float_as_uint(m) + (ez > 0.5f - d ? 1u : 0u) - (ez < -0.5f - d ? 1u : 0u);
}
__device__ __forceinline__ uint32_t pack_bytes(uint32_t a, uint32_t b, uint32_t c, uint32_t d)
{
    return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}

static inline int elem_bytes(int32_t dtype) { return dtype == PSPMM_F32 ? 4 : 2; }
static inline bool dtype_ok(int32_t dtype) { return dtype == PSPMM_F32 || dtype == PSPMM_BF16 || dtype == PSPMM_F16; }
// Whether rows of `ld` elements of `bytes` from p on all start on a multiple of `align` bytes.
static inline bool rows_aligned(const void *p, int64_t ld, int bytes, int align)
{
    return !p || ((uintptr_t)p % align == 0 && (ld * bytes) % align == 0);
}

}  // namespace feat
