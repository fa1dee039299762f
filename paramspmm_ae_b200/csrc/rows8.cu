// Activations held in 8 bits: per row and block of 128 columns
//     a = max |x|,   scale = a / 127,   q = rint(x * (127 / a))      (and back: x' = q * scale, |x' - x| <= 0.51 scale)
//
// Whole numbers rather than an 8-bit floating type: its step at the block's largest value is a / 16, here it is a / 127
// everywhere, and the error of a gradient product follows the largest steps.  Products x * (127 / a) are rounded once (fma), so
// the result is what the formula gives in 64 bits from the two 32-bit factors.
//
// Bound by HBM: one pass, a lane group per block, the maximum by shuffles between the group's lanes while the values wait
// in registers.
#include "feature_types.cuh"

namespace {
using namespace feat;

struct Rows8Args {
    const void *x;   // quantise: input; dequantise: output
    int8_t *q;
    float *scales;
    int64_t n, ld;
    int64_t units;   // n * blocks
    int32_t dim, pitch, blocks;
};

// LANES lanes share a block; each holds NV vectors of VW neighbouring columns, LANES * VW apart.  VW < 4: the lane's
// four neighbouring columns come by loads of single values (rows that are not aligned), so that bytes leave as words.
template <typename T, int VW> struct Shape {
    static constexpr int COLS = VW < 4 ? 4 : VW;      // neighbouring columns of a lane
    static constexpr int LANES = VW < 4 ? 32 : 8;
    static constexpr int NV = EIGHT_BLOCK / (LANES * COLS);
};

template <typename T, int VW>
__device__ __forceinline__ void load_cols(float (&f)[Shape<T, VW>::COLS], const T *p, int left)
{
    constexpr int COLS = Shape<T, VW>::COLS;
    if constexpr (VW < 4) {
#pragma unroll
        for (int i = 0; i < COLS; ++i)
            f[i] = i < left ? to_float(p[i]) : 0.f;
    } else {
        if (left > 0) {  // (a whole vector: dim is a multiple of VW)
            load_vec<T, VW>(f, p);
        } else {
#pragma unroll
            for (int i = 0; i < COLS; ++i)
                f[i] = 0.f;
        }
    }
}

template <typename T, int VW>
__global__ void __launch_bounds__(256) quantize_kernel(const Rows8Args a)
{
    using S = Shape<T, VW>;
    const int lane = threadIdx.x % S::LANES;
    const int64_t unit = ((int64_t)blockIdx.x * 256 + threadIdx.x) / S::LANES;
    if (unit >= a.units)
        return;
    const int64_t row = unit / a.blocks;
    const int c0 = (int)(unit % a.blocks) * EIGHT_BLOCK + lane * S::COLS;
    const T *x = static_cast<const T *>(a.x) + row * a.ld;
    float f[S::NV][S::COLS];
#pragma unroll
    for (int v = 0; v < S::NV; ++v)
        load_cols<T, VW>(f[v], x + c0 + v * S::LANES * S::COLS, a.dim - (c0 + v * S::LANES * S::COLS));
    uint32_t top = 0;
#pragma unroll
    for (int v = 0; v < S::NV; ++v)
#pragma unroll
        for (int i = 0; i < S::COLS; ++i)
            top = max(top, __float_as_uint(f[v][i]) & 0x7fffffffu);
    const uint32_t mask = S::LANES == 32 ? PSPMM_FULL_MASK : ((1u << S::LANES) - 1) << (threadIdx.x % 32 / S::LANES * S::LANES);
#pragma unroll
    for (int d = S::LANES / 2; d > 0; d >>= 1)
        top = max(top, __shfl_xor_sync(mask, top, d));
    float scale, up;
    eight_scale(top, scale, up);
    if (lane == 0)
        a.scales[unit] = scale;
    int8_t *q = a.q + row * a.pitch;
#pragma unroll
    for (int v = 0; v < S::NV; ++v) {
        const int c = c0 + v * S::LANES * S::COLS;
        if (c >= a.pitch)  // (the pitch is a multiple of 16; columns between dim and it are zeros)
            break;
        uint32_t w[S::COLS / 4];
#pragma unroll
        for (int i = 0; i < S::COLS / 4; ++i) {
            uint32_t b[4];
#pragma unroll
            for (int j = 0; j < 4; ++j)
                b[j] = eight_round(f[v][4 * i + j], up);
            w[i] = pack_bytes(b[0], b[1], b[2], b[3]);
        }
        if constexpr (S::COLS == 8)
            *reinterpret_cast<uint2 *>(q + c) = make_uint2(w[0], w[1]);
        else
            *reinterpret_cast<uint32_t *>(q + c) = w[0];
    }
}

template <typename T, int VW>
__global__ void __launch_bounds__(256) dequantize_kernel(const Rows8Args a)
{
    using S = Shape<T, VW>;
    const int lane = threadIdx.x % S::LANES;
    const int64_t unit = ((int64_t)blockIdx.x * 256 + threadIdx.x) / S::LANES;
    if (unit >= a.units)
        return;
    const int64_t row = unit / a.blocks;
    const int c0 = (int)(unit % a.blocks) * EIGHT_BLOCK + lane * S::COLS;
    const float scale = a.scales[unit];
    const int8_t *q = a.q + row * a.pitch;
    T *out = static_cast<T *>(const_cast<void *>(a.x)) + row * a.ld;
    uint32_t w[S::NV][S::COLS / 4] = {};
#pragma unroll
    for (int v = 0; v < S::NV; ++v) {
        const int c = c0 + v * S::LANES * S::COLS;
        if (c < a.pitch) {
            if constexpr (S::COLS == 8) {
                const uint2 u = *reinterpret_cast<const uint2 *>(q + c);
                w[v][0] = u.x;
                w[v][1] = u.y;
            } else {
                w[v][0] = *reinterpret_cast<const uint32_t *>(q + c);
            }
        }
    }
#pragma unroll
    for (int v = 0; v < S::NV; ++v) {
        const int c = c0 + v * S::LANES * S::COLS;
        float f[S::COLS];
#pragma unroll
        for (int i = 0; i < S::COLS; ++i)
            f[i] = (float)(int8_t)(w[v][i / 4] >> (8 * (i % 4))) * scale;
        if constexpr (VW < 4) {
#pragma unroll
            for (int i = 0; i < S::COLS; ++i)
                if (c + i < a.dim)
                    out[c + i] = from_float<T>(f[i]);
        } else if (c < a.dim) {
            store_vec<T, VW>(out + c, f);
        }
    }
}

template <typename T, int VW>
cudaError_t launch(bool quantize, const Rows8Args &a, cudaStream_t st)
{
    const int64_t ctas = (a.units * Shape<T, VW>::LANES + 255) / 256;
    if (quantize)
        quantize_kernel<T, VW><<<(unsigned)ctas, 256, 0, st>>>(a);
    else
        dequantize_kernel<T, VW><<<(unsigned)ctas, 256, 0, st>>>(a);
    return cudaGetLastError();
}

// Widest loads that the rows admit: 16 bytes, 8 bytes for 16-bit types, single values.
template <typename T>
cudaError_t launch_typed(bool quantize, const Rows8Args &a, cudaStream_t st)
{
    constexpr int WIDE = 16 / sizeof(T);
    if (a.dim % WIDE == 0 && rows_aligned(a.x, a.ld, sizeof(T), 16))
        return launch<T, WIDE>(quantize, a, st);
    if constexpr (sizeof(T) == 2)
        if (a.dim % 4 == 0 && rows_aligned(a.x, a.ld, sizeof(T), 8))
            return launch<T, 4>(quantize, a, st);
    return launch<T, 1>(quantize, a, st);
}

int rows8_run(bool quantize, const void *x, int32_t dtype, int64_t ld, int64_t n, int32_t dim, int8_t *q, int64_t pitch,
              float *scales, void *stream)
{
    if (!dtype_ok(dtype) || n < 0 || dim < 1 || ld < dim || pitch < dim || pitch % 16 != 0)
        return PSPMM_E_ARG;
    if (n == 0)
        return PSPMM_OK;
    if (!x || !q || !scales || (uintptr_t)q % 16 != 0 || (uintptr_t)scales % 4 != 0 || (uintptr_t)x % elem_bytes(dtype) != 0)
        return PSPMM_E_ARG;
    const int64_t blocks = ((int64_t)dim + EIGHT_BLOCK - 1) / EIGHT_BLOCK;
    // (bytes of q between the last column's 16 and a longer pitch belong to the caller)
    const int64_t units = n * blocks;
    if (pitch > INT32_MAX || n > ((int64_t)INT32_MAX * 8) / blocks)  // CTAs of eight blocks
        return PSPMM_E_RANGE;
    Rows8Args a = {x, q, scales, n, ld, units, dim, (int32_t)pitch, (int32_t)blocks};
    cudaError_t e = dtype == PSPMM_F32    ? launch_typed<float>(quantize, a, (cudaStream_t)stream)
                    : dtype == PSPMM_BF16 ? launch_typed<bf16>(quantize, a, (cudaStream_t)stream)
                                          : launch_typed<f16>(quantize, a, (cudaStream_t)stream);
    PSPMM_CUDA_TRY(e);
    return PSPMM_OK;
}

}  // namespace

extern "C" int pspmm_quantize_rows(const void *x, int32_t dtype, int64_t ldx, int64_t n, int32_t dim, int8_t *q, int64_t pitch,
                                   float *scales, void *stream)
{
    return rows8_run(true, x, dtype, ldx, n, dim, q, pitch, scales, stream);
}

extern "C" int pspmm_dequantize_rows(const int8_t *q, int64_t pitch, const float *scales, int32_t dtype, void *out, int64_t ld_out,
                                     int64_t n, int32_t dim, void *stream)
{
    return rows8_run(false, out, dtype, ld_out, n, dim, const_cast<int8_t *>(q), pitch, const_cast<float *>(scales), stream);
}
