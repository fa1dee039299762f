// Activations held in 8 bits: per row and block of 128 columns
//     a = max |x|,   scale = a / 127,   q = rint(x * (127 / a))      (and back: x' = q * scale, |x' - x| <= 0.51 scale)
//
// Whole numbers rather than an 8-bit floating type: its step at the block's largest value is a / 16, here it is a / 127
// everywhere, and the error of a gradient product follows the largest steps.  Products x * (127 / a) are rounded once (fma), so
// the result is what the formula gives in 64 bits from the two 32-bit factors.
//
// Bound by HBM: one pass, a lane group per block, the maximum by shuffles between the group's lanes while the values wait
// in registers.  32,768 x 4,096 bf16: 70 us (5.8 TB/s), back 58 (7.0); 400,000 x 256 fp32: 84 us (6.1 TB/s).  Odd widths are bound by
// their single loads and bytes: 89,251 x 47 fp32 8 us (2.8 TB/s), back 6.
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
    int32_t used;    // dim and the zeros to the next multiple of 16; bytes behind them belong to the caller
};

// LANES lanes share a block; each holds NV vectors of VW neighbouring columns, LANES * VW apart.  CUT = 4 or 2: rows of at most a quarter or
// a half of a block.  Few lanes with many values each take the divisions and shuffles of a scale less often, until a warp's loads
// no longer lie side by side (to 8 bits): bf16, 32,768 x 4,096 8 lanes 80 us, 4 lanes 70, 2 lanes 96, 1,500,000 x 16 4 lanes 51, 2 lanes
// 33; fp32, 600,000 x 64 8 lanes 43, 4 lanes 39; single values (rows that are not aligned), 100,000 x 1,001 32 lanes 125, 16 lanes 109,
// 600,000 x 29 8 lanes 31, 4 lanes 33.
template <int VW, int CUT> struct Shape {
    static constexpr int LANES = VW == 8 ? (CUT == 1 ? 4 : 2) : VW == 4 ? 4 : CUT == 1 ? 16 : 8;
    static constexpr int NV = EIGHT_BLOCK / (LANES * VW * CUT);
};

// Unit (a row's block) of a lane group: 32-bit division where the count admits it (64-bit division was half of the odd widths' instructions).
__device__ __forceinline__ int64_t unit_row(const Rows8Args &a, int64_t unit, int &block)
{
    if (a.blocks == 1) {
        block = 0;
        return unit;
    }
    if (a.units <= UINT32_MAX) {
        const uint32_t row = (uint32_t)unit / (uint32_t)a.blocks;
        block = (int)((uint32_t)unit - row * (uint32_t)a.blocks);
        return row;
    }
    const int64_t row = unit / a.blocks;
    block = (int)(unit - row * a.blocks);
    return row;
}

template <int VW> __device__ __forceinline__ void store_bytes(int8_t *q, const uint32_t (&b)[VW])
{
    if constexpr (VW == 8)
        *reinterpret_cast<uint2 *>(q) = make_uint2(pack_bytes(b[0], b[1], b[2], b[3]), pack_bytes(b[4], b[5], b[6], b[7]));
    else if constexpr (VW == 4)
        *reinterpret_cast<uint32_t *>(q) = pack_bytes(b[0], b[1], b[2], b[3]);
    else
        *q = (int8_t)b[0];
}

template <typename T, int VW, int CUT>
__global__ void __launch_bounds__(256) quantize_kernel(const Rows8Args a)
{
    using S = Shape<VW, CUT>;
    const int lane = threadIdx.x % S::LANES;
    const int64_t unit = ((int64_t)blockIdx.x * 256 + threadIdx.x) / S::LANES;
    if (unit >= a.units)
        return;
    int block;
    const int64_t row = unit_row(a, unit, block);
    const int c0 = block * EIGHT_BLOCK + lane * VW;
    const T *x = static_cast<const T *>(a.x) + row * a.ld;
    float f[S::NV][VW];
#pragma unroll
    for (int v = 0; v < S::NV; ++v) {
        const int c = c0 + v * S::LANES * VW;
        if (c < a.dim) {  // (a whole vector: dim is a multiple of VW)
            load_vec<T, VW>(f[v], x + c);
        } else {
#pragma unroll
            for (int i = 0; i < VW; ++i)
                f[v][i] = 0.f;
        }
    }
    float most = 0.f;
#pragma unroll
    for (int v = 0; v < S::NV; ++v)
#pragma unroll
        for (int i = 0; i < VW; ++i)
            most = max_nan(most, fabsf(f[v][i]));
    uint32_t top = __float_as_uint(most);
    const uint32_t mask = ((1u << S::LANES) - 1) << (threadIdx.x % 32 / S::LANES * S::LANES);
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
        const int c = c0 + v * S::LANES * VW;
        if (c >= a.used)
            break;
        uint32_t b[VW];
#pragma unroll
        for (int i = 0; i < VW; ++i)
            b[i] = eight_round(f[v][i], up);
        store_bytes<VW>(q + c, b);
    }
}

template <typename T, int VW, int CUT>
__global__ void __launch_bounds__(256) dequantize_kernel(const Rows8Args a)
{
    using S = Shape<VW, CUT>;
    const int lane = threadIdx.x % S::LANES;
    const int64_t unit = ((int64_t)blockIdx.x * 256 + threadIdx.x) / S::LANES;
    if (unit >= a.units)
        return;
    int block;
    const int64_t row = unit_row(a, unit, block);
    const int c0 = block * EIGHT_BLOCK + lane * VW;
    const float scale = a.scales[unit];
    const int8_t *q = a.q + row * a.pitch;
    T *out = static_cast<T *>(const_cast<void *>(a.x)) + row * a.ld;
    uint32_t w[S::NV][(VW + 3) / 4] = {};
#pragma unroll
    for (int v = 0; v < S::NV; ++v) {
        const int c = c0 + v * S::LANES * VW;
        if (c < a.dim) {
            if constexpr (VW == 8) {
                const uint2 u = *reinterpret_cast<const uint2 *>(q + c);
                w[v][0] = u.x;
                w[v][1] = u.y;
            } else if constexpr (VW == 4) {
                w[v][0] = *reinterpret_cast<const uint32_t *>(q + c);
            } else {
                w[v][0] = *reinterpret_cast<const uint8_t *>(q + c);
            }
        }
    }
#pragma unroll
    for (int v = 0; v < S::NV; ++v) {
        const int c = c0 + v * S::LANES * VW;
        float f[VW];
#pragma unroll
        for (int i = 0; i < VW; ++i)
            f[i] = (float)(int8_t)(w[v][i / 4] >> (8 * (i % 4))) * scale;
        if (c < a.dim)
            store_vec<T, VW>(out + c, f);
    }
}

template <typename T, int VW, int CUT>
cudaError_t launch_cut(bool quantize, const Rows8Args &a, cudaStream_t st)
{
    const int64_t ctas = (a.units * Shape<VW, CUT>::LANES + 255) / 256;
    if (quantize)
        quantize_kernel<T, VW, CUT><<<(unsigned)ctas, 256, 0, st>>>(a);
    else
        dequantize_kernel<T, VW, CUT><<<(unsigned)ctas, 256, 0, st>>>(a);
    return cudaGetLastError();
}

template <typename T, int VW> cudaError_t launch(bool quantize, const Rows8Args &a, cudaStream_t st)
{
    return a.dim <= EIGHT_BLOCK / 4   ? launch_cut<T, VW, 4>(quantize, a, st)
           : a.dim <= EIGHT_BLOCK / 2 ? launch_cut<T, VW, 2>(quantize, a, st)
                                      : launch_cut<T, VW, 1>(quantize, a, st);
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
    const int64_t units = n * blocks;
    if (pitch > INT32_MAX || dim > INT32_MAX - 8192 || n > ((int64_t)INT32_MAX * 8) / blocks)  // (a CTA takes 16 at least)
        return PSPMM_E_RANGE;
    Rows8Args a = {x, q, scales, n, ld, units, dim, (int32_t)pitch, (int32_t)blocks, (dim + 15) / 16 * 16};
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
