// Root-mean-square norm of a residual stream, forward and backward:
//     h = x + r,   rstd = (mean_j h_j^2 + eps)^-1/2,   y_j = h_j rstd w_j   (relu: negative y become 0)
//     g = dy w [y > 0],   n = h rstd,   dx = rstd (g - n mean_j(g_j n_j)) + dh,   dw_j = sum over rows of dy_j [y > 0] n_j
// and, where asked for, y in 8 bits (rows8.cu's form) from the same pass.
//
// Bound by HBM: every array is moved once.  A row is held in the registers of its lanes between the sum and its use: 2 to 32
// lanes (several rows per warp) with up to 24 values each (16 in the backward), a CTA of as many warps as the row needs beyond that, and two passes over a
// row wider than 8,192 columns.  Rows of a CTA wait at a barrier between their sum and its use, so each asks for the row after the next
// to be brought to L2.  x + r -> h, y in us (TB/s), alone, with y in 8 bits beside, and backward: 169,343 x 128 fp32 60 (5.8), 64, 61;
// 16,384 x 4,096 bf16 90 (6.0), 145, 105; single values, 30,000 x 2,047 fp32 172 (5.7), 219, 186, 400,000 x 250 bf16 201 (4.0), 344, 270.  The 8-bit forms of
// wide rows are bound by instructions: 43 per value and thread, 57 % of issue slots.  (Measured and left: rows brought to shared memory by bulk copies, several in
// flight per CTA, one more pass of instructions over every value, bf16 127, 210, 159; second numbers for the values next to a half
// and the largest ones alone, from memory again, which was 15 % slower than all of them from registers.)
//
// Numbers: the sum of h^2 has the bits of a 64-bit one but for what a 32-bit sum of 2^-24 of it loses; rstd is kept in 32 bits for the
// backward, whose sums are in 32 bits.  y in 8 bits is taken from a y with twice the bits of a 32-bit one, because next to a half the last bit
// of that decides which whole number it becomes; y itself is the 32-bit one with and without it.  Those bits are a second
// 32-bit number (values below 1e-30 have fewer): in 64-bit numbers the norm of 169,343 x 128 took 92 us, most of it conversions, of
// which an SM does 16 per clock.
#include "feature_types.cuh"

namespace {
using namespace feat;

struct NormArgs {
    const void *x, *r, *w;
    void *h, *y;      // either may be null
    float *rstd;
    int8_t *q;        // null: no 8-bit form
    float *scales;
    int64_t n, ld_x, ld_r, ld_h, ld_y;
    double eps;
    int32_t dim, pitch, blocks, relu;
    int32_t used;     // columns of q that are written: dim and the zeros to the next multiple of 16
};

struct NormBackArgs {
    const void *dy, *h, *w, *dh;  // dh may be null
    const float *rstd;
    void *dx;
    float *part;      // [grid][dim]
    int64_t n, ld_dy, ld_h, ld_dh, ld_dx;
    int32_t dim, relu;
};

struct WeightArgs {
    const float *part;
    void *dw;
    int32_t parts, dim, dtype;
};

constexpr int AHEAD = 2;  // rows of a lane group that are brought to L2

// TPR threads share a row; each holds VPT vectors of VW values.  TPR > 32: a CTA's threads, as many warps of the TPR / 32 as the row needs.
template <int TPR> struct Rows {
    static constexpr int MOST = TPR <= 32 ? 256 : TPR;  // threads of a CTA
    static constexpr int PER_CTA = TPR <= 32 ? 256 / TPR : 1;
    static constexpr int LANES = TPR <= 32 ? TPR : 32;  // of a warp that share a row
};

// Column of a thread's vector v: a warp's lanes side by side, a warp's vectors behind one another (so that the 128 columns of
// a scale never leave a warp).
template <int VW, int TPR, int VPT> __device__ __forceinline__ int column(int t, int v)
{
    constexpr int L = Rows<TPR>::LANES;
    return ((t / L * VPT + v) * L + t % L) * VW;
}

template <typename T, int VW> __device__ __forceinline__ void load_some(float (&f)[VW], const T *p, bool in)
{
    if (in) {
        load_vec<T, VW>(f, p);
    } else {
#pragma unroll
        for (int i = 0; i < VW; ++i)
            f[i] = 0.f;
    }
}

// A thread's values in pairs, for the packed instructions (half of what single ones take to issue).
template <int N, int VW> __device__ __forceinline__ float &at(float (&m)[N][VW], int e) { return m[e / VW][e % VW]; }
template <int N, int VW> __device__ __forceinline__ pair_t pair_of(float (&m)[N][VW], int e) { return make_pair(at(m, e), at(m, e + 1)); }
template <int N, int VW> __device__ __forceinline__ void set_pair(float (&m)[N][VW], int e, pair_t p)
{
    get_pair(p, at(m, e), at(m, e + 1));
}

template <typename S, int LANES> __device__ __forceinline__ S lanes_sum(S v, uint32_t mask)
{
#pragma unroll
    for (int d = LANES / 2; d > 0; d >>= 1)
        v += __shfl_xor_sync(mask, v, d);
    return v;
}

// Sums of a CTA's warps: two sets in turn, so that a row needs one barrier (the next row's sums leave this row's alone, and the one
// after that begins behind the next row's barrier).  What no warp writes stays 0.
template <typename S, int WARPS> struct WarpSums {
    S set[2][WARPS];
    __device__ __forceinline__ void clear()
    {
        for (int i = threadIdx.x; i < (int)(sizeof(set) / sizeof(S)); i += blockDim.x)
            set[0][i] = 0;
        __syncthreads();
    }
};

// Sum over a row's threads; `turn` alternates from row to row.
template <typename S, int TPR, int WARPS> __device__ __forceinline__ S row_sum(S v, uint32_t mask, WarpSums<S, WARPS> &sums, int &turn)
{
    v = lanes_sum<S, Rows<TPR>::LANES>(v, mask);
    if constexpr (TPR > 32) {
        S *set = sums.set[turn];
        turn ^= 1;
        if (threadIdx.x % 32 == 0)
            set[threadIdx.x / 32] = v;
        __syncthreads();
        S p[4] = {};
#pragma unroll
        for (int i = 0; i < WARPS; ++i)
            p[i % 4] += set[i];
        v = (p[0] + p[1]) + (p[2] + p[3]);
    }
    return v;
}

__device__ __forceinline__ uint32_t group_mask(int lanes)
{
    return lanes == 32 ? PSPMM_FULL_MASK : ((1u << lanes) - 1) << (threadIdx.x % 32 / lanes * lanes);
}

// 1 / sqrt(m) in 64 bits: the 32-bit one and two steps of Newton's, which double its correct bits (the library's quotient of a root
// took a third of the narrow rows' time).  Outside the 32-bit numbers' range, the library's.
__device__ __forceinline__ double inverse_root(double m)
{
    if (!(m > 1e-30 && m < 1e30))
        return 1.0 / sqrt(m);
    double r = (double)rsqrtf((float)m);
#pragma unroll
    for (int i = 0; i < 2; ++i)
        r = fma(r * 0.5, fma(-m * r, r, 1.0), r);
    return r;
}

// A row to come is brought to L2, so that its loads wait for that and not for memory.
__device__ __forceinline__ void look_ahead(const void *row, int bytes)
{
    const uintptr_t from = ((uintptr_t)row + 15) / 16 * 16, to = ((uintptr_t)row + bytes) / 16 * 16;
    if (from < to)
        asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(from), "r"((uint32_t)(to - from)) : "memory");
}

// CTAs per SM that a kernel's registers leave room for (left to itself the compiler takes more registers than its loads repay in the lane
// groups: 400,000 x 250 bf16 236 us against 205).
constexpr int ctas_for(int tpr, int values, bool eight)
{
    return tpr > 32 ? 1 : values <= 4 ? 5 - eight : values <= 8 ? 4 - eight : 2;
}

template <typename T, int VW, int TPR, int VPT, bool EIGHT>
__global__ void __launch_bounds__(Rows<TPR>::MOST, ctas_for(TPR, VW * VPT, EIGHT)) norm_kernel(const NormArgs a)
{
    using R = Rows<TPR>;
    __shared__ __align__(16) WarpSums<double, R::MOST / 32> sums;
    int turn = 0;
    if (TPR > 32)
        sums.clear();
    const int t = TPR > 32 ? threadIdx.x : threadIdx.x % R::LANES;
    const uint32_t mask = group_mask(R::LANES);
    float w[VPT][VW];
#pragma unroll
    for (int v = 0; v < VPT; ++v) {
        const int c = column<VW, TPR, VPT>(t, v);
        load_some<T, VW>(w[v], static_cast<const T *>(a.w) + c, c < a.dim);
    }
    const float least = a.relu ? 0.f : -__int_as_float(0x7f800000);
    const int64_t step = (int64_t)gridDim.x * R::PER_CTA;
    for (int64_t row = (int64_t)blockIdx.x * R::PER_CTA + (TPR > 32 ? 0 : threadIdx.x / R::LANES); row < a.n; row += step) {
        // Without r, zeros are added all the same (16,384 x 4,096 bf16 102 us with a test per value, 92 without) but where
        // registers are short and the test leaves more warps: 400,000 x 250 bf16 304 us against 215.
        constexpr bool ALWAYS = VW > 1 || (TPR > 32 && TPR < 1024);
        constexpr int VALUES = VPT * VW;
        static_assert(VALUES % 2 == 0, "values are worked on in pairs");
        float h[VPT][VW], low[VPT][VW];  // x + r in 32 bits, and what that leaves of the residual until it is added
#pragma unroll
        for (int v = 0; v < VPT; ++v) {
            const int c = column<VW, TPR, VPT>(t, v);
            load_some<T, VW>(h[v], static_cast<const T *>(a.x) + row * a.ld_x + c, c < a.dim);
        }
        if (VW > 1 || a.r) {
#pragma unroll
            for (int v = 0; v < VPT; ++v) {
                const int c = column<VW, TPR, VPT>(t, v);
                load_some<T, VW>(low[v], static_cast<const T *>(a.r) + row * a.ld_r + c, a.r && c < a.dim);
            }
        } else {
#pragma unroll
            for (int v = 0; v < VPT; ++v)
#pragma unroll
                for (int i = 0; i < VW; ++i)
                    low[v][i] = 0.f;
        }
        if (TPR > 32 && t == 0 && row + AHEAD * step < a.n) {
            look_ahead(static_cast<const T *>(a.x) + (row + AHEAD * step) * a.ld_x, a.dim * (int)sizeof(T));
            if (a.r)
                look_ahead(static_cast<const T *>(a.r) + (row + AHEAD * step) * a.ld_r, a.dim * (int)sizeof(T));
        }
        // The sum of (h + low)^2, h = x + r rounded and low the exact remainder (Knuth's): h^2 in 64 bits and h low, 2^-24 of it, in 32.  (Both
        // addends in 64 bits: two conversions per value, of which an SM does 16 per clock; 16,384 x 4,096 bf16 116 us against 102.)
        double ss = 0;
        pair_t crosses = 0;
#pragma unroll
        for (int e = 0; e < VALUES; e += 2) {
            if (ALWAYS || a.r) {
                const pair_t x = pair_of(h, e), r = pair_of(low, e), sum = add_pair(x, r), b = sub_pair(sum, x);
                const pair_t rest = add_pair(sub_pair(x, sub_pair(sum, b)), sub_pair(r, b));
                crosses = fma_pair(sum, rest, crosses);
                set_pair(h, e, sum);
                set_pair(low, e, rest);
            }
            const double h0 = at(h, e), h1 = at(h, e + 1);
            ss = fma(h1, h1, fma(h0, h0, ss));
        }
        float cross, cross1;
        get_pair(crosses, cross, cross1);
        cross += cross1;
        if (fabsf(cross) < __int_as_float(0x7f800000)) {
            ss = fma(2.0, (double)cross, ss);
        } else {  // beyond the 32-bit numbers' range, or an infinity (whose remainder is none) or a NaN among the row
#pragma unroll
            for (int v = 0; v < VPT; ++v)
#pragma unroll
                for (int i = 0; i < VW; ++i)
                    if (fabsf(low[v][i]) < __int_as_float(0x7f800000))
                        ss = fma(2.0 * (double)h[v][i], (double)low[v][i], ss);
        }
        if (a.h) {
#pragma unroll
            for (int v = 0; v < VPT; ++v) {
                const int c = column<VW, TPR, VPT>(t, v);
                if (c < a.dim)
                    store_vec<T, VW>(static_cast<T *>(a.h) + row * a.ld_h + c, h[v]);
            }
        }
        ss = row_sum<double, TPR>(ss, mask, sums, turn);
        const double rstd64 = inverse_root(ss / a.dim + a.eps);
        const float rstd = (float)rstd64;
        if (t == 0)
            a.rstd[row] = rstd;
        if (a.y) {
#pragma unroll
            for (int v = 0; v < VPT; ++v) {
                const int c = column<VW, TPR, VPT>(t, v);
                float y[VW];
                if constexpr (VW == 1) {
                    y[0] = max_nan(h[v][0] * rstd * w[v][0], least);
                } else {
#pragma unroll
                    for (int i = 0; i < VW; i += 2) {
                        get_pair(mul_pair(mul_pair(pair_of(h, v * VW + i), make_pair(rstd, rstd)), pair_of(w, v * VW + i)), y[i], y[i + 1]);
                        y[i] = max_nan(y[i], least);
                        y[i + 1] = max_nan(y[i + 1], least);
                    }
                }
                if (c < a.dim)
                    store_vec<T, VW>(static_cast<T *>(a.y) + row * a.ld_y + c, y);
            }
        }
        if constexpr (EIGHT) {
            // (h + low) rstd w as a sum of two 32-bit numbers, the first the sum rounded: products and what their rounding leaves (fma).
            // A row whose rstd is no number (NaN, or infinite) takes 0 in its place, so that the columns behind it stay zeros, and a NaN
            // among the magnitudes of each block.
            const bool number = rstd < __int_as_float(0x7f800000);
            const float by1 = number ? rstd : 0.f, rest = number ? (float)(rstd64 - rstd) : 0.f, none = number ? 0.f : __int_as_float(0x7fc00000);
            const pair_t by = make_pair(by1, by1), by_less = make_pair(-by1, -by1), by_rest = make_pair(rest, rest);
#pragma unroll
            for (int e = 0; e < VALUES; e += 2) {
                const pair_t x = pair_of(h, e), f = pair_of(w, e), n = mul_pair(x, by), less_n = mul_pair(x, by_less);
                const pair_t en = fma_pair(pair_of(low, e), by, fma_pair(x, by_rest, fma_pair(x, by, less_n)));
                const pair_t less_y = mul_pair(less_n, f), ey = fma_pair(en, f, fma_pair(n, f, less_y));
                const pair_t y = sub_pair(ey, less_y);
                set_pair(low, e, sub_pair(ey, add_pair(less_y, y)));
                set_pair(h, e, y);
                at(h, e) = max_nan(at(h, e), least);  // (the second number of a value cut to 0 is not looked at)
                at(h, e + 1) = max_nan(at(h, e + 1), least);
            }
            // A block is LB lanes wide and SB vectors deep.
            constexpr int LB = R::LANES * VW >= EIGHT_BLOCK ? EIGHT_BLOCK / VW : R::LANES;
            constexpr int DEEP = EIGHT_BLOCK / (LB * VW), SB = DEEP < VPT ? DEEP : VPT;
            static_assert(VPT % SB == 0 || R::PER_CTA > 1, "a block spans warps");
            int8_t *q = a.q + row * a.pitch;
#pragma unroll
            for (int v0 = 0; v0 < VPT; v0 += SB) {
                float most = none;
#pragma unroll
                for (int v = v0; v < v0 + SB && v < VPT; ++v)
#pragma unroll
                    for (int i = 0; i < VW; ++i)
                        most = max_nan(most, fabsf(h[v][i]));
                uint32_t top = __float_as_uint(most);
#pragma unroll
                for (int d = LB / 2; d > 0; d >>= 1)
                    top = max(top, __shfl_xor_sync(mask, top, d));
                float scale, up;
                eight_scale(top, scale, up);
                const int first = column<VW, TPR, VPT>(t, v0);
                if (first % EIGHT_BLOCK == 0 && first < a.dim)
                    a.scales[row * a.blocks + first / EIGHT_BLOCK] = scale;
#pragma unroll
                for (int v = v0; v < v0 + SB && v < VPT; ++v) {
                    const int c = column<VW, TPR, VPT>(t, v);
                    uint32_t b[VW];
                    float off[VW], most_off = 0.f;  // (fmaxf leaves out the NaN of a block without a scale)
#pragma unroll
                    for (int i = 0; i < VW; ++i) {
                        b[i] = eight_round(h[v][i], up, off[i]);
                        most_off = fmaxf(most_off, off[i]);
                    }
                    if (most_off > 0.5f - NEAR_HALF) {  // one value in 2^14
#pragma unroll
                        for (int i = 0; i < VW; ++i)
                            if (off[i] > 0.5f - NEAR_HALF)
                                b[i] = eight_round_low(h[v][i], low[v][i], up);
                    }
                    if (c < a.used) {
                        if constexpr (VW == 8)
                            *reinterpret_cast<uint2 *>(q + c) =
                                make_uint2(pack_bytes(b[0], b[1], b[2], b[3]), pack_bytes(b[4], b[5], b[6], b[7]));
                        else if constexpr (VW == 4)
                            *reinterpret_cast<uint32_t *>(q + c) = pack_bytes(b[0], b[1], b[2], b[3]);
                        else
                            q[c] = (int8_t)b[0];
                    }
                }
            }
        }
    }
}

// Rows of any width: a CTA per row, two passes, 64-bit numbers.
template <typename T, bool EIGHT>
__global__ void __launch_bounds__(1024) norm_wide_kernel(const NormArgs a)
{
    __shared__ __align__(16) WarpSums<double, 32> sums;
    int turn = 0;
    sums.clear();
    const T *w = static_cast<const T *>(a.w);
    for (int64_t row = blockIdx.x; row < a.n; row += gridDim.x) {
        const T *x = static_cast<const T *>(a.x) + row * a.ld_x;
        const T *r = a.r ? static_cast<const T *>(a.r) + row * a.ld_r : nullptr;
        double ss = 0;
        for (int c = threadIdx.x; c < a.dim; c += 1024) {
            const double h = r ? (double)to_float(x[c]) + (double)to_float(r[c]) : (double)to_float(x[c]);
            ss = fma(h, h, ss);
        }
        ss = row_sum<double, 1024>(ss, PSPMM_FULL_MASK, sums, turn);
        const double rstd64 = inverse_root(ss / a.dim + a.eps);
        const float rstd = (float)rstd64;
        if (threadIdx.x == 0)
            a.rstd[row] = rstd;
        // A warp takes 128 neighbouring columns at a time, a lane four of them.
        for (int c0 = threadIdx.x * 4; c0 < (a.dim + EIGHT_BLOCK - 1) / EIGHT_BLOCK * EIGHT_BLOCK; c0 += 4096) {
            double y64[4];
            uint32_t top = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int c = c0 + i;
                y64[i] = 0;
                if (c < a.dim) {
                    const float xi = to_float(x[c]), ri = r ? to_float(r[c]) : 0.f, wi = to_float(w[c]);
                    const float h = r ? xi + ri : xi;
                    if (a.h)
                        static_cast<T *>(a.h)[row * a.ld_h + c] = from_float<T>(h);
                    if (a.y) {
                        const float y = h * rstd * wi;
                        static_cast<T *>(a.y)[row * a.ld_y + c] = from_float<T>(a.relu && y < 0.f ? 0.f : y);
                    }
                    if constexpr (EIGHT) {
                        y64[i] = (r ? (double)xi + (double)ri : (double)xi) * rstd64 * (double)wi;
                        if (a.relu && y64[i] < 0.0)
                            y64[i] = 0.0;
                    }
                }
                top = max(top, __float_as_uint((float)y64[i]) & 0x7fffffffu);
            }
            if constexpr (EIGHT) {
                top = __reduce_max_sync(PSPMM_FULL_MASK, top);
                float scale, up;
                eight_scale(top, scale, up);
                if (threadIdx.x % 32 == 0)
                    a.scales[row * a.blocks + c0 / EIGHT_BLOCK] = scale;
                uint32_t b[4];
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    b[i] = eight_round(y64[i], (double)up);
                if (c0 < a.used)
                    *reinterpret_cast<uint32_t *>(a.q + row * a.pitch + c0) = pack_bytes(b[0], b[1], b[2], b[3]);
            }
        }
    }
}

template <typename T, int VW, int TPR, int VPT>
__global__ void __launch_bounds__(Rows<TPR>::MOST) norm_backward_kernel(const NormBackArgs a)
{
    using R = Rows<TPR>;
    extern __shared__ float warps_dw[];  // [warps][dim] where several rows share a CTA
    __shared__ __align__(16) WarpSums<float, R::MOST / 32> sums;
    int turn = 0;
    if (TPR > 32)
        sums.clear();
    const int t = TPR > 32 ? threadIdx.x : threadIdx.x % R::LANES;
    const uint32_t mask = group_mask(R::LANES);
    float w[VPT][VW], dw[VPT][VW] = {};
#pragma unroll
    for (int v = 0; v < VPT; ++v) {
        const int c = column<VW, TPR, VPT>(t, v);
        load_some<T, VW>(w[v], static_cast<const T *>(a.w) + c, c < a.dim);
    }
    const int64_t step = (int64_t)gridDim.x * R::PER_CTA;
    for (int64_t row = (int64_t)blockIdx.x * R::PER_CTA + (TPR > 32 ? 0 : threadIdx.x / R::LANES); row < a.n; row += step) {
        if (TPR > 32 && t == 0 && row + AHEAD * step < a.n) {
            look_ahead(static_cast<const T *>(a.h) + (row + AHEAD * step) * a.ld_h, a.dim * (int)sizeof(T));
            look_ahead(static_cast<const T *>(a.dy) + (row + AHEAD * step) * a.ld_dy, a.dim * (int)sizeof(T));
            if (a.dh)
                look_ahead(static_cast<const T *>(a.dh) + (row + AHEAD * step) * a.ld_dh, a.dim * (int)sizeof(T));
        }
        float n[VPT][VW], g[VPT][VW], dh[VPT][VW];
#pragma unroll
        for (int v = 0; v < VPT; ++v) {
            const int c = column<VW, TPR, VPT>(t, v);
            load_some<T, VW>(n[v], static_cast<const T *>(a.h) + row * a.ld_h + c, c < a.dim);
            load_some<T, VW>(g[v], static_cast<const T *>(a.dy) + row * a.ld_dy + c, c < a.dim);
        }
        if (a.dh) {
#pragma unroll
            for (int v = 0; v < VPT; ++v) {
                const int c = column<VW, TPR, VPT>(t, v);
                load_some<T, VW>(dh[v], static_cast<const T *>(a.dh) + row * a.ld_dh + c, c < a.dim);
            }
        }
        const float rstd = a.rstd[row];
        const pair_t by = make_pair(rstd, rstd);
        pair_t sum2 = 0;
#pragma unroll
        for (int e = 0; e < VPT * VW; e += 2) {
            const pair_t m = mul_pair(pair_of(n, e), by), f = pair_of(w, e);
            set_pair(n, e, m);
            if (a.relu) {
                float y0, y1;
                get_pair(mul_pair(m, f), y0, y1);
                if (!(y0 > 0.f))
                    at(g, e) = 0.f;
                if (!(y1 > 0.f))
                    at(g, e + 1) = 0.f;
            }
            set_pair(dw, e, fma_pair(pair_of(g, e), m, pair_of(dw, e)));
            const pair_t gw = mul_pair(pair_of(g, e), f);
            set_pair(g, e, gw);
            sum2 = fma_pair(gw, m, sum2);
        }
        float s, s1;
        get_pair(sum2, s, s1);
        s = row_sum<float, TPR>(s + s1, mask, sums, turn) / a.dim;
        const pair_t less_s = make_pair(-s, -s);
#pragma unroll
        for (int e = 0; e < VPT * VW; e += 2) {
            const pair_t o = mul_pair(fma_pair(pair_of(n, e), less_s, pair_of(g, e)), by);
            set_pair(g, e, o);
            if (a.dh) {
                at(g, e) += at(dh, e);
                at(g, e + 1) += at(dh, e + 1);
            }
        }
#pragma unroll
        for (int v = 0; v < VPT; ++v) {
            const int c = column<VW, TPR, VPT>(t, v);
            if (c < a.dim)
                store_vec<T, VW>(static_cast<T *>(a.dx) + row * a.ld_dx + c, g[v]);
        }
    }
    float *part = a.part + (int64_t)blockIdx.x * a.dim;
    if constexpr (TPR > 32) {
#pragma unroll
        for (int v = 0; v < VPT; ++v) {
            const int c = column<VW, TPR, VPT>(t, v);
#pragma unroll
            for (int i = 0; i < VW; ++i)
                if (c < a.dim)
                    part[c + i] = dw[v][i];
        }
    } else {
#pragma unroll
        for (int v = 0; v < VPT; ++v)
#pragma unroll
            for (int i = 0; i < VW; ++i)
#pragma unroll
                for (int d = 16; d >= R::LANES; d >>= 1)
                    dw[v][i] += __shfl_xor_sync(PSPMM_FULL_MASK, dw[v][i], d);
        if (threadIdx.x % 32 < R::LANES) {
#pragma unroll
            for (int v = 0; v < VPT; ++v) {
                const int c = column<VW, TPR, VPT>(t, v);
#pragma unroll
                for (int i = 0; i < VW; ++i)
                    if (c < a.dim)
                        warps_dw[threadIdx.x / 32 * a.dim + c + i] = dw[v][i];
            }
        }
        __syncthreads();
        for (int c = threadIdx.x; c < a.dim; c += R::MOST) {
            float s = 0;
#pragma unroll
            for (int i = 0; i < R::MOST / 32; ++i)
                s += warps_dw[i * a.dim + c];
            part[c] = s;
        }
    }
}

template <typename T>
__global__ void __launch_bounds__(1024) norm_wide_backward_kernel(const NormBackArgs a)
{
    __shared__ __align__(16) WarpSums<float, 32> sums;
    int turn = 0;
    sums.clear();
    const T *w = static_cast<const T *>(a.w);
    float *part = a.part + (int64_t)blockIdx.x * a.dim;
    for (int c = threadIdx.x; c < a.dim; c += 1024)
        part[c] = 0.f;
    for (int64_t row = blockIdx.x; row < a.n; row += gridDim.x) {
        const T *hp = static_cast<const T *>(a.h) + row * a.ld_h, *dy = static_cast<const T *>(a.dy) + row * a.ld_dy;
        const float rstd = a.rstd[row];
        float s = 0;
        for (int c = threadIdx.x; c < a.dim; c += 1024) {
            const float n = to_float(hp[c]) * rstd;
            float g = to_float(dy[c]);
            if (a.relu && !(n * to_float(w[c]) > 0.f))
                g = 0.f;
            part[c] = fmaf(g, n, part[c]);  // (a thread meets its own columns only)
            s = fmaf(g * to_float(w[c]), n, s);
        }
        s = row_sum<float, 1024>(s, PSPMM_FULL_MASK, sums, turn) / a.dim;
        for (int c = threadIdx.x; c < a.dim; c += 1024) {
            const float n = to_float(hp[c]) * rstd;
            float g = to_float(dy[c]) * to_float(w[c]);
            if (a.relu && !(n * to_float(w[c]) > 0.f))
                g = 0.f;
            float o = (g - n * s) * rstd;
            if (a.dh)
                o += to_float(static_cast<const T *>(a.dh)[row * a.ld_dh + c]);
            static_cast<T *>(a.dx)[row * a.ld_dx + c] = from_float<T>(o);
        }
    }
}

// dw = sum of the CTAs' parts, in a fixed order: a CTA takes 32 neighbouring columns, its warps the parts in turn.
__global__ void __launch_bounds__(1024) norm_weight_kernel(const WeightArgs a)
{
    __shared__ float sums[32][33];
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const int c = blockIdx.x * 32 + lane;
    pdl_wait();
    float s = 0.f;
    if (c < a.dim)
        for (int p = warp; p < a.parts; p += 32)
            s += a.part[(int64_t)p * a.dim + c];
    sums[warp][lane] = s;
    __syncthreads();
    if (warp == 0 && c < a.dim) {
        s = 0.f;
#pragma unroll
        for (int i = 0; i < 32; ++i)
            s += sums[i][lane];
        if (a.dtype == PSPMM_F32)
            static_cast<float *>(a.dw)[c] = s;
        else if (a.dtype == PSPMM_BF16)
            static_cast<bf16 *>(a.dw)[c] = from_float<bf16>(s);
        else
            static_cast<f16 *>(a.dw)[c] = from_float<f16>(s);
    }
}

// CTAs of a launch: as many as find a place, or as there are rows for.
template <typename K> unsigned resident_grid(K kern, int threads, size_t smem, int64_t ctas)
{
    if (ctas <= pspmm_sm_count())
        return (unsigned)ctas;
    int per_sm = 0;
    if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kern, threads, smem) != cudaSuccess || per_sm < 1)
        per_sm = 1;
    const int64_t most = (int64_t)per_sm * pspmm_sm_count();
    return (unsigned)(ctas < most ? ctas : most);
}

template <int VW, int TPR, int VPT> int threads_for(int dim)
{
    return TPR <= 32 ? 256 : (dim + 32 * VW * VPT - 1) / (32 * VW * VPT) * 32;
}

template <typename T, int VW, int TPR, int VPT, bool EIGHT> cudaError_t launch_forward(const NormArgs &a, cudaStream_t st)
{
    const int64_t ctas = (a.n + Rows<TPR>::PER_CTA - 1) / Rows<TPR>::PER_CTA;
    const int threads = threads_for<VW, TPR, VPT>(a.dim);
    auto kern = norm_kernel<T, VW, TPR, VPT, EIGHT>;
    kern<<<resident_grid(kern, threads, 0, ctas), threads, 0, st>>>(a);
    return cudaGetLastError();
}

// Parts of dw: at most this many, so that scratch can be sized without a look at the kernels.
constexpr int PARTS_PER_SM = 8;
int64_t most_parts(int64_t n) { return n < (int64_t)PARTS_PER_SM * pspmm_sm_count() ? n : (int64_t)PARTS_PER_SM * pspmm_sm_count(); }

template <typename T, int VW, int TPR, int VPT> cudaError_t launch_backward(const NormBackArgs &a, unsigned &parts, cudaStream_t st)
{
    using R = Rows<TPR>;
    auto kern = norm_backward_kernel<T, VW, TPR, VPT>;
    const int threads = threads_for<VW, TPR, VPT>(a.dim);
    const size_t smem = TPR > 32 ? 0 : (size_t)8 * a.dim * 4;  // (at most 8 x 512 columns: 16 KB)
    int64_t ctas = (a.n + R::PER_CTA - 1) / R::PER_CTA;
    ctas = ctas < most_parts(a.n) ? ctas : most_parts(a.n);
    parts = resident_grid(kern, threads, smem, ctas);
    kern<<<parts, threads, smem, st>>>(a);
    return cudaGetLastError();
}

// Three vectors per lane (THREES of so many values) fill lane groups that two or four would leave half empty, where instructions bound
// the kernel: 97,235 x 144 with y in 8 bits bf16 82 -> 53 us, fp32 74 -> 57; without them bf16 43 -> 37; the backward's 24 values
// per lane leave fewer warps, bf16 49 -> 51.
template <bool EIGHT> struct Forward {
    static constexpr int EIGHT_OF_FOUR = 4;
    template <int VW> static constexpr bool THREES = EIGHT || VW == 8;
    const NormArgs &a;
    cudaStream_t st;
    template <typename T, int VW, int TPR, int VPT> cudaError_t run() { return launch_forward<T, VW, TPR, VPT, EIGHT>(a, st); }
};
struct Backward {
    static constexpr int EIGHT_OF_FOUR = 8;  // lanes for eight vectors of four (600,000 x 32 fp32 60 us, by four lanes 71; forward 70 in 8 bits, 61)
    template <int VW> static constexpr bool THREES = false;
    const NormBackArgs &a;
    unsigned &parts;
    cudaStream_t st;
    template <typename T, int VW, int TPR, int VPT> cudaError_t run() { return launch_backward<T, VW, TPR, VPT>(a, parts, st); }
};

template <typename T, int VW, int TPR, typename L> cudaError_t three(L &l)
{
    if constexpr (L::template THREES<VW>)
        return l.template run<T, VW, TPR, 3>();
    else
        return cudaErrorInvalidValue;  // (not reached)
}

// Fewest threads that hold a row in 16 values each (8 where they come singly, 24 by THREES of eight); false beyond 8,192 columns.  (Eight lanes at the least, and
// single values by 32: 1,000,000 x 16 fp32 68 us against 49, bf16 88 against 33, 600,000 x 47 fp32 154 against 82 and in 8 bits 254
// against 113.)
// (More would spill beside the 8-bit form's second numbers, fewer leave too few loads in flight.)
template <typename T, int VW, typename L> bool by_width(int dim, L l, cudaError_t &e)
{
    const int nv = (dim + VW - 1) / VW;
    if constexpr (VW == 1) {
        if (nv <= 32) e = l.template run<T, 1, 8, 4>();
        else if (nv <= 64) e = l.template run<T, 1, 8, 8>();
        else if (nv <= 128) e = l.template run<T, 1, 16, 8>();
        else if (nv <= 256) e = l.template run<T, 1, 32, 8>();
        else if (nv <= 1024) e = l.template run<T, 1, 128, 8>();
        else if (nv <= 4096) e = l.template run<T, 1, 512, 8>();
        else if (nv <= 8192) e = l.template run<T, 1, 1024, 8>();
        else return false;
    } else if constexpr (VW == 8) {
        if (nv <= 2) e = l.template run<T, 8, 2, 1>();
        else if (nv <= 4) e = l.template run<T, 8, 2, 2>();
        else if (nv <= 8) e = l.template run<T, 8, 4, 2>();
        else if (nv <= 16) e = l.template run<T, 8, 8, 2>();
        else if (L::template THREES<8> && nv <= 24) e = three<T, 8, 8>(l);
        else if (nv <= 32) e = l.template run<T, 8, 16, 2>();
        else if (L::template THREES<8> && nv <= 48) e = three<T, 8, 16>(l);
        else if (nv <= 64) e = l.template run<T, 8, 32, 2>();
        else if (nv <= 128) e = l.template run<T, 8, 64, 2>();
        else if (nv <= 256) e = l.template run<T, 8, 128, 2>();
        else if (nv <= 512) e = l.template run<T, 8, 256, 2>();
        else if (nv <= 1024) e = l.template run<T, 8, 512, 2>();
        else return false;
    } else {
        if (nv <= 4) e = l.template run<T, VW, 4, 1>();
        else if (nv <= 8) e = l.template run<T, VW, L::EIGHT_OF_FOUR, 8 / L::EIGHT_OF_FOUR>();
        else if (nv <= 16) e = l.template run<T, VW, 4, 4>();
        else if (L::template THREES<4> && nv <= 24) e = three<T, VW, 8>(l);
        else if (nv <= 32) e = l.template run<T, VW, 8, 4>();
        else if (L::template THREES<4> && nv <= 48) e = three<T, VW, 16>(l);
        else if (nv <= 64) e = l.template run<T, VW, 16, 4>();
        else if (L::template THREES<4> && nv <= 96) e = three<T, VW, 32>(l);
        else if (nv <= 128) e = l.template run<T, VW, 32, 4>();
        else if (nv <= 256) e = l.template run<T, VW, 64, 4>();
        else if (nv <= 512) e = l.template run<T, VW, 128, 4>();
        else if (nv <= 1024) e = l.template run<T, VW, 256, 4>();
        else if (nv <= 2048) e = l.template run<T, VW, 512, 4>();
        else return false;
    }
    return true;
}

template <typename T, bool EIGHT> cudaError_t forward_typed(const NormArgs &a, cudaStream_t st)
{
    constexpr int B = sizeof(T), WIDE = 16 / B;
    auto aligned = [&](int bytes) {
        return a.dim * B % bytes == 0 && rows_aligned(a.x, a.ld_x, B, bytes) && rows_aligned(a.r, a.ld_r, B, bytes) &&
               rows_aligned(a.h, a.ld_h, B, bytes) && rows_aligned(a.y, a.ld_y, B, bytes) && rows_aligned(a.w, 0, B, bytes);
    };
    cudaError_t e = cudaSuccess;
    const Forward<EIGHT> l = {a, st};
    if (aligned(16) && by_width<T, WIDE>(a.dim, l, e))
        return e;
    if constexpr (B == 2)
        if (aligned(8) && by_width<T, 4>(a.dim, l, e))
            return e;
    if (by_width<T, 1>(a.dim, l, e))
        return e;
    const unsigned grid = (unsigned)(a.n < 2 * pspmm_sm_count() ? a.n : 2 * pspmm_sm_count());
    norm_wide_kernel<T, EIGHT><<<grid, 1024, 0, st>>>(a);
    return cudaGetLastError();
}
template <typename T> cudaError_t forward_typed(const NormArgs &a, cudaStream_t st)
{
    return a.q ? forward_typed<T, true>(a, st) : forward_typed<T, false>(a, st);
}

template <typename T> cudaError_t backward_typed(const NormBackArgs &a, unsigned &parts, cudaStream_t st)
{
    constexpr int B = sizeof(T), WIDE = 16 / B;
    auto aligned = [&](int bytes) {
        return a.dim * B % bytes == 0 && rows_aligned(a.dy, a.ld_dy, B, bytes) && rows_aligned(a.h, a.ld_h, B, bytes) &&
               rows_aligned(a.dh, a.ld_dh, B, bytes) && rows_aligned(a.dx, a.ld_dx, B, bytes) && rows_aligned(a.w, 0, B, bytes);
    };
    cudaError_t e = cudaSuccess;
    const Backward l = {a, parts, st};
    if (aligned(16) && by_width<T, WIDE>(a.dim, l, e))
        return e;
    if constexpr (B == 2)
        if (aligned(8) && by_width<T, 4>(a.dim, l, e))
            return e;
    if (by_width<T, 1>(a.dim, l, e))
        return e;
    const int64_t most = most_parts(a.n);
    parts = (unsigned)(most < 2 * pspmm_sm_count() ? most : 2 * pspmm_sm_count());
    norm_wide_backward_kernel<T><<<parts, 1024, 0, st>>>(a);
    return cudaGetLastError();
}

bool bad(const void *p, int64_t ld, int32_t dim, int bytes) { return ld < dim || (uintptr_t)p % bytes != 0; }

}  // namespace

extern "C" int pspmm_rms_norm(const void *x, int64_t ld_x, const void *residual, int64_t ld_residual, const void *weight,
                              int32_t dtype, int64_t n, int32_t dim, double eps, int32_t relu, void *h, int64_t ld_h, void *y,
                              int64_t ld_y, float *rstd, int8_t *q, int64_t pitch, float *scales, void *stream)
{
    if (!dtype_ok(dtype) || n < 0 || dim < 1 || !(eps >= 0) || ld_x < dim || (residual && ld_residual < dim) ||
        (h && ld_h < dim) || (y && ld_y < dim) || (q && (pitch < dim || pitch % 16 != 0)) || !q != !scales)
        return PSPMM_E_ARG;
    if (n == 0)
        return PSPMM_OK;
    const int B = elem_bytes(dtype);
    if (!x || !weight || !rstd || bad(x, ld_x, 0, B) || bad(residual, 0, 0, B) || bad(weight, 0, 0, B) || bad(h, 0, 0, B) ||
        bad(y, 0, 0, B) || (uintptr_t)rstd % 4 != 0 || (uintptr_t)q % 16 != 0 || (uintptr_t)scales % 4 != 0)
        return PSPMM_E_ARG;
    if (pitch > INT32_MAX - 8192 || dim > INT32_MAX - 8192)
        return PSPMM_E_RANGE;
    const NormArgs a = {x, residual, weight, h, y, rstd, q, scales, n, ld_x, ld_residual, ld_h, ld_y, eps, dim,
                        (int32_t)pitch, (dim + EIGHT_BLOCK - 1) / EIGHT_BLOCK, relu, (dim + 15) / 16 * 16};
    cudaStream_t st = (cudaStream_t)stream;
    PSPMM_CUDA_TRY(dtype == PSPMM_F32    ? forward_typed<float>(a, st)
                   : dtype == PSPMM_BF16 ? forward_typed<bf16>(a, st)
                                         : forward_typed<f16>(a, st));
    return PSPMM_OK;
}

extern "C" int pspmm_rms_norm_backward_scratch_bytes(int64_t n, int32_t dim, size_t *bytes)
{
    if (n < 0 || dim < 1 || !bytes)
        return PSPMM_E_ARG;
    *bytes = (size_t)most_parts(n) * (size_t)dim * 4;
    return PSPMM_OK;
}

extern "C" int pspmm_rms_norm_backward(const void *dy, int64_t ld_dy, const void *h, int64_t ld_h, const float *rstd,
                                       const void *weight, const void *dh, int64_t ld_dh, int32_t dtype, int64_t n, int32_t dim,
                                       int32_t relu, void *dx, int64_t ld_dx, void *dweight, void *scratch, size_t scratch_bytes,
                                       void *stream)
{
    if (!dtype_ok(dtype) || n < 0 || dim < 1 || ld_dy < dim || ld_h < dim || (dh && ld_dh < dim) || ld_dx < dim)
        return PSPMM_E_ARG;
    const int B = elem_bytes(dtype);
    if (!dweight || bad(dweight, 0, 0, B))
        return PSPMM_E_ARG;
    cudaStream_t st = (cudaStream_t)stream;
    if (n == 0) {
        PSPMM_CUDA_TRY(cudaMemsetAsync(dweight, 0, (size_t)dim * B, st));
        return PSPMM_OK;
    }
    if (!dy || !h || !rstd || !weight || !dx || !scratch || bad(dy, 0, 0, B) || bad(h, 0, 0, B) || bad(weight, 0, 0, B) ||
        bad(dh, 0, 0, B) || bad(dx, 0, 0, B) || (uintptr_t)rstd % 4 != 0 || (uintptr_t)scratch % 4 != 0 ||
        scratch_bytes < (size_t)most_parts(n) * (size_t)dim * 4)
        return PSPMM_E_ARG;
    if (dim > INT32_MAX - 8192)
        return PSPMM_E_RANGE;
    const NormBackArgs a = {dy, h, weight, dh, rstd, dx, (float *)scratch, n, ld_dy, ld_h, ld_dh, ld_dx, dim, relu};
    unsigned parts = 0;
    PSPMM_CUDA_TRY(dtype == PSPMM_F32    ? backward_typed<float>(a, parts, st)
                   : dtype == PSPMM_BF16 ? backward_typed<bf16>(a, parts, st)
                                         : backward_typed<f16>(a, parts, st));
    const WeightArgs wa = {(const float *)scratch, dweight, (int32_t)parts, dim, dtype};
    PSPMM_CUDA_TRY(launch_dependent(norm_weight_kernel, dim3((unsigned)((dim + 31) / 32)), 1024, 0, st, wa));
    return PSPMM_OK;
}
