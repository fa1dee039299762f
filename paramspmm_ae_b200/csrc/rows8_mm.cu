// Weight gradient from an activation held in 8 bits (rows8.cu), on the 5th-generation tensor cores:
//
//     C[m, n] = sum over rows i of  q[i, m] scale[i, m / 128] G[i, n],       fp32 out, fp32 accuracy.
//
// q is a whole number of at most seven bits and a sign, exact in bf16.  The scale goes to the other side: x = scale[i, b] G[i, n],
// one 32-bit rounding, is cut in registers into three bf16 parts whose sum it is (its upper, middle and lower 8 bits),
// and three products q x_l, q x_m, q x_h run as tcgen05.mma kind::f16: half of what a product of two fp32 operands takes.  A tile of
// C is 128 rows high, one block of scales, so that a row of G meets one scale per tile.
//
// Both operands lie in memory as the sum runs over their rows, so a tile's rows are contiguous along M and N.  They go to shared
// memory that way (MN-major core matrices without swizzle: 8 sum indices x 16 bytes; eight neighbouring lanes store one) and no
// transposition is needed.
//
// Accumulation.  The tensor core truncates when it adds to the accumulator, so its chains are short: one stage of 32 rows, the
// lower parts first, while the accumulator is below 2^-7 of its final size; then two truncations at full size.  Chains are added in
// registers, rounded to nearest.
//
// Structure: a CTA per tile and range of rows.  Three groups of four warps own a stage each: a group loads its next rows of q and G
// into registers, waits for its stage to be free, splits and stores.  Two warps issue the MMAs, a chain in turn; eight add
// finished chains out of TMEM (two buffers of 128 columns) and store the tile.  Ranges of rows leave partial tiles in scratch,
// which reduce_kernel adds in order.
//
// An infinity of x keeps its sign (its lower parts are zeros), a NaN stays one.  Parts below 2^-133, bf16's least, are lost.
//
// Every wait is bounded (two seconds).  When one runs out, g_rows8_mm_status is set, what was not computed becomes NaN, and the
// CTA leaves.
#include "feature_types.cuh"
#include "tensor_core.cuh"

namespace {
using namespace feat;
using tc::acc_load;
using tc::bar_arrive;
using tc::bar_init;
using tc::elect_one;
using tc::mma_commit;
using tc::smem_addr;

constexpr int BM = 128, BN = 128, BK = 32;
constexpr int STAGES = 3, ACC_BUFS = 2;
constexpr int A_BYTES = BM * BK * 2, PLANE = BN * BK * 2;
constexpr int STAGE_BYTES = A_BYTES + 3 * PLANE;
constexpr int OUT_PITCH = 36;                    // floats per row of a drainer's 32 x 32 output patch
constexpr int OUT_BYTES = 32 * OUT_PITCH * 4;
constexpr int GROUP_WARPS = 4, LOADERS = STAGES * GROUP_WARPS, DRAINERS = 8;
constexpr int MMA_WARP = LOADERS + DRAINERS;
constexpr int THREADS = (LOADERS + DRAINERS + 4) * 32;
constexpr int SMEM = STAGES * STAGE_BYTES + DRAINERS * OUT_BYTES + 1024;
constexpr int TMEM_COLS = ACC_BUFS * BN;
// Registers per thread after the split: 768 x 80 = 61,440 at launch; 384 x 80 + 256 x 104 + 128 x 32 = 61,440.
constexpr int DRAINER_REGS = 104, OTHER_REGS = 32;

__device__ unsigned g_rows8_mm_status;

struct MmArgs {
    const int8_t *q;
    const float *scales;
    const void *G;
    float *C;                  // output, or partial tiles [splits][M][N] when splits > 1
    int64_t pitch, ldG, ldC, rows;
    int64_t rows_per_split;    // a multiple of BK
    int32_t M, N, blocks;
    int32_t splits, m_tiles, n_tiles, bn;  // bn: columns per tile, a multiple of 16
    int32_t vec;               // rows of G may be read 16 bytes at a time
    uint32_t wait_ns;
    int32_t withhold;          // arrivals that no one brings: 0, or 1 to make the waits for a stage run out
};

struct ReduceArgs {
    const float *part;
    float *C;
    int64_t ldC;
    int32_t splits, M, N;
};

__device__ __forceinline__ bool bar_wait(uint32_t bar, int parity, volatile int *abort, uint32_t limit_ns)
{
    return tc::bar_wait(bar, parity, abort, limit_ns, &g_rows8_mm_status);
}

// Descriptor of an MN-major tile without swizzle: chunks of 8 neighbouring m or n 128 bytes apart, groups of 8 sum indices
// `chunks` * 128 bytes apart.
__device__ __forceinline__ uint64_t tile_desc(uint32_t addr, int chunks)
{
    return (uint64_t)((addr & 0x3ffff) >> 4) | ((uint64_t)(chunks * 8) << 16) | ((uint64_t)(128 >> 4) << 32) | (1ull << 46);
}

__device__ __forceinline__ void mma(uint32_t acc, uint64_t a, uint64_t b, uint32_t idesc, int accumulate)
{
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.s32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
                 ::"r"(acc), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}

// Four whole numbers -> bf16: 128 + (q & 127) less 128 or 256, both exact.
__device__ __forceinline__ uint32_t bf16_pair(uint32_t w, uint32_t pick)
{
    const uint32_t t = __byte_perm(w, 0x43434343u, pick);
    const uint32_t lo = t & 0x437f437fu, hi = t & 0x43804380u;
    const __nv_bfloat162 d = __hsub2(*reinterpret_cast<const __nv_bfloat162 *>(&lo), *reinterpret_cast<const __nv_bfloat162 *>(&hi));
    return *reinterpret_cast<const uint32_t *>(&d);
}

__device__ __forceinline__ uint32_t upper_halves(float x0, float x1)
{
    return __byte_perm(__float_as_uint(x0), __float_as_uint(x1), 0x7632);
}
__device__ __forceinline__ float less_upper(float x) { return x - __uint_as_float(__float_as_uint(x) & 0xffff0000u); }

// Eight values -> three 16-byte chunks, `PLANE` apart.
__device__ __forceinline__ void split_store(float (&x)[8], unsigned char *dst)
{
    uint4 h, m, l;
    h = make_uint4(upper_halves(x[0], x[1]), upper_halves(x[2], x[3]), upper_halves(x[4], x[5]), upper_halves(x[6], x[7]));
    float r[8];
#pragma unroll
    for (int i = 0; i < 8; ++i)
        r[i] = less_upper(x[i]);
    m = make_uint4(upper_halves(r[0], r[1]), upper_halves(r[2], r[3]), upper_halves(r[4], r[5]), upper_halves(r[6], r[7]));
    // (the remainder of an infinity or a NaN is a NaN)
    const float sum = ((r[0] + r[1]) + (r[2] + r[3])) + ((r[4] + r[5]) + (r[6] + r[7]));
#pragma unroll
    for (int i = 0; i < 8; ++i)
        r[i] = less_upper(r[i]);
    l = make_uint4(upper_halves(r[0], r[1]), upper_halves(r[2], r[3]), upper_halves(r[4], r[5]), upper_halves(r[6], r[7]));
    if (sum != sum) {
        uint32_t *hw = &h.x, *mw = &m.x, *lw = &l.x;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const uint32_t keep = i & 1 ? 0x0000ffffu : 0xffff0000u;
            if (!(fabsf(x[i]) < __int_as_float(0x7f800000))) {
                mw[i / 2] &= keep;
                lw[i / 2] &= keep;
                if (x[i] != x[i])
                    hw[i / 2] |= ~keep & 0x7fff7fffu;
            }
        }
    }
    *reinterpret_cast<uint4 *>(dst) = h;
    *reinterpret_cast<uint4 *>(dst + PLANE) = m;
    *reinterpret_cast<uint4 *>(dst + 2 * PLANE) = l;
}

// Eight neighbouring values of a row as they lie in memory.
template <typename T> struct Raw { uint32_t w[2 * sizeof(T)]; };

__device__ __forceinline__ uint4 load16(const void *p)
{
    uint4 v;  // volatile: the loads of the next stage are to leave before this stage's wait, not at their first use
    asm volatile("ld.global.nc.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}

template <typename T> __device__ __forceinline__ void load_raw(Raw<T> &r, const T *p, int left, bool vec)
{
    if (vec && left >= 8) {
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; ++i) {
            const uint4 v = load16(reinterpret_cast<const char *>(p) + 16 * i);
            r.w[4 * i] = v.x;
            r.w[4 * i + 1] = v.y;
            r.w[4 * i + 2] = v.z;
            r.w[4 * i + 3] = v.w;
        }
    } else if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            r.w[i] = i < left ? __float_as_uint(to_float(p[i])) : 0u;
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t lo = 2 * i < left ? *reinterpret_cast<const uint16_t *>(p + 2 * i) : 0u;
            const uint32_t hi = 2 * i + 1 < left ? *reinterpret_cast<const uint16_t *>(p + 2 * i + 1) : 0u;
            r.w[i] = lo | hi << 16;
        }
    }
}
template <typename T> __device__ __forceinline__ void raw_floats(float (&x)[8], const Raw<T> &r)
{
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        if constexpr (sizeof(T) == 4)
            x[i] = __uint_as_float(r.w[i]);
        else if constexpr (sizeof(T) == 2) {
            const uint16_t b = (uint16_t)(i & 1 ? r.w[i / 2] >> 16 : r.w[i / 2]);
            x[i] = to_float(*reinterpret_cast<const T *>(&b));
        }
    }
}

template <typename T>
__global__ void __launch_bounds__(THREADS, 1) rows8_mm_kernel(const MmArgs a)
{
    extern __shared__ __align__(1024) unsigned char smem[];
    __shared__ __align__(8) uint64_t bars[2 * STAGES + 2 * ACC_BUFS];
    __shared__ uint32_t tmem_base;
    __shared__ volatile int abort_flag;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t full = smem_addr(bars), empty = full + 8 * STAGES, acc_full = empty + 8 * STAGES,
                   acc_empty = acc_full + 8 * ACC_BUFS;
    if (threadIdx.x == 0) {
        for (int i = 0; i < STAGES; ++i) {
            bar_init(full + 8 * i, GROUP_WARPS + a.withhold);
            bar_init(empty + 8 * i, 1);
        }
        for (int i = 0; i < ACC_BUFS; ++i) {
            bar_init(acc_full + 8 * i, 1);
            bar_init(acc_empty + 8 * i, DRAINERS);
        }
        abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == MMA_WARP) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;"
                     ::"r"(smem_addr(&tmem_base)), "r"(TMEM_COLS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = tmem_base;
    pdl_launch_dependents();

    // Neighbouring CTAs take the tiles of one range of rows, which they read together.
    const int nt = blockIdx.x % a.n_tiles, mt = blockIdx.x / a.n_tiles % a.m_tiles, split = blockIdx.x / a.n_tiles / a.m_tiles;
    const int m0 = mt * BM, n0 = nt * a.bn;
    const int64_t i0 = split * a.rows_per_split;
    const int64_t i1 = a.rows - i0 > a.rows_per_split ? i0 + a.rows_per_split : a.rows;
    const int stages = (int)((i1 - i0 + BK - 1) / BK);

    if (warp < LOADERS) {
        // Group g fills stage slot g with rows 32 g .. of every 96; a warp 8 rows of them, lane (k, j) pieces j, j + 4, ... of row k.
        const int g = warp / GROUP_WARPS, octet = warp % GROUP_WARPS, k = lane & 7, j = lane >> 3;
        unsigned char *st = smem + g * STAGE_BYTES;
        const int chunks = a.bn / 8;
        const int n_end = a.N - n0 < a.bn ? a.N - n0 : a.bn;  // columns of G that exist
        uint4 qv[2];
        Raw<T> gv[4];
        float scale = 0.f;
        auto fetch = [&](int s) {
            const int64_t i = i0 + (int64_t)s * BK + octet * 8 + k;
            const bool in = i < i1;
            const int8_t *q = a.q + (in ? i * a.pitch + m0 : 0);
#pragma unroll
            for (int p = 0; p < 2; ++p) {
                const int c = (j + 4 * p) * 16;
                qv[p] = in && m0 + c < a.pitch ? load16(q + c) : make_uint4(0, 0, 0, 0);
            }
            scale = in ? a.scales[i * a.blocks + mt] : 0.f;
            const T *row = static_cast<const T *>(a.G) + (in ? i * a.ldG + n0 : 0);
#pragma unroll
            for (int p = 0; p < 4; ++p) {
                const int c = j + 4 * p;
                if (c < chunks)
                    load_raw<T>(gv[p], row + c * 8, in ? n_end - c * 8 : 0, a.vec);
            }
        };
        if (g < stages)
            fetch(g);
        int phase = 0;
        for (int s = g; s < stages; s += STAGES) {
            if (!bar_wait(empty + 8 * g, phase ^ 1, &abort_flag, a.wait_ns))
                break;
#pragma unroll
            for (int p = 0; p < 2; ++p) {
                unsigned char *dst = st + octet * (BM / 8 * 128) + (j + 4 * p) * 256 + k * 16;
                *reinterpret_cast<uint4 *>(dst) = make_uint4(bf16_pair(qv[p].x, 0x4140), bf16_pair(qv[p].x, 0x4342),
                                                             bf16_pair(qv[p].y, 0x4140), bf16_pair(qv[p].y, 0x4342));
                *reinterpret_cast<uint4 *>(dst + 128) = make_uint4(bf16_pair(qv[p].z, 0x4140), bf16_pair(qv[p].z, 0x4342),
                                                                   bf16_pair(qv[p].w, 0x4140), bf16_pair(qv[p].w, 0x4342));
            }
#pragma unroll
            for (int p = 0; p < 4; ++p) {
                const int c = j + 4 * p;
                if (c < chunks) {
                    float x[8];
                    raw_floats<T>(x, gv[p]);
#pragma unroll
                    for (int t = 0; t < 8; ++t)
                        x[t] *= scale;
                    split_store(x, st + A_BYTES + octet * (chunks * 128) + c * 128 + k * 16);
                }
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0)
                bar_arrive(full + 8 * g);
            phase ^= 1;
            if (s + STAGES < stages)
                fetch(s + STAGES);
        }
    } else if (warp >= MMA_WARP) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(OTHER_REGS));
        if (warp == MMA_WARP || warp == MMA_WARP + 2) {
            // A chain (stage) each in turn; also the accumulator buffer.
            const int m = warp == MMA_WARP ? 0 : 1;
            // D fp32, A and B bf16, both MN-major
            const uint32_t idesc = (1u << 4) | (1u << 7) | (1u << 10) | (1u << 15) | (1u << 16) | ((uint32_t)(a.bn >> 3) << 17) |
                                   ((uint32_t)(BM >> 4) << 24);
            const uint32_t acc = tmem + m * BN;
            const uint64_t desc_a = tile_desc(smem_addr(smem), BM / 8);
            const uint64_t desc_b = tile_desc(smem_addr(smem) + A_BYTES, a.bn / 8);
            for (int s = m; s < stages; s += 2) {
                const int slot = s % STAGES;
                if (!bar_wait(acc_empty + 8 * m, ((s >> 1) & 1) ^ 1, &abort_flag, a.wait_ns) ||
                    !bar_wait(full + 8 * slot, s / STAGES & 1, &abort_flag, a.wait_ns))
                    break;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                if (elect_one()) {
                    const uint64_t pa = desc_a + (uint64_t)(slot * (STAGE_BYTES >> 4));
                    const uint64_t pb = desc_b + (uint64_t)(slot * (STAGE_BYTES >> 4));
#pragma unroll
                    for (int p = 2; p >= 0; --p)  // lower, middle, upper parts
#pragma unroll
                        for (int h = 0; h < BK / 16; ++h)  // two groups of 8 sum indices each
                            mma(acc, pa + (uint64_t)(h * 2 * (BM / 8) * 8),
                                pb + (uint64_t)(p * (PLANE >> 4) + h * 2 * a.bn), idesc, p < 2 || h > 0);
                    mma_commit(empty + 8 * slot);
                    mma_commit(acc_full + 8 * m);
                }
                __syncwarp();
            }
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(DRAINER_REGS));
        // Drainer d: TMEM lanes (rows) of its quadrant, half the columns.
        const int d = warp - LOADERS;
        const int quad = warp & 3, half = d >> 2;
        const int cols = a.bn / 2;  // a multiple of 8
        float *patch = reinterpret_cast<float *>(smem + STAGES * STAGE_BYTES + d * OUT_BYTES);
        float acc[64];
#pragma unroll
        for (int t = 0; t < 64; ++t)
            acc[t] = 0.f;
        bool ok = true;
        for (int s = 0; s < stages; ++s) {
            const int buf = s & 1;
            if (!bar_wait(acc_full + 8 * buf, s >> 1 & 1, &abort_flag, a.wait_ns)) {
                ok = false;
                break;
            }
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll
            for (int q0 = 0; q0 < 8; q0 += 4) {
                if (q0 * 8 >= cols)
                    break;
                uint32_t v[4][8];
#pragma unroll
                for (int q = 0; q < 4; ++q)
                    if ((q0 + q) * 8 < cols)
                        acc_load(v[q], tmem + ((uint32_t)(quad * 32) << 16) + buf * BN + half * cols + (q0 + q) * 8);
                asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
                for (int q = 0; q < 4; ++q)
                    if ((q0 + q) * 8 < cols)
#pragma unroll
                        for (int t = 0; t < 8; ++t) {
                            asm volatile("" : "+r"(v[q][t]));  // (not read ahead of the wait)
                            acc[(q0 + q) * 8 + t] += __uint_as_float(v[q][t]);
                        }
            }
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            __syncwarp();
            if (lane == 0)
                bar_arrive(acc_empty + 8 * buf);
        }
        if (!ok) {  // a wait ran out: no stale memory passes for a result
#pragma unroll
            for (int t = 0; t < 64; ++t)
                acc[t] = __int_as_float(0x7fffffff);
        }
        const int c0 = n0 + half * cols;
        const int c1 = a.N - n0 < a.bn ? a.N : n0 + a.bn;
        float *out = a.C + ((int64_t)split * a.M + m0 + quad * 32) * a.ldC + c0;
        const int rows = a.M - m0 - quad * 32;  // of the warp's 32
        // 32 columns at a time through shared memory, so that eight lanes store 128 bytes of a row.
        const bool vec = (a.ldC & 3) == 0 && ((uintptr_t)out & 15) == 0;
#pragma unroll
        for (int j0 = 0; j0 < 64; j0 += 32) {
            if (j0 >= cols)
                break;
            __syncwarp();
#pragma unroll
            for (int t = 0; t < 32; t += 4)
                *reinterpret_cast<float4 *>(patch + lane * OUT_PITCH + t) =
                    make_float4(acc[j0 + t], acc[j0 + t + 1], acc[j0 + t + 2], acc[j0 + t + 3]);
            __syncwarp();
            for (int t = 0; t < 8; ++t) {
                const int r = (lane >> 3) + t * 4, c = (lane & 7) * 4;
                if (r >= rows)
                    break;
                const float4 v = *reinterpret_cast<const float4 *>(patch + r * OUT_PITCH + c);
                float *o = out + r * a.ldC + j0 + c;
                const int left = j0 + c < cols ? c1 - (c0 + j0 + c) : 0;
                if (vec && left >= 4) {
                    *reinterpret_cast<float4 *>(o) = v;
                } else {
                    if (left > 0)
                        o[0] = v.x;
                    if (left > 1)
                        o[1] = v.y;
                    if (left > 2)
                        o[2] = v.z;
                    if (left > 3)
                        o[3] = v.w;
                }
            }
        }
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (warp == MMA_WARP && abort_flag) {  // let the MMAs in flight end (they wait on nothing)
        for (int i = 0; i < 1000; ++i)
            __nanosleep(1000);
    }
    if (warp == MMA_WARP)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(TMEM_COLS));
}

// C = sum of the partial tiles: a block takes 32 neighbouring elements, its eight warps the splits in turn.
__global__ void __launch_bounds__(256) reduce_kernel(const ReduceArgs a)
{
    __shared__ float sums[8][33];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int64_t total = (int64_t)a.M * a.N;
    const int64_t i = (int64_t)blockIdx.x * 32 + lane;
    pdl_wait();
    float s[4] = {};
    if (i < total) {
        int t = warp;
        for (; t + 24 < a.splits; t += 32)
#pragma unroll
            for (int u = 0; u < 4; ++u)
                s[u] += a.part[(t + 8 * u) * total + i];
        for (; t < a.splits; t += 8)
            s[0] += a.part[t * total + i];
    }
    sums[warp][lane] = (s[0] + s[1]) + (s[2] + s[3]);
    __syncthreads();
    if (warp == 0 && i < total) {
        float t = 0.f;
#pragma unroll
        for (int w = 0; w < 8; ++w)
            t += sums[w][lane];
        a.C[i / a.N * a.ldC + i % a.N] = t;
    }
}

// Tiles, and ranges of rows: a launch lasts (rounds of CTAs) x (stages of a range + start and end, about 10 stages' time); cutting
// gives every SM a range and costs the partial tiles' trip through memory and one more launch (5 stages' time).
void plan(int64_t rows, int32_t M, int32_t N, MmArgs &a)
{
    a.m_tiles = (M + BM - 1) / BM;
    a.n_tiles = (N + BN - 1) / BN;
    const int32_t per = (N + a.n_tiles - 1) / a.n_tiles;
    a.bn = (per + 15) / 16 * 16;
    const int64_t tiles = (int64_t)a.m_tiles * a.n_tiles, sms = pspmm_sm_count();
    const int64_t stages = (rows + BK - 1) / BK;
    a.splits = 1;
    a.rows_per_split = stages * BK;
    double best = 1e30;
    for (int64_t rounds = 0; rounds <= 4; ++rounds) {
        int64_t splits = rounds * sms / tiles;
        splits = splits < 1 ? 1 : (splits > stages ? stages : splits);
        const int64_t len = (stages + splits - 1) / splits;
        splits = (stages + len - 1) / len;
        double cost = (double)((tiles * splits + sms - 1) / sms) * (double)(len + 10);
        if (splits > 1)
            cost += 5 + (double)splits * (double)M * (double)N * 8.0 / 2e6;
        if (cost < best) {
            best = cost;
            a.splits = (int32_t)splits;
            a.rows_per_split = len * BK;
        }
    }
}

size_t partial_bytes(const MmArgs &a, int32_t M, int32_t N)
{
    return a.splits > 1 ? (size_t)a.splits * (size_t)M * (size_t)N * sizeof(float) : 0;
}

template <typename T> cudaError_t launch(const MmArgs &a, cudaStream_t st)
{
    auto kern = rows8_mm_kernel<T>;
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM);
    if (e != cudaSuccess)
        return e;
    kern<<<(unsigned)(a.m_tiles * a.n_tiles * a.splits), THREADS, SMEM, st>>>(a);
    return cudaGetLastError();
}

int mm_run(const int8_t *q, int64_t pitch, const float *scales, int64_t rows, int32_t dim, const void *G, int32_t dtype, int64_t ldG,
           int32_t cols, float *C, int64_t ldC, void *scratch, size_t scratch_bytes, uint32_t wait_ns, int32_t withhold, void *stream)
{
    if (!dtype_ok(dtype) || rows < 0 || dim < 1 || cols < 0 || pitch < dim || pitch % 16 != 0 || ldG < cols || ldC < cols)
        return PSPMM_E_ARG;
    if (cols == 0)
        return PSPMM_OK;
    if (!C || (uintptr_t)C % 4 != 0)
        return PSPMM_E_ARG;
    if (dim > (1 << 20) || cols > (1 << 20))
        return PSPMM_E_RANGE;
    cudaStream_t st = (cudaStream_t)stream;
    if (rows == 0) {
        PSPMM_CUDA_TRY(cudaMemset2DAsync(C, (size_t)ldC * 4, 0, (size_t)cols * 4, (size_t)dim, st));
        return PSPMM_OK;
    }
    if (!q || !scales || !G || (uintptr_t)q % 16 != 0 || (uintptr_t)scales % 4 != 0 || (uintptr_t)G % elem_bytes(dtype) != 0)
        return PSPMM_E_ARG;
    if (rows > (int64_t)INT32_MAX * BK / 2)
        return PSPMM_E_RANGE;
    MmArgs a = {};
    plan(rows, dim, cols, a);
    if ((int64_t)a.m_tiles * a.n_tiles * a.splits > INT32_MAX)
        return PSPMM_E_RANGE;
    const size_t need = partial_bytes(a, dim, cols);
    if (need > 0 && (!scratch || scratch_bytes < need || (uintptr_t)scratch % 16 != 0))
        return PSPMM_E_ARG;
    a.q = q;
    a.scales = scales;
    a.G = G;
    a.C = a.splits > 1 ? (float *)scratch : C;
    a.pitch = pitch;
    a.ldG = ldG;
    a.ldC = a.splits > 1 ? cols : ldC;
    a.rows = rows;
    a.M = dim;
    a.N = cols;
    a.blocks = (dim + EIGHT_BLOCK - 1) / EIGHT_BLOCK;
    a.vec = rows_aligned(G, ldG, elem_bytes(dtype), 16);
    a.wait_ns = wait_ns;
    a.withhold = withhold;
    PSPMM_CUDA_TRY(dtype == PSPMM_F32    ? launch<float>(a, st)
                   : dtype == PSPMM_BF16 ? launch<bf16>(a, st)
                                         : launch<f16>(a, st));
    if (a.splits > 1) {
        const ReduceArgs r = {a.C, C, ldC, a.splits, dim, cols};
        PSPMM_CUDA_TRY(launch_dependent(reduce_kernel, dim3((unsigned)(((int64_t)dim * cols + 31) / 32)), 256, 0, st, r));
    }
    return PSPMM_OK;
}

}  // namespace

extern "C" int pspmm_rows8_mm_t_scratch_bytes(int64_t n, int32_t dim, int32_t cols, size_t *bytes)
{
    if (n < 0 || dim < 1 || cols < 0 || !bytes)
        return PSPMM_E_ARG;
    *bytes = 0;
    if (n == 0 || cols == 0)
        return PSPMM_OK;
    MmArgs a = {};
    plan(n, dim, cols, a);
    *bytes = partial_bytes(a, dim, cols);
    return PSPMM_OK;
}

extern "C" int pspmm_rows8_mm_t(const int8_t *q, int64_t pitch, const float *scales, int64_t n, int32_t dim, const void *G,
                                int32_t dtype, int64_t ldG, int32_t cols, float *C, int64_t ldC, void *scratch,
                                size_t scratch_bytes, void *stream)
{
    return mm_run(q, pitch, scales, n, dim, G, dtype, ldG, cols, C, ldC, scratch, scratch_bytes, 2000000000u, 0, stream);
}

extern "C" int pspmm_rows8_mm_t_stalled(const int8_t *q, int64_t pitch, const float *scales, int64_t n, int32_t dim, const void *G,
                                        int32_t dtype, int64_t ldG, int32_t cols, float *C, int64_t ldC, void *scratch,
                                        size_t scratch_bytes, void *stream)
{
    return mm_run(q, pitch, scales, n, dim, G, dtype, ldG, cols, C, ldC, scratch, scratch_bytes, 20000000u, 1, stream);
}

extern "C" int pspmm_rows8_mm_status(int32_t *status)
{
    if (!status)
        return PSPMM_E_ARG;
    unsigned v = 0;
    PSPMM_CUDA_TRY(cudaMemcpyFromSymbol(&v, g_rows8_mm_status, sizeof(v)));
    *status = (int32_t)v;
    return PSPMM_OK;
}
