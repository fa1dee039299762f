// Weight gradient from an activation held in 8 bits (rows8.cu), on the 5th-generation tensor cores:
//
//     C[m, n] = sum over rows i of  q[i, m] scale[i, m / 128] G[i, n],       fp32 out, fp32 accuracy.
//
// q is a whole number of at most seven bits and a sign, exact in bf16.  The scale goes to the other side: x = scale[i, b] G[i, n],
// one 32-bit rounding, is cut in registers into three bf16 parts whose sum it is (its upper, middle and lower 8 bits),
// and three products x_l q, x_m q, x_h q run as tcgen05.mma kind::f16: half of what a product of two fp32 operands takes.
//
// A tile is 128 columns of G (the rows of the MMA) by one block of scales (its columns), so that a row of G meets one scale.  The
// parts of x go to TMEM, where an MMA's first operand may lie: a thread has one column of G and 32 rows of a stage, so they need no
// transposition on the way.  q goes to shared memory as it lies, its rows contiguous along m
// (MN-major core matrices without swizzle: 8 sum indices x 16 bytes, one behind the other at 144 bytes so that the lanes of
// a store meet different banks).
//
// Accumulation.  The tensor core truncates when it adds to the accumulator, so its chains are short: two stages of 32 rows, in each
// the lower parts first.  Chains are added in registers, rounded to nearest.
//
// Structure: a CTA per tile and range of rows.  Four groups of four warps fill the stages; a warp has what it needs of its next two
// stages under way to shared memory of its own, as it lies: tiles by TMA, or words by cp.async where G's rows are not aligned.  (Loads
// to registers that are to outlast a stage are waited for together with the next ones, however they are ordered.)  Two warps
// issue the MMAs; eight add finished chains out of TMEM (two buffers of 128 columns) and store the tile.  Ranges of rows leave
// partial tiles in scratch, which reduce_kernel adds in order.  G with unaligned rows is copied to aligned ones first where scratch
// has room for it.
//
// No unit is full: of the issue slots, the fullest, 68 % are taken in active cycles, the tensor pipe stands at 46 %, DRAM at a third.  2,270
// instructions per stage of a tile are issued in 900 cycles, of which the MMAs take 384; cutting x takes 4 x 180 of the instructions and
// unpacking q 4 x 85, the other half, waits, copies and the adding up of chains, has not been broken down.  2,449,029 x 256 x 256 fp32: 1,075 us (1,265 in
// long runs under the power cap) against 600 for the MMAs and 480 for the bytes; one loading group that takes its rows through registers
// 1,926.  19,717 x 500 x 16: 20 us, start and the adding of partial tiles.  The copy of unaligned rows: 1,029,577 x 285 fp16 314 us.
//
// An infinity of x keeps its sign (its lower parts are zeros), a NaN stays one.  Parts below 2^-133, bf16's least, are lost.
//
// Every wait is bounded (two seconds).  When one runs out, g_rows8_mm_status is set, what was not computed becomes NaN, and the
// CTA leaves.
#include <cuda.h>

#include "feature_types.cuh"
#include "tensor_core.cuh"

namespace {
using namespace feat;
using tc::bar_arrive;
using tc::bar_init;
using tc::bar_try;
using tc::elect_one;
using tc::mma_commit;
using tc::smem_addr;

constexpr int BN = 128, BM = 128, BK = 32;       // columns of G, columns of q, rows of a stage
constexpr int GROUPS = 4, SLOTS = GROUPS;        // loading groups, each with a slot of its own for the MMAs
constexpr int AHEAD = 2;                         // stages that a loading warp has under way
constexpr int ACC_BUFS = 2;
constexpr int CHAIN = 2;                         // stages that one chain adds up
// Chunks of 8 neighbouring columns of q lie Q_CHUNK bytes apart, 128 of them used.
constexpr int Q_CHUNK = 144, Q_OCTET = BM / 8 * Q_CHUNK, Q_BYTES = BK / 8 * Q_OCTET;
constexpr int GROUP_WARPS = 4, LOADERS = GROUPS * GROUP_WARPS, DRAINERS = 8;
constexpr int MMA_WARP = LOADERS + DRAINERS;
constexpr int THREADS = (LOADERS + DRAINERS + 4) * 32;
constexpr int TMEM_X = ACC_BUFS * BM, TMEM_COLS = 512;  // the parts of x: 16 columns each, 48 per slot
// Registers per thread after the split: 896 x 72 = 64,512 at launch; 512 x 72 + 256 x 88 + 128 x 40 = 64,512.
constexpr int DRAINER_REGS = 88, OTHER_REGS = 40;
// What a warp brings in per stage, as it lies in memory: 32 columns of 32 rows of G (by words: one more than fills them, for rows that
// begin inside a word), 8 rows of q, 32 scales.
template <typename T, bool TMA> struct Raw {
    static constexpr int PITCH = 32 * sizeof(T) + (TMA || sizeof(T) == 4 ? 0 : 4);
    static constexpr int Q = (BK * PITCH + 127) / 128 * 128, SCALES = Q + 8 * BM, BYTES = SCALES + BK * 4;
    static constexpr int SMEM = SLOTS * Q_BYTES + LOADERS * AHEAD * BYTES;
    static_assert(SLOTS * Q_BYTES % 128 == 0 && BYTES % 128 == 0, "copies of tiles land on 128 bytes");
};

__device__ unsigned g_rows8_mm_status;

struct MmArgs {
    const int8_t *q;
    const float *scales;
    const void *G;
    float *C;                  // output, or partial tiles [splits][M][N] when splits > 1
    int64_t pitch, ldG, ldC, rows;
    int64_t rows_per_split;    // a multiple of BK
    int32_t M, N, blocks;
    int32_t splits, m_tiles, n_tiles;
    uint32_t wait_ns;
    int32_t withhold;          // arrivals that no one brings: 0, or 1 to make the waits for a stage run out
};

// Tiles of G (32 x 32) and q (128 x 8).
struct Maps {
    CUtensorMap G, q;
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

// Descriptor of an MN-major tile without swizzle: bytes from one chunk of 8 neighbouring columns to the next, and from one group of
// 8 sum indices to the next.
__device__ __forceinline__ uint64_t tile_desc(uint32_t addr, int chunk, int octet)
{
    return (uint64_t)((addr & 0x3ffff) >> 4) | ((uint64_t)(octet >> 4) << 16) | ((uint64_t)(chunk >> 4) << 32) | (1ull << 46);
}

// First operand in TMEM, second in shared memory.
__device__ __forceinline__ void mma(uint32_t acc, uint32_t a, uint64_t b, uint32_t idesc, int accumulate)
{
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.s32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
                 ::"r"(acc), "r"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}

// Accumulator columns of the warp's 32 TMEM lanes.
__device__ __forceinline__ void acc_load16(uint32_t (&v)[16], uint32_t addr)
{
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];\n\t"
                 "tcgen05.wait::ld.sync.aligned;"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
                   "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
                 : "r"(addr));
}
__device__ __forceinline__ void acc_load8(uint32_t (&v)[8], uint32_t addr)
{
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];\n\ttcgen05.wait::ld.sync.aligned;"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7])
                 : "r"(addr));
}

// Half a part (8 packed columns) of the warp's 32 columns of G -> TMEM.
__device__ __forceinline__ void part_store(uint32_t addr, const uint32_t (&v)[8])
{
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};"
                 ::"r"(addr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
                 : "memory");
}

// Four whole numbers -> bf16: 128 + (q & 127) less 128 or 256, both exact.
__device__ __forceinline__ uint32_t bf16_pair(uint32_t w, uint32_t pick)
{
    const uint32_t t = __byte_perm(w, 0x43434343u, pick);
    const uint32_t lo = t & 0x437f437fu, hi = t & 0x43804380u;
    const __nv_bfloat162 d = __hsub2(*reinterpret_cast<const __nv_bfloat162 *>(&lo), *reinterpret_cast<const __nv_bfloat162 *>(&hi));
    return *reinterpret_cast<const uint32_t *>(&d);
}

// The upper 16 bits of two values, cut off, as a bf16 pair; and what is left of the values.
__device__ __forceinline__ uint32_t cut_pair(pair_t &x)
{
    float x0, x1;
    get_pair(x, x0, x1);
    const uint32_t u0 = __float_as_uint(x0), u1 = __float_as_uint(x1);
    x = add_pair(x, make_pair(__uint_as_float((u0 & 0xffff0000u) ^ 0x80000000u), __uint_as_float((u1 & 0xffff0000u) ^ 0x80000000u)));
    return __byte_perm(u0, u1, 0x7632);
}

// cp.async of 16 or 4 bytes, of which the first `bytes` are read and the rest zeros.
__device__ __forceinline__ void copy16(uint32_t dst, const void *src, int bytes)
{
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void copy4(uint32_t dst, const void *src, int bytes)
{
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
// A tile from column x, row y on; what lies outside the array is zeros.
__device__ __forceinline__ void copy_tile(uint32_t dst, const CUtensorMap *map, int x, int y, uint32_t bar)
{
    asm volatile("cp.async.bulk.tensor.2d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
                 ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(bar) : "memory");
}
template <int PENDING> __device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(PENDING) : "memory"); }
// 16 rows of a thread's column -> half of each part in TMEM.  What is left of an infinity or a NaN is a NaN: `rest` adds up the
// remainders, so that one look at it tells whether all values had a split.
__device__ __forceinline__ void split_column(pair_t (&x)[8], uint32_t addr, pair_t &rest)
{
    uint32_t v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        v[i] = cut_pair(x[i]);
        rest = add_pair(rest, x[i]);
    }
    part_store(addr, v);
#pragma unroll
    for (int i = 0; i < 8; ++i)
        v[i] = cut_pair(x[i]);
    part_store(addr + 16, v);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        float x0, x1;
        get_pair(x[i], x0, x1);
        v[i] = __byte_perm(__float_as_uint(x0), __float_as_uint(x1), 0x7632);
    }
    part_store(addr + 32, v);
}
// The parts of a value of any kind: an infinity stands in the upper part alone, and a NaN is one there.
__device__ __forceinline__ uint32_t part_of(float x, int part)
{
    const bool finite = fabsf(x) < __int_as_float(0x7f800000);
    const float r = finite ? x - __uint_as_float(__float_as_uint(x) & 0xffff0000u) : 0.f;
    if (part == 0)
        return x != x ? 0x7fffu : __float_as_uint(x) >> 16;
    return __float_as_uint(part == 1 ? r : r - __uint_as_float(__float_as_uint(r) & 0xffff0000u)) >> 16;
}

template <typename T, bool TMA>
__global__ void __launch_bounds__(THREADS, 1) rows8_mm_kernel(const MmArgs a, const __grid_constant__ Maps maps)
{
    extern __shared__ __align__(1024) unsigned char smem[];
    __shared__ __align__(8) uint64_t bars[2 * SLOTS + 2 * ACC_BUFS + LOADERS * AHEAD];
    __shared__ uint32_t tmem_base;
    __shared__ volatile int abort_flag;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t full = smem_addr(bars), empty = full + 8 * SLOTS, acc_full = empty + 8 * SLOTS,
                   acc_empty = acc_full + 8 * ACC_BUFS, landed = acc_empty + 8 * ACC_BUFS;
    if (threadIdx.x == 0) {
        for (int i = 0; i < SLOTS; ++i) {
            bar_init(full + 8 * i, GROUP_WARPS + a.withhold);
            bar_init(empty + 8 * i, 1);
        }
        for (int i = 0; i < ACC_BUFS; ++i) {
            bar_init(acc_full + 8 * i, 1);
            bar_init(acc_empty + 8 * i, DRAINERS);
        }
        for (int i = 0; i < LOADERS * AHEAD; ++i)
            bar_init(landed + 8 * i, 1);
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
    const int m0 = mt * BM, n0 = nt * BN;
    const int bm = min((a.M - m0 + 15) / 16 * 16, BM);  // columns of the MMA
    const int64_t i0 = split * a.rows_per_split;
    const int64_t i1 = a.rows - i0 > a.rows_per_split ? i0 + a.rows_per_split : a.rows;
    const int stages = (int)((i1 - i0 + BK - 1) / BK);

    if (warp < LOADERS) {
        // Group g takes stages g, g + 4, ...; of each, warp w 32 columns of G (a thread one of them) and 8 rows of q.  A warp waits
        // for its own copies only.
        using R = Raw<T, TMA>;
        constexpr int SZ = sizeof(T);
        const int g = warp / GROUP_WARPS, w = warp % GROUP_WARPS, slot = g;
        const int col0 = n0 + w * 32;
        const bool some = col0 < a.N;
        // (lanes beyond the last column have it again: their rows of the tile are not stored)
        const int mine = min(lane, a.N - 1 - col0) * SZ;
        const uint32_t raw0 = smem_addr(smem) + SLOTS * Q_BYTES + warp * (AHEAD * R::BYTES);
        const uint32_t lanes_x = tmem + ((uint32_t)(w * 32) << 16) + TMEM_X;
        const uint32_t landed0 = landed + 8 * (warp * AHEAD);
        const uintptr_t g_begin = (uintptr_t)a.G, g_col = g_begin + (int64_t)col0 * SZ;
        const uintptr_t g_end = g_begin + ((a.rows - 1) * a.ldG + a.N) * SZ;
        const int64_t g_row = a.ldG * SZ;
        // Words: even and odd rows of a stage begin this far into one, the same in every stage.
        const int off[2] = {TMA || SZ == 4 ? 0 : (int)((g_col + i0 * g_row) & 2), TMA || SZ == 4 ? 0 : (int)((g_col + (i0 + 1) * g_row) & 2)};

        const float *sp = a.scales + (i0 + g * BK + lane) * a.blocks + mt;  // of the next stage's rows

        auto fetch = [&](int s, int buf) {
            if (s < stages) {
                const uint32_t raw = raw0 + buf * R::BYTES;
                const int64_t i = i0 + (int64_t)s * BK;
                if constexpr (TMA) {
                    if (elect_one()) {
                        const uint32_t bar = landed0 + 8 * buf;
                        asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;"
                                     ::"r"(bar), "r"((some ? BK * R::PITCH : 0) + 8 * BM) : "memory");
                        if (some)
                            copy_tile(raw, &maps.G, col0, (int)i, bar);
                        copy_tile(raw + R::Q, &maps.q, m0, (int)i + w * 8, bar);
                    }
                } else {
                    if (some) {
                        const uint32_t dst = raw + lane * 4;
                        uintptr_t first = g_col + i * g_row;
                        for (int k = 0; k < BK; ++k, first += g_row) {
                            const uintptr_t src = first / 4 * 4 + lane * 4;
                            if (lane * 4 >= 32 * SZ + off[k & 1])
                                continue;  // (16-bit types: 16 words, 17 where the row begins inside one)
                            if (i + k < i1 && src < g_begin) {  // G begins inside this word
                                *reinterpret_cast<uint16_t *>(smem + (dst + k * R::PITCH + 2 - smem_addr(smem))) =
                                    *reinterpret_cast<const uint16_t *>(g_begin);
                            } else {
                                const bool in = i + k < i1 && src < g_end;
                                copy4(dst + k * R::PITCH, in ? (const void *)src : a.scales, in ? SZ == 2 && src + 4 > g_end ? 2 : 4 : 0);
                            }
                        }
                    }
#pragma unroll
                    for (int p = 0; p < 2; ++p) {
                        const int row = p * 4 + lane / 8, at = lane % 8 * 16;
                        const bool in = i + w * 8 + row < i1 && m0 + at < a.pitch;
                        copy16(raw + R::Q + row * BM + at, a.q + (in ? (i + w * 8 + row) * a.pitch + m0 + at : 0), in ? 16 : 0);
                    }
                }
                const bool in = i + lane < i1;
                copy4(raw + R::SCALES + lane * 4, in ? sp : a.scales, in ? 4 : 0);
                sp += (int64_t)a.blocks * (GROUPS * BK);
            }
            asm volatile("cp.async.commit_group;" ::: "memory");  // (an empty one keeps the count)
        };
        auto value = [&](const unsigned char *raw, int k) {
            return to_float(*reinterpret_cast<const T *>(raw + k * R::PITCH + off[k & 1] + mine));
        };
        // x of a stage value by value, where some have no split.  (Stores to TMEM are not ordered among themselves: the parts that
        // went there before are waited for, or a NaN of theirs might land last.)
        auto store_slowly = [&](const unsigned char *raw, uint32_t to) {
            asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
#pragma unroll 1
            for (int k = 0; k < BK; k += 2) {
                const float x[2] = {value(raw, k) * *reinterpret_cast<const float *>(raw + R::SCALES + k * 4),
                                    value(raw, k + 1) * *reinterpret_cast<const float *>(raw + R::SCALES + k * 4 + 4)};
#pragma unroll
                for (int part = 0; part < 3; ++part)
                    asm volatile("tcgen05.st.sync.aligned.32x32b.x1.b32 [%0], {%1};"
                                 ::"r"(to + part * 16 + k / 2), "r"(part_of(x[0], part) | part_of(x[1], part) << 16) : "memory");
            }
        };
#pragma unroll
        for (int t = 0; t < AHEAD; ++t)
            fetch(g + t * GROUPS, t);
        int buf = 0, phase = 0, landed_phase = 0, s = g;
        for (; s < stages; s += GROUPS) {
            copies_wait<AHEAD - 1>();
            __syncwarp();
            if ((TMA && !bar_wait(landed0 + 8 * buf, landed_phase, &abort_flag, a.wait_ns)) ||
                !bar_wait(empty + 8 * slot, phase ^ 1, &abort_flag, a.wait_ns))
                break;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const unsigned char *raw = smem + SLOTS * Q_BYTES + (warp * AHEAD + buf) * R::BYTES;
#pragma unroll
            for (int p = 0; p < 4; ++p) {
                const int half = lane >> 4, qc = lane & 15;
                const uint2 v = *reinterpret_cast<const uint2 *>(raw + R::Q + (half + 2 * p) * BM + qc * 8);
                *reinterpret_cast<uint4 *>(smem + slot * Q_BYTES + w * Q_OCTET + qc * Q_CHUNK + (half + 2 * p) * 16) =
                    make_uint4(bf16_pair(v.x, 0x4140), bf16_pair(v.x, 0x4342), bf16_pair(v.y, 0x4140), bf16_pair(v.y, 0x4342));
            }
            if (some) {
                pair_t rest = 0;
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    pair_t x[8];
#pragma unroll
                    for (int k = 0; k < 16; k += 4) {
                        const int row = half * 16 + k;
                        const float4 v = *reinterpret_cast<const float4 *>(raw + R::SCALES + row * 4);
                        x[k / 2] = mul_pair(make_pair(value(raw, row), value(raw, row + 1)), make_pair(v.x, v.y));
                        x[k / 2 + 1] = mul_pair(make_pair(value(raw, row + 2), value(raw, row + 3)), make_pair(v.z, v.w));
                    }
                    split_column(x, lanes_x + slot * 48 + half * 8, rest);
                }
                float rest0, rest1;
                get_pair(rest, rest0, rest1);
                if (__any_sync(PSPMM_FULL_MASK, rest0 + rest1 != rest0 + rest1))
                    store_slowly(raw, lanes_x + slot * 48);
            }
            __syncwarp();
            fetch(s + AHEAD * GROUPS, buf);
            asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0)
                bar_arrive(full + 8 * slot);
            phase ^= 1;
            if (++buf == AHEAD) {
                buf = 0;
                landed_phase ^= 1;
            }
        }
        copies_wait<0>();
        if (TMA && s < stages) {  // a wait ran out: the tiles under way land before the memory is given back
            for (int t = 0; t < AHEAD && s < stages; ++t, s += GROUPS) {
                for (int n = 0; n < 1000 && !bar_try(landed0 + 8 * buf, landed_phase); ++n)
                    __nanosleep(1000);
                if (++buf == AHEAD) {
                    buf = 0;
                    landed_phase ^= 1;
                }
            }
        }
    } else if (warp >= MMA_WARP) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(OTHER_REGS));
        if (warp < MMA_WARP + 2) {
            // Two warps issue, a chain in turn: what one waits and issues for a stage takes longer than its MMAs.  Chain c has accumulator
            // c & 1 and slots 2 (c & 1) and the next, so that a warp meets every phase of its barriers.
            static_assert(CHAIN == 2 && SLOTS == 2 * CHAIN && ACC_BUFS == 2, "a warp's slots are its own");
            const int m = warp - MMA_WARP;
            // D fp32, both operands bf16, the second one MN-major
            const uint32_t idesc = (1u << 4) | (1u << 7) | (1u << 10) | (1u << 16) | ((uint32_t)(bm >> 3) << 17) | ((uint32_t)(BN >> 4) << 24);
            const uint64_t desc_q = tile_desc(smem_addr(smem) + m * CHAIN * Q_BYTES, Q_CHUNK, Q_OCTET);
            const uint32_t acc = tmem + m * BM, x0 = tmem + TMEM_X + m * CHAIN * 48;
            int phase = 0;
            bool ok = true;
            for (int s = m * CHAIN; ok && s < stages; s += SLOTS) {
                ok = bar_wait(acc_empty + 8 * m, phase ^ 1, &abort_flag, a.wait_ns);
#pragma unroll
                for (int at = 0; at < CHAIN; ++at) {
                    if (!ok || s + at >= stages)
                        break;
                    ok = bar_wait(full + 8 * (m * CHAIN + at), phase, &abort_flag, a.wait_ns);
                    if (!ok)
                        break;
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    if (elect_one()) {
#pragma unroll
                        for (int p = 2; p >= 0; --p)  // lower, middle, upper parts
#pragma unroll
                            for (int h = 0; h < BK / 16; ++h)  // two groups of 8 sum indices each
                                mma(acc, x0 + at * 48 + p * 16 + h * 8,
                                    desc_q + (uint64_t)(at * (Q_BYTES >> 4) + h * 2 * (Q_OCTET >> 4)), idesc, at > 0 || p < 2 || h > 0);
                        mma_commit(empty + 8 * (m * CHAIN + at));
                        if (at == CHAIN - 1 || s + at == stages - 1)
                            mma_commit(acc_full + 8 * m);
                    }
                    __syncwarp();
                }
                phase ^= 1;
            }
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(DRAINER_REGS));
        // Drainer d: TMEM lanes (columns of G) of its quadrant, half the columns of q.
        const int d = warp - LOADERS;
        const int quad = warp & 3, half = d >> 2;
        const int cols = bm / 2;  // a multiple of 8
        pair_t acc[32];
#pragma unroll
        for (int t = 0; t < 32; ++t)
            acc[t] = 0;
        bool ok = true;
        const int chains = (stages + CHAIN - 1) / CHAIN;
        for (int s = 0; s < chains; ++s) {
            const int buf = s & 1;
            if (!bar_wait(acc_full + 8 * buf, s >> 1 & 1, &abort_flag, a.wait_ns)) {
                ok = false;
                break;
            }
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const uint32_t from = tmem + ((uint32_t)(quad * 32) << 16) + buf * BM + half * cols;
            if (cols == BM / 2) {
#pragma unroll
                for (int c = 0; c < 64; c += 16) {
                    uint32_t v[16];
                    acc_load16(v, from + c);
#pragma unroll
                    for (int t = 0; t < 16; t += 2)
                        acc[(c + t) / 2] = add_pair(acc[(c + t) / 2], make_pair(__uint_as_float(v[t]), __uint_as_float(v[t + 1])));
                }
            } else {
#pragma unroll
                for (int c = 0; c < 64; c += 8) {
                    if (c >= cols)
                        break;
                    uint32_t v[8];
                    acc_load8(v, from + c);
#pragma unroll
                    for (int t = 0; t < 8; t += 2)
                        acc[(c + t) / 2] = add_pair(acc[(c + t) / 2], make_pair(__uint_as_float(v[t]), __uint_as_float(v[t + 1])));
                }
            }
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            __syncwarp();
            if (lane == 0)
                bar_arrive(acc_empty + 8 * buf);
        }
        const int n = n0 + quad * 32 + lane, m = m0 + half * cols;
        float *out = a.C + ((int64_t)split * a.M + m) * a.ldC + n;
        if (n < a.N) {  // (neighbouring lanes store neighbouring elements)
#pragma unroll
            for (int t = 0; t < 64; ++t)
                if (t < cols && m + t < a.M) {
                    float v[2];
                    get_pair(acc[t / 2], v[0], v[1]);
                    // where a wait ran out, no stale memory passes for a result
                    out[t * a.ldC] = ok ? v[t & 1] : __int_as_float(0x7fffffff);
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

struct PadArgs {
    const void *src;
    void *dst;
    int64_t rows, ld, pitch;
    int32_t cols;
};

// Rows of G moved to 16-byte boundaries, zeros behind them: a warp takes four rows at a time.
template <typename T> __global__ void __launch_bounds__(256) pad_kernel(const PadArgs a)
{
    const int lane = threadIdx.x & 31;
    const int64_t warps = (int64_t)gridDim.x * 8;
    for (int64_t r0 = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); r0 < a.rows; r0 += 4 * warps) {
        for (int c = lane; c < a.pitch; c += 32) {
            T v[4];
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                const int64_t r = r0 + t * warps;
                v[t] = r < a.rows && c < a.cols ? static_cast<const T *>(a.src)[r * a.ld + c] : from_float<T>(0.f);
            }
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                const int64_t r = r0 + t * warps;
                if (r < a.rows)
                    static_cast<T *>(a.dst)[r * a.pitch + c] = v[t];
            }
        }
    }
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
    return a.splits > 1 ? ((size_t)a.splits * (size_t)M * (size_t)N * sizeof(float) + 255) / 256 * 256 : 0;
}
// A copy of G with rows of whole 16 bytes.
int64_t padded_cols(int32_t N, int bytes) { return ((int64_t)N * bytes + 15) / 16 * 16 / bytes; }
size_t padded_bytes(int64_t rows, int32_t N, int bytes) { return (size_t)rows * (size_t)padded_cols(N, bytes) * bytes; }

// The driver's function that describes an array to TMA (the library links the runtime only); null where there is none.
typedef CUresult (*EncodeTiled)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *,
                                const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle,
                                CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeTiled encode_tiled()
{
    static const EncodeTiled fn = [] {
        void *p = nullptr;
        cudaDriverEntryPointQueryResult found;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &found) != cudaSuccess ||
            found != cudaDriverEntryPointSuccess)
            return (EncodeTiled) nullptr;
        return (EncodeTiled)p;
    }();
    return fn;
}

// A matrix of `width` elements of `bytes` bytes per row, in tiles of w x h elements.
bool describe(CUtensorMap &map, const void *p, int bytes, int64_t width, int64_t rows, int64_t ld, int w, int h)
{
    const cuuint64_t size[2] = {(cuuint64_t)width, (cuuint64_t)rows}, stride[1] = {(cuuint64_t)(ld * bytes)};
    const cuuint32_t box[2] = {(cuuint32_t)w, (cuuint32_t)h}, step[2] = {1, 1};
    const CUtensorMapDataType type = bytes == 4   ? CU_TENSOR_MAP_DATA_TYPE_UINT32
                                     : bytes == 2 ? CU_TENSOR_MAP_DATA_TYPE_UINT16
                                                  : CU_TENSOR_MAP_DATA_TYPE_UINT8;
    return encode_tiled()(&map, type, 2, const_cast<void *>(p), size, stride, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                          CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                          CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T, bool TMA> cudaError_t launch_loads(const MmArgs &a, const Maps &maps, cudaStream_t st)
{
    auto kern = rows8_mm_kernel<T, TMA>;
    constexpr int SMEM = Raw<T, TMA>::SMEM;
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM);
    if (e != cudaSuccess)
        return e;
    kern<<<(unsigned)(a.m_tiles * a.n_tiles * a.splits), THREADS, SMEM, st>>>(a, maps);
    return cudaGetLastError();
}

// Tiles by TMA where the rows of both operands begin on 16 bytes (its strides are below 2^40 and its coordinates 32 bits).
template <typename T> cudaError_t launch(MmArgs a, void *padded, cudaStream_t st)
{
    if (padded) {
        const PadArgs p = {a.G, padded, a.rows, a.ldG, padded_cols(a.N, sizeof(T)), a.N};
        const int64_t ctas = (a.rows + 31) / 32, most = (int64_t)pspmm_sm_count() * 16;
        pad_kernel<T><<<(unsigned)(ctas < most ? ctas : most), 256, 0, st>>>(p);
        cudaError_t e = cudaGetLastError();
        if (e != cudaSuccess)
            return e;
        a.G = padded;
        a.ldG = p.pitch;
    }
    Maps maps = {};
    if (rows_aligned(a.G, a.ldG, sizeof(T), 16) && a.rows < INT32_MAX - 1024 && a.ldG * (int64_t)sizeof(T) < 1ll << 40 && encode_tiled() &&
        describe(maps.G, a.G, sizeof(T), a.N, a.rows, a.ldG, 32, BK) && describe(maps.q, a.q, 1, a.pitch, a.rows, a.pitch, BM, 8))
        return launch_loads<T, true>(a, maps, st);
    return launch_loads<T, false>(a, maps, st);
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
    if (dim > (1 << 20) || cols > (1 << 20) || (int64_t)dim * cols > (int64_t)INT32_MAX * 32)
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
    a.wait_ns = wait_ns;
    a.withhold = withhold;
    const int B = elem_bytes(dtype);
    void *padded = nullptr;  // (scratch that has no room for the copy is used without it)
    if (!rows_aligned(G, ldG, B, 16) && scratch && scratch_bytes >= need + padded_bytes(rows, cols, B) && (uintptr_t)scratch % 16 == 0)
        padded = (char *)scratch + need;
    PSPMM_CUDA_TRY(dtype == PSPMM_F32    ? launch<float>(a, padded, st)
                   : dtype == PSPMM_BF16 ? launch<bf16>(a, padded, st)
                                         : launch<f16>(a, padded, st));
    if (a.splits > 1) {
        const ReduceArgs r = {a.C, C, ldC, a.splits, dim, cols};
        PSPMM_CUDA_TRY(launch_dependent(reduce_kernel, dim3((unsigned)(((int64_t)dim * cols + 31) / 32)), 256, 0, st, r));
    }
    return PSPMM_OK;
}

}  // namespace

extern "C" int pspmm_rows8_mm_t_scratch_bytes(int64_t n, int32_t dim, int32_t cols, int32_t dtype, int32_t aligned, size_t *bytes)
{
    if (n < 0 || dim < 1 || cols < 0 || !dtype_ok(dtype) || !bytes)
        return PSPMM_E_ARG;
    *bytes = 0;
    if (n == 0 || cols == 0)
        return PSPMM_OK;
    MmArgs a = {};
    plan(n, dim, cols, a);
    *bytes = partial_bytes(a, dim, cols) + (aligned ? 0 : padded_bytes(n, cols, elem_bytes(dtype)));
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

extern "C" int pspmm_rows8_mm_status(int32_t *status) { return pspmm_read_status(g_rows8_mm_status, status); }
