// Rows of a table looked up by id and scaled, and the table's gradient:
//     out[i] = s T[id_i],      dT[t] = s * sum over {i : id_i = t} G[i]
//
// Lookup: a gather, bound by HBM (each row of the table once if ids repeat close together, each row of `out`).
//
// Gradient: the ids are sorted with their positions (stable, so that a row's sum has one order whatever the timing), and every
// row of the table is then written once, zeros included, by one lane group that gathers the rows of G in the order of their
// positions.  Ids that occur more than `run` times are cut into chunks of `run` sorted positions, whose sums are left in scratch and
// added up by a dependent launch: no atomics on values, and the hottest id does not hold the launch up.
// Up to RANK_MAX ids are sorted by counting, one launch; more by least-significant-digit passes of 8 bits (as many as the table's
// size needs), three launches each.
// Ids outside the table: NaN rows in the lookup, nothing in the gradient, and pspmm_embedding_status tells.
#include "feature_types.cuh"

namespace {
using namespace feat;

__device__ unsigned g_embedding_status;

constexpr int RANK_MAX = 2048;
constexpr int TILE_THREADS = 256, TILE_KEYS = 8, TILE = TILE_THREADS * TILE_KEYS;  // keys of a CTA in a digit pass
constexpr int WARPS = TILE_THREADS / 32;
constexpr int MOST_TOKENS = 256;  // rows of the table that a CTA writes

struct LookupArgs {
    const void *ids, *table;
    void *out;
    int64_t n, n_rows, ld_table, ld_out;
    int32_t ids64, vecs, lanes;  // vectors per row, lanes that share a row
    float scale;
};

struct Ids {
    const void *ids;
    int64_t n, n_rows, padding;  // padding: the id without a gradient (-1: none)
    int32_t ids64;
};

struct SortArgs {
    Ids in;
    const uint32_t *key_in;  // null: the first pass, from `in`
    const uint32_t *pos_in;
    uint32_t *key_out, *pos_out;
    uint32_t *counts;  // [256][tiles], turned into each tile's first place inside its digit
    uint32_t *totals;  // [256]
    int32_t tiles, shift;
};

struct GradArgs {
    const uint32_t *keys, *pos;  // sorted
    const void *grad;
    void *out;
    float *part;     // [chunks][2][cols]: the piece that begins before the chunk or with it, and the one that begins inside
    int64_t n, n_rows, ld_grad, ld_out;
    int64_t units;   // chunks * slices
    int32_t chunk_ctas;  // the first CTAs of the launch take chunks
    int32_t run, vecs, lanes, slices, tokens, cols;
    float scale;
};

__device__ __forceinline__ int64_t load_id(const void *ids, int ids64, int64_t i)
{
    return ids64 ? static_cast<const int64_t *>(ids)[i] : (int64_t)static_cast<const int32_t *>(ids)[i];
}
// Sort key of position i: its id, or n_rows (the last key) where no row takes the gradient.
__device__ __forceinline__ uint32_t load_key(const Ids &a, int64_t i)
{
    const int64_t id = load_id(a.ids, a.ids64, i);
    const bool in = id >= 0 && id < a.n_rows;
    if (!in)
        g_embedding_status = 1;
    return (uint32_t)(in && id != a.padding ? id : a.n_rows);
}

// `lanes` lanes share a row, ROWS rows of a lane group are in flight together.
template <typename T, int VW, int ROWS>
__global__ void __launch_bounds__(256) lookup_kernel(const LookupArgs a)
{
    const int gl = threadIdx.x % a.lanes;
    const int64_t groups = (int64_t)gridDim.x * (256 / a.lanes);
    const int64_t group = (int64_t)blockIdx.x * (256 / a.lanes) + threadIdx.x / a.lanes;
    const float nan = __int_as_float(0x7fc00000);
    for (int64_t i0 = group; i0 < a.n; i0 += groups * ROWS) {
        int64_t id[ROWS];
#pragma unroll
        for (int r = 0; r < ROWS; ++r) {
            const int64_t i = i0 + r * groups;
            id[r] = i < a.n ? load_id(a.ids, a.ids64, i) : -1;
            if (i < a.n && (id[r] < 0 || id[r] >= a.n_rows)) {
                id[r] = -1;
                g_embedding_status = 1;
            }
        }
        for (int v = gl; v < a.vecs; v += a.lanes) {
            float f[ROWS][VW];
#pragma unroll
            for (int r = 0; r < ROWS; ++r) {
                if (id[r] >= 0) {
                    load_vec<T, VW>(f[r], static_cast<const T *>(a.table) + id[r] * a.ld_table + (int64_t)v * VW);
                } else {
#pragma unroll
                    for (int j = 0; j < VW; ++j)
                        f[r][j] = nan;
                }
            }
#pragma unroll
            for (int r = 0; r < ROWS; ++r) {
#pragma unroll
                for (int j = 0; j < VW; ++j)
                    f[r][j] *= a.scale;
                const int64_t i = i0 + r * groups;
                if (i < a.n)
                    store_vec<T, VW>(static_cast<T *>(a.out) + i * a.ld_out + (int64_t)v * VW, f[r]);
            }
        }
    }
}

// ---- sorting -------------------------------------------------------------------------------------------------------

// Few ids: the place of a key is the number of smaller ones and of equal ones before it; a warp counts for one key.
__global__ void __launch_bounds__(256) rank_kernel(const SortArgs a)
{
    __shared__ uint32_t keys[RANK_MAX];
    const int n = (int)a.in.n, lane = threadIdx.x % 32;
    for (int i = threadIdx.x; i < n; i += 256)
        keys[i] = load_key(a.in, i);
    __syncthreads();
    const int i = blockIdx.x * 8 + threadIdx.x / 32;
    if (i >= n)
        return;
    const uint32_t key = keys[i];
    int before = 0;
    for (int j = lane; j < n; j += 32)
        before += keys[j] < key || (keys[j] == key && j < i);
    before = __reduce_add_sync(PSPMM_FULL_MASK, before);
    if (lane == 0) {
        a.key_out[before] = key;
        a.pos_out[before] = (uint32_t)i;
    }
}

__device__ __forceinline__ uint32_t sort_key(const SortArgs &a, int64_t i)
{
    return a.key_in ? a.key_in[i] : load_key(a.in, i);
}

__global__ void __launch_bounds__(TILE_THREADS) digit_count_kernel(const SortArgs a)
{
    __shared__ uint32_t bins[256];
    bins[threadIdx.x] = 0;
    __syncthreads();
    for (int k = 0; k < TILE_KEYS; ++k) {
        const int64_t i = (int64_t)blockIdx.x * TILE + k * TILE_THREADS + threadIdx.x;
        if (i < a.in.n)
            atomicAdd(&bins[sort_key(a, i) >> a.shift & 255], 1u);
    }
    __syncthreads();
    a.counts[(int64_t)threadIdx.x * a.tiles + blockIdx.x] = bins[threadIdx.x];
}

// Sum over the threads before this one, in a CTA of 256; `warps` is scratch of 8.
__device__ __forceinline__ uint32_t exclusive_256(uint32_t v, uint32_t *warps, uint32_t &total)
{
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
    uint32_t s = v;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const uint32_t t = __shfl_up_sync(PSPMM_FULL_MASK, s, d);
        if (lane >= d)
            s += t;
    }
    __syncthreads();
    if (lane == 31)
        warps[warp] = s;
    __syncthreads();
    uint32_t before = 0;
    total = 0;
#pragma unroll
    for (int w = 0; w < 8; ++w) {
        before += w < warp ? warps[w] : 0;
        total += warps[w];
    }
    return before + s - v;
}

// A CTA per digit: its counts over the tiles -> places inside the digit, and the digit's total.
__global__ void __launch_bounds__(256) digit_scan_kernel(const SortArgs a)
{
    __shared__ uint32_t warps[8];
    uint32_t *c = a.counts + (int64_t)blockIdx.x * a.tiles;
    uint32_t carry = 0;
    for (int t0 = 0; t0 < a.tiles; t0 += 256) {
        const int t = t0 + threadIdx.x;
        const uint32_t v = t < a.tiles ? c[t] : 0;
        uint32_t total;
        const uint32_t before = exclusive_256(v, warps, total);
        if (t < a.tiles)
            c[t] = carry + before;
        carry += total;
    }
    if (threadIdx.x == 0)
        a.totals[blockIdx.x] = carry;
}

// Stable: a warp takes 256 neighbouring keys, 32 at a time; equal digits among the 32 find one another by a match, and a
// count per warp and digit carries on from one 32 to the next.
__global__ void __launch_bounds__(TILE_THREADS) digit_scatter_kernel(const SortArgs a)
{
    __shared__ uint32_t seen[WARPS][256];
    __shared__ uint32_t first[256];
    __shared__ uint32_t warps[8];
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
    uint32_t total;
    first[threadIdx.x] = exclusive_256(a.totals[threadIdx.x], warps, total) +
                         a.counts[(int64_t)threadIdx.x * a.tiles + blockIdx.x];
    for (int w = 0; w < WARPS; ++w)
        seen[w][threadIdx.x] = 0;
    __syncthreads();
    uint32_t key[TILE_KEYS], pos[TILE_KEYS], rank[TILE_KEYS];
    const int64_t i0 = (int64_t)blockIdx.x * TILE + warp * (32 * TILE_KEYS) + lane;
#pragma unroll
    for (int k = 0; k < TILE_KEYS; ++k) {
        const int64_t i = i0 + k * 32;
        key[k] = i < a.in.n ? sort_key(a, i) : 0xffffffffu;
        pos[k] = i < a.in.n ? (a.pos_in ? a.pos_in[i] : (uint32_t)i) : 0;
    }
#pragma unroll
    for (int k = 0; k < TILE_KEYS; ++k) {
        const bool in = i0 + k * 32 < a.in.n;
        const uint32_t d = in ? key[k] >> a.shift & 255 : 256;  // (lanes beyond the end match one another only)
        const uint32_t same = __match_any_sync(PSPMM_FULL_MASK, d);
        const uint32_t below = __popc(same & ((1u << lane) - 1));
        rank[k] = in ? seen[warp][d] + below : 0;
        __syncwarp();
        if (in && below == 0)
            seen[warp][d] += __popc(same);
        __syncwarp();
    }
    __syncthreads();
    uint32_t before = first[threadIdx.x];
    for (int w = 0; w < WARPS; ++w) {
        const uint32_t c = seen[w][threadIdx.x];
        seen[w][threadIdx.x] = before;
        before += c;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < TILE_KEYS; ++k)
        if (i0 + k * 32 < a.in.n) {
            const uint32_t to = seen[warp][key[k] >> a.shift & 255] + rank[k];
            a.key_out[to] = key[k];
            a.pos_out[to] = pos[k];
        }
}

// ---- sums ----------------------------------------------------------------------------------------------------------

// First position in [lo, hi) whose key is not below `key` (hi: none).
__device__ __forceinline__ int64_t lower_bound(const uint32_t *keys, uint32_t key, int64_t lo, int64_t hi)
{
    while (lo < hi) {
        const int64_t mid = (lo + hi) >> 1;
        if (keys[mid] < key)
            lo = mid + 1;
        else
            hi = mid;
    }
    return lo;
}

// The same over all keys by a whole warp, 32 probes a step.
__device__ __forceinline__ int64_t warp_lower_bound(const uint32_t *keys, uint32_t key, int64_t n)
{
    const int lane = threadIdx.x % 32;
    int64_t lo = 0, hi = n;  // the answer lies in [lo, hi]
    while (hi - lo > 32) {
        const int64_t step = (hi - lo + 31) / 32;
        const int64_t at = lo + lane * step;
        const bool below = at < hi && keys[at] < key;
        const int c = __popc(__ballot_sync(PSPMM_FULL_MASK, below));
        if (c == 0)
            return lo;
        const int64_t from = lo + (c - 1) * step;
        lo = from + 1;
        hi = from + step < hi ? from + step : hi;
    }
    const bool below = lo + lane < hi && keys[lo + lane] < key;
    return lo + __popc(__ballot_sync(PSPMM_FULL_MASK, below));
}

// Sum of the rows of G at sorted positions [p, e), one vector of columns.
template <typename T, int VW>
__device__ __forceinline__ void gather_sum(float (&acc)[VW], const GradArgs &a, int64_t p, int64_t e, int v)
{
    constexpr int U = 4;
    const T *g = static_cast<const T *>(a.grad) + (int64_t)v * VW;
#pragma unroll
    for (int j = 0; j < VW; ++j)
        acc[j] = 0.f;
    for (; p + U <= e; p += U) {
        float f[U][VW];
#pragma unroll
        for (int u = 0; u < U; ++u)
            load_vec<T, VW>(f[u], g + (int64_t)a.pos[p + u] * a.ld_grad);
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int j = 0; j < VW; ++j)
                acc[j] += f[u][j];
    }
    for (; p < e; ++p) {
        float f[VW];
        load_vec<T, VW>(f, g + (int64_t)a.pos[p] * a.ld_grad);
#pragma unroll
        for (int j = 0; j < VW; ++j)
            acc[j] += f[j];
    }
}

template <typename T, int VW>
__device__ __forceinline__ void chunk_part(const GradArgs &a, int64_t chunk, int slot, int64_t p, int64_t e, int v)
{
    float acc[VW];
    gather_sum<T, VW>(acc, a, p, e, v);
    float *part = a.part + (chunk * 2 + slot) * a.cols + (int64_t)v * VW;
#pragma unroll
    for (int j = 0; j < VW; ++j)
        part[j] = acc[j];
}

// Whether the id at position p, the first of its run, occurs more than `run` times.
__device__ __forceinline__ bool is_long(const GradArgs &a, int64_t p)
{
    return p + a.run < a.n && a.keys[p + a.run] == a.keys[p];
}

template <typename T, int VW>
__global__ void __launch_bounds__(256) grad_kernel(const GradArgs a)
{
    __shared__ int64_t start[MOST_TOKENS + 1];
    __shared__ int64_t range[2];
    pdl_launch_dependents();
    pdl_wait();
    const int gl = threadIdx.x % a.lanes, group = threadIdx.x / a.lanes, groups = 256 / a.lanes;
    if ((int)blockIdx.x < a.chunk_ctas) {  // a lane group per chunk and slice of columns
        const int64_t unit = (int64_t)blockIdx.x * groups + group;
        if (unit >= a.units)
            return;
        const int64_t chunk = unit / a.slices;
        const int v = (int)(unit % a.slices) * a.lanes + gl;
        if (v >= a.vecs)
            return;
        const int64_t begin = chunk * a.run, end = begin + a.run < a.n ? begin + a.run : a.n;
        const uint32_t head = a.keys[begin], tail = a.keys[end - 1];
        if (head < a.n_rows) {
            const int64_t from = begin > a.run ? begin - a.run : 0;
            const int64_t s = lower_bound(a.keys, head, from, begin);
            // (a run that reaches `run` places back is long; so is one whose first position says so)
            if ((s == from && begin - from == a.run) || is_long(a, s))
                chunk_part<T, VW>(a, chunk, 0, begin, lower_bound(a.keys, head + 1, begin, end), v);
        }
        if (tail != head && tail < a.n_rows) {
            const int64_t s = lower_bound(a.keys, tail, begin, end);
            if (is_long(a, s))
                chunk_part<T, VW>(a, chunk, 1, s, end, v);
        }
        return;
    }
    const int64_t t0 = (int64_t)(blockIdx.x - a.chunk_ctas) * a.tokens;
    const int tokens = a.n_rows - t0 < a.tokens ? (int)(a.n_rows - t0) : a.tokens;
    if (threadIdx.x < 64) {
        const int64_t at = warp_lower_bound(a.keys, (uint32_t)(t0 + (threadIdx.x < 32 ? 0 : tokens)), a.n);
        if (threadIdx.x % 32 == 0)
            range[threadIdx.x / 32] = at;
    }
    __syncthreads();
    for (int t = threadIdx.x; t <= tokens; t += 256)
        start[t] = lower_bound(a.keys, (uint32_t)(t0 + t), range[0], range[1]);
    __syncthreads();
    for (int t = group; t < tokens; t += groups) {
        const int64_t s = start[t], e = start[t + 1];
        if (e - s > a.run)
            continue;  // cut into chunks
        T *out = static_cast<T *>(a.out) + (t0 + t) * a.ld_out;
        for (int v = gl; v < a.vecs; v += a.lanes) {
            float acc[VW];
            gather_sum<T, VW>(acc, a, s, e, v);
#pragma unroll
            for (int j = 0; j < VW; ++j)
                acc[j] *= a.scale;
            store_vec<T, VW>(out + (int64_t)v * VW, acc);
        }
    }
}

// The chunks' sums of each long run, added in order: a CTA looks at 256 chunks for runs that begin there.
template <typename T>
__global__ void __launch_bounds__(256) combine_kernel(const GradArgs a)
{
    __shared__ int64_t begins[256];
    __shared__ int64_t ends;
    __shared__ int found;
    __shared__ float sums[256];
    if (threadIdx.x == 0)
        found = 0;
    __syncthreads();
    pdl_wait();
    const int64_t chunks = (a.n + a.run - 1) / a.run;
    const int64_t chunk = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (chunk < chunks) {
        // A run that begins in a chunk and is long reaches the chunk's end.
        const int64_t begin = chunk * a.run, end = begin + a.run < a.n ? begin + a.run : a.n;
        const uint32_t tail = a.keys[end - 1];
        if (tail < a.n_rows) {
            const int64_t s = lower_bound(a.keys, tail, begin, end);
            if ((s > begin || s == 0 || a.keys[s - 1] != tail) && is_long(a, s))
                begins[atomicAdd(&found, 1)] = s;
        }
    }
    __syncthreads();
    // Threads: `wide` columns side by side, 256 / wide shares of a run's chunks.
    int wide = 256;
    while (wide / 2 >= a.cols)
        wide /= 2;
    const int shares = 256 / wide, share = threadIdx.x / wide;
    for (int f = 0; f < found; ++f) {
        const int64_t s = begins[f];
        const uint32_t key = a.keys[s];
        if (threadIdx.x < 32) {
            const int64_t e = warp_lower_bound(a.keys, key + 1, a.n);
            if (threadIdx.x == 0)
                ends = e;
        }
        __syncthreads();
        const int64_t c0 = s / a.run, c1 = (ends - 1) / a.run;
        const int64_t per = (c1 - c0 + shares) / shares;  // chunks of a share, of c1 - c0 + 1
        const int64_t from = c0 + share * per, to = from + per <= c1 ? from + per : c1 + 1;
        for (int col0 = 0; col0 < a.cols; col0 += wide) {
            const int col = col0 + threadIdx.x % wide;
            float sum = 0.f;
            if (col < a.cols)
                for (int64_t c = from; c < to; ++c)
                    sum += a.part[(c * 2 + (c == c0 && s != c0 * a.run ? 1 : 0)) * a.cols + col];
            sums[threadIdx.x] = sum;
            __syncthreads();
            if (share == 0 && col < a.cols) {
                for (int i = 1; i < shares; ++i)
                    sum += sums[i * wide + threadIdx.x];
                static_cast<T *>(a.out)[(int64_t)key * a.ld_out + col] = from_float<T>(sum * a.scale);
            }
            __syncthreads();
        }
    }
}

// ---- host ----------------------------------------------------------------------------------------------------------

int lanes_for(int64_t vecs)
{
    int l = 1;
    while (l < 32 && l < vecs)
        l *= 2;
    return l;
}

template <typename T, int VW> cudaError_t launch_lookup(LookupArgs a, int32_t dim, cudaStream_t st)
{
    a.vecs = dim / VW;
    a.lanes = lanes_for(a.vecs);
    const int64_t per_cta = 256 / a.lanes * 4;
    int64_t ctas = (a.n + per_cta - 1) / per_cta;
    const int64_t most = (int64_t)pspmm_sm_count() * 64;
    ctas = ctas < most ? ctas : most;
    lookup_kernel<T, VW, 4><<<(unsigned)ctas, 256, 0, st>>>(a);
    return cudaGetLastError();
}

template <typename T> cudaError_t lookup_typed(const LookupArgs &a, int32_t dim, cudaStream_t st)
{
    constexpr int B = sizeof(T), WIDE = 16 / B;
    auto aligned = [&](int bytes) {
        return dim * B % bytes == 0 && rows_aligned(a.table, a.ld_table, B, bytes) && rows_aligned(a.out, a.ld_out, B, bytes);
    };
    if (aligned(16))
        return launch_lookup<T, WIDE>(a, dim, st);
    if constexpr (B == 2)
        if (aligned(8))
            return launch_lookup<T, 4>(a, dim, st);
    return launch_lookup<T, 1>(a, dim, st);
}

// Positions of a chunk: short ones spread a small call over the GPU, long ones leave fewer sums of a hot id to add up.
int32_t run_for(int64_t n) { return n <= (1 << 16) ? 32 : n <= (1 << 18) ? 64 : n <= (1 << 20) ? 128 : 256; }

size_t round_up(size_t v) { return (v + 255) / 256 * 256; }

struct GradScratch {
    size_t keys[2], pos[2], counts, totals, part, bytes;
};
GradScratch grad_scratch(int64_t n, int32_t dim)
{
    GradScratch s;
    size_t at = 0;
    const size_t tiles = (size_t)((n + TILE - 1) / TILE);
    auto take = [&](size_t bytes) {
        const size_t p = at;
        at += round_up(bytes);
        return p;
    };
    for (int i = 0; i < 2; ++i) {
        s.keys[i] = take((size_t)n * 4);
        s.pos[i] = take((size_t)n * 4);
    }
    s.counts = take(n > RANK_MAX ? tiles * 256 * 4 : 0);
    s.totals = take(256 * 4);
    const int64_t run = run_for(n);
    s.part = take(n > run ? (size_t)((n + run - 1) / run) * 2 * (size_t)dim * 4 : 0);
    s.bytes = at;
    return s;
}

template <typename T, int VW> cudaError_t launch_grad(GradArgs a, int32_t dim, cudaStream_t st)
{
    a.vecs = dim / VW;
    a.lanes = lanes_for(a.vecs);
    a.slices = (a.vecs + a.lanes - 1) / a.lanes;
    const int64_t chunks = a.n > a.run ? (a.n + a.run - 1) / a.run : 0;
    a.units = chunks * a.slices;
    const int64_t per_cta = 256 / a.lanes;
    a.chunk_ctas = (int32_t)((a.units + per_cta - 1) / per_cta);
    // about 32 KB of the table per CTA
    int64_t tokens = (32 << 10) / ((int64_t)dim * sizeof(T));
    a.tokens = (int32_t)(tokens < per_cta ? per_cta : tokens > MOST_TOKENS ? MOST_TOKENS : tokens);
    const int64_t ctas = a.chunk_ctas + (a.n_rows + a.tokens - 1) / a.tokens;
    cudaError_t e = launch_dependent(grad_kernel<T, VW>, dim3((unsigned)ctas), 256, 0, st, a);
    if (e == cudaSuccess && chunks > 0)
        e = launch_dependent(combine_kernel<T>, dim3((unsigned)((chunks + 255) / 256)), 256, 0, st, a);
    return e;
}

template <typename T> cudaError_t grad_typed(const GradArgs &a, int32_t dim, cudaStream_t st)
{
    constexpr int B = sizeof(T), WIDE = 16 / B;
    auto aligned = [&](int bytes) {
        return dim * B % bytes == 0 && rows_aligned(a.grad, a.ld_grad, B, bytes) && rows_aligned(a.out, a.ld_out, B, bytes);
    };
    if (aligned(16))
        return launch_grad<T, WIDE>(a, dim, st);
    if constexpr (B == 2)
        if (aligned(8))
            return launch_grad<T, 4>(a, dim, st);
    return launch_grad<T, 1>(a, dim, st);
}

bool misaligned(const void *p, int bytes) { return (uintptr_t)p % bytes != 0; }

}  // namespace

extern "C" int pspmm_embedding(const void *ids, int32_t ids64, int64_t n, const void *table, int32_t dtype, int64_t n_rows,
                               int32_t dim, int64_t ld_table, float scale, void *out, int64_t ld_out, void *stream)
{
    if (!dtype_ok(dtype) || n < 0 || n_rows < 0 || dim < 1 || ld_table < dim || ld_out < dim)
        return PSPMM_E_ARG;
    if (n == 0)
        return PSPMM_OK;
    const int B = elem_bytes(dtype);
    if (!ids || (!table && n_rows > 0) || !out || misaligned(ids, ids64 ? 8 : 4) || misaligned(table, B) || misaligned(out, B))
        return PSPMM_E_ARG;
    const LookupArgs a = {ids, table, out, n, n_rows, ld_table, ld_out, ids64 != 0, 0, 0, scale};
    cudaStream_t st = (cudaStream_t)stream;
    PSPMM_CUDA_TRY(dtype == PSPMM_F32    ? lookup_typed<float>(a, dim, st)
                   : dtype == PSPMM_BF16 ? lookup_typed<bf16>(a, dim, st)
                                         : lookup_typed<f16>(a, dim, st));
    return PSPMM_OK;
}

extern "C" int pspmm_embedding_grad_scratch_bytes(int64_t n, int32_t dim, size_t *bytes)
{
    if (n < 0 || dim < 1 || !bytes)
        return PSPMM_E_ARG;
    *bytes = n > 0 ? grad_scratch(n, dim).bytes : 0;
    return PSPMM_OK;
}

extern "C" int pspmm_embedding_grad(const void *ids, int32_t ids64, int64_t n, const void *grad, int32_t dtype, int64_t ld_grad,
                                    int64_t n_rows, int32_t dim, float scale, int64_t padding, void *out, int64_t ld_out,
                                    void *scratch, size_t scratch_bytes, void *stream)
{
    if (!dtype_ok(dtype) || n < 0 || n_rows < 0 || dim < 1 || ld_grad < dim || ld_out < dim)
        return PSPMM_E_ARG;
    if (n_rows == 0)
        return PSPMM_OK;
    const int B = elem_bytes(dtype);
    if (!out || misaligned(out, B))
        return PSPMM_E_ARG;
    // (CTAs take at least 8 rows of the table, at least a lane group per chunk and slice)
    if (n > INT32_MAX - 65536 || n_rows > (int64_t)UINT32_MAX - 1 || dim > (1 << 24) ||
        (n / run_for(n) + 1) * ((int64_t)dim / 32 + 1) + n_rows > INT32_MAX - 65536)
        return PSPMM_E_RANGE;
    cudaStream_t st = (cudaStream_t)stream;
    if (n == 0) {
        PSPMM_CUDA_TRY(cudaMemset2DAsync(out, (size_t)ld_out * B, 0, (size_t)dim * B, (size_t)n_rows, st));
        return PSPMM_OK;
    }
    const GradScratch lay = grad_scratch(n, dim);
    if (!ids || !grad || !scratch || scratch_bytes < lay.bytes || misaligned(ids, ids64 ? 8 : 4) || misaligned(grad, B) ||
        misaligned(scratch, 16))
        return PSPMM_E_ARG;
    char *base = (char *)scratch;
    uint32_t *keys[2], *pos[2];
    for (int i = 0; i < 2; ++i) {
        keys[i] = (uint32_t *)(base + lay.keys[i]);
        pos[i] = (uint32_t *)(base + lay.pos[i]);
    }
    SortArgs s = {{ids, n, n_rows, padding, ids64 != 0}, nullptr, nullptr, keys[0], pos[0], (uint32_t *)(base + lay.counts),
                  (uint32_t *)(base + lay.totals), (int32_t)((n + TILE - 1) / TILE), 0};
    int last = 0;
    if (n <= RANK_MAX) {
        rank_kernel<<<(unsigned)((n + 7) / 8), 256, 0, st>>>(s);
        PSPMM_CUDA_TRY(cudaGetLastError());
    } else {
        int bits = 1;
        while (bits < 32 && (n_rows >> bits) != 0)
            ++bits;  // keys are 0 .. n_rows
        for (int p = 0; p * 8 < bits; ++p) {
            s.key_in = p ? keys[last] : nullptr;
            s.pos_in = p ? pos[last] : nullptr;
            last = p ? last ^ 1 : 0;
            s.key_out = keys[last];
            s.pos_out = pos[last];
            s.shift = 8 * p;
            digit_count_kernel<<<s.tiles, TILE_THREADS, 0, st>>>(s);
            PSPMM_CUDA_TRY(cudaGetLastError());
            digit_scan_kernel<<<256, 256, 0, st>>>(s);
            PSPMM_CUDA_TRY(cudaGetLastError());
            digit_scatter_kernel<<<s.tiles, TILE_THREADS, 0, st>>>(s);
            PSPMM_CUDA_TRY(cudaGetLastError());
        }
    }
    const GradArgs a = {keys[last], pos[last], grad, out, (float *)(base + lay.part), n, n_rows, ld_grad, ld_out, 0, 0,
                        run_for(n), 0, 0, 0, 0, dim, scale};
    PSPMM_CUDA_TRY(dtype == PSPMM_F32    ? grad_typed<float>(a, dim, st)
                   : dtype == PSPMM_BF16 ? grad_typed<bf16>(a, dim, st)
                                         : grad_typed<f16>(a, dim, st));
    return PSPMM_OK;
}

extern "C" int pspmm_embedding_status(int32_t *status)
{
    if (!status)
        return PSPMM_E_ARG;
    unsigned v = 0;
    PSPMM_CUDA_TRY(cudaMemcpyFromSymbol(&v, g_embedding_status, sizeof(v)));
    *status = (int32_t)v;
    return PSPMM_OK;
}
