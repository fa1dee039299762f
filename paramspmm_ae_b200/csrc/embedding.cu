// Rows of a table looked up by id and scaled, and the table's gradient:
//     out[i] = s T[id_i],      dT[t] = s * sum over {i : id_i = t} G[i]
//
// Lookup: a gather, bound by HBM (each row of the table once if ids repeat close together, each row of `out`).
//
// Gradient: the ids are sorted with their positions (stable, so that a row's sum has one order whatever the timing).  Lane groups then
// take equal chunks of sorted positions, gather the rows of G in that order and store a row of dT where an id's run of positions ends.
// Runs that cross the border of a chunk leave their pieces in scratch, which a dependent launch adds in order: no atomics
// on values, and the hottest id does not hold the launch up.  The rows that no id names are zeroed, with all others, by CTAs of the
// sorting kernels, which leave the memory system idle.
// Up to RANK_MAX ids are sorted by counting, one launch; more by least-significant-digit passes of up to 9 bits, as many as the
// table's size needs, one or two launches each: a pass counts the digits of the next one while it places its keys.
// Lookup and gradient in us: 1,000,003 ids of 2,449,029 rows of 64 fp32 77 + 245, of which 90 write the zeros of dT; 32,768 ids into
// 50,021 rows of 1,024 bf16 21 + 66; 200,003 ids into 100,003 rows of 47 fp32 17 + 53, of which 31 sort.
// Ids outside the table: NaN rows in the lookup, nothing in the gradient, and pspmm_embedding_status tells.
#include "feature_types.cuh"

namespace {
using namespace feat;

__device__ unsigned g_embedding_status;

constexpr int RANK_MAX = 2048;
constexpr int TILE_THREADS = 256, TILE_KEYS = 8, TILE = TILE_THREADS * TILE_KEYS;  // keys of a CTA in a digit pass
constexpr int WARPS = TILE_THREADS / 32;
constexpr int DIGIT_BITS = 9, DIGITS = 1 << DIGIT_BITS;  // at most (nine: a table of 2^17 to 2^18 rows in two passes, not three)
constexpr int SCAN_TILES = 32;
constexpr int HOT = 64;  // chunks from which on a run's pieces are added by a CTA

struct LookupArgs {
    const void *ids, *table;
    void *out;
    int64_t n, n_rows, ld_table, ld_out;
    int32_t ids64, cols;
    float scale;
};

struct Ids {
    const void *ids;
    int64_t n, n_rows, padding;  // padding: the id without a gradient (-1: none)
    int32_t ids64;
};

// Memory that the sorting kernels zero beside their work: a share of it each.
struct Fill {
    char *p;
    int64_t bytes;
    int32_t share, shares, ctas;  // shares done, and in all
    int32_t now;                  // shares of this launch
};

// Sorted and unsorted ids are pairs: sort key in x, position in y.
struct SortArgs {
    Ids in;
    const uint2 *from;  // null: the first pass, from `in`
    uint2 *to;
    uint32_t *counts;   // keys of each digit and tile; where scanned, each tile's first place inside its digit
    uint32_t *totals;   // [digits] of a scanned pass; null: the tiles add up the counts before them on their own
    uint32_t *next;     // counts of the next pass, added up while this one's keys are placed; null: there is none
    int32_t tiles, shift;
    int32_t passes, bits, mask;  // of a digit
    int32_t work;       // CTAs that sort; those behind them fill
    Fill fill;
};

struct GradArgs {
    const uint2 *ids;   // sorted
    const void *grad;
    void *out;
    float *part;        // [chunks][2][cols]: the piece that begins with the chunk, and the one that begins inside and goes on
    int64_t n, n_rows, ld_grad, ld_out;
    int64_t units;      // chunks * slices
    int32_t run, vecs, slices, cols;
    int32_t hot_ctas;   // combine: the first CTAs take runs of more than HOT chunks
    float scale;
};

__device__ __forceinline__ int64_t load_id(const void *ids, int ids64, int64_t i)
{
    return ids64 ? static_cast<const int64_t *>(ids)[i] : (int64_t)static_cast<const int32_t *>(ids)[i];
}
// A store that does not displace what the caches hold.
template <typename T, int VW> __device__ __forceinline__ void store_past(T *p, const Vec<T, VW> &v)
{
    if constexpr (sizeof(v) == 16)
        __stcs(reinterpret_cast<uint4 *>(p), *reinterpret_cast<const uint4 *>(&v));
    else if constexpr (sizeof(v) == 8)
        __stcs(reinterpret_cast<uint2 *>(p), *reinterpret_cast<const uint2 *>(&v));
    else if constexpr (sizeof(v) == 4)
        __stcs(reinterpret_cast<uint32_t *>(p), *reinterpret_cast<const uint32_t *>(&v));
    else
        __stcs(reinterpret_cast<unsigned short *>(p), *reinterpret_cast<const unsigned short *>(&v));
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

// L lanes share a row; a lane group takes ROWS neighbouring rows of the output and has them in flight together.  A warp's ids are looked at
// by a lane each (by all of them: 52 instructions per 32 values of rows of 47, 24 us against 17).  Stored past the caches' order, so that the
// table's rows stay.
template <typename T, int VW, int L, int ROWS>
__global__ void __launch_bounds__(256) lookup_kernel(const LookupArgs a)
{
    typedef Vec<T, VW> V;
    constexpr int PER_WARP = 32 / L * ROWS;
    static_assert(PER_WARP <= 32, "a lane per row");
    const int lane = threadIdx.x % 32;
    const int64_t first = ((int64_t)blockIdx.x * 8 + threadIdx.x / 32) * PER_WARP;
    if (first >= a.n)
        return;
    int64_t at = -1;
    if (lane < PER_WARP && first + lane < a.n) {
        const int64_t id = load_id(a.ids, a.ids64, first + lane);
        if (id >= 0 && id < a.n_rows)
            at = id * a.ld_table;
        else
            g_embedding_status = 1;
    }
    int64_t from[ROWS];
#pragma unroll
    for (int r = 0; r < ROWS; ++r)
        from[r] = __shfl_sync(PSPMM_FULL_MASK, at, lane / L * ROWS + r);
    const int64_t i0 = first + lane / L * ROWS;
    const int rows = a.n - i0 < ROWS ? (int)(a.n - i0) : ROWS;
    const float nan = __int_as_float(0x7fc00000);
    const T *table = static_cast<const T *>(a.table);
    T *out = static_cast<T *>(a.out) + i0 * a.ld_out;
    for (int c = lane % L * VW; c < a.cols; c += L * VW) {
        V f[ROWS];
#pragma unroll
        for (int r = 0; r < ROWS; ++r) {
            if (from[r] >= 0) {
                f[r] = *reinterpret_cast<const V *>(table + from[r] + c);
            } else {
#pragma unroll
                for (int j = 0; j < VW; ++j)
                    f[r].v[j] = from_float<T>(nan);
            }
        }
#pragma unroll
        for (int r = 0; r < ROWS; ++r) {
#pragma unroll
            for (int j = 0; j < VW; ++j)
                f[r].v[j] = from_float<T>(to_float(f[r].v[j]) * a.scale);
            if (r < rows)
                store_past(out + r * a.ld_out + c, f[r]);
        }
    }
}

// ---- sorting -------------------------------------------------------------------------------------------------------

// A share of the memory, cut at 16 bytes, by the CTAs from `work` on.
__device__ __forceinline__ void fill_zeros(const Fill &f, int cta)
{
    const int64_t lead = min((int64_t)(-(uintptr_t)f.p & 15), f.bytes), whole = (f.bytes - lead) / 16;
    uint4 *p = reinterpret_cast<uint4 *>(f.p + lead);
    const int64_t from = whole * f.share / f.shares, to = whole * (f.share + f.now) / f.shares;
    for (int64_t i = from + (int64_t)cta * 256 + threadIdx.x; i < to; i += (int64_t)f.ctas * 256)
        p[i] = make_uint4(0, 0, 0, 0);
    if (f.share == 0 && cta == 0) {  // the ends (elements of 2 or 4 bytes)
        uint16_t *q = reinterpret_cast<uint16_t *>(f.p);
        for (int64_t i = threadIdx.x; i < lead / 2; i += 256)
            q[i] = 0;
        for (int64_t i = (lead + whole * 16) / 2 + threadIdx.x; i < f.bytes / 2; i += 256)
            q[i] = 0;
    }
}

// Counts lie by tile where the tiles read them all, else by digit.
__device__ __forceinline__ int64_t count_at(const SortArgs &a, int64_t tile, uint32_t digit)
{
    return a.totals ? digit * (int64_t)a.tiles + tile : (tile << a.bits) + digit;
}

// Few ids: the place of a key is the number of smaller ones and of equal ones before it; a warp counts for one key.
__global__ void __launch_bounds__(256) rank_kernel(const SortArgs a)
{
    __shared__ uint32_t keys[RANK_MAX];
    pdl_launch_dependents();
    if ((int)blockIdx.x >= a.work) {
        fill_zeros(a.fill, blockIdx.x - a.work);
        return;
    }
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
    if (lane == 0)
        a.to[before] = make_uint2(key, (uint32_t)i);
}

__device__ __forceinline__ uint2 sort_pair(const SortArgs &a, int64_t i)
{
    return a.from ? a.from[i] : make_uint2(load_key(a.in, i), (uint32_t)i);
}

// Of the first pass; the others are counted by the pass before.
__global__ void __launch_bounds__(TILE_THREADS) digit_count_kernel(const SortArgs a)
{
    __shared__ uint32_t bins[DIGITS];
    pdl_launch_dependents();
    if ((int)blockIdx.x >= a.work) {
        fill_zeros(a.fill, blockIdx.x - a.work);
        return;
    }
    for (int d = threadIdx.x; d <= a.mask; d += TILE_THREADS) {
        bins[d] = 0;
        for (int p = 1; p < a.passes; ++p)
            a.counts[(((int64_t)p * a.tiles + blockIdx.x) << a.bits) + d] = 0;
    }
    __syncthreads();
    uint32_t key[TILE_KEYS];
#pragma unroll
    for (int k = 0; k < TILE_KEYS; ++k) {
        const int64_t i = (int64_t)blockIdx.x * TILE + k * TILE_THREADS + threadIdx.x;
        key[k] = i < a.in.n ? load_key(a.in, i) : 0;
    }
#pragma unroll
    for (int k = 0; k < TILE_KEYS; ++k)
        if ((int64_t)blockIdx.x * TILE + k * TILE_THREADS + threadIdx.x < a.in.n)
            atomicAdd(&bins[key[k] >> a.shift & a.mask], 1u);
    __syncthreads();
    for (int d = threadIdx.x; d <= a.mask; d += TILE_THREADS)
        a.counts[count_at(a, blockIdx.x, d)] = bins[d];
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
    pdl_launch_dependents();
    if ((int)blockIdx.x >= a.work) {
        fill_zeros(a.fill, blockIdx.x - a.work);
        return;
    }
    pdl_wait();
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

// Stable: a warp takes 256 neighbouring keys, 32 at a time; equal digits among the 32 find one another by a ballot per bit
// (which was faster than one match instruction), and a count per warp and digit carries on from one 32 to the next.  The tile is put in
// order in shared memory, so that equal digits leave side by side.  Bound by latency: 8 dependent rounds per warp, 10 to 17 us per pass of
// 200,003 keys with its scan.
// PER neighbouring digits per thread.
template <int PER>
__global__ void __launch_bounds__(TILE_THREADS) digit_scatter_kernel(const SortArgs a)
{
    __shared__ uint32_t seen[WARPS][256 * PER];
    __shared__ uint32_t away[256 * PER];  // from a key's place in the tile to its place among all
    __shared__ uint32_t warps[8];
    __shared__ uint2 tile[TILE];
    pdl_launch_dependents();
    if ((int)blockIdx.x >= a.work) {
        fill_zeros(a.fill, blockIdx.x - a.work);
        return;
    }
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
    for (int i = threadIdx.x; i < WARPS * 256 * PER; i += TILE_THREADS)
        (&seen[0][0])[i] = 0;
    __syncthreads();
    pdl_wait();
    uint2 pair[TILE_KEYS];
    uint32_t rank[TILE_KEYS];
    const int64_t i0 = (int64_t)blockIdx.x * TILE + warp * (32 * TILE_KEYS) + lane;
#pragma unroll
    for (int k = 0; k < TILE_KEYS; ++k)
        if (i0 + k * 32 < a.in.n)
            pair[k] = sort_pair(a, i0 + k * 32);
    // keys of this thread's digits: in all tiles, in those before this one
    uint32_t total, all[PER] = {}, earlier[PER] = {}, sum = 0;
#pragma unroll
    for (int e = 0; e < PER; ++e) {
        const int d = threadIdx.x * PER + e;
        if (d > a.mask) {
        } else if (a.totals) {
            all[e] = a.totals[d];
            earlier[e] = a.counts[count_at(a, blockIdx.x, d)];
        } else {
#pragma unroll 16
            for (int t = 0; t < a.tiles; ++t) {
                const uint32_t c = a.counts[(t << a.bits) + d];
                all[e] += c;
                earlier[e] += t < (int)blockIdx.x ? c : 0;
            }
        }
        sum += all[e];
    }
    uint32_t first = exclusive_256(sum, warps, total);
#pragma unroll
    for (int k = 0; k < TILE_KEYS; ++k) {
        const bool in = i0 + k * 32 < a.in.n;
        const uint32_t d = in ? pair[k].x >> a.shift & a.mask : 0;
        uint32_t same = __ballot_sync(PSPMM_FULL_MASK, in);
        for (int b = 0; b < a.bits; ++b) {
            const uint32_t set = __ballot_sync(PSPMM_FULL_MASK, d >> b & 1);
            same &= d >> b & 1 ? set : ~set;
        }
        const uint32_t below = __popc(same & ((1u << lane) - 1));
        rank[k] = in ? seen[warp][d] + below : 0;
        __syncwarp();
        if (in && below == 0)
            seen[warp][d] += __popc(same);
        __syncwarp();
    }
    __syncthreads();
    uint32_t mine = 0;
#pragma unroll
    for (int e = 0; e < PER; ++e)
        for (int w = 0; w < WARPS; ++w)
            mine += seen[w][threadIdx.x * PER + e];
    uint32_t before = exclusive_256(mine, warps, total);
#pragma unroll
    for (int e = 0; e < PER; ++e) {
        const int d = threadIdx.x * PER + e;
        away[d] = first + earlier[e] - before;
        first += all[e];
        for (int w = 0; w < WARPS; ++w) {
            const uint32_t c = seen[w][d];
            seen[w][d] = before;
            before += c;
        }
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < TILE_KEYS; ++k)
        if (i0 + k * 32 < a.in.n)
            tile[seen[warp][pair[k].x >> a.shift & a.mask] + rank[k]] = pair[k];
    __syncthreads();
#pragma unroll
    for (int k = 0; k < TILE_KEYS; ++k) {
        const uint32_t j = k * TILE_THREADS + threadIdx.x;
        uint32_t place = 0xffffffffu;
        if (j < total) {
            const uint2 v = tile[j];
            const uint32_t to = away[v.x >> a.shift & a.mask] + j;
            a.to[to] = v;
            place = (uint32_t)count_at(a, to / TILE, v.x >> (a.shift + a.bits) & a.mask);
        }
        if (a.next) {
            // A hot id's keys lie side by side: one addition for neighbours with one place (in turn, additions to a place take 50 ns each).
            const uint32_t left = __shfl_up_sync(PSPMM_FULL_MASK, place, 1);
            const uint32_t heads = __ballot_sync(PSPMM_FULL_MASK, lane == 0 || place != left);
            if (place != 0xffffffffu && (heads >> lane & 1)) {
                const uint32_t behind = lane == 31 ? 0 : heads >> (lane + 1);
                atomicAdd(&a.next[place], behind ? (uint32_t)__ffs(behind) : (uint32_t)(32 - lane));
            }
        }
    }
}

// ---- sums ----------------------------------------------------------------------------------------------------------

// First position in [lo, n) whose key is not below `key` (n: none), by a whole warp, 32 probes a step.
__device__ __forceinline__ int64_t warp_lower_bound(const uint2 *ids, uint32_t key, int64_t lo, int64_t n)
{
    const int lane = threadIdx.x % 32;
    int64_t hi = n;  // the answer lies in [lo, hi]
    while (hi - lo > 32) {
        const int64_t step = (hi - lo + 31) / 32;
        const int64_t at = lo + lane * step;
        const bool below = at < hi && ids[at].x < key;
        const int c = __popc(__ballot_sync(PSPMM_FULL_MASK, below));
        if (c == 0)
            return lo;
        const int64_t from = lo + (c - 1) * step;
        lo = from + 1;
        hi = from + step < hi ? from + step : hi;
    }
    const bool below = lo + lane < hi && ids[lo + lane].x < key;
    return lo + __popc(__ballot_sync(PSPMM_FULL_MASK, below));
}

// A group of L lanes per chunk and slice of columns, a vector per lane, U rows in flight; a lane looks at a position, and the places of the
// rows and of the runs' beginnings go round by shuffles and a ballot.  Bound by the latency of its gathers: 64 registers and 32 warps per SM were
// faster than 80 and 24, spills and all (32,768 ids, rows of 1,024 bf16, sorting and all: 72 -> 67 us).
template <typename T, int VW, int L>
__global__ void __launch_bounds__(256, 4) grad_kernel(const GradArgs a)
{
    constexpr int U = L < 8 ? L : sizeof(T) * VW <= 4 && L >= 16 ? 16 : 8;
    typedef Vec<T, VW> V;
    pdl_launch_dependents();
    const int64_t unit = (int64_t)blockIdx.x * (256 / L) + threadIdx.x / L;
    if (unit >= a.units)
        return;
    const int lane = threadIdx.x % 32, group = lane / L * L, look = lane % U;
    const uint32_t mask = L == 32 ? PSPMM_FULL_MASK : ((1u << L) - 1) << group;
    const int64_t chunk = unit / a.slices;
    const int v = (int)(unit % a.slices) * L + lane % L;
    const int64_t begin = chunk * a.run, end = begin + a.run < a.n ? begin + a.run : a.n;
    // (lanes beyond the row's vectors load the last one again)
    const T *grad = static_cast<const T *>(a.grad) + (int64_t)min(v, a.vecs - 1) * VW;
    const bool mine = v < a.vecs;
    float acc[VW] = {};
    pdl_wait();
    uint32_t key = a.ids[begin].x;
    const bool goes_on = end < a.n && a.ids[end - 1].x == a.ids[end].x;  // the last run, behind the chunk
    bool whole = begin == 0 || a.ids[begin - 1].x != key, head = true;   // of the run at hand: begins here; with the chunk
    auto finish = [&](bool ends) {
        if (key >= a.n_rows || !mine)
            return;
        if (whole && ends) {
#pragma unroll
            for (int j = 0; j < VW; ++j)
                acc[j] *= a.scale;
            store_vec<T, VW>(static_cast<T *>(a.out) + (int64_t)key * a.ld_out + (int64_t)v * VW, acc);
        } else {
            float *part = a.part + (chunk * 2 + (head ? 0 : 1)) * a.cols + (int64_t)v * VW;
#pragma unroll
            for (int j = 0; j < VW; ++j)
                part[j] = acc[j];
        }
    };
    for (int64_t p = begin; p < end; p += U) {
        const uint2 id = a.ids[p + look < end ? p + look : end - 1];
        const uint32_t before = __shfl_up_sync(mask, id.x, 1);
        const uint32_t begins = __ballot_sync(mask, id.x != (look == 0 ? key : before)) >> group;
        const int64_t at = (int64_t)id.y * a.ld_grad;
        V f[U];
#pragma unroll
        for (int u = 0; u < U; ++u)
            f[u] = *reinterpret_cast<const V *>(grad + __shfl_sync(mask, at, group + u));
        const int here = end - p < U ? (int)(end - p) : U;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (u >= here)
                break;
            if (begins >> u & 1) {
                finish(true);
                key = __shfl_sync(mask, id.x, group + u);
                whole = true;
                head = false;
#pragma unroll
                for (int j = 0; j < VW; ++j)
                    acc[j] = 0.f;
            }
#pragma unroll
            for (int j = 0; j < VW; ++j)
                acc[j] += to_float(f[u].v[j]);
        }
    }
    finish(!goes_on);
}

// The pieces of each run that crosses chunks, added in order.  A warp per chunk and 128 columns looks for the run that begins in the
// chunk and goes on; one of more than HOT chunks is left to a CTA per HOT chunks and 16 columns, sixteen shares of the pieces each.
template <typename T>
__global__ void __launch_bounds__(256) combine_kernel(const GradArgs a)
{
    __shared__ float sums[16][17];
    const int64_t chunks = (a.n + a.run - 1) / a.run;
    const uint2 *ids = a.ids;
    pdl_wait();
    if ((int)blockIdx.x < a.hot_ctas) {
        const int tiles = (a.cols + 15) / 16;
        const int64_t first = (int64_t)(blockIdx.x / tiles) * HOT * a.run, next = first + (int64_t)HOT * a.run;
        if (next >= a.n)
            return;
        const uint32_t key = ids[next].x;
        if (key >= a.n_rows || ids[next - 1].x != key)
            return;
        const int64_t s = warp_lower_bound(ids, key, first, next);
        if (s == first && first > 0 && ids[first - 1].x == key)
            return;
        const int64_t c0 = s / a.run;
        if ((c0 + HOT) * a.run >= a.n || ids[(c0 + HOT) * a.run].x != key)
            return;
        const int64_t c1 = (warp_lower_bound(ids, key + 1, next, a.n) - 1) / a.run;
        const int col = (int)(blockIdx.x % tiles) * 16 + threadIdx.x % 16, share = threadIdx.x / 16;
        const int64_t per = (c1 - c0 + 16) / 16;
        const int64_t from = c0 + share * per, to = from + per <= c1 ? from + per : c1 + 1;
        float sum = 0.f;
        if (col < a.cols) {
            const int inside = s != c0 * a.run ? 1 : 0;
#pragma unroll 8
            for (int64_t c = from; c < to; ++c)
                sum += a.part[(c * 2 + (c == c0 ? inside : 0)) * a.cols + col];
        }
        sums[share][threadIdx.x % 16] = sum;
        __syncthreads();
        if (share == 0 && col < a.cols) {
#pragma unroll
            for (int i = 1; i < 16; ++i)
                sum += sums[i][threadIdx.x];
            static_cast<T *>(a.out)[(int64_t)key * a.ld_out + col] = from_float<T>(sum * a.scale);
        }
        return;
    }
    const int tiles = (a.cols + 127) / 128, lane = threadIdx.x % 32;
    const int64_t unit = (int64_t)(blockIdx.x - a.hot_ctas) * 8 + threadIdx.x / 32;
    const int64_t chunk = unit / tiles;
    if (chunk >= chunks)
        return;
    const int64_t begin = chunk * a.run, end = begin + a.run;
    if (end >= a.n)
        return;
    const uint32_t key = ids[end].x;
    if (key >= a.n_rows || ids[end - 1].x != key)
        return;
    const int64_t s = warp_lower_bound(ids, key, begin, end);
    if (s == begin && begin > 0 && ids[begin - 1].x == key)
        return;
    const int64_t far = (chunk + HOT) * a.run;
    if (far < a.n && ids[far].x == key)
        return;
    const int64_t c1 = (warp_lower_bound(ids, key + 1, end, far < a.n ? far : a.n) - 1) / a.run;
    const int col = (int)(unit % tiles) * 128 + lane;
    float sum[4] = {};
    for (int64_t c0 = chunk; c0 <= c1; c0 += 4) {
        float f[4][4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int64_t c = c0 + u;
            const float *part = a.part + (c * 2 + (c == chunk && s != begin ? 1 : 0)) * a.cols + col;
#pragma unroll
            for (int t = 0; t < 4; ++t)
                f[u][t] = c <= c1 && col + 32 * t < a.cols ? part[32 * t] : 0.f;
        }
#pragma unroll
        for (int u = 0; u < 4; ++u)
#pragma unroll
            for (int t = 0; t < 4; ++t)
                sum[t] += f[u][t];
    }
#pragma unroll
    for (int t = 0; t < 4; ++t)
        if (col + 32 * t < a.cols)
            static_cast<T *>(a.out)[(int64_t)key * a.ld_out + col + 32 * t] = from_float<T>(sum[t] * a.scale);
}

// ---- host ----------------------------------------------------------------------------------------------------------

template <typename T, int VW, int L> cudaError_t launch_lookup_lanes(const LookupArgs &a, cudaStream_t st)
{
    const int64_t groups = 256 / L, ctas = (a.n + groups - 1) / groups, enough = 4 * (int64_t)pspmm_sm_count();
    // several rows per lane group where that still leaves every SM some CTAs
    if (L >= 8 && ctas >= 8 * enough)
        lookup_kernel<T, VW, L, L < 8 ? L : 8><<<(unsigned)((ctas + 7) / 8), 256, 0, st>>>(a);
    else if (ctas >= 4 * enough)
        lookup_kernel<T, VW, L, 4><<<(unsigned)((ctas + 3) / 4), 256, 0, st>>>(a);
    else
        lookup_kernel<T, VW, L, 1><<<(unsigned)ctas, 256, 0, st>>>(a);
    return cudaGetLastError();
}

template <typename T, int VW> cudaError_t launch_lookup(const LookupArgs &a, int32_t dim, cudaStream_t st)
{
    const int vecs = dim / VW;
    return vecs <= 4    ? launch_lookup_lanes<T, VW, 4>(a, st)
           : vecs <= 8  ? launch_lookup_lanes<T, VW, 8>(a, st)
           : vecs <= 16 ? launch_lookup_lanes<T, VW, 16>(a, st)
                        : launch_lookup_lanes<T, VW, 32>(a, st);
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

// Positions of a chunk: short ones spread a small call over the GPU, long ones leave fewer pieces to add.
int32_t run_for(int64_t n) { return n <= (1 << 12) ? 8 : n <= (1 << 16) ? 32 : n <= (1 << 20) ? 64 : 128; }

size_t round_up(size_t v) { return (v + 255) / 256 * 256; }

struct GradScratch {
    size_t pairs[2], counts, totals, part, bytes;
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
    for (int i = 0; i < 2; ++i)
        s.pairs[i] = take(i == 0 || n > RANK_MAX ? (size_t)n * 8 : 0);
    s.counts = take(n > RANK_MAX ? 4 * tiles * DIGITS * 4 : 0);  // of up to four passes
    s.totals = take(n > RANK_MAX ? DIGITS * 4 : 0);
    const int64_t run = run_for(n);
    s.part = take(n > run ? (size_t)((n + run - 1) / run) * 2 * (size_t)dim * 4 : 0);
    s.bytes = at;
    return s;
}

template <typename T, int VW, int L> cudaError_t launch_grad_lanes(GradArgs a, cudaStream_t st)
{
    a.slices = (a.vecs + L - 1) / L;
    const int64_t chunks = (a.n + a.run - 1) / a.run, per_cta = 256 / L;
    a.units = chunks * a.slices;
    cudaError_t e = launch_dependent(grad_kernel<T, VW, L>, dim3((unsigned)((a.units + per_cta - 1) / per_cta)), 256, 0, st, a);
    if (e != cudaSuccess || chunks == 1)
        return e;
    a.hot_ctas = (int32_t)(chunks / HOT * ((a.cols + 15) / 16));
    const int64_t warps = chunks * ((a.cols + 127) / 128);
    return launch_dependent(combine_kernel<T>, dim3((unsigned)(a.hot_ctas + (warps + 7) / 8)), 256, 0, st, a);
}

template <typename T, int VW> cudaError_t launch_grad(GradArgs a, int32_t dim, cudaStream_t st)
{
    a.vecs = dim / VW;
    return a.vecs <= 4    ? launch_grad_lanes<T, VW, 4>(a, st)
           : a.vecs <= 8  ? launch_grad_lanes<T, VW, 8>(a, st)
           : a.vecs <= 16 ? launch_grad_lanes<T, VW, 16>(a, st)
                          : launch_grad_lanes<T, VW, 32>(a, st);
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
    if (dim > (1 << 24) || n > (int64_t)INT32_MAX * 8)
        return PSPMM_E_RANGE;
    const LookupArgs a = {ids, table, out, n, n_rows, ld_table, ld_out, ids64 != 0, dim, scale};
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
    const int64_t chunks = n / run_for(n) + 1;  // (a warp per chunk and 32 columns at most, a CTA per HOT chunks and 16)
    if (n > INT32_MAX - 65536 || n_rows > (int64_t)UINT32_MAX - 2 || dim > (1 << 24) ||
        chunks * ((int64_t)dim / 32 + 1) + chunks / HOT * ((int64_t)dim / 16 + 1) > INT32_MAX - 65536)
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
    uint2 *pairs[2] = {(uint2 *)(base + lay.pairs[0]), (uint2 *)(base + lay.pairs[1])};
    const int32_t tiles = (int32_t)((n + TILE - 1) / TILE);
    uint32_t *counts = (uint32_t *)(base + lay.counts);
    int bits = 1;
    while (bits < 32 && (n_rows >> bits) != 0)
        ++bits;  // keys are 0 .. n_rows
    const int passes = n <= RANK_MAX ? 0 : (bits + DIGIT_BITS - 1) / DIGIT_BITS, digit = passes ? (bits + passes - 1) / passes : 0;
    // The counts before a tile: read by each up to this many tiles (tiles^2 or twice as many KB in all), else scanned by a launch of its own.
    const bool scan = tiles > SCAN_TILES;
    SortArgs s = {{ids, n, n_rows, padding, ids64 != 0}, nullptr, pairs[0], counts, scan ? (uint32_t *)(base + lay.totals) : nullptr,
                  nullptr, tiles, 0, passes, digit, (1 << digit) - 1, 0, {}};
    s.fill = {(char *)out, n_rows * dim * B, 0, passes ? 1 + (scan ? 3 : 2) * passes : 1, 0, 1};
    if (ld_out != dim) {  // (rows apart from one another)
        PSPMM_CUDA_TRY(cudaMemset2DAsync(out, (size_t)ld_out * B, 0, (size_t)dim * B, (size_t)n_rows, st));
        s.fill.bytes = 0;
    }
    // CTAs that fill: 16 KB each, or four per SM.  The passes' placing takes longest and has two shares.
    const int64_t fill = (s.fill.bytes / s.fill.shares + (16 << 10) - 1) >> 14, most = 4 * (int64_t)pspmm_sm_count();
    s.fill.ctas = (int32_t)(fill < 1 ? 1 : fill < most ? fill : most);
    // (the first launch waits for all before it; the others, for one another where they need to)
    auto first = [&](void (*kern)(const SortArgs), int work) {
        s.work = work;
        kern<<<(unsigned)(work + s.fill.ctas), 256, 0, st>>>(s);
        ++s.fill.share;
        return cudaGetLastError();
    };
    auto then = [&](void (*kern)(const SortArgs), int work, int shares) {
        s.work = work;
        s.fill.now = shares;
        const cudaError_t e = launch_dependent(kern, dim3((unsigned)(work + s.fill.ctas)), 256, 0, st, s);
        s.fill.share += shares;
        return e;
    };
    PSPMM_CUDA_TRY(passes ? first(digit_count_kernel, tiles) : first(rank_kernel, (int)((n + 7) / 8)));
    int last = 0;
    for (int p = 0; p < passes; ++p) {
        s.from = p ? pairs[last] : nullptr;
        last = p ? last ^ 1 : 0;
        s.to = pairs[last];
        s.shift = digit * p;
        s.counts = counts + ((int64_t)p * tiles << digit);
        s.next = p + 1 < passes ? s.counts + ((int64_t)tiles << digit) : nullptr;
        if (scan)
            PSPMM_CUDA_TRY(then(digit_scan_kernel, 1 << digit, 1));
        PSPMM_CUDA_TRY(then(digit > 8 ? digit_scatter_kernel<2> : digit_scatter_kernel<1>, tiles, 2));
    }
    const GradArgs a = {pairs[last], grad, out, (float *)(base + lay.part), n, n_rows, ld_grad, ld_out, 0, run_for(n), 0, 0, dim, 0, scale};
    PSPMM_CUDA_TRY(dtype == PSPMM_F32    ? grad_typed<float>(a, dim, st)
                   : dtype == PSPMM_BF16 ? grad_typed<bf16>(a, dim, st)
                                         : grad_typed<f16>(a, dim, st));
    return PSPMM_OK;
}

extern "C" int pspmm_embedding_status(int32_t *status) { return pspmm_read_status(g_embedding_status, status); }
