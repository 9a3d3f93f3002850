// Pages of a cache from the requests' lengths: blocks of new tokens take pages off a stack of free
// ones, and give them back.
//
// Whole numbers, a few bytes for each sequence, page and row: the launches' latency bounds them.
// Which page a block takes follows from a running sum of the blocks that the sequences before it
// want, so one workgroup goes through the sequences, 1024 at a time, and then through their new
// blocks, each thread finding its block's sequence by bisection of the sums in LDS; no order of
// threads or atomics changes a result.  The positions and slots of many rows are a launch of their
// own (kExtendRows); of few they follow in the first.  A token each of 256 sequences 6.3 us; 32
// prompts of up to 521 rows, taken and given back in three launches, 12 us (15 with a second running
// sum a launch and sums of 64 bits), 8 clips of up to 19200 rows (2400 pages) as much; groups of 256
// threads are as fast but for the clips, 14.4.
#include "kv.h"

namespace h3mi {
namespace {

constexpr int kPageThreads = 1024;
constexpr int kPageWaves = kPageThreads / 64;

struct Pool {
    int32_t *free, *count;
    int pages;
};

// The sum of v over the workgroup's threads up to this one; `all` is that of all of them.  (Sums of blocks: a table has fewer
// than 2^31 entries.)
__device__ __forceinline__ int running_sum(int v, int* waves, int& all) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int o = __shfl_up(v, d);
        if (lane >= d) v += o;
    }
    __syncthreads();  // what the last call left has been read
    if (lane == 63) waves[wave] = v;
    __syncthreads();
    int before = 0;
    all = 0;
#pragma unroll
    for (int w = 0; w < kPageWaves; ++w) {
        const int x = waves[w];
        before += w < wave ? x : 0;
        all += x;
    }
    return before + v;
}

// The sequence of 1024 whose items hold item j: ends[s] items up to sequence s, its own among them.
__device__ __forceinline__ int owner(const int* ends, int j) {
    int at = 0;
#pragma unroll
    for (int step = kPageThreads / 2; step; step >>= 1)
        if (ends[at + step - 1] <= j) at += step;
    return at;
}

struct Extend {
    Pool pool;
    int32_t *tables, *lens;
    const int32_t* counts;
    int n, blocks, rows;
    int32_t *granted, *positions;
    int64_t* slots;
};

__device__ __forceinline__ void place_row(const Extend& e, uint32_t x) {
    const int i = static_cast<int>(x / static_cast<uint32_t>(e.rows)), r = static_cast<int>(x - static_cast<uint32_t>(i) * e.rows);
    const int c = e.granted[i];
    int at = -1;
    int64_t slot = -1;
    if (r < c) {
        at = e.lens[i] - c + r;
        const int page = e.tables[static_cast<int64_t>(i) * e.blocks + at / kKvBlock];
        if (page >= 0 && page < e.pool.pages) slot = static_cast<int64_t>(page) * kKvBlock + at % kKvBlock;
    }
    e.positions[x] = at;
    e.slots[x] = slot;
}

// One workgroup.  whole: the rows' positions and slots too.
__global__ __launch_bounds__(kPageThreads) void kv_extend_kernel(Extend e, int whole) {
    __shared__ int waves[kPageWaves], ends[kPageThreads], have[kPageThreads], cut;
    const int t = threadIdx.x;
    int free = *e.pool.count;
    free = free < 0 ? 0 : free > e.pool.pages ? e.pool.pages : free;
    int wanted = 0, taken = 0;  // blocks of the sequences before: wanted, given
    for (int i0 = 0; i0 < e.n; i0 += kPageThreads) {
        const int i = i0 + t;
        int c = 0, old = 0, held = 0, want = 0;
        bool fits = false;
        if (i < e.n) {
            c = e.counts ? e.counts[i] : e.rows;
            c = c < 0 ? 0 : c > e.rows ? e.rows : c;
            old = e.lens[i];
            old = old < 0 ? 0 : old;
            const int64_t end = static_cast<int64_t>(old) + c;
            fits = end <= static_cast<int64_t>(kKvBlock) * e.blocks;
            held = static_cast<int>((static_cast<int64_t>(old) + kKvBlock - 1) / kKvBlock);
            if (fits) want = static_cast<int>((end + kKvBlock - 1) / kKvBlock) - held;
        }
        int all;
        const int upto = running_sum(want, waves, all);
        // Once a sequence is not given its pages none after it is given any: what is given ends before the first of them.
        const bool given = fits && (want == 0 || upto <= free - wanted);
        if (i < e.n) {
            e.granted[i] = given ? c : 0;
            e.lens[i] = given ? old + c : old;
        }
        const int left = free - wanted;
        if (t == 0) cut = left < 0 ? 0 : all;
        ends[t] = upto;
        have[t] = held;
        __syncthreads();
        if (upto > left && upto - want <= left && left >= 0) cut = upto - want;
        __syncthreads();
        const int got = cut;
        for (int j = t; j < got; j += kPageThreads) {
            const int s = owner(ends, j), b = have[s] + j - (s ? ends[s - 1] : 0);
            e.tables[static_cast<int64_t>(i0 + s) * e.blocks + b] = e.pool.free[free - 1 - taken - j];
        }
        wanted += all;
        taken += got;
        __syncthreads();
    }
    if (t == 0) *e.pool.count = free - taken;
    if (!whole) return;
    const uint32_t rows = static_cast<uint32_t>(e.n) * e.rows;
    for (uint32_t x = t; x < rows; x += kPageThreads) place_row(e, x);
}

__global__ __launch_bounds__(256) void kv_places_kernel(Extend e, uint32_t rows) {
    const uint32_t x = blockIdx.x * 256u + threadIdx.x;
    if (x < rows) place_row(e, x);
}

struct Release {
    Pool pool;
    int32_t *tables, *lens;
    const int32_t* keep;
    int n, blocks;
};

constexpr int kReleaseEach = 4;  // blocks that a thread takes at a time

// One workgroup.
__global__ __launch_bounds__(kPageThreads) void kv_release_kernel(Release e) {
    __shared__ int waves[kPageWaves], ends[kPageThreads], first[kPageThreads];
    const int t = threadIdx.x;
    int count = *e.pool.count;
    count = count < 0 ? 0 : count > e.pool.pages ? e.pool.pages : count;
    for (int i0 = 0; i0 < e.n; i0 += kPageThreads) {
        const int i = i0 + t;
        int from = 0, gone = 0;
        if (i < e.n) {
            const int old = e.lens[i] < 0 ? 0 : e.lens[i];
            int left = e.keep ? e.keep[i] : 0;
            left = left < 0 ? 0 : left > old ? old : left;
            from = static_cast<int>((static_cast<int64_t>(left) + kKvBlock - 1) / kKvBlock);
            int to = static_cast<int>((static_cast<int64_t>(old) + kKvBlock - 1) / kKvBlock);
            if (to > e.blocks) to = e.blocks;
            gone = to > from ? to - from : 0;
            e.lens[i] = left;
        }
        int taken;
        ends[t] = running_sum(gone, waves, taken);
        first[t] = from;
        __syncthreads();
        for (int64_t j0 = 0; j0 < taken; j0 += kPageThreads * kReleaseEach) {
            int page[kReleaseEach], good = 0;
            int64_t at[kReleaseEach];
#pragma unroll
            for (int x = 0; x < kReleaseEach; ++x) {
                page[x] = -1, at[x] = -1;
                if (j0 + t * kReleaseEach + x < taken) {
                    const int j = static_cast<int>(j0) + t * kReleaseEach + x, s = owner(ends, j);
                    at[x] = static_cast<int64_t>(i0 + s) * e.blocks + first[s] + j - (s ? ends[s - 1] : 0);
                    page[x] = e.tables[at[x]];
                    good += page[x] >= 0 && page[x] < e.pool.pages;
                }
            }
            int back;
            int to = count + running_sum(good, waves, back) - good;
#pragma unroll
            for (int x = 0; x < kReleaseEach; ++x) {
                if (at[x] < 0) continue;
                e.tables[at[x]] = -1;
                if (page[x] < 0 || page[x] >= e.pool.pages) continue;
                if (to < e.pool.pages) e.pool.free[to] = page[x];
                ++to;
            }
            count = count + back < e.pool.pages ? count + back : e.pool.pages;
        }
        __syncthreads();
    }
    if (t == 0) *e.pool.count = count;
}

// Rows up to which the first launch writes positions and slots.
constexpr int64_t kExtendRows = 4096;

int check(const char* what, const h3mi_kv_pool* p, const int32_t* tables, const int32_t* lens, int64_t n, int64_t blocks) {
    if (!p) return fail(H3MI_EINVAL, "%s: null pool", what);
    if (p->pages < 0 || p->pages > (1 << 30)) return fail(H3MI_EINVAL, "%s: pages=%lld", what, (long long)p->pages);
    if (n < 0 || n > 0x7FFFFFFF - kPageThreads || blocks < 0 || blocks >= (int64_t{1} << 25))
        return fail(H3MI_EINVAL, "%s: bad sequences n=%lld blocks=%lld", what, (long long)n, (long long)blocks);
    if (n * blocks > 0x7FFFFFFF) return fail(H3MI_EINVAL, "%s: tables of 2^31 entries and more", what);
    if (n == 0) return H3MI_OK;
    if (!p->count || (p->pages > 0 && !p->free)) return fail(H3MI_EINVAL, "%s: null free or count", what);
    if (!lens || (blocks > 0 && !tables)) return fail(H3MI_EINVAL, "%s: null tables or lens", what);
    if (!aligned(p->free, 4) || !aligned(p->count, 4) || !aligned(tables, 4) || !aligned(lens, 4))
        return fail(H3MI_EALIGN, "%s: free, count, tables and lens must be 4-byte aligned", what);
    return H3MI_OK;
}

struct Bytes {
    const void* p;
    size_t bytes;
};

// Whether two of them overlap (null: not there).
template <int N>
bool any_overlap(const Bytes (&s)[N]) {
    for (int x = 1; x < N; ++x)
        for (int y = 0; y < x; ++y)
            if (s[x].p && s[y].p && overlap(s[x].p, s[x].bytes, s[y].p, s[y].bytes)) return true;
    return false;
}

}  // namespace
}  // namespace h3mi

using namespace h3mi;

extern "C" int h3mi_kv_extend(const h3mi_kv_pool* pool, int32_t* tables, int32_t* lens, const int32_t* counts, int64_t n,
                              int64_t blocks, int64_t rows, int32_t* granted, int32_t* positions, int64_t* slots, void* stream) {
    if (int e = check("kv_extend", pool, tables, lens, n, blocks)) return e;
    if (rows < 0 || rows > (1 << 30)) return fail(H3MI_EINVAL, "kv_extend: rows=%lld", (long long)rows);
    const int64_t all = n * rows;
    if (all > 0x7FFFFFFF) return fail(H3MI_EINVAL, "kv_extend: too many rows for one call");
    if (n == 0) return ok();
    if (!granted || (rows > 0 && (!positions || !slots))) return fail(H3MI_EINVAL, "kv_extend: null granted, positions or slots");
    if (!aligned(counts, 4) || !aligned(granted, 4) || !aligned(positions, 4) || !aligned(slots, 8))
        return fail(H3MI_EALIGN, "kv_extend: counts, granted and positions must be 4-byte aligned, slots 8-byte");
    const size_t each = 4 * static_cast<size_t>(n);
    const Bytes spans[] = {{pool->free, 4 * static_cast<size_t>(pool->pages)}, {pool->count, 4}, {tables, each * blocks}, {lens, each},
                           {counts, each}, {granted, each}, {positions, 4 * static_cast<size_t>(all)}, {slots, 8 * static_cast<size_t>(all)}};
    if (any_overlap(spans)) return fail(H3MI_EALIAS, "kv_extend: two of the call's tensors overlap");
    const Extend e = {{pool->free, pool->count, static_cast<int>(pool->pages)}, tables, lens, counts, static_cast<int>(n),
                      static_cast<int>(blocks), static_cast<int>(rows), granted, positions, slots};
    const bool whole = all <= kExtendRows;
    hipLaunchKernelGGL(kv_extend_kernel, dim3(1), dim3(kPageThreads), 0, as_stream(stream), e, whole);
    if (int rc = check_launch("kv_extend")) return rc;
    if (whole) return ok();
    hipLaunchKernelGGL(kv_places_kernel, dim3(static_cast<unsigned>((all + 255) / 256)), dim3(256), 0, as_stream(stream), e,
                       static_cast<uint32_t>(all));
    return check_launch("kv_extend");
}

extern "C" int h3mi_kv_release(const h3mi_kv_pool* pool, int32_t* tables, int32_t* lens, const int32_t* keep, int64_t n, int64_t blocks,
                               void* stream) {
    if (int e = check("kv_release", pool, tables, lens, n, blocks)) return e;
    if (n == 0) return ok();
    if (!aligned(keep, 4)) return fail(H3MI_EALIGN, "kv_release: keep must be 4-byte aligned");
    const size_t each = 4 * static_cast<size_t>(n);
    const Bytes spans[] = {{pool->free, 4 * static_cast<size_t>(pool->pages)}, {pool->count, 4}, {tables, each * blocks}, {lens, each}, {keep, each}};
    if (any_overlap(spans)) return fail(H3MI_EALIAS, "kv_release: two of the call's tensors overlap");
    const Release e = {{pool->free, pool->count, static_cast<int>(pool->pages)}, tables, lens, keep, static_cast<int>(n), static_cast<int>(blocks)};
    hipLaunchKernelGGL(kv_release_kernel, dim3(1), dim3(kPageThreads), 0, as_stream(stream), e);
    return check_launch("kv_release");
}
