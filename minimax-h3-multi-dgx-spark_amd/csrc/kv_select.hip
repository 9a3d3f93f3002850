// Selecting a sequence's blocks of keys for tiles of queries.
//
// A tile's score of a block is a product of whole numbers (the pooled queries as 11-bit
// integers, the sum of the block's 8-bit keys as 16-bit ones), exact in int32: |qi| <=
// 1023, |k_sum| <= 64 * 127 and dim <= 256 keep it below 2^31.  The pooled queries are
// summed in 64 bits: the sum of N bf16 values (128 rows of the heads of a group) is exact
// where the largest is below 2^(45 - log2 N) times the least that is not 0, 2^38 for one
// head, 2^30 to 256 heads.  So neither the order of a sum nor the split of the work changes
// a selection; of values further apart the last bits of 53 may, and with them a selection
// whose scores lie next to each other.
//
// A workgroup takes one tile of one kv head: it pools the queries, scores every block
// (dim / 8 lanes a block, 16 bytes of k_sum each, v_dot2_i32_i16), keeps the scores as
// ordered 32-bit keys in LDS, finds the last selected key by up to four passes over 8 bits
// of it, and writes the selected blocks in order.  Few tiles over long tables, whose scoring
// would wait on a few CUs' loads, score in a launch of their own, a workgroup for every
// kChunk blocks, and the keys pass through memory.  1064 tiles of 609 blocks take 28 us (25
// again and again, its inputs in the caches; 34 MB of queries and 9 MB of sums would be 9), half
// of it the queries' pooling, and then each tile reads all the sums of its head; 32 tiles of
// 2048 blocks 15 us in two launches.
#include "kv.h"

namespace h3mi {
namespace {

constexpr int kMaxSelect = 32768;  // blocks: their keys fill 128 KiB of LDS
constexpr int kBatch = 8;  // blocks whose sums a lane has in flight; at most the lanes of a block

// Sum over groups of CH lanes, by DPP moves within 16: a neighbour, the other pair, the mirrored other four, the other eight.
template <int CH>
__device__ __forceinline__ int lane_sum(int v) {
    v += __builtin_amdgcn_update_dpp(0, v, 0xB1, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x4E, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x141, 0xF, 0xF, false);
    if constexpr (CH >= 16) v += __builtin_amdgcn_update_dpp(0, v, 0x128, 0xF, 0xF, false);
    if constexpr (CH >= 32) v += __shfl_xor(v, 16);
    return v;
}

typedef short s16x2 __attribute__((ext_vector_type(2)));

// Keys ordered as scores: 0 is kept for blocks that are not there.  NaN becomes the
// lowest key of a block, and -0 (a negative product times a zero scale) is 0.
__device__ __forceinline__ uint32_t key_of(float s) {
    if (__builtin_isnan(s)) return 1u;
    const uint32_t b = __float_as_uint(s + 0.0f);
    const uint32_t k = (b & 0x80000000u) ? ~b : b | 0x80000000u;
    return k < 2u ? 2u : k;
}

enum Part { kWhole, kScores, kSelection };
constexpr int kChunk = 256;

template <int D, int THREADS, Part PART>
__global__ __launch_bounds__(THREADS) void kv_select_kernel(const uint16_t* __restrict__ q, int64_t ld, int64_t bs, KvCache c,
                                                            KvSeqs s, int rows, int heads, int top, int causal, int tiles, int chunks,
                                                            uint32_t* __restrict__ all_keys, int32_t* __restrict__ out) {
    constexpr int CH = D / 8, kSelWaves = THREADS / 64;
    constexpr int GROUPS = THREADS / CH;  // row groups while pooling, blocks at once while scoring
    extern __shared__ uint32_t keys[];
    __shared__ double part[kSelWaves][D];
    __shared__ double pool[D];
    __shared__ __align__(16) int16_t qi[D];
    __shared__ uint32_t hist[256];
    __shared__ uint32_t pick[3];
    __shared__ int wsum[2][kSelWaves];
    __shared__ double wmax[kSelWaves];

    const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
    // an XCD takes whole heads, whose sums its L2 then holds for every tile
    const int at_all = xcd_item() / chunks, chunk = xcd_item() % chunks;
    uint32_t* const my_keys = all_keys + static_cast<int64_t>(at_all) * s.blocks;
    const int tile = at_all % tiles, h = at_all / tiles % c.heads, i = at_all / tiles / c.heads;
    int32_t* const to = out + ((static_cast<int64_t>(i) * tiles + tile) * c.heads + h) * top;
    const int len = s.len(i), count = s.count(i, rows), group = heads / c.heads;
    const int r0 = tile * kKvTile, live = count - r0 < kKvTile ? count - r0 : kKvTile;
    // the tile's own tokens, and the blocks it sees
    const int first = s.end(i) - count + r0, last = first + live - 1;
    int seen = (len + kKvBlock - 1) / kKvBlock;
    if (causal && last < len) seen = last < 0 ? 0 : block_of(last) + 1;
    if (live <= 0 || c.pages == 0) seen = 0;
    if (seen == 0) {
        if constexpr (PART != kScores)
            for (int j = t; j < top; j += THREADS) to[j] = -1;
        return;
    }
    if constexpr (PART == kSelection) {
        for (int b = t; b < seen; b += THREADS) keys[b] = my_keys[b];
    } else {
        // the blocks to score: keys[0] is block low's
        const int low = chunk * kChunk, high = PART == kScores && low + kChunk < seen ? low + kChunk : seen;
        if (low >= high) return;
        const int ch = t % CH, grp = t / CH;
        {
            double p[8] = {};
            // four rows in flight (1064 tiles 24.5 -> 23.8 us; eight 23.6, but 20 tiles of 22 rows of 5 heads 10.5 -> 11.2)
            for (int x0 = grp; x0 < live * group; x0 += GROUPS * 4) {
                uint4 w[4];
#pragma unroll
                for (int y = 0; y < 4; ++y) {
                    const int x = x0 + y * GROUPS, r = x / group, hq = h * group + x - r * group;
                    w[y] = make_uint4(0, 0, 0, 0);
                    if (x < live * group)
                        w[y] = *reinterpret_cast<const uint4*>(q + i * bs + (r0 + r) * ld + static_cast<int64_t>(hq) * D + ch * 8);
                }
#pragma unroll
                for (int y = 0; y < 4; ++y) {
                    const uint32_t a[4] = {w[y].x, w[y].y, w[y].z, w[y].w};
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        p[2 * j] += bf16_lo(a[j]);
                        p[2 * j + 1] += bf16_hi(a[j]);
                    }
                }
            }
            // the row groups of a wave, then the waves through LDS
#pragma unroll
            for (int j = 0; j < 8; ++j) {
#pragma unroll
                for (int m = 32; m >= CH; m >>= 1) p[j] += __shfl_xor(p[j], m);
                if (lane < CH) part[wave][ch * 8 + j] = p[j];
            }
        }
        __syncthreads();
        if (t < D) {
            double p = 0.0;
#pragma unroll
            for (int w = 0; w < kSelWaves; ++w) p += part[w][t];
            pool[t] = p;
        }
        __syncthreads();
        double m = t < D ? fabs(pool[t]) : 0.0;
        bool bad = !(m < __builtin_inf());  // a NaN or an infinity
#pragma unroll
        for (int x = 32; x; x >>= 1) m = fmax(m, __shfl_xor(m, x));
        bad = __any(bad);
        if (lane == 0) wmax[wave] = bad ? __builtin_inf() : m;
        __syncthreads();
        m = 0.0;
#pragma unroll
        for (int w = 0; w < kSelWaves; ++w) m = fmax(m, wmax[w]);
        if (t < D) qi[t] = m > 0.0 && m < __builtin_inf() ? static_cast<int16_t>(rint(pool[t] * 1023.0 / m)) : int16_t{0};
        __syncthreads();

        const uint4 qw = *reinterpret_cast<const uint4*>(qi + ch * 8);
        const int own = first < 0 ? 0 : block_of(first);
        // The blocks' pages first, so that nothing but the sums' own latency stands in the way of kBatch of them at once.
        for (int b = low + t; b < high; b += THREADS) keys[b - low] = static_cast<uint32_t>(s.page(i, b, c.pages));
        __syncthreads();
        const int up = low + (high - low + GROUPS - 1) / GROUPS * GROUPS;  // whole groups, so that every lane takes part
        for (int b0 = low + grp; b0 < up; b0 += GROUPS * kBatch) {
            uint4 k[kBatch];
#pragma unroll
            for (int x = 0; x < kBatch; ++x) {
                const int b = b0 + x * GROUPS, page = b < high ? static_cast<int>(keys[b - low]) : -1;
                // (a page that is not there: page 0's, not used)
                k[x] = *reinterpret_cast<const uint4*>(c.ksum + (static_cast<int64_t>(page < 0 ? 0 : page) * c.heads + h) * D + ch * 8);
            }
            // every lane of a group has the sums; lane x makes the key of the group's block x
            const int b = b0 + ch * GROUPS, page = ch < kBatch && b < high ? static_cast<int>(keys[b - low]) : -1;
            const float ks = page < 0 ? 0.0f : c.ks[static_cast<int64_t>(page) * c.heads + h];
            int mine = 0;
#pragma unroll
            for (int x = 0; x < kBatch; ++x) {
                int dot = __builtin_amdgcn_sdot2(__builtin_bit_cast(s16x2, qw.x), __builtin_bit_cast(s16x2, k[x].x), 0, false);
                dot = __builtin_amdgcn_sdot2(__builtin_bit_cast(s16x2, qw.y), __builtin_bit_cast(s16x2, k[x].y), dot, false);
                dot = __builtin_amdgcn_sdot2(__builtin_bit_cast(s16x2, qw.z), __builtin_bit_cast(s16x2, k[x].z), dot, false);
                dot = __builtin_amdgcn_sdot2(__builtin_bit_cast(s16x2, qw.w), __builtin_bit_cast(s16x2, k[x].w), dot, false);
                dot = lane_sum<CH>(dot);
                mine = ch == x ? dot : mine;
            }
            if (ch < kBatch && b < high) {
                const int held = len - b * kKvBlock < kKvBlock ? len - b * kKvBlock : kKvBlock;
                const float score = static_cast<float>(mine) * (ks / static_cast<float>(held));
                const uint32_t key = page < 0 ? 0u : causal && b >= own ? 0xFFFFFFFFu : key_of(score);
                if constexpr (PART == kScores) my_keys[b] = key;
                else keys[b] = key;
            }
        }
        if constexpr (PART == kScores) return;
    }
    __syncthreads();

    // The least key taken (thr), and how many of the blocks that have it (need).
    uint32_t thr = 1u;
    int need = top;
    if (seen > top) {
        uint32_t prefix = 0;
        int want = top;
        for (int shift = 24; shift >= 0; shift -= 8) {
            for (int x = t; x < 256; x += THREADS) hist[x] = 0;
            __syncthreads();
            for (int b = t; b < seen; b += THREADS)
                if (shift == 24 || (keys[b] >> (shift + 8)) == prefix) atomicAdd(&hist[(keys[b] >> shift) & 255u], 1u);
            __syncthreads();
            if (wave == 0) {
                // suffix sums of four bins a lane: the highest bin at which `want` blocks are reached
                uint32_t n[4], sum = 0;
#pragma unroll
                for (int j = 3; j >= 0; --j) n[j] = hist[255 - (4 * lane + 3 - j)];
                // lane 0 holds the highest four bins, n[3] the highest of them
                sum = n[0] + n[1] + n[2] + n[3];
                uint32_t before = sum;
#pragma unroll
                for (int x = 1; x < 64; x <<= 1) {
                    const uint32_t o = __shfl_up(before, x);
                    if (lane >= x) before += o;
                }
                before -= sum;  // blocks in higher bins than this lane's
                const uint32_t w = static_cast<uint32_t>(want);
                if (before < w && before + sum >= w) {
                    uint32_t run = before;
                    int bin = 255 - 4 * lane;
#pragma unroll
                    for (int j = 3; j >= 0; --j, --bin) {
                        if (run + n[j] >= w) break;
                        run += n[j];
                    }
                    pick[0] = static_cast<uint32_t>(bin);
                    pick[1] = run;
                    pick[2] = hist[bin];
                }
            }
            __syncthreads();
            prefix = (prefix << 8) | pick[0];
            want -= static_cast<int>(pick[1]);
            thr = prefix << shift;
            // The bin's blocks are as many as are wanted, mostly after two passes or three: all of them (150 blocks 8.5 -> 8.0 us,
            // 2048 15.4 -> 14.8).
            if (pick[2] == static_cast<uint32_t>(want)) break;
            __syncthreads();
        }
        need = want;
        if (thr == 0) thr = 1u, need = top;  // fewer blocks are there than wanted: all of them
    }

    // In order: blocks above thr, and the first `need` at it.
    int done = 0, ties = 0;
    for (int b0 = 0; b0 < seen; b0 += THREADS) {
        const int b = b0 + t;
        const uint32_t key = b < seen ? keys[b] : 0u;
        const bool over = key > thr, tie = key == thr;
        const uint64_t mo = __ballot(over), mt = __ballot(tie), below = (uint64_t{1} << lane) - 1;
        if (lane == 0) wsum[0][wave] = __popcll(mo), wsum[1][wave] = __popcll(mt);
        __syncthreads();
        int o = __popcll(mo & below), e = ties + __popcll(mt & below), all_o = 0, all_e = 0;
#pragma unroll
        for (int w = 0; w < kSelWaves; ++w) {
            if (w < wave) o += wsum[0][w], e += wsum[1][w];
            all_o += wsum[0][w];
            all_e += wsum[1][w];
        }
        // blocks taken before this one: those above thr, and the ties before it that were taken
        const int t0 = ties < need ? ties : need, te = e < need ? e : need;
        if (over || (tie && e < need)) to[done + o + te - t0] = b;
        const int t1 = ties + all_e < need ? ties + all_e : need;
        done += all_o + t1 - t0;
        ties += all_e;
        __syncthreads();
    }
    for (int j = done + t; j < top; j += THREADS) to[j] = -1;
}

}  // namespace
}  // namespace h3mi

using namespace h3mi;

namespace {

// Whether the tiles are few and their tables long: 32 tiles of 2048 blocks 21 us in one launch, 15 in two.
bool scores_apart(int64_t groups, int64_t blocks) { return 2 * groups <= cu_count() && blocks >= 2 * kChunk; }

int64_t key_bytes(int64_t groups, int64_t blocks) { return scores_apart(groups, blocks) ? groups * blocks * 4 : 0; }

template <int D>
void launch(Part part, int threads, int64_t groups, size_t lds, hipStream_t st, const uint16_t* q, int64_t ld, int64_t bs, const KvCache& c,
            const KvSeqs& s, int rows, int heads, int top, int causal, int tiles, int chunks, uint32_t* keys, int32_t* out) {
    const auto fn = part == kScores ? kv_select_kernel<D, 256, kScores>
                    : part == kSelection ? kv_select_kernel<D, 1024, kSelection>
                    : threads == 1024 ? kv_select_kernel<D, 1024, kWhole> : kv_select_kernel<D, 256, kWhole>;
    hipLaunchKernelGGL(fn, dim3(static_cast<unsigned>(groups)), dim3(threads), static_cast<unsigned>(lds), st, q, ld, bs, c, s, rows, heads, top,
                       causal, tiles, chunks, keys, out);
}

}  // namespace

extern "C" int64_t h3mi_kv_select_workspace(int64_t n, int64_t rows, int64_t kv_heads, int64_t blocks) {
    int64_t groups;
    if (n <= 0 || rows <= 0 || kv_heads <= 0 || blocks <= 0 || blocks > kMaxSelect || rows > (1 << 30)) return 0;
    if (!launchable(n, (rows + kKvTile - 1) / kKvTile, kv_heads, 1024, &groups)) return 0;
    return key_bytes(groups, blocks);
}

extern "C" int h3mi_kv_select(const uint16_t* q, int64_t rows, int64_t heads, int64_t ld_q, int64_t bs_q,
                              const h3mi_kv_cache* cache, const h3mi_kv_seqs* seqs, int64_t top, int causal, int32_t* blocks,
                              void* workspace, int64_t workspace_bytes, void* stream) {
    if (int e = kv_check("kv_select", cache, seqs)) return e;
    if (heads <= 0 || heads > 65536 || heads % cache->heads)
        return fail(H3MI_EINVAL, "kv_select: heads=%lld must be a multiple of the cache's %lld", (long long)heads, (long long)cache->heads);
    if (int e = kv_check_rows("kv_select", "q", q, rows, heads, cache->dim, seqs->n, ld_q, bs_q)) return e;
    if (top < 1 || top > kMaxSelect) return fail(H3MI_EINVAL, "kv_select: top=%lld must be in [1, %d]", (long long)top, kMaxSelect);
    if (seqs->blocks > kMaxSelect)
        return fail(H3MI_EINVAL, "kv_select: %lld blocks a sequence, at most %d", (long long)seqs->blocks, kMaxSelect);
    if (seqs->n == 0 || rows == 0) return ok();
    if (!blocks) return fail(H3MI_EINVAL, "kv_select: null blocks");
    if (!aligned(blocks, 4)) return fail(H3MI_EALIGN, "kv_select: blocks must be 4-byte aligned");
    const int64_t tiles = (rows + kKvTile - 1) / kKvTile;
    int64_t groups;
    if (!launchable(seqs->n, tiles, cache->heads, 1024, &groups)) return fail(H3MI_EINVAL, "kv_select: too many rows for one call");
    const size_t bytes = static_cast<size_t>(groups) * top * 4;
    if (overlap(blocks, bytes, q, kv_span(seqs->n, rows, heads, cache->dim, ld_q, bs_q)) || kv_overlaps(blocks, bytes, *cache))
        return fail(H3MI_EALIAS, "kv_select: blocks overlaps q or the cache");
    if (kv_seqs_overlap(blocks, bytes, *seqs)) return fail(H3MI_EALIAS, "kv_select: blocks overlaps tables, lens or counts");
    const int64_t need = key_bytes(groups, seqs->blocks);
    if (need > 0 && (!workspace || workspace_bytes < need))
        return fail(H3MI_EINVAL, "kv_select: workspace of %lld bytes, %lld needed", (long long)(workspace ? workspace_bytes : 0), (long long)need);
    if (!aligned(workspace, 4)) return fail(H3MI_EALIGN, "kv_select: workspace must be 4-byte aligned");
    if (need > 0 && (overlap(workspace, need, blocks, bytes) || overlap(workspace, need, q, kv_span(seqs->n, rows, heads, cache->dim, ld_q, bs_q)) ||
                     kv_overlaps(workspace, need, *cache) || kv_seqs_overlap(workspace, need, *seqs)))
        return fail(H3MI_EALIAS, "kv_select: the workspace overlaps blocks or an input");
    const auto go = cache->dim == 64 ? launch<64> : cache->dim == 128 ? launch<128> : launch<256>;
    const auto run = [&](Part part, int threads, int64_t in_launch, int64_t chunks, int64_t keys_held) {
        go(part, threads, in_launch, keys_held * 4, as_stream(stream), q, ld_q, bs_q, kv_cache(*cache), kv_seqs(*seqs), static_cast<int>(rows),
           static_cast<int>(heads), static_cast<int>(top), causal, static_cast<int>(tiles), static_cast<int>(chunks),
           static_cast<uint32_t*>(workspace), blocks);
        return check_launch("kv_select");
    };
    if (need > 0) {
        const int64_t chunks = (seqs->blocks + kChunk - 1) / kChunk;
        if (int e = run(kScores, 256, groups * chunks, chunks, kChunk)) return e;
        return run(kSelection, 1024, groups, 1, seqs->blocks);
    }
    // few workgroups: more of their own waves (150 blocks, 240 groups 11.2 us so, 8.3 with 256 threads; 609 blocks, 1064
    // groups 25.3 with 256, 29.3 with 512)
    return run(kWhole, 2 * groups <= cu_count() ? 1024 : 256, groups, 1, seqs->blocks);
}
