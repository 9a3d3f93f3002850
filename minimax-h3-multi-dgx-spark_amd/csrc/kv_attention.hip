// Attention over the 8-bit key/value cache.
#include "kv.h"

namespace h3mi {
namespace {

// One wave: one query row of one head; a lane scores a token of each block.
template <int D>
__global__ __launch_bounds__(64) void kv_attention_kernel(const uint16_t* __restrict__ q, int64_t ld, int64_t bs, KvCache c,
                                                          KvSeqs s, int rows, int heads, float scale, int causal,
                                                          const int32_t* __restrict__ list, int top, uint16_t* __restrict__ out) {
    __shared__ float qs[D];
    __shared__ float ps[kKvBlock];
    const int lane = threadIdx.x;
    const int hq = blockIdx.x % heads;
    const int64_t item = blockIdx.x / heads;
    const int i = static_cast<int>(item / rows), r = static_cast<int>(item % rows);
    const int h = hq / (heads / c.heads);
    const int len = s.len(i), count = s.count(i, rows);
    const int at = s.end(i) - count + r;
    int last = len - 1;  // the last token seen
    if (causal && at < last) last = at;
    if (r >= count) last = -1;
    const int64_t row = i * bs + static_cast<int64_t>(r) * ld + static_cast<int64_t>(hq) * D;
    for (int d = lane; d < D; d += 64) qs[d] = bf16_f32(q[row + d]) * scale;
    __syncthreads();
    const int tiles = (rows + kKvTile - 1) / kKvTile;
    const int32_t* const mine = list ? list + ((static_cast<int64_t>(i) * tiles + r / kKvTile) * c.heads + h) * top : nullptr;
    const int nb = last < 0 ? 0 : block_of(last) + 1;
    const int steps = mine ? (nb ? top : 0) : nb;
    float m = -__builtin_inff(), l = 0.0f, o[D / 64] = {};
    for (int x = 0; x < steps; ++x) {
        const int b = mine ? mine[x] : x;
        if (b < 0 || b >= nb) continue;
        const int page = s.page(i, b, c.pages);
        if (page < 0) continue;
        const int64_t tile = static_cast<int64_t>(page) * c.heads + h;
        const int8_t* const k = c.k + tile * (kKvBlock * D) + lane * D;
        float dot = 0.0f;
        for (int d = 0; d < D; d += 16) {
            const uint4 w = *reinterpret_cast<const uint4*>(k + d);
            const uint32_t a[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
            for (int j = 0; j < 16; ++j) dot += qs[d + j] * static_cast<float>(static_cast<int8_t>(a[j >> 2] >> (8 * (j & 3))));
        }
        const bool there = b * kKvBlock + lane <= last;
        const float x0 = there ? dot * c.ks[tile] : -__builtin_inff();
        float bm = x0;
#pragma unroll
        for (int y = 32; y; y >>= 1) bm = fmaxf(bm, __shfl_xor(bm, y));
        const float mn = fmaxf(m, bm), fix = __expf(m - mn);
        const float p = there ? __expf(x0 - mn) : 0.0f;
        float sum = p;
#pragma unroll
        for (int y = 32; y; y >>= 1) sum += __shfl_xor(sum, y);
        l = l * fix + sum;
        m = mn;
        ps[lane] = p * c.vs[tile];
        __syncthreads();
#pragma unroll
        for (int e = 0; e < D / 64; ++e) {
            const int8_t* const v = c.v + tile * (kKvBlock * D) + (e * 64 + lane) * kKvBlock;
            float acc = 0.0f;
            for (int y = 0; y < kKvBlock; ++y) acc += ps[y] * static_cast<float>(v[y]);
            o[e] = o[e] * fix + acc;
        }
        __syncthreads();
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
    for (int e = 0; e < D / 64; ++e) out[(item * heads + hq) * D + e * 64 + lane] = bf16_bits(o[e] * inv);
}

}  // namespace
}  // namespace h3mi

using namespace h3mi;

extern "C" int64_t h3mi_kv_attention_workspace(int64_t, int64_t, int64_t, int64_t, int64_t, int64_t, int64_t) { return 0; }

extern "C" int h3mi_kv_attention_bf16(const uint16_t* q, int64_t rows, int64_t heads, int64_t ld_q, int64_t bs_q,
                                      const h3mi_kv_cache* cache, const h3mi_kv_seqs* seqs, float scale, int causal,
                                      const int32_t* blocks, int64_t top, uint16_t* out, void* workspace,
                                      int64_t workspace_bytes, void* stream) {
    if (int e = kv_check("kv_attention", cache, seqs)) return e;
    if (heads <= 0 || heads > 65536 || heads % cache->heads)
        return fail(H3MI_EINVAL, "kv_attention: heads=%lld must be a multiple of the cache's %lld", (long long)heads, (long long)cache->heads);
    if (int e = kv_check_rows("kv_attention", "q", q, rows, heads, cache->dim, seqs->n, ld_q, bs_q)) return e;
    if (!(scale == scale) || scale - scale != 0.0f) return fail(H3MI_EINVAL, "kv_attention: scale is not finite");
    if (blocks && (top < 1 || top > 0x7FFFFFFF)) return fail(H3MI_EINVAL, "kv_attention: top=%lld", (long long)top);
    if (seqs->n == 0 || rows == 0) return ok();
    if (!out) return fail(H3MI_EINVAL, "kv_attention: null out");
    if (!aligned(out, 16) || !aligned(blocks, 4)) return fail(H3MI_EALIGN, "kv_attention: out must be 16-byte aligned, blocks 4-byte");
    const int D = static_cast<int>(cache->dim);
    int64_t groups;
    if (!launchable(seqs->n, rows, heads, 64, &groups)) return fail(H3MI_EINVAL, "kv_attention: too many rows for one call");
    const auto fn = D == 64 ? kv_attention_kernel<64> : D == 128 ? kv_attention_kernel<128> : kv_attention_kernel<256>;
    hipLaunchKernelGGL(fn, dim3(static_cast<unsigned>(groups)), dim3(64), 0, as_stream(stream), q, ld_q, bs_q, kv_cache(*cache),
                       kv_seqs(*seqs), static_cast<int>(rows), static_cast<int>(heads), scale, causal, blocks,
                       static_cast<int>(top), out);
    return check_launch("kv_attention");
}
