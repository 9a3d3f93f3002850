// Writing the 4-bit key/value cache and reading it back.
//
// 32 elements of a token share a factor 2^e, the least of e = -125 .. 125 with max |x| <= 7 2^e,
// and are rounded to 0, 0.5, 1, 1.5, 2, 3, 4, 6 times it, to the nearest, to the even place between
// two.  The values lie 2 apart from 4 on, so that 6 is the nearest to all that is up to 7, and no
// error is more than half the distance of its neighbours (above 7 2^125, bf16's last quarter of a
// binade, 6 2^125 is the nearest there is).  x 2^-e is exact, and what a value stands for is a
// bf16: the one rounding is that to 4 bits.  A token's own scales: what was written is never
// rounded again, and a write touches the bytes of its own tokens alone.
//
// Both kernels move 2 + 17/32 bytes an element and do little with them, so HBM bounds them.  A
// workgroup takes one block of 64 tokens of one head, keys and values: a thread holds 4 tokens of
// 8 elements, 4 lanes a group, so that a wave's accesses are whole rows of a head, of 128 to 512
// bytes in bf16 and 32 to 128 in 4 bits.  The scales, bytes 64 apart from group to group, are
// gathered in LDS and stored four tokens at a time.  4-bit rows are stored through the L2, which makes
// whole lines of them (a clip of 19200 tokens of 56 x 128 written and read back 264 us past it, 218
// so); bf16 rows go past it, and large inputs past the memory-side cache, as in 8 bits.
#include "kv.h"

namespace h3mi {
namespace {

// The scale code of a group whose largest magnitude has bf16 bits a: 2^(code - 127).
__device__ __forceinline__ int four_code(uint32_t a) {
    const int e = static_cast<int>(a >> 7), code = e - 2 + ((a & 127u) > 96u);  // 1.75 = 1 + 96 / 128
    if (e == 255) return 255;
    return code < 2 ? 2 : code > 252 ? 252 : code;
}

__device__ __forceinline__ uint32_t pack_four(const uint4& x, int code) {
    typedef __bf16 bf2 __attribute__((ext_vector_type(2)));
    const float s = four_scale(code);
    uint32_t w = 0;
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w, __builtin_bit_cast(bf2, x.x), s, 0);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w, __builtin_bit_cast(bf2, x.y), s, 1);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w, __builtin_bit_cast(bf2, x.z), s, 2);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w, __builtin_bit_cast(bf2, x.w), s, 3);
    return code == 255 ? 0u : w;
}

// The largest magnitude (bf16 bits; a NaN's are above an infinity's) of the 32 elements that 4 neighbouring lanes hold.
__device__ __forceinline__ uint32_t group_max(const uint4& x) {
    uint32_t m = max_mag(max_mag(x.x & 0x7FFF7FFFu, x.y & 0x7FFF7FFFu), max_mag(x.z & 0x7FFF7FFFu, x.w & 0x7FFF7FFFu));
    m = max_mag(m, m >> 16) & 0xFFFFu;
    m = max_mag(m, static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(static_cast<int>(m), 0xB1, 0xF, 0xF, true)));  // lane ^ 1
    return max_mag(m, static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(static_cast<int>(m), 0x4E, 0xF, 0xF, true)));  // lane ^ 2
}

// One workgroup: one of the blocks that a sequence's new tokens touch, one head.  2 D threads.
template <int D, bool STREAM>
__global__ __launch_bounds__(2 * D) void kv4_write_kernel(Rows kin, Rows vin, KvCache4 c, KvSeqs s, int rows, int touched) {
    constexpr int CH = D / 8, G = D / kFourGroup;
    __shared__ __attribute__((aligned(4))) uint8_t codes[2][G][kKvBlock];
    const int at_all = xcd_item(), h = at_all % c.heads, item = at_all / c.heads;
    const int i = item / touched;
    const int len = s.len(i), count = s.count(i, rows), start = s.end(i) - count;
    const int b = block_of(start < 0 ? 0 : start) + item % touched;
    const int base = b * kKvBlock;
    if (count == 0 || base >= len) return;
    const int page = s.page(i, b, c.pages);
    if (page < 0) return;
    const int64_t tile = static_cast<int64_t>(page) * c.heads + h;
    const int t = threadIdx.x, ch = t % CH, line = t / CH;
    uint4 x[2][4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int at = base + 16 * j + line;
        x[0][j] = x[1][j] = make_uint4(0, 0, 0, 0);
        if (at >= start && at < len) {
            const int64_t row = at - start;
            x[0][j] = load_row<STREAM>(kin.p + i * kin.bs + row * kin.ld + h * D + ch * 8);
            x[1][j] = load_row<STREAM>(vin.p + i * vin.bs + row * vin.ld + h * D + ch * 8);
        }
    }
#pragma unroll
    for (int w = 0; w < 2; ++w) {
        uint8_t* const out = (w ? c.v : c.k) + tile * (kKvBlock * D / 2);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int tok = 16 * j + line, at = base + tok;
            const int code = four_code(group_max(x[w][j]));
            if (ch % 4 == 0) codes[w][ch / 4][tok] = static_cast<uint8_t>(code);
            if (at >= start && at < len) *reinterpret_cast<uint32_t*>(out + tok * (D / 2) + ch * 4) = pack_four(x[w][j], code);
        }
    }
    __syncthreads();
    if (t >= 2 * G * (kKvBlock / 4)) return;
    const int w = t / (G * (kKvBlock / 4)), word = t % (G * (kKvBlock / 4)), tok = word % (kKvBlock / 4) * 4;
    uint8_t* const to = (w ? c.vs : c.ks) + tile * (G * kKvBlock) + word * 4;
    const uint8_t* const from = &codes[w][0][0] + word * 4;
    if (base + tok >= start && base + tok + 4 <= len) {
        *reinterpret_cast<uint32_t*>(to) = *reinterpret_cast<const uint32_t*>(from);
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (base + tok + j >= start && base + tok + j < len) to[j] = from[j];
    }
}

// One workgroup: one cache block of those that a sequence's tokens starts .. starts + length - 1 lie in, one head.
// STREAM: loads past the caches too, where the call's own output is more than the memory-side cache holds (a clip of 19200 tokens
// of 56 x 128 written and read back 252 us without, 237 so; where nothing came between, and the cache still holds it, 218).
template <int D, bool STREAM>
__global__ __launch_bounds__(2 * D) void kv4_read_kernel(uint16_t* __restrict__ kout, uint16_t* __restrict__ vout,
                                                         const int32_t* __restrict__ starts, KvCache4 c, KvSeqs s, int length,
                                                         int touched) {
    constexpr int CH = D / 8, G = D / kFourGroup;
    const int at_all = xcd_item(), h = at_all % c.heads, item = at_all / c.heads;
    const int i = item / touched;
    const int start = starts ? starts[i] : 0;
    const int64_t b = static_cast<int64_t>(block_of(start)) + item % touched;
    const int len = s.len(i);
    const int64_t base = b * kKvBlock, from = base - start;  // of the block's first token in the output
    if (from >= length) return;
    const int page = base < len ? s.page(i, static_cast<int>(b), c.pages) : -1;
    const int t = threadIdx.x, ch = t % CH, line = t / CH;
    const int64_t tile = static_cast<int64_t>(page < 0 ? 0 : page) * c.heads + h;
    uint32_t q[2][4] = {};
    int code[2][4] = {};
    if (page >= 0) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int tok = 16 * j + line;
#pragma unroll
            for (int w = 0; w < 2; ++w) {
                const uint32_t* const p = reinterpret_cast<const uint32_t*>((w ? c.v : c.k) + tile * (kKvBlock * D / 2) + tok * (D / 2) + ch * 4);
                q[w][j] = STREAM ? __builtin_nontemporal_load(p) : *p;
                code[w][j] = (w ? c.vs : c.ks)[tile * (G * kKvBlock) + ch / 4 * kKvBlock + tok];
            }
        }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int64_t r = from + 16 * j + line, at = base + 16 * j + line;
        if (r < 0 || r >= length) continue;
        const int64_t o = ((i * static_cast<int64_t>(length) + r) * c.heads + h) * D + ch * 8;
        const bool there = page >= 0 && at < len;
#pragma unroll
        for (int w = 0; w < 2; ++w) {
            uint4 y = make_uint4(0, 0, 0, 0);
            if (there)
                y = code[w][j] >= kFourBad ? make_uint4(0x7FC07FC0u, 0x7FC07FC0u, 0x7FC07FC0u, 0x7FC07FC0u)
                                           : four_bf16x8(q[w][j], four_scale(code[w][j]));
            store_past((w ? vout : kout) + o, y);
        }
    }
}

}  // namespace
}  // namespace h3mi

using namespace h3mi;

extern "C" int h3mi_kv_write_mx4(const uint16_t* k, const uint16_t* v, int64_t rows, int64_t ld_k, int64_t bs_k, int64_t ld_v,
                                 int64_t bs_v, const h3mi_kv_cache4* cache, const h3mi_kv_seqs* seqs, void* stream) {
    if (int e = kv_check("kv_write", cache, seqs)) return e;
    if (int e = kv_check_rows("kv_write", "k", k, rows, cache->heads, cache->dim, seqs->n, ld_k, bs_k)) return e;
    if (int e = kv_check_rows("kv_write", "v", v, rows, cache->heads, cache->dim, seqs->n, ld_v, bs_v)) return e;
    if (seqs->n == 0 || rows == 0 || seqs->blocks == 0 || cache->pages == 0) return ok();
    int64_t touched = (rows + 2 * kKvBlock - 2) / kKvBlock;
    if (touched > seqs->blocks) touched = seqs->blocks;
    const int D = static_cast<int>(cache->dim);
    int64_t groups;
    if (!launchable(seqs->n, touched, cache->heads, 2 * D, &groups)) return fail(H3MI_EINVAL, "kv_write: too many tokens for one call");
    for (int x = 0; x < 2; ++x) {
        const size_t bytes = kv_span(seqs->n, rows, cache->heads, cache->dim, x ? ld_v : ld_k, x ? bs_v : bs_k);
        if (kv_overlaps(x ? v : k, bytes, *cache)) return fail(H3MI_EALIAS, "kv_write: the rows overlap the cache");
    }
    if (kv_seqs_overlap(*cache, *seqs)) return fail(H3MI_EALIAS, "kv_write: tables, lens or counts overlap the cache");
    const bool stream_in = seqs->n * rows * cache->heads * D * 4 > kMemoryCache;
    const auto fn = stream_in ? (D == 64 ? kv4_write_kernel<64, true> : D == 128 ? kv4_write_kernel<128, true> : kv4_write_kernel<256, true>)
                              : (D == 64 ? kv4_write_kernel<64, false> : D == 128 ? kv4_write_kernel<128, false> : kv4_write_kernel<256, false>);
    hipLaunchKernelGGL(fn, dim3(static_cast<unsigned>(groups)), dim3(2 * D), 0, as_stream(stream), Rows{k, ld_k, bs_k},
                       Rows{v, ld_v, bs_v}, kv_cache(*cache), kv_seqs(*seqs), static_cast<int>(rows), static_cast<int>(touched));
    return check_launch("kv_write");
}

extern "C" int h3mi_kv_read_mx4_bf16(uint16_t* k, uint16_t* v, const int32_t* starts, int64_t length, const h3mi_kv_cache4* cache,
                                     const h3mi_kv_seqs* seqs, void* stream) {
    if (int e = kv_check("kv_read", cache, seqs)) return e;
    if (length < 0 || length > (1 << 30)) return fail(H3MI_EINVAL, "kv_read: length=%lld", (long long)length);
    if (seqs->n == 0 || length == 0) return ok();
    if (!k || !v) return fail(H3MI_EINVAL, "kv_read: null k or v");
    if (!aligned(k, 16) || !aligned(v, 16) || !aligned(starts, 4))
        return fail(H3MI_EALIGN, "kv_read: k and v must be 16-byte aligned, starts 4-byte");
    const int D = static_cast<int>(cache->dim);
    const int64_t touched = starts ? (length + 2 * kKvBlock - 2) / kKvBlock : (length + kKvBlock - 1) / kKvBlock;
    int64_t groups;
    if (!launchable(seqs->n, touched, cache->heads, 2 * D, &groups)) return fail(H3MI_EINVAL, "kv_read: too many tokens for one call");
    const size_t bytes = static_cast<size_t>(seqs->n) * length * cache->heads * cache->dim * 2;
    if (overlap(k, bytes, v, bytes) || kv_overlaps(k, bytes, *cache) || kv_overlaps(v, bytes, *cache))
        return fail(H3MI_EALIAS, "kv_read: k, v and the cache overlap");
    for (const uint16_t* x : {k, v})
        if (kv_seqs_overlap(x, bytes, *seqs) || (starts && overlap(x, bytes, starts, 4 * static_cast<size_t>(seqs->n))))
            return fail(H3MI_EALIAS, "kv_read: k or v overlaps tables, lens, counts or starts");
    const bool stream_in = 2 * bytes > static_cast<size_t>(kMemoryCache);
    const auto fn = stream_in ? (D == 64 ? kv4_read_kernel<64, true> : D == 128 ? kv4_read_kernel<128, true> : kv4_read_kernel<256, true>)
                              : (D == 64 ? kv4_read_kernel<64, false> : D == 128 ? kv4_read_kernel<128, false> : kv4_read_kernel<256, false>);
    hipLaunchKernelGGL(fn, dim3(static_cast<unsigned>(groups)), dim3(2 * D), 0, as_stream(stream), k, v, starts,
                       kv_cache(*cache), kv_seqs(*seqs), static_cast<int>(length), static_cast<int>(touched));
    return check_launch("kv_read");
}
