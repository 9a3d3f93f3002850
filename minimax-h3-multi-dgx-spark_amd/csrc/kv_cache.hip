// Writing the 8-bit key/value cache and reading it back.
//
// Both move 3 bytes an element (2 in bf16, 1 in 8 bits) and do little with them, so
// HBM bounds them.  A workgroup takes one block of 64 tokens of one head, keys and
// values: a thread holds 4 tokens of 8 elements, so that a wave's loads and stores
// of bf16 rows are whole 128- to 512-byte rows of the head, the block's maximum
// needs one barrier, and four tokens of an element are one word of the transposed
// values, which pass through LDS so that their global rows are written (read) whole.
// Consecutive blocks and heads run on one XCD (a clip of 19200 tokens of 56 x 128 written
// in 155 us against 161 with heads dealt over the XCDs, read back in 154 against 160), and
// what is written goes past the L2 (161 against 167, 160 against 168; 2401 tokens 19.0
// against 25.0 and 17.3 against 20.4).  With the inputs past the caches too the clip is written
// in 150 us and read back in 157, 5.5 and 5.3 TB/s.
#include "kv.h"

namespace h3mi {

namespace {

int check_sizes(const char* what, int64_t pages, int64_t heads, int64_t dim, const h3mi_kv_seqs* s) {
    if (dim != 64 && dim != 128 && dim != 256)
        return fail(H3MI_EINVAL, "%s: dim=%lld must be 64, 128 or 256", what, (long long)dim);
    if (heads <= 0 || heads > 65536 || pages < 0 || pages > 0x7FFFFFFF)
        return fail(H3MI_EINVAL, "%s: bad cache sizes heads=%lld pages=%lld", what, (long long)heads, (long long)pages);
    if (s->n < 0 || s->n > 0x7FFFFFFF || s->blocks < 0 || s->blocks >= (int64_t{1} << 25))
        return fail(H3MI_EINVAL, "%s: bad sequences n=%lld blocks=%lld", what, (long long)s->n, (long long)s->blocks);
    return H3MI_OK;
}

int check_seqs(const char* what, const h3mi_kv_seqs* s) {
    if (!aligned(s->tables, 4) || !aligned(s->lens, 4) || !aligned(s->counts, 4))
        return fail(H3MI_EALIGN, "%s: tables, lens and counts must be 4-byte aligned", what);
    return H3MI_OK;
}

}  // namespace

int kv_check(const char* what, const h3mi_kv_cache* c, const h3mi_kv_seqs* s) {
    if (!c || !s) return fail(H3MI_EINVAL, "%s: null cache or sequences", what);
    if (int e = check_sizes(what, c->pages, c->heads, c->dim, s)) return e;
    if (s->n == 0) return H3MI_OK;
    if (c->pages > 0 && (!c->k || !c->v || !c->k_scale || !c->v_scale || !c->k_sum))
        return fail(H3MI_EINVAL, "%s: null cache pointer", what);
    if (!s->lens || (s->blocks > 0 && !s->tables)) return fail(H3MI_EINVAL, "%s: null tables or lens", what);
    if (!aligned(c->k, 16) || !aligned(c->v, 16) || !aligned(c->k_sum, 16) || !aligned(c->k_scale, 4) || !aligned(c->v_scale, 4))
        return fail(H3MI_EALIGN, "%s: the cache must be 16-byte aligned", what);
    const size_t bytes = static_cast<size_t>(c->pages) * c->heads * c->dim * kKvBlock;
    if (overlap(c->k, bytes, c->v, bytes)) return fail(H3MI_EALIAS, "%s: the cache's k and v overlap", what);
    return check_seqs(what, s);
}

int kv_check(const char* what, const h3mi_kv_cache4* c, const h3mi_kv_seqs* s) {
    if (!c || !s) return fail(H3MI_EINVAL, "%s: null cache or sequences", what);
    if (int e = check_sizes(what, c->pages, c->heads, c->dim, s)) return e;
    if (s->n == 0) return H3MI_OK;
    if (c->pages > 0 && (!c->k || !c->v || !c->k_scale || !c->v_scale)) return fail(H3MI_EINVAL, "%s: null cache pointer", what);
    if (!s->lens || (s->blocks > 0 && !s->tables)) return fail(H3MI_EINVAL, "%s: null tables or lens", what);
    if (!aligned(c->k, 16) || !aligned(c->v, 16) || !aligned(c->k_scale, 16) || !aligned(c->v_scale, 16))
        return fail(H3MI_EALIGN, "%s: the cache must be 16-byte aligned", what);
    if (kv_self_overlaps(*c)) return fail(H3MI_EALIAS, "%s: the cache's tensors overlap", what);
    return check_seqs(what, s);
}

int kv_check_rows(const char* what, const char* name, const uint16_t* p, int64_t rows, int64_t heads, int64_t dim,
                  int64_t n, int64_t ld, int64_t bs) {
    if (rows < 0 || rows > (1 << 30)) return fail(H3MI_EINVAL, "%s: rows=%lld", what, (long long)rows);
    if (rows == 0 || n == 0) return H3MI_OK;
    if (!p) return fail(H3MI_EINVAL, "%s: null %s", what, name);
    if ((rows > 1 && ld < heads * dim) || bs < 0 || (n > 1 && bs < heads * dim))
        return fail(H3MI_EINVAL, "%s: %s strides %lld, %lld are shorter than a row", what, name, (long long)ld, (long long)bs);
    if (!aligned(p, 16) || ld % 8 || bs % 8)
        return fail(H3MI_EALIGN, "%s: %s must be 16-byte aligned with strides that are multiples of 8", what, name);
    return H3MI_OK;
}

size_t kv_span(int64_t n, int64_t rows, int64_t heads, int64_t dim, int64_t ld, int64_t bs) {
    if (n == 0 || rows == 0) return 0;
    return 2 * (static_cast<size_t>(n - 1) * bs + static_cast<size_t>(rows - 1) * ld + static_cast<size_t>(heads) * dim);
}

namespace {

struct Span {
    const void* p;
    size_t bytes;
};

// A cache's tensors.
struct Spans {
    Span s[5];
    int count;
    explicit Spans(const h3mi_kv_cache& c) : count(5) {
        const size_t tiles = static_cast<size_t>(c.pages) * c.heads, kv = tiles * c.dim * kKvBlock;
        s[0] = {c.k, kv}, s[1] = {c.v, kv}, s[2] = {c.k_scale, 4 * tiles}, s[3] = {c.v_scale, 4 * tiles}, s[4] = {c.k_sum, 2 * tiles * c.dim};
    }
    explicit Spans(const h3mi_kv_cache4& c) : count(4) {
        const size_t all = static_cast<size_t>(c.pages) * c.heads * c.dim * kKvBlock;
        s[0] = {c.k, all / 2}, s[1] = {c.v, all / 2}, s[2] = {c.k_scale, all / kFourGroup}, s[3] = {c.v_scale, all / kFourGroup};
    }
    bool meet(const void* p, size_t bytes) const {
        for (int x = 0; x < count; ++x)
            if (overlap(p, bytes, s[x].p, s[x].bytes)) return true;
        return false;
    }
    bool meet_each_other() const {
        for (int x = 1; x < count; ++x)
            for (int y = 0; y < x; ++y)
                if (overlap(s[x].p, s[x].bytes, s[y].p, s[y].bytes)) return true;
        return false;
    }
    bool meet(const h3mi_kv_seqs& q) const {
        for (int x = 0; x < count; ++x)
            if (kv_seqs_overlap(s[x].p, s[x].bytes, q)) return true;
        return false;
    }
};

}  // namespace

bool kv_overlaps(const void* p, size_t bytes, const h3mi_kv_cache& c) { return Spans(c).meet(p, bytes); }
bool kv_overlaps(const void* p, size_t bytes, const h3mi_kv_cache4& c) { return Spans(c).meet(p, bytes); }
bool kv_self_overlaps(const h3mi_kv_cache& c) { return Spans(c).meet_each_other(); }
bool kv_self_overlaps(const h3mi_kv_cache4& c) { return Spans(c).meet_each_other(); }
bool kv_seqs_overlap(const h3mi_kv_cache& c, const h3mi_kv_seqs& s) { return Spans(c).meet(s); }
bool kv_seqs_overlap(const h3mi_kv_cache4& c, const h3mi_kv_seqs& s) { return Spans(c).meet(s); }

bool kv_seqs_overlap(const void* p, size_t bytes, const h3mi_kv_seqs& s) {
    const size_t each = 4 * static_cast<size_t>(s.n);
    return (s.blocks && overlap(p, bytes, s.tables, each * s.blocks)) || overlap(p, bytes, s.lens, each) || (s.counts && overlap(p, bytes, s.counts, each));
}

namespace {

// Words of a head's transposed block in LDS: 16 words of 4 tokens a row, one row's
// words off the next's banks.
constexpr int kVtStride = 17;

// A block's new scale and what becomes of its old values: old ints times mul, 0 if it is 0.
struct Scale {
    float s, mul;
};

__device__ __forceinline__ Scale grow(float a, float old, bool fresh) {
#pragma clang fp contract(off)
    const float want = a * (1.0f / 127.0f);
    if (fresh || old == 0.0f) return {want, 0.0f};
    if (!__builtin_isfinite(old)) return {old, 0.0f};
    const float r = want / old;
    if (!(r <= 256.0f)) return {want, 0.0f};
    int k = 0;
    if (r > 1.0f) {
        int e;
        const float m = __builtin_frexpf(r, &e);  // r = m 2^e, m in [0.5, 1)
        k = m == 0.5f ? e - 1 : e;
    }
    return {__builtin_ldexpf(old, k), __builtin_ldexpf(1.0f, -k)};
}

// Four signed bytes times mul (a power of two, 0 or 1), rounded to nearest even.
__device__ __forceinline__ uint32_t refit(uint32_t w, float mul) {
    if (mul == 1.0f) return w;
    uint32_t r = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int q = static_cast<int8_t>(w >> (8 * j));
        r |= (static_cast<uint32_t>(static_cast<int>(rintf(static_cast<float>(q) * mul))) & 0xFFu) << (8 * j);
    }
    return r;
}

// Bytes of four tokens of 8 elements (lo, hi words of each token) -> words of four
// tokens for each element.
__device__ __forceinline__ void transpose4(const uint2 (&t)[4], uint32_t (&w)[8]) {
#pragma unroll
    for (int p = 0; p < 2; ++p) {
        const uint32_t a = p ? t[0].y : t[0].x, b = p ? t[1].y : t[1].x, c = p ? t[2].y : t[2].x, d = p ? t[3].y : t[3].x;
        const uint32_t ab0 = __builtin_amdgcn_perm(b, a, 0x05010400u), ab1 = __builtin_amdgcn_perm(b, a, 0x07030602u);
        const uint32_t cd0 = __builtin_amdgcn_perm(d, c, 0x05010400u), cd1 = __builtin_amdgcn_perm(d, c, 0x07030602u);
        w[4 * p + 0] = __builtin_amdgcn_perm(cd0, ab0, 0x05040100u);
        w[4 * p + 1] = __builtin_amdgcn_perm(cd0, ab0, 0x07060302u);
        w[4 * p + 2] = __builtin_amdgcn_perm(cd1, ab1, 0x05040100u);
        w[4 * p + 3] = __builtin_amdgcn_perm(cd1, ab1, 0x07060302u);
    }
}

// One workgroup: one of the blocks that a sequence's new tokens touch, one head.  2 D threads.
// STREAM: the rows are loaded past the caches as well (a clip of 19200 tokens 150 us against
// 155), unless they fit the memory-side cache and may still be there (2401 tokens 22.6 us so,
// 19.0 cached).
template <int D, bool STREAM>
__global__ __launch_bounds__(2 * D) void kv_write_kernel(Rows kin, Rows vin, KvCache c, KvSeqs s, int rows, int touched) {
    constexpr int CH = D / 8;  // 16-byte chunks of a row
    constexpr int WAVES = 2 * D / 64;
    __shared__ uint32_t vt[D * kVtStride];
    __shared__ uint32_t part[2][WAVES];
    __shared__ int sums[D];

    const int at_all = xcd_item(), h = at_all % c.heads, item = at_all / c.heads;
    const int i = item / touched;
    const int len = s.len(i), count = s.count(i, rows), start = s.end(i) - count;
    // a negative start: tokens before the sequence's first are dropped
    const int b = block_of(start < 0 ? 0 : start) + item % touched;
    const int base = b * kKvBlock;
    if (count == 0 || base >= len) return;
    const int page = s.page(i, b, c.pages);
    if (page < 0) return;
    const int64_t tile = static_cast<int64_t>(page) * c.heads + h;

    const int t = threadIdx.x, col = (t % CH) * 8, quad = t / CH;
    uint4 kx[4], vx[4];
    bool fresh[4], kept[4];
    uint32_t km = 0, vm = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int at = base + 4 * quad + j;
        fresh[j] = at >= start && at < len;
        kept[j] = at < start;
        kx[j] = vx[j] = make_uint4(0, 0, 0, 0);
        if (fresh[j]) {
            const int64_t row = at - start;
            kx[j] = load_row<STREAM>(kin.p + i * kin.bs + row * kin.ld + h * D + col);
            vx[j] = load_row<STREAM>(vin.p + i * vin.bs + row * vin.ld + h * D + col);
        }
    }
    const bool first = start <= base;  // no token of the block is older
    int8_t* const kout = c.k + tile * (kKvBlock * D);
    int8_t* const vout = c.v + tile * (kKvBlock * D);
    // what an older block held, asked for before the maximum is known
    float old_k = 0.0f, old_v = 0.0f;
    uint2 ko[4] = {};
    uint32_t vo[8] = {};
    if (!first) {
        old_k = c.ks[tile], old_v = c.vs[tile];
        if (base + 4 * quad < start) {
#pragma unroll
            for (int j = 0; j < 4; ++j) ko[j] = *reinterpret_cast<const uint2*>(kout + (4 * quad + j) * D + col);
#pragma unroll
            for (int p = 0; p < 8; ++p) vo[p] = *reinterpret_cast<const uint32_t*>(vout + (col + p) * kKvBlock + 4 * quad);
        }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const uint32_t a[4] = {kx[j].x, kx[j].y, kx[j].z, kx[j].w}, e[4] = {vx[j].x, vx[j].y, vx[j].z, vx[j].w};
#pragma unroll
        for (int p = 0; p < 4; ++p) {
            km = max_mag(km, a[p] & 0x7FFF7FFFu);
            vm = max_mag(vm, e[p] & 0x7FFF7FFFu);
        }
    }
    uint32_t km1 = km & 0xFFFFu, vm1 = vm & 0xFFFFu;
    km1 = km1 > (km >> 16) ? km1 : km >> 16;
    vm1 = vm1 > (vm >> 16) ? vm1 : vm >> 16;
    // (16-bit patterns as whole numbers in fp32)
    km1 = static_cast<uint32_t>(wave_max(static_cast<float>(km1)));
    vm1 = static_cast<uint32_t>(wave_max(static_cast<float>(vm1)));
    if ((t & 63) == 0) part[0][t >> 6] = km1, part[1][t >> 6] = vm1;
    if (t < D) sums[t] = 0;
    __syncthreads();
    km1 = vm1 = 0;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
        km1 = km1 > part[0][w] ? km1 : part[0][w];
        vm1 = vm1 > part[1][w] ? vm1 : part[1][w];
    }
    const Scale sk = grow(wave_uniform(bf16_f32(km1)), old_k, first), sv = grow(wave_uniform(bf16_f32(vm1)), old_v, first);
    if (t == 0) c.ks[tile] = sk.s, c.vs[tile] = sv.s;

    // s is fl(a c), c = fl(1 / 127), of some bf16 a times a power of two, and no x is above that a and power: quant8
    // rounds every such x / s as the divide does (tests/test_kv_quant_exact.py)
    const float rk = 1.0f / sk.s, rv = 1.0f / sv.s;
    const bool live_k = sk.s > 0.0f && __builtin_isfinite(sk.s), live_v = sv.s > 0.0f && __builtin_isfinite(sv.s);
    const bool exact_k = quot_exact(sk.s, rk), exact_v = quot_exact(sv.s, rv);
    int acc[8] = {};
    uint2 vq[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int tok = 4 * quad + j;
        uint2 q = make_uint2(0, 0);
        vq[j] = q;
        if (fresh[j]) {
            const uint32_t a[4] = {kx[j].x, kx[j].y, kx[j].z, kx[j].w}, e[4] = {vx[j].x, vx[j].y, vx[j].z, vx[j].w};
            if (live_k) q = quant8(a, sk.s, rk, exact_k);
            if (live_v) vq[j] = quant8(e, sv.s, rv, exact_v);
        } else if (kept[j] && live_k && sk.mul != 0.0f) {
            q = make_uint2(refit(ko[j].x, sk.mul), refit(ko[j].y, sk.mul));
        }
        store_past(kout + tok * D + col, q);
#pragma unroll
        for (int p = 0; p < 4; ++p) {
            acc[p] += static_cast<int8_t>(q.x >> (8 * p));
            acc[4 + p] += static_cast<int8_t>(q.y >> (8 * p));
        }
    }
    uint32_t w[8];
    transpose4(vq, w);
    const bool olds = live_v && sv.mul != 0.0f;
    uint32_t mask = 0;  // bytes of the tokens kept
#pragma unroll
    for (int j = 0; j < 4; ++j) mask |= kept[j] ? 0xFFu << (8 * j) : 0u;
#pragma unroll
    for (int p = 0; p < 8; ++p) {
        if (olds && mask) w[p] |= refit(vo[p], sv.mul) & mask;
        vt[(col + p) * kVtStride + quad] = w[p];
        atomicAdd(&sums[col + p], acc[p]);
    }
    __syncthreads();
    // 4 D 16-byte pieces of the transposed values, two a thread
#pragma unroll
    for (int p = 0; p < 2; ++p) {
        const int piece = t + p * 2 * D, row = piece >> 2, at = (piece & 3) * 4;
        const uint32_t* const src = vt + row * kVtStride + at;
        store_past(vout + piece * 16, make_uint4(src[0], src[1], src[2], src[3]));
    }
    if (t < D) c.ksum[tile * D + t] = static_cast<int16_t>(sums[t]);
}

// 8 signed bytes times s, as 8 bf16.
__device__ __forceinline__ uint4 widen(uint2 q, float s) {
    float f[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = static_cast<float>(static_cast<int8_t>((j < 4 ? q.x : q.y) >> (8 * (j & 3)))) * s;
    return make_uint4(bf16x2_bits(f[0], f[1]), bf16x2_bits(f[2], f[3]), bf16x2_bits(f[4], f[5]), bf16x2_bits(f[6], f[7]));
}

// One workgroup: one cache block of those that a sequence's tokens starts .. starts + length - 1 lie in, one head.
template <int D>
__global__ __launch_bounds__(2 * D) void kv_read_kernel(uint16_t* __restrict__ kout, uint16_t* __restrict__ vout,
                                                        const int32_t* __restrict__ starts, KvCache c, KvSeqs s, int length,
                                                        int touched) {
    constexpr int CH = D / 8;
    __shared__ uint32_t vt[D * kVtStride];
    const int at_all = xcd_item(), h = at_all % c.heads, item = at_all / c.heads;
    const int i = item / touched;
    const int start = starts ? starts[i] : 0;
    const int64_t b = static_cast<int64_t>(block_of(start)) + item % touched;
    const int len = s.len(i);
    const int64_t base = b * kKvBlock, from = base - start;  // of the block's first token in the output
    if (from >= length) return;
    const int page = base < len ? s.page(i, static_cast<int>(b), c.pages) : -1;
    const int t = threadIdx.x, col = (t % CH) * 8, quad = t / CH;
    const int64_t tile = static_cast<int64_t>(page < 0 ? 0 : page) * c.heads + h;
    float ks = 0.0f, vs = 0.0f;
    uint2 kq[4];
    if (page >= 0) {
        ks = c.ks[tile], vs = c.vs[tile];
        const int8_t* const kin = c.k + tile * (kKvBlock * D);
        const int8_t* const vin = c.v + tile * (kKvBlock * D);
#pragma unroll
        for (int j = 0; j < 4; ++j) kq[j] = *reinterpret_cast<const uint2*>(kin + (4 * quad + j) * D + col);
#pragma unroll
        for (int p = 0; p < 2; ++p) {
            const int piece = t + p * 2 * D, row = piece >> 2, at = (piece & 3) * 4;
            const uint4 w = *reinterpret_cast<const uint4*>(vin + piece * 16);
            uint32_t* const dst = vt + row * kVtStride + at;
            dst[0] = w.x, dst[1] = w.y, dst[2] = w.z, dst[3] = w.w;
        }
    }
    __syncthreads();
    uint32_t w[8];
#pragma unroll
    for (int p = 0; p < 8; ++p) w[p] = page < 0 ? 0u : vt[(col + p) * kVtStride + quad];
    const uint2 lo[4] = {make_uint2(w[0], w[4]), make_uint2(w[1], w[5]), make_uint2(w[2], w[6]), make_uint2(w[3], w[7])};
    uint32_t x[8];  // x[j], x[4 + j]: elements 0..3 and 4..7 of token j
    transpose4(lo, x);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int64_t r = from + 4 * quad + j, at = base + 4 * quad + j;
        if (r < 0 || r >= length) continue;
        const int64_t o = ((i * static_cast<int64_t>(length) + r) * c.heads + h) * D + col;
        const bool there = page >= 0 && at < len;
        const uint4 none = make_uint4(0, 0, 0, 0);
        store_past(kout + o, there ? widen(kq[j], ks) : none);
        store_past(vout + o, there ? widen(make_uint2(x[j], x[4 + j]), vs) : none);
    }
}

}  // namespace
}  // namespace h3mi

using namespace h3mi;

extern "C" int h3mi_kv_write_i8(const uint16_t* k, const uint16_t* v, int64_t rows, int64_t ld_k, int64_t bs_k, int64_t ld_v,
                                int64_t bs_v, const h3mi_kv_cache* cache, const h3mi_kv_seqs* seqs, void* stream) {
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
    if (kv_self_overlaps(*cache)) return fail(H3MI_EALIAS, "kv_write: the cache's tensors overlap");
    if (kv_seqs_overlap(*cache, *seqs)) return fail(H3MI_EALIAS, "kv_write: tables, lens or counts overlap the cache");
    const bool stream_in = seqs->n * rows * cache->heads * D * 4 > kMemoryCache;
    const auto fn = stream_in ? (D == 64 ? kv_write_kernel<64, true> : D == 128 ? kv_write_kernel<128, true> : kv_write_kernel<256, true>)
                              : (D == 64 ? kv_write_kernel<64, false> : D == 128 ? kv_write_kernel<128, false> : kv_write_kernel<256, false>);
    hipLaunchKernelGGL(fn, dim3(static_cast<unsigned>(groups)), dim3(2 * D), 0, as_stream(stream), Rows{k, ld_k, bs_k},
                       Rows{v, ld_v, bs_v}, kv_cache(*cache), kv_seqs(*seqs), static_cast<int>(rows), static_cast<int>(touched));
    return check_launch("kv_write");
}

extern "C" int h3mi_kv_read_bf16(uint16_t* k, uint16_t* v, const int32_t* starts, int64_t length, const h3mi_kv_cache* cache,
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
    const auto fn = D == 64 ? kv_read_kernel<64> : D == 128 ? kv_read_kernel<128> : kv_read_kernel<256>;
    hipLaunchKernelGGL(fn, dim3(static_cast<unsigned>(groups)), dim3(2 * D), 0, as_stream(stream), k, v, starts,
                       kv_cache(*cache), kv_seqs(*seqs), static_cast<int>(length), static_cast<int>(touched));
    return check_launch("kv_read");
}
