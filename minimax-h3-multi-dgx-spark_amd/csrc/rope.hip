// Rotary positions: pairs (a, b) of a head's first `rot` elements become, with w = freqs[pair],
//   (a c - b s, a s + b c),  c = amplitude cos(p w), s = amplitude sin(p w)   (inverse: s negated)
// for a row at position p.  The transpose of that matrix, which a gradient is multiplied by, is
// the inverse.  Pairs are (i, i + rot / 2), or (2 i, 2 i + 1) where they are interleaved.
//
// p w is formed in turns in 64 bits and reduced there, as p has up to 31 bits and a bf16 result
// wants the angle to a few thousandths whatever p is; what is left, half a turn at most, goes
// through fp32 sine and cosine.  Products and sums are fp32, and a result is rounded once.
//
// It moves 4 bytes a turned element and does 3 operations with it, so HBM bounds it, and the
// sines, one for each row and pair whatever the heads, are formed once for a workgroup's share of
// the row's heads and kept in LDS.  A workgroup takes a few whole rows, or where there are few
// rows a share of one's heads.  A thread takes 8 pairs of a head (4 interleaved ones): 16-byte
// accesses whose lanes lie side by side, or as many bytes as the turned part (or its half) divides
// into.
#include "kv.h"

namespace h3mi {
namespace {

struct RopeRows {
    const uint16_t* in;
    uint16_t* out;
    int heads;
    int64_t ld_in, bs_in, ld_out, bs_out;
};

struct RopeCall {
    RopeRows q, k;  // k.heads 0: none
    const int32_t* positions;
    const double* freqs;
    uint32_t rows, all;   // of a sequence; of all
    int dim, rot, tokens; // tokens: rows of a workgroup
    int parts;            // workgroups of such rows
    int turned, units;    // units of a head: turned ones, and with those that are copied (at most 256)
    float amplitude, sign;
    bool in_place;
};

constexpr int kRopeThreads = 256;
constexpr int kRopeAhead = 4;   // units that a thread has in flight (2 and 8: 1% and 4% slower)
constexpr int kRopeTokens = 16;

// How rows go through the caches.  kCached: rows in place that the memory-side cache may hold.  kStore: new tensors, written past
// the L2 (2401 rows of 112 heads, the memory-side cache full of others 31.5 us, 28.6 so; else 24.2 and 24.6).  kPast: rows that
// are more than that cache holds beside others, read past it too (19200 in place 217 us, 191 so; 2401 of 48 heads of 4 sequences
// into new tensors 51 and 47; but 4801 rows in place, which it holds, 43 and 52).
enum RopeWay { kCached, kStore, kPast };
constexpr int64_t kRopePast = kMemoryCache / 4 * 3;

// V neighbouring elements, one access.
template <int V>
struct Run {
    uint32_t w[V == 1 ? 1 : V / 2];
    template <bool PAST>
    __device__ __forceinline__ void load(const uint16_t* p) {
        if constexpr (V == 8) {
            const uint4 x = load_row<PAST>(p);
            w[0] = x.x, w[1] = x.y, w[2] = x.z, w[3] = x.w;
        } else if constexpr (V == 4) {
            const uint2 x = *reinterpret_cast<const uint2*>(p);
            w[0] = x.x, w[1] = x.y;
        } else if constexpr (V == 2) {
            w[0] = *reinterpret_cast<const uint32_t*>(p);
        } else {
            w[0] = *p;
        }
    }
    template <bool PAST>
    __device__ __forceinline__ void store(uint16_t* p) const {
        if constexpr (V == 8) {
            const uint4 x = make_uint4(w[0], w[1], w[2], w[3]);
            if constexpr (PAST) store_past(p, x);
            else *reinterpret_cast<uint4*>(p) = x;
        } else if constexpr (V == 4) {
            *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
        } else if constexpr (V == 2) {
            *reinterpret_cast<uint32_t*>(p) = w[0];
        } else {
            *p = static_cast<uint16_t>(w[0]);
        }
    }
};

__device__ __forceinline__ void turn(float x, float y, float2 cs, float& u, float& v) {
    u = __builtin_fmaf(x, cs.x, -(y * cs.y));
    v = __builtin_fmaf(x, cs.y, y * cs.x);
}

// A unit's pairs; tab: (c, s) of its first.  PAIRS: neighbours in a, else a and b.
template <bool PAIRS, int V>
__device__ __forceinline__ void turn(Run<V>& a, Run<V>& b, const float2* tab) {
    if constexpr (PAIRS) {
#pragma unroll
        for (int j = 0; j < V / 2; ++j) {
            float u, v;
            turn(bf16_lo(a.w[j]), bf16_hi(a.w[j]), tab[j], u, v);
            a.w[j] = bf16x2_bits(u, v);
        }
    } else if constexpr (V == 1) {
        float u, v;
        turn(bf16_f32(a.w[0]), bf16_f32(b.w[0]), tab[0], u, v);
        a.w[0] = bf16_bits(u), b.w[0] = bf16_bits(v);
    } else {
#pragma unroll
        for (int j = 0; j < V / 2; ++j) {
            float u0, v0, u1, v1;
            turn(bf16_lo(a.w[j]), bf16_lo(b.w[j]), tab[2 * j], u0, v0);
            turn(bf16_hi(a.w[j]), bf16_hi(b.w[j]), tab[2 * j + 1], u1, v1);
            a.w[j] = bf16x2_bits(u0, u1);
            b.w[j] = bf16x2_bits(v0, v1);
        }
    }
}

// A unit: V pairs of halves, V / 2 of neighbours, or as many elements that are copied.
template <bool PAIRS, int V, RopeWay W>
__global__ __launch_bounds__(kRopeThreads) void rope_kernel(RopeCall c) {
    extern __shared__ float2 tab[];  // [tokens, rot / 2]: (c, s)
    __shared__ bool real[kRopeTokens];  // rows that a position was given for
    const int half = c.rot / 2, t = threadIdx.x;
    const uint32_t first = blockIdx.x / c.parts * c.tokens, left = c.all - first;
    const int part = blockIdx.x % c.parts, tokens = left < static_cast<uint32_t>(c.tokens) ? static_cast<int>(left) : c.tokens;
    if (t < tokens) real[t] = c.positions[first + t] >= 0;
    for (int x = t; x < tokens * half; x += kRopeThreads) {
        const int tok = x / half, i = x - tok * half, p = c.positions[first + tok];
        float2 cs = make_float2(1.0f, 0.0f);
        if (p >= 0) {
            constexpr double kTurn = 0.15915494309189533577;  // 1 / (2 pi)
            double a = p * (c.freqs[i] * kTurn);
            a -= __builtin_rint(a);
            float s, o;
            sincospif(2.0f * static_cast<float>(a), &s, &o);
            cs = make_float2(o * c.amplitude, s * c.sign);
        }
        tab[x] = cs;
    }
    __syncthreads();

    // (row, head) pairs of the workgroup's share, kRopeThreads / units at a time
    const int heads = c.q.heads + c.k.heads, share = (heads + c.parts - 1) / c.parts;
    const int h0 = part * share, h1 = h0 + share < heads ? h0 + share : heads, mine = h1 - h0;
    if (mine <= 0) return;
    const int lanes = kRopeThreads / c.units, unit = t % c.units, lane = t / c.units;
    if (lane >= lanes) return;
    const bool turned = unit < c.turned;
    // its elements: a at `at`, and of halves b at `at + apart`
    const int at = turned ? V * unit : c.rot + (PAIRS ? V : 2 * V) * (unit - c.turned), apart = turned ? half : V;
    const bool two = !PAIRS && at + apart < c.dim;  // (the last copied unit may have V elements alone)
    for (int x0 = lane; x0 < tokens * mine; x0 += lanes * kRopeAhead) {
        Run<V> y[kRopeAhead], z[kRopeAhead];
        uint16_t* to[kRopeAhead];
        int tok[kRopeAhead];
#pragma unroll
        for (int j = 0; j < kRopeAhead; ++j) {
            const int x = x0 + j * lanes;
            to[j] = nullptr;
            if (x >= tokens * mine) continue;
            tok[j] = x / mine;
            const int h = h0 + x - tok[j] * mine;
            const uint32_t row = first + tok[j], i = row / c.rows, r = row - i * c.rows;
            if (c.in_place && !real[tok[j]]) continue;
            const bool of_q = h < c.q.heads;
            const RopeRows& rows = of_q ? c.q : c.k;
            const int64_t el = static_cast<int64_t>(of_q ? h : h - c.q.heads) * c.dim + at;
            const uint16_t* const from = rows.in + i * rows.bs_in + r * rows.ld_in + el;
            to[j] = rows.out + i * rows.bs_out + r * rows.ld_out + el;
            if (!(turned && real[tok[j]])) tok[j] = -1;
            y[j].template load<W == kPast>(from);
            if (two) z[j].template load<W == kPast>(from + apart);
        }
#pragma unroll
        for (int j = 0; j < kRopeAhead; ++j) {
            if (!to[j]) continue;
            if (tok[j] >= 0) turn<PAIRS, V>(y[j], z[j], tab + tok[j] * half + unit * (PAIRS ? V / 2 : V));
            y[j].template store<W != kCached>(to[j]);
            if (two) z[j].template store<W != kCached>(to[j] + apart);
        }
    }
}

size_t span_of(const h3mi_rope_rows& x, bool out, int64_t n, int64_t rows, int64_t dim) {
    const int64_t ld = out ? x.ld_out : x.ld_in, bs = out ? x.bs_out : x.bs_in;
    return 2 * (static_cast<size_t>(n - 1) * bs + static_cast<size_t>(rows - 1) * ld + static_cast<size_t>(x.heads) * dim);
}

int check_rows(const char* name, const h3mi_rope_rows& x, int64_t n, int64_t rows, int64_t dim) {
    const int64_t e = x.heads * dim;
    if (!x.in || !x.out) return fail(H3MI_EINVAL, "rope: null %s", name);
    if (x.heads <= 0 || x.heads > 65536) return fail(H3MI_EINVAL, "rope: %s has %lld heads", name, (long long)x.heads);
    for (int64_t ld : {x.ld_in, x.ld_out})
        if (rows > 1 && ld < e) return fail(H3MI_EINVAL, "rope: %s strides are shorter than a row", name);
    for (int64_t bs : {x.bs_in, x.bs_out})
        if (n > 1 && bs < e) return fail(H3MI_EINVAL, "rope: %s strides are shorter than a row", name);
    if (!aligned(x.in, 16) || !aligned(x.out, 16) || (rows > 1 && (x.ld_in % 8 || x.ld_out % 8)) || (n > 1 && (x.bs_in % 8 || x.bs_out % 8)))
        return fail(H3MI_EALIGN, "rope: %s must be 16-byte aligned with strides that are multiples of 8", name);
    // rows that overlap would be turned twice
    if (n > 1 && rows > 1 && x.bs_out < (rows - 1) * x.ld_out + e && x.ld_out < (n - 1) * x.bs_out + e)
        return fail(H3MI_EALIAS, "rope: rows of %s overlap", name);
    if (x.in == x.out && ((rows > 1 && x.ld_in != x.ld_out) || (n > 1 && x.bs_in != x.bs_out)))
        return fail(H3MI_EALIAS, "rope: %s in place with other strides", name);
    if (x.in != x.out && overlap(x.in, span_of(x, false, n, rows, dim), x.out, span_of(x, true, n, rows, dim)))
        return fail(H3MI_EALIAS, "rope: %s overlaps its result", name);
    return H3MI_OK;
}

// Whether runs of run_a elements every `step` of them meet runs of run_b that lie d behind.
bool runs_meet(int64_t d, int64_t step, int64_t run_a, int64_t run_b) {
    d %= step;
    if (d < 0) d += step;
    return d < run_a || d + run_b > step;
}

// Whether rows of a and b share an element; of one buffer they are known not to in views of a projection's output, and where
// whole sequences, or what all sequences have of a token, lie apart.
bool rows_meet(const uint16_t* a, int64_t ha, int64_t lda, int64_t bsa, const uint16_t* b, int64_t hb, int64_t ldb, int64_t bsb,
               int64_t n, int64_t rows, int64_t dim) {
    const h3mi_rope_rows x = {a, nullptr, ha, lda, bsa, 0, 0}, y = {b, nullptr, hb, ldb, bsb, 0, 0};
    if (!overlap(a, span_of(x, false, n, rows, dim), b, span_of(y, false, n, rows, dim))) return false;
    const int64_t d = (reinterpret_cast<intptr_t>(b) - reinterpret_cast<intptr_t>(a)) / 2, ea = ha * dim, eb = hb * dim;
    if (n > 1 && bsa == bsb && !runs_meet(d, bsa, (rows - 1) * lda + ea, (rows - 1) * ldb + eb)) return false;
    if (rows > 1 && lda == ldb && !runs_meet(d, lda, (n - 1) * bsa + ea, (n - 1) * bsb + eb)) return false;
    // equal strides, one a multiple of the other: rows between each other's
    if (n == 1 || rows == 1 || lda != ldb || bsa != bsb) return true;
    const int64_t step = lda < bsa ? lda : bsa;
    return (lda + bsa - step) % step || runs_meet(d, step, ea, eb);
}

}  // namespace
}  // namespace h3mi

using namespace h3mi;

extern "C" int h3mi_rope_bf16(const h3mi_rope_rows* q, const h3mi_rope_rows* k, const int32_t* positions, const double* freqs,
                              int64_t n, int64_t rows, int64_t dim, int64_t rot, int interleaved, int inverse, float amplitude,
                              void* stream) {
    if (!q) return fail(H3MI_EINVAL, "rope: null q");
    if (dim < 8 || dim > 512 || dim % 8) return fail(H3MI_EINVAL, "rope: dim=%lld must be a multiple of 8 up to 512", (long long)dim);
    if (rot < 2 || rot > dim || rot % 2) return fail(H3MI_EINVAL, "rope: rot=%lld must be even, 2 to dim", (long long)rot);
    if (n < 0 || rows < 0 || n > 0x7FFFFFFF || rows > 0x7FFFFFFF || n * rows > 0x7FFFFFFF)
        return fail(H3MI_EINVAL, "rope: bad sizes n=%lld rows=%lld", (long long)n, (long long)rows);
    if (!(amplitude - amplitude == 0.0f)) return fail(H3MI_EINVAL, "rope: amplitude is not finite");
    if (n == 0 || rows == 0) return ok();
    if (!positions || !freqs) return fail(H3MI_EINVAL, "rope: null positions or freqs");
    if (!aligned(positions, 4) || !aligned(freqs, 8)) return fail(H3MI_EALIGN, "rope: positions must be 4-byte aligned, freqs 8-byte");
    if (int e = check_rows("q", *q, n, rows, dim)) return e;
    if (k)
        if (int e = check_rows("k", *k, n, rows, dim)) return e;
    const size_t pos_bytes = 4 * static_cast<size_t>(n) * rows, freq_bytes = 4 * static_cast<size_t>(rot);
    for (const h3mi_rope_rows* x : {q, k}) {
        if (!x) continue;
        if (overlap(x->out, span_of(*x, true, n, rows, dim), positions, pos_bytes) || overlap(x->out, span_of(*x, true, n, rows, dim), freqs, freq_bytes))
            return fail(H3MI_EALIAS, "rope: a result overlaps positions or freqs");
    }
    if (k && (rows_meet(q->out, q->heads, q->ld_out, q->bs_out, k->out, k->heads, k->ld_out, k->bs_out, n, rows, dim) ||
              (k->in != k->out && rows_meet(q->out, q->heads, q->ld_out, q->bs_out, k->in, k->heads, k->ld_in, k->bs_in, n, rows, dim)) ||
              (q->in != q->out && rows_meet(k->out, k->heads, k->ld_out, k->bs_out, q->in, q->heads, q->ld_in, q->bs_in, n, rows, dim))))
        return fail(H3MI_EALIAS, "rope: q and k overlap");
    if (k && (k->in == k->out) != (q->in == q->out)) return fail(H3MI_EINVAL, "rope: q and k must both be in place, or neither");

    // The widest accesses that the turned part fills, or each of its halves (2261 rows in place of 80 heads of 256, 128 of them
    // turned: 20 us in 8; 120, in 4: 23; 124: in pairs, by 4, 28, else by 2 27; 126: pairs by 2 37, else singly 39, which is
    // what all but the first took singly, 40 to 45.  Into new tensors, whose copied elements go by the same width, 128 takes 38 to
    // 43, 120 43 to 50, 124 62, 126 85 to 93; at a copy's rate all would take 38).
    const int64_t run = interleaved ? rot : rot / 2, V = run % 8 == 0 ? 8 : run % 4 == 0 ? 4 : run % 2 == 0 ? 2 : 1;
    RopeCall c = {};
    const auto side = [](const h3mi_rope_rows& x) { return RopeRows{x.in, x.out, static_cast<int>(x.heads), x.ld_in, x.bs_in, x.ld_out, x.bs_out}; };
    c.q = side(*q);
    if (k) c.k = side(*k);
    c.positions = positions, c.freqs = freqs;
    c.rows = static_cast<uint32_t>(rows), c.all = static_cast<uint32_t>(n * rows);
    c.dim = static_cast<int>(dim), c.rot = static_cast<int>(rot);
    c.amplitude = amplitude, c.sign = inverse ? -amplitude : amplitude;
    c.in_place = q->in == q->out;
    c.turned = static_cast<int>(run / V);
    const int64_t rest = c.in_place ? 0 : dim - rot;
    c.units = c.turned + static_cast<int>(interleaved ? rest / V : (rest + 2 * V - 1) / (2 * V));
    // Rows until a thread has kRopeAhead units, as far as there are workgroups for every CU; else a share of a row's heads.
    const int64_t heads = q->heads + (k ? k->heads : 0), a_round = kRopeThreads / c.units, want = a_round * kRopeAhead, cus = cu_count();
    int64_t tokens = want / heads;
    if (tokens > c.all / (4 * cus)) tokens = c.all / (4 * cus);
    if (tokens > kRopeTokens) tokens = kRopeTokens;
    if (tokens < 1) tokens = 1;
    int64_t parts = 1;
    if (tokens == 1) {
        parts = 4 * cus / c.all;
        if (parts > (heads + a_round - 1) / a_round) parts = (heads + a_round - 1) / a_round;
        if (parts < (heads + 4 * want - 1) / (4 * want)) parts = (heads + 4 * want - 1) / (4 * want);
    }
    c.tokens = static_cast<int>(tokens), c.parts = static_cast<int>(parts);
    const int64_t groups = (c.all + tokens - 1) / tokens * parts;
    if (groups * kRopeThreads >= (int64_t{1} << 32)) return fail(H3MI_EINVAL, "rope: too many rows for one call");
    const size_t lds = static_cast<size_t>(tokens) * (rot / 2) * 8;
    const RopeWay way = c.all * heads * dim * (c.in_place ? 2 : 4) > kRopePast ? kPast : c.in_place ? kCached : kStore;
    const auto wide = interleaved ? (way == kCached ? rope_kernel<true, 8, kCached> : way == kStore ? rope_kernel<true, 8, kStore> : rope_kernel<true, 8, kPast>)
                                  : (way == kCached ? rope_kernel<false, 8, kCached> : way == kStore ? rope_kernel<false, 8, kStore> : rope_kernel<false, 8, kPast>);
    const auto fn = V == 8 ? wide
                  : V == 4 ? (interleaved ? rope_kernel<true, 4, kCached> : rope_kernel<false, 4, kCached>)
                  : V == 2 ? (interleaved ? rope_kernel<true, 2, kCached> : rope_kernel<false, 2, kCached>)
                           : rope_kernel<false, 1, kCached>;
    hipLaunchKernelGGL(fn, dim3(static_cast<unsigned>(groups)), dim3(kRopeThreads), lds, as_stream(stream), c);
    return check_launch("rope");
}
