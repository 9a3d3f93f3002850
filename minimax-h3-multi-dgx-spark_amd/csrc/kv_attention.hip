// Attention over the key/value caches of 8 and of 4 bits.
//
// One pass over a sequence's blocks of 64 tokens with the running maximum m and sum l of
// the softmax, in base 2:  x = (q . k) c_b, c_b = k_scale scale log2(e);  p = 2^(x - m);
// l += sum p;  o += sum p v.  Keys and values are 8-bit integers, which bf16 holds
// exactly, so the products run on bf16 MFMAs with the integers themselves: a block's key
// scale is a factor of its scores (one fma with the subtraction of m), and its value scale
// a term of the exponent, p v_scale = 2^(x - m + log2 v_scale), which costs nothing per
// score; l takes the sum times 1 / v_scale.  Scores and sums are fp32; a probability is
// rounded once, to the bf16 that the second product multiplies.  That is off by 2^-8 of it at
// most, as the output's own rounding is: outputs are 1.8e-3 off (rms) where a few tokens outweigh
// the rest, 2.4e-3 where thousands weigh alike, and 1.7e-3 is what the output's rounding leaves
// with probabilities in 32 bits.  A second MFMA for the remainder would add half of all products
// of a tile.  Of few queries, which memory bounds, it costs (4 bits, 16 queries) 2% at 128 and 256
// elements and 8 to 10% at 64, with 32 queries of 128 21% (8 x 20 rows 61.6 us, 74.5 so); left
// out there too, so that a row's result is as good whatever rows it comes with.
//
// Both products are formed transposed, S^T = K Q^T and O^T = V^T P^T: a query is then a
// column, whose scores lie in the registers of two (four) lanes, so that the maximum needs
// one (two) lane exchanges a block, and the lanes that hold a query's probabilities are
// those that the second product wants them in.  Rows of K are taken in the order that
// makes the probabilities' registers whole runs of tokens; V is stored transposed, so that
// its rows are runs of tokens too.  P never leaves the registers.
//
// In 4 bits a factor is a power of two and a value has two bits, so that their products are
// exact in bf16 too and go into the MFMAs as they are: no factors of blocks, c = scale log2(e).
// Values lie token by token there, and are transposed on their way, in pairs by permutes.
//
// Two kernels: tiles of 128 or 256 query rows of a head, bound by the MFMAs and the
// softmax, and up to 64, 32 or 16 queries (of 64, 128, 256 elements) of a kv head's group,
// bound by the cache's bytes.
#include <type_traits>

#include "kv.h"

namespace h3mi {
namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr float kLog2e = 1.44269504088896341f;
// The running maximum's start: finite, so that a row that has seen nothing has differences
// that are numbers, and below every finite score that counts.
constexpr float kLowest = -3.4028234663852886e38f;
// A row keeps its reference until a score passes it by 2^kSlack (then p <= 2^kSlack, which
// fp32 sums and bf16 probabilities hold as well as p <= 1): the accumulators are rescaled a
// few times a sequence, not once a block.
constexpr float kSlack = 8.0f;
// Value scales whose log2 goes into the exponent: 2^(+-60) keeps p v_scale a normal number
// for every p above 2^-66.  Others (zero, not finite) multiply p afterwards, as in a block
// whose key scale is not finite.
constexpr float kFoldLow = 0x1p-60f, kFoldHigh = 0x1p+60f;

// 8 signed bytes as 8 bf16.
__device__ __forceinline__ uint4 ints_bf16(uint2 q) {
    float f[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = static_cast<float>(static_cast<int8_t>((j < 4 ? q.x : q.y) >> (8 * (j & 3))));
    return make_uint4(bf16x2_bits(f[0], f[1]), bf16x2_bits(f[2], f[3]), bf16x2_bits(f[4], f[5]), bf16x2_bits(f[6], f[7]));
}

__device__ __forceinline__ bf16x8 frag(uint4 w) { return __builtin_bit_cast(bf16x8, w); }

// 8 query elements, with the sign of the scale.
__device__ __forceinline__ bf16x8 query_frag(const uint16_t* p, float scale) {
    uint4 w = *reinterpret_cast<const uint4*>(p);
    const uint32_t flip = scale < 0.0f ? 0x80008000u : 0u;
    w.x ^= flip, w.y ^= flip, w.z ^= flip, w.w ^= flip;
    return frag(w);
}

// 8 probabilities, rounded to nearest even.
__device__ __forceinline__ bf16x8 pack(const float (&x)[8]) {
    return frag(make_uint4(bf16x2_bits(x[0], x[1]), bf16x2_bits(x[2], x[3]), bf16x2_bits(x[4], x[5]), bf16x2_bits(x[6], x[7])));
}

__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ float uniform(float v) { return __int_as_float(__builtin_amdgcn_readfirstlane(__float_as_int(v))); }

// The larger of lanes l and l ^ 32.
__device__ __forceinline__ float max_halves(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

// The larger of lanes l and l ^ 16.
__device__ __forceinline__ float max_quads(float v) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

__device__ __forceinline__ float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }

// What a block's scores and probabilities are multiplied by.
struct Factors {
    float c;         // scores: k_scale |scale| log2(e), the sign being the queries'; never 0, so that a masked score's
                     // -inf stays one: 2^-126 makes as much of a score as 0 does
    float lv, iv;    // the exponent's term, and what a sum of probabilities is multiplied by
    float vs;        // probabilities are multiplied by it where iv is 0
};

__device__ __forceinline__ Factors factors(float ks, float vs, float scale) {
    const float c = ks * fabsf(scale);
    const bool fold = vs >= kFoldLow && vs <= kFoldHigh && __builtin_isfinite(c);
    // (both within an ulp, of a scale far from where they flush)
    return {c < 0x1p-126f ? 0x1p-126f : c, fold ? __builtin_amdgcn_logf(vs) : 0.0f, fold ? __builtin_amdgcn_rcpf(vs) : 0.0f, vs};
}

// Whether one of four scale codes stands for no number: bytes of kFourBad and more.
__device__ __forceinline__ bool four_bad(uint32_t codes) {
    static_assert(kFourBad == 253, "125 + 3 = 2^7");
    return (((codes & 0x7F7F7F7Fu) + 0x03030303u) & codes & 0x80808080u) != 0;
}

struct Queries {
    const uint16_t* p;
    int64_t ld, bs;
    int rows, heads;
};

struct Lists {
    const int32_t* p;  // [n, tiles, kv heads, top], or null
    int top, tiles;
};

// Partial results of the items whose blocks are split: for each (item, split, row of the
// item) dim sums, and (m, l).  A split without a token writes l = 0 and no sums.
struct Partial {
    float* o;
    float2* ml;
    int splits, rows;  // of an item
    __device__ __forceinline__ int64_t at(int64_t item, int split, int row) const { return (item * splits + split) * rows + row; }
};

// ------------------------------------------------------------------ tiles of queries

// W waves of 32 query rows.  The block's keys and values go through LDS as bf16, converted
// once a workgroup, in two buffers each.  A wave's step y has two halves: the products of
// block y's keys and of block y - 1's values (MFMA, while a later block's bytes are loaded),
// then block y's softmax and that later block's conversion (VALU).  With 4 waves there is a
// barrier a step, and the workgroups that share a CU fall out of step by themselves.  Of 8
// waves the second four run half a step behind the first, with a barrier after each half: of
// the two waves on a SIMD one is in its products while the other is in its softmax; they
// convert their share of a block one step earlier in turn, so that it is there in time.
//
// Rows in LDS are 16-byte chunks whose index is XORed with row bits, so that 16 lanes of an
// access lie on the 16 different 16-byte groups of LDS's 256 bytes of banks, both for the
// writes (rows) and for the MFMA operands' reads (columns); by three row bits instead of four
// 43% of LDS's cycles were conflicts, and 2.88 ms were 2.63.  (16% are now, with
// threads that stage two neighbouring chunks, which took the 256-element kernel from 434 us to 404.)
//
// Measured: 4800 rows over 19721 tokens of 56 x 128 in 2.6 ms, 1040 TFLOP/s, 86% of what a
// large bf16 product reaches on the card; the power limit holds it there (1.93 GHz, 52% of
// MFMA issue).  56 heads of 2401 rows over lists of 100 blocks in 0.51 ms, 860 TFLOP/s.

// The place of chunk ch of a row of CH chunks (8: two rows share the banks).
template <int CH>
__device__ __forceinline__ int chunk_at(int row, int ch) {
    return CH == 8 ? ch ^ ((row >> 1) & 7) : ch ^ (row & 15);
}

constexpr int kSchedMfma = 0x8, kSchedLdsRead = 0x100;  // instruction classes of sched_group_barrier

template <int D, int W>
struct TileShape {
    static constexpr int kThreads = 64 * W;
    static constexpr int kRows = 32 * W;
    static constexpr int kKeyBytes = kKvBlock * D * 2;
    static constexpr int kLds = 4 * kKeyBytes;
    static constexpr int kGroups = W == 8 ? 2 : 1;
    // MFMAs that an operand is read ahead; 8 waves step together, and 4 there cost them 0.5%, 8 elsewhere gain nothing
    static constexpr int kAhead = W == 8 ? 8 : 4;
    static constexpr int kLoads = kKvBlock * D / 16 / kThreads;  // 16-byte pieces of K (and of V) a thread
};

// A block's keys (values) in 4 bits and their scales as buffers, which end behind the block: nothing is loaded of one that is not
// there (page < 0).  (By address 4800 rows over 19721 tokens take 2635 us, so 2650; 300 rows over 4000 tokens 47.3, so 46.2.)
struct FourPlace {
    __amdgpu_buffer_rsrc_t values, codes;
    __device__ __forceinline__ FourPlace(const uint8_t* v, const uint8_t* s, int heads, int h, int dim, int page) {
        const int64_t tile = static_cast<int64_t>(page < 0 ? 0 : page) * heads + h;
        values = span_bytes(v + tile * (kKvBlock * dim / 2), page < 0 ? 0 : kKvBlock * dim / 2);
        codes = span_bytes(s + tile * (kKvBlock * dim / kFourGroup), page < 0 ? 0 : kKvBlock * dim / kFourGroup);
    }
};

constexpr int kNonTemporal = 2;  // of a buffer load, as load_once (a query of 56 heads over 19721 tokens 34.3 us without, 30.4 so)

template <class T, int WAY>
__device__ __forceinline__ T load_from(__amdgpu_buffer_rsrc_t b, int at) {
    if constexpr (sizeof(T) == 16) return __builtin_bit_cast(T, __builtin_amdgcn_raw_buffer_load_b128(b, at, 0, WAY));
    else if constexpr (sizeof(T) == 8) return __builtin_bit_cast(T, __builtin_amdgcn_raw_buffer_load_b64(b, at, 0, WAY));
    else if constexpr (sizeof(T) == 4) return __builtin_amdgcn_raw_buffer_load_b32(b, at, 0, WAY);
    else if constexpr (sizeof(T) == 2) return __builtin_amdgcn_raw_buffer_load_b16(b, at, 0, WAY);
    else return __builtin_amdgcn_raw_buffer_load_b8(b, at, 0, WAY);
}
template <class T>
__device__ __forceinline__ T load_past(__amdgpu_buffer_rsrc_t b, int at) { return load_from<T, kNonTemporal>(b, at); }

// What a thread loads and stages of a block in 4 bits.  Keys: pieces of 16 elements of a token, half a group's, as in 8 bits.
// Values lie as they were written, token by token, and the second product wants runs of tokens: a thread takes 8 elements of
// 4 (2) neighbouring tokens, whose pairs of elements, converted (one instruction for two, exact), change places with a permute
// each and are 8 (4) bytes of 8 rows in LDS.
template <int D, int W>
struct FourTile {
    static constexpr int kThreads = 64 * W;
    static constexpr int kPieces = kKvBlock * D / 16 / kThreads;
    static constexpr int kEach = kKvBlock * D / kThreads;     // elements a thread
    static constexpr int kTok = kEach >= 32 ? 4 : 2, kUnits = kEach / (8 * kTok);

    struct Keys {
        uint2 w[kPieces];
        uint8_t code[kPieces];
        __device__ __forceinline__ void load(const KvCache4& c, int h, int page, int t) {
            const FourPlace p(c.k, c.ks, c.heads, h, D, page);
#pragma unroll
            for (int j = 0; j < kPieces; ++j) {
                const int piece = t + j * kThreads, line = piece / (D / 16), g = piece % (D / 16) / 2;
                w[j] = load_from<uint2, 0>(p.values, piece * 8);
                code[j] = load_from<uint8_t, 0>(p.codes, g * kKvBlock + line);
            }
        }
        __device__ __forceinline__ void stage(uint8_t* buf, int t) const {
            constexpr int CH = D / 8;
#pragma unroll
            for (int j = 0; j < kPieces; ++j) {
                const int piece = t + j * kThreads, line = piece / (CH / 2), ch = piece % (CH / 2) * 2;
                // token bits 2 and 3 change places, as in 8 bits
                const int row = (line & ~12) | ((line & 4) << 1) | ((line & 8) >> 1);
                uint8_t* const to_row = buf + row * (CH * 16);
                // (a NaN of every element: a factor of 2^128 is none, whatever is not 0 times it)
                const bool bad = code[j] >= kFourBad;
                const float f = four_scale(bad ? 255 : code[j]);
                const uint32_t some = bad ? 0x11111111u : 0u;
                *reinterpret_cast<uint4*>(to_row + chunk_at<CH>(row, ch) * 16) = four_bf16x8(w[j].x | some, f);
                *reinterpret_cast<uint4*>(to_row + chunk_at<CH>(row, ch + 1) * 16) = four_bf16x8(w[j].y | some, f);
            }
        }
    };

    // The place of chunk ch (8 tokens) of element `row` in LDS: two rows on the 256 bytes of banks, 16-byte chunks whose index is
    // XORed so that 16 lanes lie on different ones where they read neighbouring rows; where 32 (64) lanes write all tokens of
    // rows r and r + 8, bit 3 puts these on the two halves.
    static __device__ __forceinline__ uint32_t value_at(int row, int ch) {
        return (row >> 1) * 256 + (((((row & 1) << 3) | ch) ^ ((row >> 1) & 7) ^ (row & 8)) * 16);
    }

    struct Values {
        uint32_t w[kUnits][kTok], codes[kUnits];
        // A unit's 8 elements and its first token: all tokens of two neighbouring runs of elements, then of the next two.
        static __device__ __forceinline__ void place(uint32_t unit, uint32_t& ch, uint32_t& tok) {
            tok = (unit >> 1) % (kKvBlock / kTok) * kTok;
            ch = unit / (2 * kKvBlock / kTok) * 2 + (unit & 1);
        }
        __device__ __forceinline__ void load(const KvCache4& c, int h, int page, int t) {
            const FourPlace p(c.v, c.vs, c.heads, h, D, page);
#pragma unroll
            for (int j = 0; j < kUnits; ++j) {
                uint32_t ch, tok;
                place(t + j * kThreads, ch, tok);
#pragma unroll
                for (int x = 0; x < kTok; ++x) w[j][x] = load_from<uint32_t, 0>(p.values, (tok + x) * (D / 2) + ch * 4);
                codes[j] = load_from<std::conditional_t<kTok == 4, uint32_t, uint16_t>, 0>(p.codes, ch / 4 * kKvBlock + tok);
            }
        }
        __device__ __forceinline__ void stage(uint8_t* buf, int t, int* poison) {
#pragma unroll
            for (int j = 0; j < kUnits; ++j) {
                uint32_t ch, tok;
                place(t + j * kThreads, ch, tok);
                // value_at(8 ch + 2 e + z, tok / 8) = (to ^ (16 e + 128 z)) + 256 e, opaque, so that the loop does not keep eight
                uint32_t to = ch * 1024 + ((tok / 8) ^ (12 * (ch & 1))) * 16 + tok % 8 * 2;
                asm("" : "+v"(to));
                if (four_bad(codes[j])) {
#pragma unroll
                    for (int x = 0; x < kTok; ++x) {
                        if ((codes[j] >> (8 * x) & 255) < kFourBad) continue;
                        w[j][x] = 0;
                        codes[j] &= ~(255u << (8 * x));
                    }
                    *poison = 1;
                }
                float f[kTok];
#pragma unroll
                for (int x = 0; x < kTok; ++x) f[x] = four_scale(codes[j] >> (8 * x) & 255);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    uint32_t y[kTok];
#pragma unroll
                    for (int x = 0; x < kTok; ++x)
                        y[x] = e == 0 ? four_bf16<0>(w[j][x], f[x]) : e == 1 ? four_bf16<1>(w[j][x], f[x]) : e == 2 ? four_bf16<2>(w[j][x], f[x]) : four_bf16<3>(w[j][x], f[x]);
#pragma unroll
                    for (int z = 0; z < 2; ++z) {
                        const uint32_t sel = z ? 0x07060302u : 0x05040100u;
                        uint8_t* const p = buf + (to ^ (16 * e + 128 * z)) + 256 * e;
                        if constexpr (kTok == 4)
                            *reinterpret_cast<uint2*>(p) = make_uint2(__builtin_amdgcn_perm(y[1], y[0], sel), __builtin_amdgcn_perm(y[kTok - 1], y[kTok - 2], sel));
                        else
                            *reinterpret_cast<uint32_t*>(p) = __builtin_amdgcn_perm(y[1], y[0], sel);
                    }
                }
            }
        }
    };
};

// The items of a launch: tiles of the queries of a head, or (pack > 1) of the queries of all
// heads that share a kv head, in the order of rows, then heads.  The first `whole` take one
// workgroup each, a multiple of what the card holds at once; the rest, which would leave a
// last round part empty, are split over their blocks to fill it.
struct Items {
    int tiles, heads;  // of a head (or a kv head's group); heads (groups) of a sequence
    int pack, rows;    // query heads and queries of an item
    uint32_t per_pack; // ceil(2^32 / pack)
    int count, whole, chunk, rest_chunk;
    bool flat, last_first;
    int seqs;
    // Consecutive items on one XCD, whose L2 then holds their head's blocks.  flat (one round, every workgroup at once):
    // dealt out in order.
    __device__ __forceinline__ int of(int block, int tail_splits, int& split, int& splits) const {
        if (block < whole) {
            split = 0, splits = 1;
            return flat ? block : (block & 7) * chunk + (block >> 3);
        }
        const int x = flat ? block - whole : ((block - whole) & 7) * rest_chunk + ((block - whole) >> 3);
        splits = tail_splits;
        split = x % splits;
        return whole + x / splits;
    }
    // x / pack: x < 128 pack where pack > 1, so that x times what per_pack is over 2^32 / pack stays below 2^32 / pack for
    // pack <= kMaxPack.
    __device__ __forceinline__ int row_of(int x) const { return pack == 1 ? x : static_cast<int>(__umulhi(static_cast<uint32_t>(x), per_pack)); }
    // Of causal items those of a head's last rows, the longest, come first: first of all in a flat launch.  MIX: where items are
    // dealt out in runs those of a head's sequences are consecutive, not those of a sequence's heads, so that the XCDs' shares are
    // alike however uneven the sequences are (over 4 bits 8 of 1176 rows and up to 10228 tokens 1800 -> 1086 us, 16 of 2560 rows over
    // themselves of 256 elements 2122 -> 1514; over 8 bits it was not tried).
    template <bool MIX>
    __device__ __forceinline__ void place(int item, int& seq, int& head, int& tile) const {
        const int all = count / tiles, nh = flat ? item % all : item / tiles;
        tile = flat ? item / all : item % tiles;
        if (last_first) tile = tiles - 1 - tile;
        if (MIX && !flat) {
            seq = nh % seqs;
            head = nh / seqs;
        } else {
            seq = nh / heads;
            head = nh % heads;
        }
    }
};

// (64 elements leave registers, 164 of 168, and LDS for three workgroups a CU: 4800 x 19200 831 us with two, 680 so.)
template <class C, int D, int W>
__global__ __launch_bounds__(64 * W, D == 256 ? 1 : D == 64 ? 3 : 2) void kv_tile_kernel(Queries q, C c, KvSeqs s, float scale, int causal,
                                                                          Lists list, uint16_t* __restrict__ out, Partial part,
                                                                          Items items) {
    using T = TileShape<D, W>;
    constexpr bool kFour = std::is_same_v<C, KvCache4>;
    constexpr bool kFar = kFour && D == 256;
    constexpr int NT = D / 32;            // tiles of 32 elements of the output
    constexpr int KC = D / 8, VC = 8;     // 16-byte chunks of a row of K, of V
    extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
    __shared__ int2 entry[T::kThreads + 3];  // (page, block) of the blocks at hand
    __shared__ Factors fact[kFour ? 1 : T::kThreads + 1];
    __shared__ int wcount[W];
    __shared__ int poison;  // kFour: a value's scale stands for no number

    int split, splits;
    const int item = items.of(blockIdx.x, part.splits, split, splits);
    if (item >= items.count) return;
    int i, head, tile;
    items.place<kFour>(item, i, head, tile);
    const int h = head * items.pack / (q.heads / c.heads);
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6, col = lane & 31, half = lane >> 5;

    const int len = s.len(i), count = s.count(i, q.rows), start = s.end(i) - count, queries = count * items.pack;
    // this lane's query, its row and its head
    const int r0 = tile * T::kRows, w0 = r0 + wave * 32, query = w0 + col;
    const int row = items.row_of(query), hq = head * items.pack + query - row * items.pack;
    // the last token that this lane's query, the wave's last and the workgroup's last see
    auto last_of = [&](int x) {
        const int y = start + items.row_of(x), most = causal && y < len - 1 ? y : len - 1;
        return x < queries ? most : -1;
    };
    const int last = last_of(query);
    const int wave_query = w0 + 31 < queries ? w0 + 31 : queries - 1;
    const int wave_last = wave_query >= w0 ? last_of(wave_query) : -1;
    const int tile_query = r0 + T::kRows - 1 < queries ? r0 + T::kRows - 1 : queries - 1;
    const int tile_last = tile_query >= r0 ? last_of(tile_query) : -1;
    // below this every query of the wave that is one sees a whole block
    const int wave_full = wave_last >= 0 ? last_of(w0) + 1 : 0;
    const int blocks = tile_last < 0 ? 0 : block_of(tile_last) + 1;

    bf16x8 qf[D / 16];
    {
        const int64_t at = i * q.bs + static_cast<int64_t>(row) * q.ld + static_cast<int64_t>(hq) * D + half * 8;
#pragma unroll
        for (int k = 0; k < D / 16; ++k)
            qf[k] = last >= 0 ? query_frag(q.p + at + k * 16, scale) : frag(make_uint4(0, 0, 0, 0));
    }
    f32x16 o[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[n][r] = 0.0f;
    float m = kLowest, l = 0.0f;

    const int32_t* const mine =
        list.p ? list.p + ((static_cast<int64_t>(i) * list.tiles + items.row_of(r0) / kKvTile) * c.heads + h) * list.top : nullptr;
    const int total = blocks == 0 ? 0 : mine ? list.top : blocks;
    // an even share: total < 2^25, splits <= 64
    const uint32_t share = static_cast<uint32_t>(total), of = static_cast<uint32_t>(splits);
    const int from = splits == 1 ? 0 : static_cast<int>(share * split / of);
    const int to = splits == 1 ? total : static_cast<int>(share * (split + 1) / of);

    // Bytes of a block into registers, and as bf16 into LDS: 8 of them a chunk.
    using Four = FourTile<D, W>;
    std::conditional_t<kFour, typename Four::Keys, uint4[T::kLoads]> kr;
    std::conditional_t<kFour, typename Four::Values, uint4[T::kLoads]> vr;
    if (kFour && t == 0) poison = 0;  // (barriers follow before it is set)
    auto load = [&](const auto* from_pages, int page, auto& to_regs) __attribute__((always_inline)) {
        if constexpr (kFour) {
            to_regs.load(c, h, page, t);
        } else {
            const int8_t* const at = from_pages + (static_cast<int64_t>(page) * c.heads + h) * (kKvBlock * D);  // uniform
#pragma unroll
            for (int j = 0; j < T::kLoads; ++j) to_regs[j] = *reinterpret_cast<const uint4*>(at + static_cast<uint32_t>(t + j * T::kThreads) * 16);
        }
    };
    auto stage = [&](uint8_t* buf, const auto& regs, auto chunks, auto swap) __attribute__((always_inline)) {
        constexpr int CH = chunks;
#pragma unroll
        for (int j = 0; j < T::kLoads; ++j) {
            const int piece = t + j * T::kThreads, line = piece / (CH / 2), ch = piece % (CH / 2) * 2;
            // token bits 2 and 3 change places: an MFMA row's registers are then runs of 8 tokens
            const int row = swap ? (line & ~12) | ((line & 4) << 1) | ((line & 8) >> 1) : line;
            uint8_t* const to_row = buf + row * (CH * 16);
            *reinterpret_cast<uint4*>(to_row + chunk_at<CH>(row, ch) * 16) = ints_bf16(make_uint2(regs[j].x, regs[j].y));
            *reinterpret_cast<uint4*>(to_row + chunk_at<CH>(row, ch + 1) * 16) = ints_bf16(make_uint2(regs[j].z, regs[j].w));
        }
    };
    auto stage_k = [&](int which) __attribute__((always_inline)) {
        if constexpr (kFour) kr.stage(smem + (which & 1) * T::kKeyBytes, t);
        else stage(smem + (which & 1) * T::kKeyBytes, kr, std::integral_constant<int, KC>{}, std::true_type{});
    };
    auto stage_v = [&](int which) __attribute__((always_inline)) {
        if constexpr (kFour) vr.stage(smem + (2 + (which & 1)) * T::kKeyBytes, t, &poison);
        else stage(smem + (2 + (which & 1)) * T::kKeyBytes, vr, std::integral_constant<int, VC>{}, std::false_type{});
    };
    auto arrive = [&]() __attribute__((always_inline)) {
        wait_lgkm0();
        __builtin_amdgcn_sched_barrier(0);
        wg_barrier();
        __builtin_amdgcn_sched_barrier(0);
    };
    // A wave without a query that sees anything converts its share of the blocks and no more.  (Not among 8 waves of 128
    // elements, whose registers the branch would overflow: 2000 rows 139 -> 158 us; of 256 it made 404 us 354.)
    const bool working = (W == 8 && D == 128) || uniform(wave_last) >= 0;
    const int behind = T::kGroups == 2 && __builtin_amdgcn_readfirstlane(wave) >= W / 2;

    for (int x0 = from; x0 < to; x0 += T::kThreads) {
        // the pages and factors of the next kThreads blocks, those that are not there left out
        __syncthreads();
        {
            const int x = x0 + t;
            const int b = x < to ? (mine ? mine[x] : x) : -1;
            const int page = b >= 0 && b < blocks ? s.page(i, b, c.pages) : -1;
            const uint64_t got = __ballot(page >= 0);
            if (lane == 0) wcount[wave] = __popcll(got);
            __syncthreads();
            int at = __popcll(got & ((uint64_t{1} << lane) - 1));
            for (int w = 0; w < wave; ++w) at += wcount[w];
            if (page >= 0) {
                entry[at] = make_int2(page, b);
                if constexpr (!kFour) {
                    const int64_t p = static_cast<int64_t>(page) * c.heads + h;
                    fact[at] = factors(c.ks[p], c.vs[p], scale * kLog2e);
                }
            }
        }
        __syncthreads();
        int n = 0;
#pragma unroll
        for (int w = 0; w < W; ++w) n += wcount[w];
        if (n == 0) continue;
        load(c.k, uniform(entry[0].x), kr);
        stage_k(0);
        arrive();
        if (behind) {
            load(c.v, uniform(entry[0].x), vr);
            if (n > 1) {
                load(c.k, uniform(entry[1].x), kr);
                stage_k(1);
            }
            stage_v(0);
            arrive();
        }
        // What a step needs to know of its blocks is read a step ahead: the pages that it loads, and its own block and factors.
        int page_k = uniform(entry[1 + behind].x), page_v = uniform(entry[behind].x), base = uniform(entry[0].y) * kKvBlock;
        // (4 bits: the same for all)
        Factors f = kFour ? factors(1.0f, 1.0f, scale * kLog2e) : fact[0];
        if constexpr (!kFour) f = {uniform(f.c), uniform(f.lv), uniform(f.iv), uniform(f.vs)};
        // Step y's halves.  The products take their operands from LDS kAhead MFMAs ahead.
        bf16x8 p[4];
        f32x16 sc[2];
        auto products = [&](int y, auto keys, auto values) __attribute__((always_inline)) {
            constexpr int NK = keys ? D / 8 : 0, N = NK + (values ? 4 * NT : 0);
            const uint8_t* const kb = smem + (y & 1) * T::kKeyBytes;
            const uint8_t* const vb = smem + (3 - (y & 1)) * T::kKeyBytes;
            // At 64 and 256 elements a row's chunk 2 k + half is found from chunk `half` by an XOR, opaque, so that the loop
            // does not keep a register for every k (256: 1200 rows over 9000 tokens 458 -> 434 us; 64, 500 rows: 23.7 -> 22.0;
            // at 128, where they fit, the XORs took 2000 rows from 137 to 142 us).
            uint32_t kx = col * (D * 2) + chunk_at<KC>(col, half) * 16, vx = kFour ? Four::value_at(col, half) : col * (kKvBlock * 2) + chunk_at<VC>(col, half) * 16;
            if constexpr (D != 128) asm("" : "+v"(kx), "+v"(vx));
            auto fetch = [&](int x) __attribute__((always_inline)) {
                if (x < NK) {
                    const int row = x % 2 * 32 + col;
                    const uint32_t at = D != 128 ? (kx ^ (x / 2 * 32)) + x % 2 * (32 * D * 2) : row * (D * 2) + chunk_at<KC>(row, x / 2 * 2 + half) * 16;
                    return frag(*reinterpret_cast<const uint4*>(kb + at));
                }
                const int d = (x - NK) % NT, w = (x - NK) / NT, row = d * 32 + col;
                if constexpr (kFour) {
                    const uint32_t at = D != 128 ? (vx ^ (w * 32)) + d * (32 * kKvBlock * 2) : Four::value_at(row, 2 * w + half);
                    return frag(*reinterpret_cast<const uint4*>(vb + at));
                }
                const uint32_t at = D != 128 ? (vx ^ (w * 32)) + d * (32 * kKvBlock * 2) : row * (kKvBlock * 2) + chunk_at<VC>(row, 2 * w + half) * 16;
                return frag(*reinterpret_cast<const uint4*>(vb + at));
            };
            bf16x8 a[T::kAhead];
#pragma unroll
            for (int x = 0; x < T::kAhead; ++x) a[x] = fetch(x);
            if constexpr (NK > 0) {
#pragma unroll
                for (int r = 0; r < 16; ++r) sc[0][r] = sc[1][r] = 0.0f;
            }
#pragma unroll
            for (int x = 0; x < N; ++x) {
                if (x < NK)
                    sc[x % 2] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[x % T::kAhead], qf[x / 2], sc[x % 2], 0, 0, 0);
                else
                    o[(x - NK) % NT] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[x % T::kAhead], p[(x - NK) / NT], o[(x - NK) % NT], 0, 0, 0);
                if (x + T::kAhead < N) a[x % T::kAhead] = fetch(x + T::kAhead);
            }
            __builtin_amdgcn_sched_group_barrier(kSchedLdsRead, T::kAhead, 0);
#pragma unroll
            for (int x = 0; x < N; ++x) {
                __builtin_amdgcn_sched_group_barrier(kSchedMfma, 1, 0);
                if (x + T::kAhead < N) __builtin_amdgcn_sched_group_barrier(kSchedLdsRead, 1, 0);
            }
        };
        auto softmax = [&]() __attribute__((always_inline)) {
            // register r of sc[u]: token base + 32 u + 16 (r / 8) + 8 half + r % 8
            if (base + kKvBlock > wave_full) {
#pragma unroll
                for (int u = 0; u < 2; ++u)
#pragma unroll
                    for (int r = 0; r < 16; ++r)
                        if (base + 32 * u + 16 * (r / 8) + 8 * half + r % 8 > last) sc[u][r] = -__builtin_inff();
            }
            float best = -__builtin_inff();
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int r = 0; r < 16; ++r) best = fmaxf(best, sc[u][r]);
            best = max_halves(best) * f.c;
            if (__any(best > m + kSlack)) {
                const float mn = fmaxf(m, best), fix = exp2_hw(m - mn);
                m = mn;
                l *= fix;
#pragma unroll
                for (int d = 0; d < NT; ++d)
#pragma unroll
                    for (int r = 0; r < 16; ++r) o[d][r] *= fix;
            }
            const float off = kFour ? -m : f.lv - m;
            if (kFour || f.iv != 0.0f) {
                float sum = 0.0f;
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                    float x[8];
#pragma unroll
                    for (int r = 0; r < 8; ++r) {
                        x[r] = exp2_hw(__builtin_fmaf(sc[w / 2][w % 2 * 8 + r], f.c, off));
                        sum += x[r];
                    }
                    p[w] = pack(x);
                }
                l = kFour ? l + sum : __builtin_fmaf(sum, f.iv, l);
            } else {
                // a scale that is no ordinary number: what a row does not see must not reach it, and a NaN or an infinity
                // must where a probability underflows
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                    float x[8];
#pragma unroll
                    for (int r = 0; r < 8; ++r) {
                        const uint32_t sees = (base + 16 * w + 8 * half + r - 1 - last) >> 31;  // all bits, or none
                        x[r] = __uint_as_float(__float_as_uint(exp2_hw(__builtin_fmaf(sc[w / 2][w % 2 * 8 + r], f.c, off))) & sees);
                        l += x[r];
                        x[r] = __uint_as_float(__float_as_uint(x[r] * f.vs) & sees);
                    }
                    p[w] = pack(x);
                }
            }
        };
        auto step = [&](int y, auto values) __attribute__((always_inline)) {
            const int next_k = y + 1 + behind, next_v = y + behind;
            if (next_k < n) load(c.k, page_k, kr);
            if (next_v < n) load(c.v, page_v, vr);
            // (past the last block: whatever the arrays hold, which is then not used)
            const int2 after = entry[next_k + 1];
            const int block = entry[y + 1].y;
            const Factors next = kFour ? f : fact[y + 1];
            if (working) {
                __builtin_amdgcn_s_setprio(1);
                products(y, std::true_type{}, values);
                __builtin_amdgcn_s_setprio(0);
            }
            if constexpr (T::kGroups == 2) arrive();
            if (working) softmax();
            if (next_k < n) stage_k(next_k);
            if (next_v < n) stage_v(next_v);
            page_v = page_k;
            page_k = uniform(after.x);
            base = uniform(block) * kKvBlock;
            if constexpr (!kFour) f = {uniform(next.c), uniform(next.lv), uniform(next.iv), uniform(next.vs)};
            arrive();
        };
        if constexpr (kFar) {
            // One wave a SIMD, with registers to spare: the bytes of block y + 2 (values: y + 1) are asked for in step y, into one of
            // two sets.  Every load is issued, of nothing behind the last block, so that the wait for one does not have to be
            // for those after it.  (1000 rows of 20 heads over 4000 tokens 190 us a step later, 182 so; of 128 elements, where two
            // waves are on a SIMD, prompts of 512 rows 22.5 and 23.0.)
            typename Four::Keys k1;
            typename Four::Values v1;
            page_k = n > 2 ? uniform(entry[2].x) : -1, page_v = n > 1 ? uniform(entry[1].x) : -1;
            load(c.k, page_v, kr);
            load(c.v, uniform(entry[0].x), vr);
            auto far_step = [&](int y, auto values, auto& k_to, auto& v_to, auto& k_from, auto& v_from) __attribute__((always_inline)) {
                load(c.k, page_k, k_to);
                load(c.v, page_v, v_to);
                const int2 after = entry[y + 3];
                const int block = entry[y + 1].y;
                if (working) {
                    __builtin_amdgcn_s_setprio(1);
                    products(y, std::true_type{}, values);
                    __builtin_amdgcn_s_setprio(0);
                    softmax();
                }
                if (y + 1 < n) k_from.stage(smem + ((y + 1) & 1) * T::kKeyBytes, t);
                v_from.stage(smem + (2 + (y & 1)) * T::kKeyBytes, t, &poison);
                page_v = page_k;
                page_k = y + 3 < n ? uniform(after.x) : -1;
                base = uniform(block) * kKvBlock;
                arrive();
            };
            far_step(0, std::false_type{}, k1, v1, kr, vr);
            for (int y = 1; y < n;) {
                far_step(y, std::true_type{}, kr, vr, k1, v1);
                if (++y >= n) break;
                far_step(y, std::true_type{}, k1, v1, kr, vr);
                ++y;
            }
        } else {
            step(0, std::false_type{});
            for (int y = 1; y < n; ++y) step(y, std::true_type{});
        }
        if (working) products(n, std::false_type{}, std::true_type{});
        if (T::kGroups == 2 && !behind) arrive();
    }

    // 4 bits: the values of a token whose scale stands for no number went in as zeros; they make NaNs of their elements,
    // 32 of the output, in the rows that see the token.  Its blocks are looked through again, in a launch that met one.
    if constexpr (kFour) {
        if (poison) {
            for (int x = from; x < to; ++x) {
                const int b = mine ? mine[x] : x;
                const int page = b >= 0 && b < blocks ? s.page(i, b, c.pages) : -1;
                if (page < 0) continue;
                const uint8_t* const codes = c.vs + (static_cast<int64_t>(page) * c.heads + h) * (NT * kKvBlock);
#pragma unroll
                for (int d = 0; d < NT; ++d) {
                    bool hit = false;
#pragma unroll 1
                    for (int x2 = 0; x2 < kKvBlock; ++x2) hit |= codes[d * kKvBlock + x2] >= kFourBad && b * kKvBlock + x2 <= last;
#pragma unroll
                    for (int r = 0; r < 16; ++r) o[d][r] = hit ? __builtin_nanf("") : o[d][r];
                }
            }
        }
    }

    l += __shfl_xor(l, 32);
    if (row >= q.rows) return;
    if (last < 0) {  // padding, or a row that sees nothing: what the registers hold is no result
        l = 0.0f;
#pragma unroll
        for (int d = 0; d < NT; ++d)
#pragma unroll
            for (int r = 0; r < 16; ++r) o[d][r] = 0.0f;
    }
    const int64_t to_row = (static_cast<int64_t>(i) * q.rows + row) * q.heads + hq;
    // register r of o[d]: element 32 d + 8 (r / 4) + 4 half + r % 4 of the query's output
    if (splits > 1) {
        const int64_t at = part.at(item - items.whole, split, query - r0);
        if (half == 0) part.ml[at] = make_float2(m, l);
        if (from >= to) return;
#pragma unroll
        for (int d = 0; d < NT; ++d)
#pragma unroll
            for (int g = 0; g < 4; ++g)
                *reinterpret_cast<float4*>(part.o + at * D + 32 * d + 8 * g + 4 * half) =
                    make_float4(o[d][4 * g], o[d][4 * g + 1], o[d][4 * g + 2], o[d][4 * g + 3]);
        return;
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
    for (int d = 0; d < NT; ++d)
#pragma unroll
        for (int g = 0; g < 4; ++g)
            *reinterpret_cast<uint2*>(out + to_row * D + 32 * d + 8 * g + 4 * half) =
                make_uint2(bf16x2_bits(o[d][4 * g] * inv, o[d][4 * g + 1] * inv), bf16x2_bits(o[d][4 * g + 2] * inv, o[d][4 * g + 3] * inv));
}

// ------------------------------------------------------------------ few queries

// A load of what no other workgroup reads, past the caches: 537 MB of cache in 87 us against 99.
__device__ __forceinline__ uint4 load_once(const int8_t* p) {
    return __builtin_bit_cast(uint4, __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(p)));
}

// LDS operations of a wave are done in order: what the compiler may not change here.
__device__ __forceinline__ void wave_order() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_wave_barrier();
    asm volatile("" ::: "memory");
}

// What a lane (column col, lanes 16 quad ..) loads of a block in 4 bits, and the operands that it makes of them.  Of the keys,
// rows of the first product's MFMAs: column 4 q + r has token 16 u + 4 r + q for MFMA set u, of it a quarter of each 128
// elements (of 64), one scale each (half of one).  So a query's probabilities of tokens 16 u + 4 r + quad are in a lane, and of
// the values it takes these, D / 16 neighbouring elements each, whose pairs change places by a permute; MFMA e takes element e
// of each lane's.  Each load's lanes then lie on whole cache lines, which no other load touches (but keys of 256 elements):
// where two did, the second waited in the L1 for the first's line (43% of cycles).  Scales are loaded once a wave, in order, and
// go through LDS to the lanes that want them.  A query of 56 heads over 19721 tokens (150 MB) 33.2 us with neighbouring tokens
// in a lane, 30.4 so, the join's 4.6 among them; 16 sequences of up to 32768 tokens of 8 heads, one draw of lengths, 58.9 and
// 53.2 (eight draws, 244593 to 380465 tokens, 266 to 414 MB: 53 to 73 us, 5.0 to 5.7 TB/s).
template <int D>
struct FourFew {
    static constexpr int kRun = D >= 128 ? 32 : 16;       // neighbouring elements of a key
    static constexpr int kRuns = D / (4 * kRun);
    static constexpr int kWords = kRun / 8;               // words of a run
    static constexpr int kWide = D / 16;                  // neighbouring elements of a value
    static constexpr int kBytes = kWide / 2;
    static constexpr int kCodes = D / kFourGroup * kKvBlock / 4;  // words of a block's scales

    // A wave's place in LDS for the scales of a block's keys and of its values.
    struct Scratch {
        uint32_t k[kCodes], v[kCodes];
    };

    // first of the 8 elements of first-product operand k
    static __device__ __forceinline__ int element(int quad, int k) { return k / kWords * (4 * kRun) + quad * kRun + k % kWords * 8; }
    // the element of register r of output tile e
    static __device__ __forceinline__ int out_element(int quad, int r, int e) { return kWide * (4 * quad + r) + e; }

    // Byte q of a word of scale codes where a factor's exponent is; what else is in it a conversion does not read.
    static __device__ __forceinline__ float factor(uint32_t word, int q) {
        return __uint_as_float(__builtin_amdgcn_alignbit(word, word, 8 * q + 9));
    }
    static __device__ __forceinline__ bool bad(uint32_t word, int q) { return (word >> (8 * q) & 255) >= kFourBad; }

    // A block's scale codes, a word (two) a lane.
    struct Codes {
        static constexpr int N = kCodes > 64 ? kCodes / 64 : 1;
        uint32_t w[N];
        __device__ __forceinline__ void load(__amdgpu_buffer_rsrc_t b, int lane) {
#pragma unroll
            for (int n = 0; n < N; ++n) w[n] = load_past<uint32_t>(b, (n * 64 + lane) * 4);
        }
        // Into LDS; whether any of them stands for no number.
        __device__ __forceinline__ bool put(uint32_t* to, int lane) const {
            bool any = false;
            wave_order();
#pragma unroll
            for (int n = 0; n < N; ++n) {
                if (kCodes >= 64 || lane < kCodes) to[n * 64 + lane] = w[n];
                any |= four_bad(w[n]);
            }
            wave_order();
            return __any(any);
        }
    };

    struct Keys {
        uint32_t w[4][kRuns * kWords], c[kRuns][4];
        Codes codes;
        __device__ __forceinline__ void load(const KvCache4& cache, int h, int page, int col, int quad) {
            const FourPlace p(cache.k, cache.ks, cache.heads, h, D, page);
            codes.load(p.codes, 16 * quad + col);
            const int tok = 4 * (col & 3) + (col >> 2);
#pragma unroll
            for (int u = 0; u < 4; ++u)
#pragma unroll
                for (int n = 0; n < kRuns; ++n) {
                    const int at = (16 * u + tok) * (D / 2) + element(quad, n * kWords) / 2;
                    if constexpr (kWords == 4) {
                        const uint4 x = load_past<uint4>(p.values, at);
                        w[u][4 * n] = x.x, w[u][4 * n + 1] = x.y, w[u][4 * n + 2] = x.z, w[u][4 * n + 3] = x.w;
                    } else {
                        const uint2 x = load_past<uint2>(p.values, at);
                        w[u][2 * n] = x.x, w[u][2 * n + 1] = x.y;
                    }
                }
        }
        // The scales; NaNs of every element where one stands for no number: a factor of 2^128 is none, whatever is not 0 times it.
        __device__ __forceinline__ void ready(Scratch& scratch, int col, int quad) {
            const bool any = codes.put(scratch.k, 16 * quad + col);
#pragma unroll
            for (int n = 0; n < kRuns; ++n)
#pragma unroll
                for (int u = 0; u < 4; ++u)
                    c[n][u] = scratch.k[element(quad, n * kWords) / kFourGroup * (kKvBlock / 4) + 4 * u + (col & 3)];
            if (!any) return;
#pragma unroll
            for (int n = 0; n < kRuns; ++n)
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    if (!bad(c[n][u], col >> 2)) continue;
                    c[n][u] = ~0u;
#pragma unroll
                    for (int k = 0; k < kWords; ++k) w[u][n * kWords + k] |= 0x11111111u;
                }
        }
        __device__ __forceinline__ bf16x8 operand(int u, int k, int col) const {
            return frag(four_bf16x8(w[u][k], factor(c[k / kWords][u], col >> 2)));
        }
    };

    struct Values {
        static constexpr int N = kBytes < 4 ? 1 : kBytes / 4;
        uint32_t w[16][N], c[16];
        Codes codes;
        __device__ __forceinline__ void load(const KvCache4& cache, int h, int page, int col, int quad) {
            const FourPlace p(cache.v, cache.vs, cache.heads, h, D, page);
            codes.load(p.codes, 16 * quad + col);
            const int at = quad * (D / 2) + col * kBytes;
#pragma unroll
            for (int x = 0; x < 16; ++x) {
                if constexpr (kBytes == 2) {
                    w[x][0] = load_past<uint16_t>(p.values, at + x * (4 * D / 2));
                } else if constexpr (kBytes == 4) {
                    w[x][0] = load_past<uint32_t>(p.values, at + x * (4 * D / 2));
                } else {
                    const uint2 y = load_past<uint2>(p.values, at + x * (4 * D / 2));
                    w[x][0] = y.x, w[x][N - 1] = y.y;
                }
            }
        }
        // The scales; zeros for the values of tokens whose scale stands for no number; whether the block has any.
        __device__ __forceinline__ bool ready(Scratch& scratch, int col, int quad) {
            const bool any = codes.put(scratch.v, 16 * quad + col);
#pragma unroll
            for (int x = 0; x < 16; x += 4) {
                const uint4 y = *reinterpret_cast<const uint4*>(&scratch.v[kWide * col / kFourGroup * (kKvBlock / 4) + x]);
                c[x] = y.x, c[x + 1] = y.y, c[x + 2] = y.z, c[x + 3] = y.w;
            }
            if (!any) return false;
#pragma unroll
            for (int x = 0; x < 16; ++x) {
                if (!bad(c[x], quad)) continue;
                c[x] = 0;
#pragma unroll
                for (int n = 0; n < N; ++n) w[x][n] = 0;
            }
            return true;
        }
        // The second product's operands of elements 2 e and 2 e + 1 (a[0], a[1]) with each half of the tokens' probabilities.
        __device__ __forceinline__ void operands(int e, int quad, bf16x8 (&a)[2][2]) const {
            uint32_t y[16];
#pragma unroll
            for (int x = 0; x < 16; ++x) {
                const float f = factor(c[x], quad);
                const uint32_t v = w[x][e / 4];
                y[x] = e % 4 == 0 ? four_bf16<0>(v, f) : e % 4 == 1 ? four_bf16<1>(v, f) : e % 4 == 2 ? four_bf16<2>(v, f) : four_bf16<3>(v, f);
            }
#pragma unroll
            for (int z = 0; z < 2; ++z) {
                const uint32_t sel = z ? 0x07060302u : 0x05040100u;
#pragma unroll
                for (int h = 0; h < 2; ++h)
                    a[z][h] = frag(make_uint4(__builtin_amdgcn_perm(y[8 * h + 1], y[8 * h], sel), __builtin_amdgcn_perm(y[8 * h + 3], y[8 * h + 2], sel),
                                              __builtin_amdgcn_perm(y[8 * h + 5], y[8 * h + 4], sel), __builtin_amdgcn_perm(y[8 * h + 7], y[8 * h + 6], sel)));
            }
        }
    };
};

constexpr int kFew = 16;  // queries: the columns of a 16x16 MFMA
constexpr int kFewWaves = 4;
constexpr int kFewThreads = 64 * kFewWaves;

// How a launch's workgroups share the blocks of all sequences of a kv head, laid end to end: even shares, whatever the
// sequences' lengths, `shares` for each kv head (0: a workgroup a sequence and kv head).  A piece, what a share has of one
// sequence, leaves partial sums: sequence i's piece of share w is piece w + i, as from one piece to the next either the
// share or the sequence is another.  spans[i]: the first and the last share with blocks of sequence i.
struct Shares {
    int shares;
    int2* spans;
};

// A workgroup: up to 16 NQ queries of one kv head's group, one share of the blocks.  Its
// waves take whole blocks in turn, straight from memory into the operands' registers (no
// LDS, no barrier; a block's bytes are converted once for all queries), and are joined once
// for each sequence.  HBM bounds it: a query of 56 heads over 19721 tokens takes 50 us, 5.7 TB/s, 17
// to 32 rows of 8 x 56 heads over 4000 tokens 87 us, where the 40 that go by tiles, 16 KB a
// workgroup at a time, take 129; 16 sequences of 1 to 32768 tokens of 8 heads (780 MB) 128, where
// shares of their own for each, a quarter of the longest, took 146.  Without shares (plan_of) a
// workgroup reads a whole sequence, and the launch takes as long as the longest.
// Workgroups of a CU that registers are kept for: left to itself the compiler schedules 16 queries over 4 bits a little worse
// (a query of 56 heads over 19721 tokens 31.1 us, 30.4 so; registers for three spill, 48).
template <class C, int D, int NQ>
constexpr int few_groups() {
    return std::is_same_v<C, KvCache4> && NQ == 1 && D < 256 ? 2 : 1;
}

template <class C, int D, int NQ>
__global__ __launch_bounds__(64 * kFewWaves, (few_groups<C, D, NQ>())) void kv_few_kernel(Queries q, C c, KvSeqs s, float scale, int causal, Lists list,
                                                                uint16_t* __restrict__ out, Partial part, Shares shares) {
    constexpr bool kFour = std::is_same_v<C, KvCache4>;
    using Four = FourFew<D>;
    constexpr int KL = D / 64;   // 16-byte pieces of a key row a lane
    constexpr int NT = D / 16;   // tiles of 16 elements of the output
    __shared__ float jo[kFewWaves][kFew][D + 4];
    __shared__ float2 jml[kFewWaves][kFew];
    __shared__ __attribute__((aligned(16))) std::conditional_t<kFour, typename Four::Scratch, int> scratch[kFewWaves];
    __shared__ int ends[kFewThreads + 1];  // blocks of the sequences up to each
    __shared__ int wave_sum[kFewWaves];

    const int h = blockIdx.x % c.heads, w = blockIdx.x / c.heads;
    const int group = q.heads / c.heads, queries = q.rows * group;
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6, col = lane & 15, quad = lane >> 4;

    // what sequence i's queries see: tokens, its first row's token and its rows
    struct Seen {
        int len, start, count;
        __device__ __forceinline__ int last_of(int r, int causal) const {
            int x = len - 1;
            if (causal && start + r < x) x = start + r;
            return r < count ? x : -1;
        }
    };
    __shared__ Seen seen[kFewThreads];
    auto seen_of = [&](int i) {
        const int count = s.count(i, q.rows);
        return Seen{s.len(i), s.end(i) - count, count};
    };
    auto blocks_of = [&](const Seen& n) {
        const int most = n.count > 0 ? n.last_of(n.count - 1, causal) : -1;
        return most < 0 ? 0 : block_of(most) + 1;
    };
    int i = w, at = 0, share_end = 0;
    if (shares.shares) {
        Seen mine = {};
        if (t < s.n) mine = seen_of(t);
        seen[t] = mine;
        int sum = blocks_of(mine);
        if (sum > 0 && list.p) sum = list.top;
        const int own = sum;
        for (int x = 1; x < 64 && x < s.n; x <<= 1) {
            const int o = __shfl_up(sum, x);
            if (lane >= x) sum += o;
        }
        if (s.n > 64) {
            if (lane == 63) wave_sum[wave] = sum;
            __syncthreads();
            for (int x = 0; x < wave; ++x) sum += wave_sum[x];
        }
        if (t < s.n) ends[t + 1] = sum;
        if (t == 0) ends[0] = 0;
        __syncthreads();
        const int all = uniform(ends[s.n]);
        const int per = all == 0 ? 1 : static_cast<int>((static_cast<uint32_t>(all) + shares.shares - 1) / shares.shares);
        if (blockIdx.x == 0 && t < s.n)
            shares.spans[t] = own == 0 ? make_int2(0, -1) : make_int2((sum - own) / per, (sum - 1) / per);
        at = uniform(w * per);
        share_end = uniform(at + per < all ? at + per : all);
        if (at >= all) return;
        // the sequence of the share's first block
        for (int x = 0; x < s.n; x += 64) {
            const uint64_t past = __ballot(x + lane < s.n && ends[x + lane + 1] > at);
            if (past) {
                i = x + __builtin_ctzll(past);
                break;
            }
        }
    }

    for (bool again = false;; again = true) {
        Seen seq;
        if (shares.shares) {
            const Seen x = seen[i];
            seq = {uniform(x.len), uniform(x.start), uniform(x.count)};
        } else {
            seq = seen_of(i);
        }
        const int blocks = blocks_of(seq);
        // below this every query that is one sees a whole block
        const int full = seq.count > 0 ? seq.last_of(0, causal) + 1 : 0;
        // query 16 g + col of each set g
        int last[NQ];
        bf16x8 qf[NQ][2 * KL];
        f32x4 o[NQ][NT];
        float m[NQ], l[NQ];
#pragma unroll
        for (int g = 0; g < NQ; ++g) {
            const int query = g * kFew + col, row = query / group, hq = h * group + query % group;
            last[g] = query < queries ? seq.last_of(row, causal) : -1;
            const int64_t to_q = i * q.bs + static_cast<int64_t>(row) * q.ld + static_cast<int64_t>(hq) * D + quad * 16;
#pragma unroll
            for (int k = 0; k < 2 * KL; ++k)
                qf[g][k] = last[g] < 0 ? frag(make_uint4(0, 0, 0, 0))
                           : kFour     ? query_frag(q.p + to_q - quad * 16 + Four::element(quad, k), scale)
                                       : query_frag(q.p + to_q + (k >> 1) * 64 + (k & 1) * 8, scale);
#pragma unroll
            for (int n = 0; n < NT; ++n) o[g][n] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
            m[g] = kLowest, l[g] = 0.0f;
        }

        const int32_t* const mine = list.p ? list.p + (static_cast<int64_t>(i) * list.tiles * c.heads + h) * list.top : nullptr;
        const int total = blocks == 0 ? 0 : mine ? list.top : blocks;
        int from = 0, to = total;
        if (shares.shares) {
            const int begin = uniform(ends[i]), last_end = uniform(ends[i + 1]), end = last_end < share_end ? last_end : share_end;
            from = at - begin, to = end - begin;
            at = end;
        }

        std::conditional_t<kFour, typename Four::Keys, uint4[4][KL]> kr;
        std::conditional_t<kFour, typename Four::Values, uint4[NT]> vr;
        bool poison = false;  // kFour: a value's scale stands for no number
        auto load_k = [&](int page) {
            if constexpr (kFour) {
                kr.load(c, h, page, col, quad);
            } else {
            const int8_t* const p = c.k + (static_cast<int64_t>(page) * c.heads + h) * (kKvBlock * D);
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const int tok = 16 * (col >> 2) + 4 * u + (col & 3);
#pragma unroll
                for (int k = 0; k < KL; ++k) kr[u][k] = load_once(p + tok * D + 64 * k + 16 * quad);
            }
            }
        };
        auto load_v = [&](int page) {
            if constexpr (kFour) {
                vr.load(c, h, page, col, quad);
            } else {
            const int8_t* const p = c.v + (static_cast<int64_t>(page) * c.heads + h) * (kKvBlock * D);
#pragma unroll
            for (int d = 0; d < NT; ++d) vr[d] = load_once(p + (16 * d + col) * kKvBlock + 16 * quad);
            }
        };

        // a lane holds the page and the factors of one of the wave's next 64 blocks
        for (int x0 = from; x0 < to; x0 += 64 * kFewWaves) {
            const int x = x0 + lane * kFewWaves + wave;
            const int b = x < to ? (mine ? mine[x] : x) : -1;
            const int page = b >= 0 && b < blocks ? s.page(i, b, c.pages) : -1;
            uint64_t left = __ballot(page >= 0);
            if (!left) continue;
            Factors f = {};
            if constexpr (kFour) {
                f = factors(1.0f, 1.0f, scale * kLog2e);
            } else if (page >= 0) {
                const int64_t p = static_cast<int64_t>(page) * c.heads + h;
                f = factors(c.ks[p], c.vs[p], scale * kLog2e);
            }
            int y = __builtin_ctzll(left);
            int now = __builtin_amdgcn_readlane(page, y);
            load_k(now);
            load_v(now);
            while (left) {
                left &= left - 1;
                const int z = left ? __builtin_ctzll(left) : y;
                const int next = __builtin_amdgcn_readlane(page, z);
                const int base = __builtin_amdgcn_readlane(b, y) * kKvBlock;
                const float fc = kFour ? f.c : __int_as_float(__builtin_amdgcn_readlane(__float_as_int(f.c), y));
                const float flv = kFour ? 0.0f : __int_as_float(__builtin_amdgcn_readlane(__float_as_int(f.lv), y));
                const float fiv = kFour ? 1.0f : __int_as_float(__builtin_amdgcn_readlane(__float_as_int(f.iv), y));
                const float fvs = kFour ? 1.0f : __int_as_float(__builtin_amdgcn_readlane(__float_as_int(f.vs), y));
                f32x4 sc[NQ][4];
                if constexpr (kFour) kr.ready(scratch[wave], col, quad);
#pragma unroll
                for (int u = 0; u < 4; ++u) {
#pragma unroll
                    for (int g = 0; g < NQ; ++g) sc[g][u] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
                    if constexpr (kFour) {
#pragma unroll
                        for (int k = 0; k < D / 32; ++k) {
                            const bf16x8 a = kr.operand(u, k, col);
#pragma unroll
                            for (int g = 0; g < NQ; ++g) sc[g][u] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, qf[g][k], sc[g][u], 0, 0, 0);
                        }
                    } else
#pragma unroll
                    for (int k = 0; k < KL; ++k) {
                        const uint4 w = kr[u][k];
                        const bf16x8 lo = frag(ints_bf16(make_uint2(w.x, w.y))), hi = frag(ints_bf16(make_uint2(w.z, w.w)));
#pragma unroll
                        for (int g = 0; g < NQ; ++g) {
                            sc[g][u] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(lo, qf[g][2 * k], sc[g][u], 0, 0, 0);
                            sc[g][u] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(hi, qf[g][2 * k + 1], sc[g][u], 0, 0, 0);
                        }
                    }
                }
                // (4 bits: loads that are always issued, of nothing behind the last, let the others' waits count them)
                if constexpr (kFour) load_k(left ? next : -1);
                else if (left) load_k(next);
                // register r of sc[g][u]: token base + 16 quad + 4 u + r (4 bits: 16 u + 4 r + quad)
                const bool mask = base + kKvBlock > full;
                bf16x8 p[NQ][2];
#pragma unroll
                for (int g = 0; g < NQ; ++g) {
                    float best = -__builtin_inff();
                    if constexpr (kFour) {
                        if (mask) {
                            const int most = last[g] - base - quad;
#pragma unroll
                            for (int u = 0; u < 4; ++u)
#pragma unroll
                                for (int r = 0; r < 4; ++r) sc[g][u][r] = 16 * u + 4 * r > most ? -__builtin_inff() : sc[g][u][r];
                        }
#pragma unroll
                        for (int u = 0; u < 4; ++u)
#pragma unroll
                            for (int r = 0; r < 4; ++r) best = fmaxf(best, sc[g][u][r]);
                    } else
#pragma unroll
                    for (int u = 0; u < 4; ++u)
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            if (mask && base + 16 * quad + 4 * u + r > last[g]) sc[g][u][r] = -__builtin_inff();
                            best = fmaxf(best, sc[g][u][r]);
                        }
                    if constexpr (kFour) {
                        best = max_halves(max_quads(best)) * fc;
                    } else {
                        best = fmaxf(best, __shfl_xor(best, 16));
                        best = fmaxf(best, __shfl_xor(best, 32)) * fc;
                    }
                    if (__any(best > m[g] + kSlack)) {
                        const float mn = fmaxf(m[g], best), fix = exp2_hw(m[g] - mn);
                        m[g] = mn;
                        l[g] *= fix;
#pragma unroll
                        for (int d = 0; d < NT; ++d) o[g][d] *= fix;
                    }
                    const float off = flv - m[g];
                    float sum = 0.0f;
#pragma unroll
                    for (int u = 0; u < 4; ++u)
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            sc[g][u][r] = exp2_hw(__builtin_fmaf(sc[g][u][r], fc, off));
                            sum += sc[g][u][r];
                        }
                    if (kFour || fiv != 0.0f) {
                        l[g] = kFour ? l[g] + sum : __builtin_fmaf(sum, fiv, l[g]);
                    } else {
                        // a scale that is no ordinary number: what a row does not see must not reach it, and a NaN or an
                        // infinity must where a probability underflows
#pragma unroll
                        for (int u = 0; u < 4; ++u)
#pragma unroll
                            for (int r = 0; r < 4; ++r) {
                                const bool sees = base + 16 * quad + 4 * u + r <= last[g];
                                l[g] += sees ? sc[g][u][r] : 0.0f;
                                sc[g][u][r] = sees ? sc[g][u][r] * fvs : 0.0f;
                            }
                    }
#pragma unroll
                    for (int w = 0; w < 2; ++w) {
                        const f32x4 a = sc[g][2 * w], e = sc[g][2 * w + 1];
                        p[g][w] = frag(make_uint4(bf16x2_bits(a[0], a[1]), bf16x2_bits(a[2], a[3]), bf16x2_bits(e[0], e[1]), bf16x2_bits(e[2], e[3])));
                    }
                }
                if constexpr (kFour) {
                    poison |= vr.ready(scratch[wave], col, quad);
#pragma unroll
                    for (int e = 0; e < NT / 2; ++e) {
                        bf16x8 a[2][2];
                        vr.operands(e, quad, a);
#pragma unroll
                        for (int z = 0; z < 2; ++z)
#pragma unroll
                            for (int g = 0; g < NQ; ++g) {
                                o[g][2 * e + z] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[z][0], p[g][0], o[g][2 * e + z], 0, 0, 0);
                                o[g][2 * e + z] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[z][1], p[g][1], o[g][2 * e + z], 0, 0, 0);
                            }
                    }
                } else
#pragma unroll
                for (int d = 0; d < NT; ++d) {
                    const bf16x8 lo = frag(ints_bf16(make_uint2(vr[d].x, vr[d].y))), hi = frag(ints_bf16(make_uint2(vr[d].z, vr[d].w)));
#pragma unroll
                    for (int g = 0; g < NQ; ++g) {
                        o[g][d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(lo, p[g][0], o[g][d], 0, 0, 0);
                        o[g][d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(hi, p[g][1], o[g][d], 0, 0, 0);
                    }
                }
                if constexpr (kFour) load_v(left ? next : -1);
                else if (left) load_v(next);
                y = z;
            }
        }

        // as in kv_tile_kernel: a wave that has met such a value looks through its blocks again
        if constexpr (kFour) {
            if (poison) {
                for (int x = from + wave; x < to; x += kFewWaves) {
                    const int b = mine ? mine[x] : x;
                    const int page = b >= 0 && b < blocks ? s.page(i, b, c.pages) : -1;
                    if (page < 0) continue;
                    const uint8_t* const codes = c.vs + (static_cast<int64_t>(page) * c.heads + h) * (D / kFourGroup * kKvBlock);
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        int first = 0x7FFFFFFF;  // token with such a scale of this register's elements
#pragma unroll 1
                        for (int x2 = kKvBlock - 1; x2 >= 0; --x2)
                            if (codes[Four::out_element(quad, r, 0) / kFourGroup * kKvBlock + x2] >= kFourBad) first = b * kKvBlock + x2;
#pragma unroll
                        for (int g = 0; g < NQ; ++g)
#pragma unroll
                            for (int e = 0; e < NT; ++e) o[g][e][r] = first <= last[g] ? __builtin_nanf("") : o[g][e][r];
                    }
                }
            }
        }

        // register r of o[g][d]: element 16 d + 4 quad + r of query 16 g + col (4 bits: out_element)
#pragma unroll
        for (int g = 0; g < NQ; ++g) {
            if (g * kFew >= queries) break;
            l[g] += __shfl_xor(l[g], 16);
            l[g] += __shfl_xor(l[g], 32);
            const bool sees = last[g] >= 0;  // else padding, or a row that sees nothing: what the registers hold is no result
            if (g > 0 || again) __syncthreads();
            if (quad == 0) jml[wave][col] = make_float2(m[g], sees ? l[g] : 0.0f);
            if constexpr (kFour) {
#pragma unroll
                for (int r = 0; r < 4; ++r)
#pragma unroll
                    for (int e = 0; e < NT; e += 4)
                        *reinterpret_cast<float4*>(&jo[wave][col][Four::out_element(quad, r, e)]) =
                            sees ? make_float4(o[g][e][r], o[g][e + 1][r], o[g][e + 2][r], o[g][e + 3][r]) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            } else
#pragma unroll
            for (int d = 0; d < NT; ++d)
                *reinterpret_cast<float4*>(&jo[wave][col][16 * d + 4 * quad]) =
                    sees ? make_float4(o[g][d][0], o[g][d][1], o[g][d][2], o[g][d][3]) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            __syncthreads();
            const int here = queries - g * kFew < kFew ? queries - g * kFew : kFew;
            for (int e = t; e < here * (D / 4); e += 64 * kFewWaves) {
                const int qn = e / (D / 4), d = e % (D / 4) * 4, query = g * kFew + qn;
                float top = kLowest;
#pragma unroll
                for (int w = 0; w < kFewWaves; ++w) top = fmaxf(top, jml[w][qn].x);
                float sum = 0.0f, a[4] = {};
#pragma unroll
                for (int w = 0; w < kFewWaves; ++w) {
                    const float2 ml = jml[w][qn];
                    const float fix = exp2_hw(ml.x - top);
                    sum += ml.y * fix;
                    const float4 x = *reinterpret_cast<const float4*>(&jo[w][qn][d]);
                    a[0] += x.x * fix, a[1] += x.y * fix, a[2] += x.z * fix, a[3] += x.w * fix;
                }
                if (shares.shares) {
                    const int64_t to_part = part.at(h, w + i, query);
                    if (d == 0) part.ml[to_part] = make_float2(top, sum);
                    *reinterpret_cast<float4*>(part.o + to_part * D + d) = make_float4(a[0], a[1], a[2], a[3]);
                } else {
                    const int64_t to_row = (static_cast<int64_t>(i) * q.rows + query / group) * q.heads + h * group + query % group;
                    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
                    *reinterpret_cast<uint2*>(out + to_row * D + d) = make_uint2(bf16x2_bits(a[0] * inv, a[1] * inv), bf16x2_bits(a[2] * inv, a[3] * inv));
                }
            }
        }
        if (at >= share_end) return;
        // the next sequence that has blocks: there is one, as the share goes on
        do ++i;
        while (uniform(ends[i + 1]) == at);
    }
}

// ------------------------------------------------------------------ joining splits

constexpr int kMaxSplits = 64;  // of a tile, a lane of the join's wave each

// D / 4 lanes take a row of an item. FEW: at most kFewSplits splits, whose sums a lane adds up; else a wave a row, 256 / D
// splits at once.  (Two splits of 30720 rows of 64 elements: a wave a row 17.8 us, so 5.9.)
constexpr int kFewSplits = 8;

template <int D, bool FEW, bool MIX>
__global__ __launch_bounds__(256) void kv_join_kernel(Partial part, Queries q, Items items, uint32_t all,
                                                      uint16_t* __restrict__ out) {
    constexpr int L = D / 4, SG = 64 / L;
    const uint32_t x = FEW ? blockIdx.x * (256 / L) + threadIdx.x / L : blockIdx.x * 4 + (threadIdx.x >> 6);
    if (x >= all) return;
    const int lane = threadIdx.x & 63, d = lane % L * 4, sg = lane / L;
    const uint32_t per = part.rows;
    const int item = static_cast<int>(x / per), r = static_cast<int>(x % per);
    int i, head, tile;
    items.place<MIX>(items.whole + item, i, head, tile);
    const int y = tile * part.rows + r, row = items.row_of(y);
    if (row >= q.rows) return;
    const int64_t query = (static_cast<int64_t>(i) * q.rows + row) * q.heads + head * items.pack + y - row * items.pack;
    float sum = 0.0f, a[4] = {};
    if constexpr (FEW) {
        float2 ml[kFewSplits];
        float4 v[kFewSplits];
        float top = kLowest;
#pragma unroll
        for (int z = 0; z < kFewSplits; ++z) {
            ml[z] = z < part.splits ? part.ml[part.at(item, z, r)] : make_float2(kLowest, 0.0f);
            // a split without a token wrote no sums: its l of 0 leaves them out below
            v[z] = z < part.splits ? *reinterpret_cast<const float4*>(part.o + part.at(item, z, r) * D + d) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            top = fmaxf(top, ml[z].x);
        }
#pragma unroll
        for (int z = 0; z < kFewSplits; ++z) {
            if (ml[z].y == 0.0f) continue;
            const float f = exp2_hw(ml[z].x - top);
            sum += ml[z].y * f;
            a[0] += v[z].x * f, a[1] += v[z].y * f, a[2] += v[z].z * f, a[3] += v[z].w * f;
        }
    } else {
        const float2 ml = lane < part.splits ? part.ml[part.at(item, lane, r)] : make_float2(kLowest, 0.0f);
        float top = ml.x;
#pragma unroll
        for (int y2 = 32; y2; y2 >>= 1) top = fmaxf(top, __shfl_xor(top, y2));
        const float fix = ml.y == 0.0f ? 0.0f : exp2_hw(ml.x - top);
        const uint64_t held = __ballot(ml.y != 0.0f);  // the splits that wrote sums
        sum = ml.y * fix;
#pragma unroll
        for (int y2 = 32; y2; y2 >>= 1) sum += __shfl_xor(sum, y2);
        for (int s0 = 0; s0 < part.splits; s0 += 4 * SG) {
            float f[4];
            float4 v[4];
#pragma unroll
            for (int z = 0; z < 4; ++z) {
                const int sp = s0 + z * SG + sg;
                f[z] = __shfl(fix, sp & 63);
                v[z] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                // (what a factor of 0 makes of a NaN or an infinity is part of the sum)
                if (held >> (sp & 63) & 1) v[z] = *reinterpret_cast<const float4*>(part.o + part.at(item, sp, r) * D + d);
            }
#pragma unroll
            for (int z = 0; z < 4; ++z) a[0] += v[z].x * f[z], a[1] += v[z].y * f[z], a[2] += v[z].z * f[z], a[3] += v[z].w * f[z];
        }
#pragma unroll
        for (int y2 = 32; y2 >= L; y2 >>= 1)
#pragma unroll
            for (int z = 0; z < 4; ++z) a[z] += __shfl_xor(a[z], y2);
        if (sg != 0) return;
    }
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
    *reinterpret_cast<uint2*>(out + query * D + d) = make_uint2(bf16x2_bits(a[0] * inv, a[1] * inv), bf16x2_bits(a[2] * inv, a[3] * inv));
}

// A row of kv_few_kernel's pieces: a workgroup, D / 4 lanes for every 1024 / D-th piece, as one sequence may have most of
// the launch's.
template <int D>
__global__ __launch_bounds__(256) void kv_join_pieces_kernel(Partial part, Shares shares, Queries q, int kv, uint16_t* __restrict__ out) {
    constexpr int L = D / 4, G = 256 / L, kAhead = 4;
    __shared__ float4 sums[G][L];
    __shared__ float2 parts[G];
    const int t = threadIdx.x, d = t % L * 4, g = t / L;
    // rows in the order of sequences, kv heads, queries of a group
    const int query = blockIdx.x % part.rows, nh = blockIdx.x / part.rows, h = nh % kv, i = nh / kv;
    const int2 span = shares.spans[i];
    float top = kLowest, sum = 0.0f, a[4] = {};
    for (int w0 = span.x + g; w0 <= span.y; w0 += G * kAhead) {
        float2 ml[kAhead];
        float4 v[kAhead];
        float best = top;
#pragma unroll
        for (int x = 0; x < kAhead; ++x) {
            const int w = w0 + x * G;
            const int64_t at = part.at(h, w + i, query);
            ml[x] = make_float2(kLowest, 0.0f);
            v[x] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            if (w <= span.y) ml[x] = part.ml[at], v[x] = *reinterpret_cast<const float4*>(part.o + at * D + d);
        }
#pragma unroll
        for (int x = 0; x < kAhead; ++x) best = fmaxf(best, ml[x].x);
        const float fix = exp2_hw(top - best);
        top = best;
        sum *= fix;
#pragma unroll
        for (int j = 0; j < 4; ++j) a[j] *= fix;
#pragma unroll
        for (int x = 0; x < kAhead; ++x) {
            const float f = exp2_hw(ml[x].x - top);
            sum += ml[x].y * f;
            a[0] += v[x].x * f, a[1] += v[x].y * f, a[2] += v[x].z * f, a[3] += v[x].w * f;
        }
    }
    sums[g][t % L] = make_float4(a[0], a[1], a[2], a[3]);
    if (t % L == 0) parts[g] = make_float2(top, sum);
    __syncthreads();
    if (g > 0) return;
#pragma unroll
    for (int x = 0; x < G; ++x) top = fmaxf(top, parts[x].x);
    sum = a[0] = a[1] = a[2] = a[3] = 0.0f;
#pragma unroll
    for (int x = 0; x < G; ++x) {
        const float4 v = sums[x][t];
        const float f = exp2_hw(parts[x].x - top);
        sum += parts[x].y * f;
        a[0] += v.x * f, a[1] += v.y * f, a[2] += v.z * f, a[3] += v.w * f;
    }
    const int group = q.heads / kv;
    const int64_t to_row = (static_cast<int64_t>(i) * q.rows + query / group) * q.heads + h * group + query % group;
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
    *reinterpret_cast<uint2*>(out + to_row * D + d) = make_uint2(bf16x2_bits(a[0] * inv, a[1] * inv), bf16x2_bits(a[2] * inv, a[3] * inv));
}

// ------------------------------------------------------------------ what a call runs

// Queries of a kv head's group that kv_few_kernel holds in registers: 64 of 64 elements, 32 of 128 (64 spilled, and took
// 230 us where 32 take 87), 16 of 256.
constexpr int64_t few_queries(int64_t dim) { return 64 * kFew / dim * 4; }

constexpr int64_t kMaxPack = 4096;

struct Plan {
    bool few, flat;
    int waves;          // of a tile's workgroup
    int pack;           // query heads of an item
    int splits;         // of a split item
    int shares;         // of a kv head's blocks (few), 0: none
    int64_t rows;       // queries of an item
    int64_t heads, tiles, items, whole;  // items of one workgroup each come first
    int64_t spans;          // rows' worth of the shares' spans
    int64_t part_rows() const { return shares ? heads * (shares + items / heads) * rows + spans : splits > 1 ? (items - whole) * splits * rows : 0; }
};

// How many pieces the blocks of `rest` items are split into over 4 bits: the least of what this makes of the launch, in us.  A block
// takes a tile 1.0, 1.8 or 2.8 (64, 128, 256 elements), alone on its CU or with as many beside it as fit; a piece costs 4 beside its
// blocks, a join 7 and its bytes.  One sequence's items are alike and go in rounds; of several, whose lengths are not known here,
// the lists are taken to be six tenths of the longest, the pieces to be dealt out evenly, and the last one to come on top.  The
// partial sums are at most what the memory-side cache holds.  Against as many pieces as fill one round: 1000 rows of 20 heads of
// 256 over 4000 tokens 182 -> 141 us, 3 sequences of 300 rows and up to 30000 tokens of 24 heads of 64 214 -> 145, of 150 rows and
// up to 9000 of 56 of 128 231 -> 165.  Sequences that are equally long, and lists, are taken for uneven too, and get more pieces
// than they need (2 of 19721 tokens, 56 heads of 128: 450 rows in 8 pieces 673 us and 239 MB of partial sums, unsplit 576; 800 rows
// in 10 970, in 3 962, unsplit 1054; 2401 rows in 13 2543, in 4 2535, unsplit 2673; 600 rows over lists of 100 blocks in 10 256,
// in 4 259, unsplit 345).
int64_t four_splits(int64_t n, int64_t rest, int64_t slots, int64_t longest, int64_t dim, int64_t item_bytes) {
    const double block = dim == 64 ? 1.0 : dim == 128 ? 1.8 : 2.8;
    int64_t best = 1;
    double least = 0.0;
    for (int64_t s = 1; s <= kMaxSplits && (s == 1 || (longest / s >= 4 && rest * s * item_bytes <= kMemoryCache)); ++s) {
        const int64_t rounds = (rest * s + slots - 1) / slots;
        const double piece = block * ((longest + s - 1) / s) + 4.0;
        double cost = n == 1 ? rounds * piece : piece + (rounds > 1 ? rest * (0.6 * block * longest + 4.0 * s) / slots : 0.0);
        if (s > 1) cost += 7.0 + rest * s * item_bytes / 7e6;
        if (s == 1 || cost < least) best = s, least = cost;
    }
    return best;
}

// Sizes checked by the caller.  four: of a cache in 4 bits.
Plan plan_of(bool four, int64_t n, int64_t rows, int64_t heads, int64_t kv, int64_t dim, int64_t blocks, int64_t top) {
    Plan p = {};
    const int64_t cus = cu_count(), group = heads / kv;
    const int64_t longest = top > 0 ? top : blocks;  // blocks that a query may read
    p.few = rows * group <= few_queries(dim);
    if (p.few) {
        p.pack = static_cast<int>(group);
        p.rows = rows * group;
        p.heads = kv;
        p.tiles = 1;
        p.items = n * kv;
        p.splits = 1;
        // As many workgroups as the CUs hold at once, by the registers that the queries take, of at least two blocks a wave,
        // where they are half as many again as the sequences: a piece and its place in the join cost 3 us (448 workgroups of
        // 17 rows unsplit 88 us, 512 shares 108; but 8 x 20 heads of 256 unsplit 68 us, 240 shares 55).
        int64_t shares = ((p.rows + kFew - 1) / kFew * dim >= 256 ? 1 : 2) * cus / kv;
        if (n <= kFewThreads && n * longest < (int64_t{1} << 30)) {
            if (shares > n * longest / (2 * kFewWaves)) shares = n * longest / (2 * kFewWaves);
            if (shares > n && 2 * shares >= 3 * n) p.shares = static_cast<int>(shares), p.spans = (8 * n + 4 * dim + 7) / (4 * dim + 8);
        }
        return p;
    }
    // Rows that leave a tile part empty share it with the other heads of their group (a list is a kv head's).
    p.pack = rows < kKvTile && group <= kMaxPack ? static_cast<int>(group) : 1;
    p.heads = heads / p.pack;
    // Tiles of 4 waves, two a CU, balance themselves; 8 waves in step are ahead where the work is long and even: 128
    // elements, 128 blocks and 1024 rows on (4800 x 19721 2661 us, 2746 with 4; 2000 x 9000 562 and 583; but 2000 x 2000
    // causal 138 and 104, 4800 x 19200 of 64 elements 927 and 837).  A list is 128 rows'.
    const int64_t queries = rows * p.pack, tiles8 = (queries + 255) / 256, tiles4 = (queries + 127) / 128;
    p.waves = dim == 128 && top == 0 && blocks >= 128 && queries >= 1024 && n * p.heads * tiles8 >= cus ? 8 : 4;
    p.rows = 32 * p.waves;
    p.tiles = p.waves == 8 ? tiles8 : tiles4;
    p.items = n * p.heads * p.tiles;
    const int64_t slots = (p.waves == 8 || dim == 256 ? 1 : dim == 64 ? 3 : 2) * (cus < 8 ? 8 : cus / 8 * 8);  // whole XCDs' worth
    p.flat = p.items <= slots;
    p.whole = p.items / slots * slots;
    const int64_t rest = p.items - p.whole;
    // A split pays for its join (5 us and the sums' bytes) by the blocks that it saves (1.3 us each, alone on a CU): a CU
    // each, or a slot each where lists are long (240 tiles of 38 blocks 47.9 us unsplit, 44.0 so; 168 tiles of 15 blocks
    // 27.9 us, and 35.9 split).
    int64_t splits = rest > 0 ? (longest >= 24 ? slots : cus) / rest : 1;
    if (splits > longest / 4) splits = longest / 4;
    if (splits > kMaxSplits) splits = kMaxSplits;
    if (four && rest > 0) splits = four_splits(n, rest, slots, longest, dim, p.rows * (dim * 4 + 8));
    if (splits <= 1) p.whole = p.items / 8 * 8, splits = 1;
    p.splits = static_cast<int>(splits);
    return p;
}

bool sizes_ok(int64_t n, int64_t rows, int64_t heads, int64_t kv, int64_t dim, int64_t blocks, int64_t top) {
    int64_t q;
    return n >= 0 && rows >= 0 && heads > 0 && kv > 0 && heads % kv == 0 && heads <= 65536 && (dim == 64 || dim == 128 || dim == 256) &&
           blocks >= 0 && top >= 0 && rows <= (1 << 30) && n <= 0x7FFFFFFF && !__builtin_mul_overflow(n, rows * heads, &q) && q < (int64_t{1} << 40);
}

}  // namespace
}  // namespace h3mi

using namespace h3mi;

namespace {

int64_t workspace_of(bool four, int64_t n, int64_t rows, int64_t heads, int64_t kv_heads, int64_t dim, int64_t blocks, int64_t top) {
    if (!sizes_ok(n, rows, heads, kv_heads, dim, blocks, top) || n == 0 || rows == 0) return 0;
    return plan_of(four, n, rows, heads, kv_heads, dim, blocks, top).part_rows() * (dim * 4 + 8);
}

}  // namespace

extern "C" int64_t h3mi_kv_attention_workspace(int64_t n, int64_t rows, int64_t heads, int64_t kv_heads, int64_t dim, int64_t blocks,
                                               int64_t top) {
    return workspace_of(false, n, rows, heads, kv_heads, dim, blocks, top);
}

extern "C" int64_t h3mi_kv_attention_mx4_workspace(int64_t n, int64_t rows, int64_t heads, int64_t kv_heads, int64_t dim, int64_t blocks,
                                                   int64_t top) {
    return workspace_of(true, n, rows, heads, kv_heads, dim, blocks, top);
}

namespace {

template <class C, int D, int W>
int launch_tiles(const Items& items, const Queries& q, const C& c, const KvSeqs& s, float scale, int causal, const Lists& list,
                 uint16_t* out, const Partial& part, hipStream_t stream) {
    int64_t groups;
    if (!launchable(items.whole + int64_t{8} * items.rest_chunk, 1, 1, 64 * W, &groups))
        return fail(H3MI_EINVAL, "kv_attention: too many rows for one call");
    const auto fn = kv_tile_kernel<C, D, W>;
    constexpr int lds = TileShape<D, W>::kLds;
    hipLaunchKernelGGL(fn, dim3(static_cast<unsigned>(groups)), dim3(64 * W), lds, stream, q, c, s, scale, causal, list, out, part, items);
    return check_launch("kv_attention");
}

// A call over a cache of 8 or of 4 bits.
template <class Cache>
int attention(const uint16_t* q, int64_t rows, int64_t heads, int64_t ld_q, int64_t bs_q, const Cache* cache, const h3mi_kv_seqs* seqs,
              float scale, int causal, const int32_t* blocks, int64_t top, uint16_t* out, void* workspace, int64_t workspace_bytes,
              void* stream) {
    using C = decltype(kv_cache(*cache));
    if (int e = kv_check("kv_attention", cache, seqs)) return e;
    if (heads <= 0 || heads > 65536 || heads % cache->heads)
        return fail(H3MI_EINVAL, "kv_attention: heads=%lld must be a multiple of the cache's %lld", (long long)heads, (long long)cache->heads);
    if (int e = kv_check_rows("kv_attention", "q", q, rows, heads, cache->dim, seqs->n, ld_q, bs_q)) return e;
    if (!(scale == scale) || scale - scale != 0.0f) return fail(H3MI_EINVAL, "kv_attention: scale is not finite");
    if (!blocks) top = 0;
    if (blocks && (top < 1 || top >= (1 << 25))) return fail(H3MI_EINVAL, "kv_attention: top=%lld", (long long)top);
    if (seqs->n == 0 || rows == 0) return ok();
    if (!out) return fail(H3MI_EINVAL, "kv_attention: null out");
    if (!aligned(out, 16) || !aligned(blocks, 4)) return fail(H3MI_EALIGN, "kv_attention: out must be 16-byte aligned, blocks 4-byte");
    const int64_t n = seqs->n, dim = cache->dim;
    if (!sizes_ok(n, rows, heads, cache->heads, dim, seqs->blocks, top)) return fail(H3MI_EINVAL, "kv_attention: too many rows for one call");
    constexpr bool kFour = std::is_same_v<C, KvCache4>;
    const Plan p = plan_of(kFour, n, rows, heads, cache->heads, dim, seqs->blocks, top);
    const int64_t part_rows = p.part_rows(), need = part_rows * (dim * 4 + 8);
    const int64_t rest = (p.items - p.whole) * p.splits;
    if (p.items > (1 << 30) || rest > (1 << 30)) return fail(H3MI_EINVAL, "kv_attention: too many rows for one call");
    const size_t bytes = static_cast<size_t>(n) * rows * heads * dim * 2;
    if (overlap(out, bytes, q, kv_span(n, rows, heads, dim, ld_q, bs_q)) || kv_overlaps(out, bytes, *cache))
        return fail(H3MI_EALIAS, "kv_attention: out overlaps q or the cache");
    const size_t list_bytes = static_cast<size_t>(n) * ((rows + kKvTile - 1) / kKvTile) * cache->heads * top * 4;
    if (kv_seqs_overlap(out, bytes, *seqs) || (blocks && overlap(out, bytes, blocks, list_bytes)))
        return fail(H3MI_EALIAS, "kv_attention: out overlaps tables, lens, counts or blocks");
    if (need > 0 && (!workspace || workspace_bytes < need))
        return fail(H3MI_EINVAL, "kv_attention: workspace of %lld bytes, %lld needed", (long long)(workspace ? workspace_bytes : 0), (long long)need);
    if (!aligned(workspace, 16)) return fail(H3MI_EALIGN, "kv_attention: workspace must be 16-byte aligned");
    if (need > 0 && (overlap(workspace, need, out, bytes) || overlap(workspace, need, q, kv_span(n, rows, heads, dim, ld_q, bs_q)) ||
                     kv_overlaps(workspace, need, *cache) || kv_seqs_overlap(workspace, need, *seqs) ||
                     (blocks && overlap(workspace, need, blocks, list_bytes))))
        return fail(H3MI_EALIAS, "kv_attention: the workspace overlaps out or an input");
    const Queries qs = {q, ld_q, bs_q, static_cast<int>(rows), static_cast<int>(heads)};
    const Lists list = {blocks, static_cast<int>(top), static_cast<int>((rows + kKvTile - 1) / kKvTile)};
    Partial part = {static_cast<float*>(workspace), nullptr, p.shares ? p.shares + static_cast<int>(n) : p.splits, static_cast<int>(p.rows)};
    const Items items = {static_cast<int>(p.tiles), static_cast<int>(p.heads), p.pack, static_cast<int>(p.rows),
                         p.pack == 1 ? 0u : static_cast<uint32_t>(((uint64_t{1} << 32) + p.pack - 1) / p.pack), static_cast<int>(p.items),
                         static_cast<int>(p.whole), static_cast<int>(p.whole / 8), static_cast<int>((rest + 7) / 8), p.flat, causal != 0, static_cast<int>(n)};
    if (need > 0) part.ml = reinterpret_cast<float2*>(part.o + (part_rows - p.spans) * dim);
    const C c = kv_cache(*cache);
    const KvSeqs s = kv_seqs(*seqs);
    const hipStream_t st = as_stream(stream);
    int rc;
    if (p.few) {
        int64_t groups;
        const Shares shares = {p.shares, p.shares ? reinterpret_cast<int2*>(part.ml + part_rows - p.spans) : nullptr};
        if (!launchable(p.shares ? p.shares * p.heads : p.items, 1, 1, kFewThreads, &groups)) return fail(H3MI_EINVAL, "kv_attention: too many rows for one call");
        const int sets = static_cast<int>((p.rows + kFew - 1) / kFew);
        const auto fn = dim == 64    ? (sets == 1 ? kv_few_kernel<C, 64, 1> : sets == 2 ? kv_few_kernel<C, 64, 2> : kv_few_kernel<C, 64, 4>)
                        : dim == 128 ? (sets == 1 ? kv_few_kernel<C, 128, 1> : kv_few_kernel<C, 128, 2>)
                                     : kv_few_kernel<C, 256, 1>;
        hipLaunchKernelGGL(fn, dim3(static_cast<unsigned>(groups)), dim3(kFewThreads), 0, st, qs, c, s, scale, causal, list, out, part,
                           shares);
        rc = check_launch("kv_attention");
        if (rc || !p.shares) return rc;
        if (!launchable(p.items, p.rows, 1, 256, &groups)) return fail(H3MI_EINVAL, "kv_attention: too many rows for one call");
        const auto join = dim == 64 ? kv_join_pieces_kernel<64> : dim == 128 ? kv_join_pieces_kernel<128> : kv_join_pieces_kernel<256>;
        hipLaunchKernelGGL(join, dim3(static_cast<unsigned>(groups)), dim3(256), 0, st, part, shares, qs, c.heads, out);
        return check_launch("kv_attention");
    } else if (dim == 64) {
        rc = launch_tiles<C, 64, 4>(items, qs, c, s, scale, causal, list, out, part, st);
    } else if (dim == 128) {
        rc = p.waves == 8 ? launch_tiles<C, 128, 8>(items, qs, c, s, scale, causal, list, out, part, st)
                          : launch_tiles<C, 128, 4>(items, qs, c, s, scale, causal, list, out, part, st);
    } else {
        rc = launch_tiles<C, 256, 4>(items, qs, c, s, scale, causal, list, out, part, st);
    }
    if (rc || p.splits == 1) return rc;
    const int64_t all = (p.items - p.whole) * p.rows;
    int64_t groups;
    const bool few = p.splits <= kFewSplits;
    const int64_t a_group = few ? 1024 / dim : 4;
    if (!launchable((all + a_group - 1) / a_group, 1, 1, 256, &groups)) return fail(H3MI_EINVAL, "kv_attention: too many rows for one call");
    const auto join = few ? (dim == 64 ? kv_join_kernel<64, true, kFour> : dim == 128 ? kv_join_kernel<128, true, kFour> : kv_join_kernel<256, true, kFour>)
                          : (dim == 64 ? kv_join_kernel<64, false, kFour> : dim == 128 ? kv_join_kernel<128, false, kFour> : kv_join_kernel<256, false, kFour>);
    hipLaunchKernelGGL(join, dim3(static_cast<unsigned>(groups)), dim3(256), 0, st, part, qs, items,
                       static_cast<uint32_t>(all), out);
    return check_launch("kv_attention");
}

}  // namespace

extern "C" int h3mi_kv_attention_bf16(const uint16_t* q, int64_t rows, int64_t heads, int64_t ld_q, int64_t bs_q,
                                      const h3mi_kv_cache* cache, const h3mi_kv_seqs* seqs, float scale, int causal,
                                      const int32_t* blocks, int64_t top, uint16_t* out, void* workspace,
                                      int64_t workspace_bytes, void* stream) {
    return attention(q, rows, heads, ld_q, bs_q, cache, seqs, scale, causal, blocks, top, out, workspace, workspace_bytes, stream);
}

extern "C" int h3mi_kv_attention_mx4_bf16(const uint16_t* q, int64_t rows, int64_t heads, int64_t ld_q, int64_t bs_q,
                                          const h3mi_kv_cache4* cache, const h3mi_kv_seqs* seqs, float scale, int causal,
                                          const int32_t* blocks, int64_t top, uint16_t* out, void* workspace,
                                          int64_t workspace_bytes, void* stream) {
    return attention(q, rows, heads, ld_q, bs_q, cache, seqs, scale, causal, blocks, top, out, workspace, workspace_bytes, stream);
}
