// The 8-bit key/value cache: what its writer, reader, selection and attention share.
#pragma once

#include "common.h"

namespace h3mi {

constexpr int kKvBlock = H3MI_KV_BLOCK;
constexpr int kKvTile = H3MI_KV_TILE;

// Checks of a cache and of a call's sequences, named `what` in the messages.
int kv_check(const char* what, const h3mi_kv_cache* c, const h3mi_kv_seqs* s);
// Checks of [n, rows, heads, dim] bf16 rows.
int kv_check_rows(const char* what, const char* name, const uint16_t* p, int64_t rows, int64_t heads, int64_t dim,
                  int64_t n, int64_t ld, int64_t bs);
// Bytes of [n, rows, heads, dim] bf16 rows, from the first to the last.
size_t kv_span(int64_t n, int64_t rows, int64_t heads, int64_t dim, int64_t ld, int64_t bs);
// Whether `bytes` at p overlap the cache's keys, values, scales or sums.
bool kv_overlaps(const void* p, size_t bytes, const h3mi_kv_cache& c);
// Whether two of the cache's keys, values, scales and sums overlap.
bool kv_self_overlaps(const h3mi_kv_cache& c);
// Whether `bytes` at p overlap the sequences' tables, lens or counts.
bool kv_seqs_overlap(const void* p, size_t bytes, const h3mi_kv_seqs& s);
// groups = a b c workgroups, if HIP takes a launch of so many with `threads` threads each: it refuses 2^32 threads and more.
inline bool launchable(int64_t a, int64_t b, int64_t c, int64_t threads, int64_t* groups) {
    int64_t g, all;
    if (__builtin_mul_overflow(a, b, &g) || __builtin_mul_overflow(g, c, &g) || __builtin_mul_overflow(g, threads, &all)) return false;
    *groups = g;
    return all < (int64_t{1} << 32);
}

struct KvCache {
    int8_t *k, *v;
    float *ks, *vs;
    int16_t* ksum;
    int64_t pages;
    int heads;
};

struct KvSeqs {
    const int32_t *tables, *lens, *counts;
    int n, blocks;

    // tokens of sequence i, and those of them that its table has blocks for (blocks < 2^25)
    __device__ __forceinline__ int end(int i) const { return lens[i] < 0 ? 0 : lens[i]; }
    __device__ __forceinline__ int len(int i) const {
        const int e = end(i), most = blocks * kKvBlock;
        return e > most ? most : e;
    }
    __device__ __forceinline__ int count(int i, int rows) const {
        if (!counts) return rows;
        const int c = counts[i];
        return c < 0 ? 0 : c > rows ? rows : c;
    }
    // page of block b of sequence i, or -1 where it is not there
    __device__ __forceinline__ int page(int i, int b, int64_t pages) const {
        if (b < 0 || b >= blocks) return -1;
        const int p = tables[static_cast<int64_t>(i) * blocks + b];
        return p < 0 || p >= pages ? -1 : p;
    }
};

// The item of a workgroup such that an XCD's workgroups, every eighth of the launch, take consecutive items.
__device__ __forceinline__ int xcd_item() {
    const int all = gridDim.x, per = all >> 3, more = all & 7, xcd = blockIdx.x & 7, at = blockIdx.x >> 3;
    return xcd * per + (xcd < more ? xcd : more) + at;
}

inline KvCache kv_cache(const h3mi_kv_cache& c) {
    return {c.k, c.v, c.k_scale, c.v_scale, c.k_sum, c.pages, static_cast<int>(c.heads)};
}
inline KvSeqs kv_seqs(const h3mi_kv_seqs& s) {
    return {s.tables, s.lens, s.counts, static_cast<int>(s.n), static_cast<int>(s.blocks)};
}

// floor(a / 64) of any int
__device__ __forceinline__ int block_of(int a) { return a >> 6; }

}  // namespace h3mi
