// kv_cache.hpp - a cache of K and V rows in fp16 or fp32: layout, device
// addressing, the tree of a draft, enqueue functions.
//
// K and V are planes [layers][S][Hkv][R][D], S sequences of R rows, or S blocks
// of R rows behind a block table: the layouts of attention_gqa's K and V, of a
// session's caches and of the paged attention. In a paged cache R % 16 == 0
// keeps 16 keys of a matrix tile in one block; a contiguous one has any R.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "../../include/aljabr_rocm.h"

namespace aljabr {

struct KvView {
    char *k, *v;             // of the layer
    const int *table;        // null: contiguous
    int B, H, D, R, num_blocks, max_blocks;
    int f16;
};

// ALJABR_ROCM_OK and the view of a layer, or the status of a cache description that no operator takes.
int kv_view(const aljabr_rocm_kv_cache *c, int layer, const char *who, KvView &v);

// Rows a sequence can hold.
__host__ __device__ inline int kv_capacity(const KvView &v) { return v.table ? v.R * v.max_blocks : v.R; }

// The plane index (sequence or block) and row of position pos of sequence b;
// false when the cache has no such row.
__device__ __forceinline__ bool kv_locate(const KvView &v, int b, long long pos, int &s, int &row) {
    if (pos < 0 || pos >= kv_capacity(v)) return false;
    if (!v.table) {
        s = b;
        row = static_cast<int>(pos);
        return true;
    }
    const int p = static_cast<int>(pos), blk = p / v.R;
    s = v.table[static_cast<long long>(b) * v.max_blocks + blk];
    row = p - blk * v.R;
    return s >= 0 && s < v.num_blocks;
}

constexpr int kTreeMost = 256;               // rows of a tree
constexpr int kTreeWords = kTreeMost / 32;

// A draft's tree in LDS: of row i, mask[w * kTreeMost + i] are bits 32w .. 32w + 31 of the rows that are i or its
// ancestors, depth[i] is the number of its ancestors.
struct Tree {
    uint32_t mask[kTreeWords * kTreeMost];
    int depth[kTreeMost];
};

// The row whose parent a thread gives fill_tree: of up to 64 rows every wave holds all.
__device__ __forceinline__ int tree_row(int n) { return n <= 64 ? threadIdx.x & 63 : threadIdx.x; }

// Fills the tree of rows [0, n), n <= kTreeMost, from the parent of each thread's row (a number that is not an earlier
// row's stands for none). With a window > 0, of a row's line only its last `window` rows are kept in mask. By a workgroup
// of kTreeMost threads, none of which waits for another where n <= 64: each wave then writes the whole tree, and what it
// reads is its own.
//
// After step s a row knows the 2^(s+1) last rows of its line and the row before them: log2(n) steps whatever the depth,
// each a row's masks joined with those of the row where its own end. A window is taken in parts of powers of two: the
// steps whose bit it has, each from where the one before ended.
__device__ __forceinline__ void fill_tree(Tree &t, int parent, int n, int window) {
    const int i = threadIdx.x, words = (n + 31) >> 5;
    const bool mine = i < n;
    const int limit = window > 0 && window < n ? window : 0;
    if (n <= 64) {
        const int lane = i & 63;
        int to = lane < n && parent >= 0 && parent < lane ? parent : -1, at = lane;
        uint32_t lo = lane < 32 ? 1u << lane : 0, hi = lane < 32 ? 0 : 1u << (lane - 32), in_lo = 0, in_hi = 0;
        for (int s = 0; 1 << s < n; ++s) {
            if (limit >> s & 1) {
                const uint32_t x = __shfl(lo, at), y = __shfl(hi, at);
                const int z = __shfl(to, at);
                if (at >= 0) {
                    in_lo |= x;
                    in_hi |= y;
                    at = z;
                }
            }
            const uint32_t x = __shfl(lo, to), y = __shfl(hi, to);
            const int z = __shfl(to, to);
            if (to >= 0) {
                lo |= x;
                hi |= y;
                to = z;
            }
        }
        t.depth[lane] = __builtin_popcount(lo) + __builtin_popcount(hi) - 1;
        t.mask[lane] = limit ? in_lo : lo;
        t.mask[kTreeMost + lane] = limit ? in_hi : hi;
        t.mask[2 * kTreeMost + lane] = 0;                  // a word of zeros behind the last
        return;
    }
    int jump = -1, cur = mine ? i : -1;
    uint32_t own[kTreeWords], part[kTreeWords];
    if (mine && parent >= 0 && parent < i) jump = parent;
#pragma unroll
    for (int w = 0; w < kTreeWords; ++w) {
        own[w] = i >> 5 == w && mine ? 1u << (i & 31) : 0;
        part[w] = 0;
        if (w <= words) t.mask[w * kTreeMost + i] = own[w];      // and a word of zeros behind the last
    }
    t.depth[i] = jump;
    __syncthreads();
    for (int s = 0; 1 << s < n; ++s) {
        if (limit >> s & 1 && cur >= 0) {
#pragma unroll
            for (int w = 0; w < kTreeWords; ++w)
                if (w < words) part[w] |= t.mask[w * kTreeMost + cur];
            cur = t.depth[cur];
        }
        const int from = jump;
        if (from >= 0) {
#pragma unroll
            for (int w = 0; w < kTreeWords; ++w)
                if (w < words) own[w] |= t.mask[w * kTreeMost + from];
            jump = t.depth[from];
        }
        __syncthreads();
        if (from >= 0) {
#pragma unroll
            for (int w = 0; w < kTreeWords; ++w)
                if (w < words) t.mask[w * kTreeMost + i] = own[w];
            t.depth[i] = jump;
        }
        __syncthreads();
    }
    int depth = -1;
#pragma unroll
    for (int w = 0; w < kTreeWords; ++w) {
        depth += __builtin_popcount(own[w]);
        if (limit && w < words) t.mask[w * kTreeMost + i] = part[w];
    }
    t.depth[i] = depth;
    __syncthreads();
}

struct KvAppend {
    float *q_out;            // [B][T][Hq][D], or null with q
    const void *q, *k, *v;   // rows of `f16` ? fp16 : fp32, element strides of a sequence, a token and a head
    const int *positions, *counts, *angles;
    const float *divisors;   // [rot / 2], or null
    int T, Hq, f16;
    long long q_sb, q_st, q_sh, kv_sb, kv_st, kv_sh;
    int rot, interleaved;    // rot 0: no rotation
    double base;
};
int enqueue_kv_append(const KvView &v, const KvAppend &a);

struct KvTreeAttention {
    float *out;              // [B][T][Hq][D]
    const float *q;          // as out
    const int *lens;         // [B] cached keys, the rows' own among them
    const int *counts;       // [B] rows of each sequence (null: T)
    const int *parents;      // [B][T], or null: row t - 1
    int T, Hq;
    float scale;             // > 0
    int window;
    float soft_cap;
    float *scratch;          // split partials; null: the stream's scratch
    size_t scratch_bytes;
};
int enqueue_kv_tree_attention(const KvView &v, const KvTreeAttention &a);
// Bytes of scratch with which enqueue_kv_tree_attention splits as it likes.
size_t kv_tree_attention_scratch_bytes(const KvView &v, int T, int Hq);

}  // namespace aljabr
