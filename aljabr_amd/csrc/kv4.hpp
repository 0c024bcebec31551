// kv4.hpp - the 4-bit KV cache: layout, device addressing, enqueue functions.
//
// A K or V row of D values is D/32 blocks of 32 four-bit codes with one fp16
// scale each; value = (code - 8) * scale, an fp16 number (the writer's scales
// have 8 significant bits, so the product has 11; any other scale's product is
// rounded to fp16). Codes and scales are separate planes:
//   codes   u8  [S][Hkv][R][D/2]   (byte j of a block: code j | code j+16 << 4, Q4_0's order)
//   scales  f16 [S][Hkv][D/32][R]
// so that a row's codes are whole 16-byte loads and the scales of four
// consecutive keys, which the attention takes as packed pairs, are one 8-byte
// load. S sequences of R rows, or S blocks of R rows behind a block table;
// R % 16 == 0 keeps 16 keys of a matrix tile in one block.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "../../include/aljabr_rocm.h"

namespace aljabr {

struct Kv4View {
    uint8_t *kc, *vc;
    uint16_t *ks, *vs;
    const int *table;        // null: contiguous
    int B, H, D, R, num_blocks, max_blocks;
};

// ALJABR_ROCM_OK, or the status of a cache description that no operator takes.
int kv4_view(const aljabr_rocm_kv4_cache *c, const char *who, Kv4View &v);

// Rows a sequence can hold.
__host__ __device__ inline int kv4_capacity(const Kv4View &v) { return v.table ? v.R * v.max_blocks : v.R; }

// The plane index (sequence or block) and row of position pos of sequence b;
// false when the cache has no such row.
__device__ __forceinline__ bool kv4_locate(const Kv4View &v, int b, long long pos, int &s, int &row) {
    if (pos < 0 || pos >= kv4_capacity(v)) return false;
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

// K and V rows [B][T][H][D] (element strides; type F32 or F16) into the cache
// at positions[b] + t for t < counts[b] (null: T).
int enqueue_kv4_write(const Kv4View &v, const void *k, const void *vv, const int *positions, const int *counts, int T,
                      long long sb, long long st, long long sh, int type);
int enqueue_kv4_read(const Kv4View &v, void *k, void *vv, const int *positions, const int *counts, int T, long long sb,
                     long long st, long long sh, int type);

struct Kv4Attention {
    float *out;              // [B][T][Hq][D]
    const float *q;          // as out
    const int *lens;         // [B] cached keys, the rows' own among them
    const int *counts;       // [B] rows of each sequence (null: T)
    int T, Hq;
    float scale;             // > 0
    int causal, window;
    float soft_cap;
    float *scratch;          // split partials; null: the stream's scratch
    size_t scratch_bytes;
};
int enqueue_kv4_attention(const Kv4View &v, const Kv4Attention &a);
// Bytes of scratch with which enqueue_kv4_attention splits as it likes.
size_t kv4_attention_scratch_bytes(const Kv4View &v, int T, int Hq);

}  // namespace aljabr
