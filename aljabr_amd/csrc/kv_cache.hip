// kv_cache.hip - rows rotated and appended to a cache, and a draft's accepted
// rows moved together (layout: kv_cache.hpp).
//
// Append: row t of a token has the pairs (x_i, x_i+r/2), or (x_2i, x_2i+1)
// interleaved, turned by theta = a base^(-2i/r) / divisor_i, the rest of the
// row is copied. The angle is computed in fp64 as quarter turns, a times
// base^(-2i/r) / divisor_i / (pi/2): its nearest integer picks the quadrant
// exactly, and the rest, at most half a quarter, is what fp32 series take. The
// product and the frequency are rounded a few times by 2^-53 of the angle: at
// a = 2^30, where fp32 angles would be off by whole turns, about 2^-22 radians.
//
// A row is D/8 lanes with two units of four values each, so that both halves
// of four pairs meet in a lane; the row is on its way before its position and
// angles are known. Bound by the bytes: 4 x 2048 tokens of 32 + 8 + 8 heads of
// 128, fp32 to an fp16 cache, 66 us (369 MB, 5.6 TB/s, what a copy reaches;
// four prompts of up to 2048, 231 MB in the mean, 36 to 51 us, part of it from
// the last-level cache); one token of a sequence 3.5 to 4.3 us, a launch.
//
// Accept: a row is kept when it and all its ancestors up to row 0 agree with
// the model, which the tree's masks say for all rows at once; a kept row's
// depth is its place. Every workgroup works this out for itself, then a wave
// moves the rows of one (layer, head, K or V). A row never moves behind one
// that is still to move (place i <= row path[i], both increasing), so rows go
// in batches in order, each read whole before it is written. Bound by the chain
// of launch, parents, choices, tree and rows: a tree of 64 rows over 32 layers
// of 8 KV heads 4.7 us, of 26 rows in 32 sequences, 10 MB of rows, 7 us.
#include <cmath>

#include "device.hpp"
#include "internal.hpp"
#include "kv_cache.hpp"
#include "kv_chunks.hpp"

namespace aljabr {
namespace {

constexpr int kThreads = 256;
static_assert(kThreads == kTreeMost, "fill_tree takes a thread a row");

struct AppendParams {
    KvView v;
    KvAppend a;
    kv::FastDiv by_heads;    // Hq + 2 H, a token's rows
    double quarter;          // 2 / pi
    double step;             // log2(base) * -2 / rot
};

template <bool WIDE>
__device__ __forceinline__ float4 load_row4(const void *base, long long at, int f16) {
    float4 x;
    if (f16) {
        const uint16_t *s = static_cast<const uint16_t *>(base) + at;
        if constexpr (WIDE) {
            const uint2 u = *reinterpret_cast<const uint2 *>(s);
            x.x = f16_bits_to_f32(u.x & 0xffffu);
            x.y = f16_bits_to_f32(u.x >> 16);
            x.z = f16_bits_to_f32(u.y & 0xffffu);
            x.w = f16_bits_to_f32(u.y >> 16);
        } else {
            x.x = f16_bits_to_f32(s[0]);
            x.y = f16_bits_to_f32(s[1]);
            x.z = f16_bits_to_f32(s[2]);
            x.w = f16_bits_to_f32(s[3]);
        }
    } else {
        const float *s = static_cast<const float *>(base) + at;
        if constexpr (WIDE) {
            x = *reinterpret_cast<const float4 *>(s);
        } else {
            x = make_float4(s[0], s[1], s[2], s[3]);
        }
    }
    return x;
}

__device__ __forceinline__ uint32_t half_bits(float x) { return __builtin_bit_cast(uint16_t, static_cast<_Float16>(x)); }

__device__ __forceinline__ void store_row4(char *plane, long long at, const float4 &x, int f16) {
    if (f16)
        *reinterpret_cast<uint2 *>(plane + 2 * at) =
            make_uint2(half_bits(x.x) | half_bits(x.y) << 16, half_bits(x.z) | half_bits(x.w) << 16);
    else
        *reinterpret_cast<float4 *>(plane + 4 * at) = x;
}

// Cosine and sine of `quarters` quarter turns: the Taylor series on [-pi/4, pi/4], whose next terms are below 2^-29.
__device__ __forceinline__ void cos_sin(double quarters, float &c, float &s) {
    const double whole = rint(quarters);
    const float x = static_cast<float>((quarters - whole) * 1.5707963267948966), x2 = x * x;
    float p = fmaf(x2, 1.0f / 362880, -1.0f / 5040);
    p = fmaf(x2, p, 1.0f / 120);
    p = fmaf(x2, p, -1.0f / 6);
    const float sn = fmaf(x * x2, p, x);
    float q = fmaf(x2, -1.0f / 3628800, 1.0f / 40320);
    q = fmaf(x2, q, -1.0f / 720);
    q = fmaf(x2, q, 1.0f / 24);
    q = fmaf(x2, q, -0.5f);
    const float cs = fmaf(x2, q, 1.0f);
    const int quad = static_cast<int>(static_cast<long long>(whole) & 3);
    c = quad & 1 ? sn : cs;
    s = quad & 1 ? cs : sn;
    if (quad == 1 || quad == 2) c = -c;
    if (quad >= 2) s = -s;
}

__device__ __forceinline__ void turn(float &x, float &y, float c, float s) {
    const float a = x, b = y;
    x = fmaf(a, c, -(b * s));
    y = fmaf(a, s, b * c);
}

template <int D, bool WIDE>
__global__ __launch_bounds__(kThreads) void kv_append_kernel(AppendParams p) {
    constexpr int LPR = D / 8, GPB = kThreads / LPR;
    const KvAppend &a = p.a;
    const int b = blockIdx.y, l = threadIdx.x % LPR;
    const int group = blockIdx.x * GPB + threadIdx.x / LPR;      // below 2^29
    const int heads = a.Hq + 2 * p.v.H, t = p.by_heads(group), h = group - t * heads;
    if (t >= (a.counts ? min(a.counts[b], a.T) : a.T)) return;
    const bool is_q = h < a.Hq, is_k = !is_q && h < a.Hq + p.v.H;
    const void *src = is_q ? a.q : is_k ? a.k : a.v;
    if (!src) return;
    const int kv = is_q ? h : is_k ? h - a.Hq : h - a.Hq - p.v.H;

    // This lane's two units: of the rotated part l and its partner half a part on, behind it two neighbours.
    const int rot = a.rot, pairs = rot / 8;
    const bool turned = l < pairs;
    const int u0 = turned ? 4 * l : rot + 8 * (l - pairs), u1 = turned ? u0 + rot / 2 : u0 + 4;
    const long long at = is_q ? b * a.q_sb + t * a.q_st + h * a.q_sh : b * a.kv_sb + t * a.kv_st + kv * a.kv_sh;
    float4 x = load_row4<WIDE>(src, at + u0, a.f16), y = load_row4<WIDE>(src, at + u1, a.f16);
    const long long pos = static_cast<long long>(a.positions[b]) + t;
    int s = 0, row = 0;
    if (!is_q && !kv_locate(p.v, b, pos, s, row)) return;
    if (turned && (is_q || is_k)) {
        const double quarters = static_cast<double>(a.angles ? a.angles[static_cast<long long>(b) * a.T + t] : pos) * p.quarter;
        // Pairs 4l .. 4l + 3, or interleaved 2l, 2l + 1 and the same a quarter of the part on.
        const int first = a.interleaved ? 2 * l : 4 * l, skip = a.interleaved ? rot / 4 - 2 : 0;
        float c[4], sn[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int i = first + j + (j >= 2 ? skip : 0);
            double f = exp2(p.step * i);
            if (a.divisors && a.divisors[i] > 0.0f) f /= static_cast<double>(a.divisors[i]);
            cos_sin(quarters * f, c[j], sn[j]);
        }
        if (a.interleaved) {
            turn(x.x, x.y, c[0], sn[0]);
            turn(x.z, x.w, c[1], sn[1]);
            turn(y.x, y.y, c[2], sn[2]);
            turn(y.z, y.w, c[3], sn[3]);
        } else {
            turn(x.x, y.x, c[0], sn[0]);
            turn(x.y, y.y, c[1], sn[1]);
            turn(x.z, y.z, c[2], sn[2]);
            turn(x.w, y.w, c[3], sn[3]);
        }
    }
    if (is_q) {
        float *dst = a.q_out + ((static_cast<long long>(b) * a.T + t) * a.Hq + h) * D;
        *reinterpret_cast<float4 *>(dst + u0) = x;
        *reinterpret_cast<float4 *>(dst + u1) = y;
    } else {
        const long long to = ((static_cast<long long>(s) * p.v.H + kv) * p.v.R + row) * D;
        store_row4(is_k ? p.v.k : p.v.v, to + u0, x, p.v.f16);
        store_row4(is_k ? p.v.k : p.v.v, to + u1, y, p.v.f16);
    }
}

struct AcceptParams {
    KvView v;
    int layers, row_bytes;
    long long layer_bytes;
    const int *lens, *counts, *parents, *tokens, *choices;
    int *new_lens, *path, *accepted, *next;
    int T;
};

constexpr int kBatch = 4;                    // 16-byte pieces that a lane holds at once

__global__ __launch_bounds__(kThreads) void kv_tree_accept_kernel(AcceptParams p) {
    __shared__ Tree tree;
    __shared__ int first[kTreeMost], line[kTreeMost], block[kTreeMost], in_block[kTreeMost], count, last;
    __shared__ uint32_t disagree[kTreeWords];
    const int i = threadIdx.x, b = blockIdx.y;
    const int n = max(p.lens[b], 0);                             // past the cache too: its rows lie where it says
    const int cnt = p.counts ? min(max(p.counts[b], 0), p.T) : p.T;
    const long long row0 = static_cast<long long>(b) * p.T;
    int up = -1;
    bool agrees = i == 0;
    if (i < cnt && i > 0) {
        up = p.parents ? p.parents[row0 + i] : i - 1;
        if (up < 0 || up >= i) up = -1;
        agrees = up >= 0 && p.tokens[row0 + i] == p.choices[row0 + up];
    }
    int s = -1, row = 0;                                         // where the draft's row i lies, or nowhere
    if (i < cnt && !kv_locate(p.v, b, static_cast<long long>(n) - cnt + i, s, row)) s = -1;
    block[i] = s;
    in_block[i] = row;
    first[i] = kTreeMost;
    line[i] = -1;
    if (i < kTreeWords) disagree[i] = 0;
    if (i == 0) count = last = 0;
    __syncthreads();
    if (i > 0 && i < cnt && agrees) atomicMin(&first[up], i);    // of a row's children that agree, the first
    __syncthreads();
    if (i > 0 && i < cnt && (!agrees || first[up] != i)) atomicOr(&disagree[i >> 5], 1u << (i & 31));
    if (p.parents) {
        const int row = tree_row(cnt);
        fill_tree(tree, row < cnt ? p.parents[row0 + row] : -1, cnt, 0);
        __syncthreads();
    } else {
        tree.depth[i] = i;
#pragma unroll
        for (int w = 0; w < kTreeWords; ++w)
            tree.mask[w * kTreeMost + i] = i >= 32 * w + 31 ? 0xffffffffu : i >= 32 * w ? (2u << (i & 31)) - 1 : 0;
        __syncthreads();
    }
    if (i < cnt && tree.mask[i] & 1) {                           // row 0 is in its line
        uint32_t against = 0;
#pragma unroll
        for (int w = 0; w < kTreeWords; ++w)
            if (w <= (cnt - 1) >> 5) against |= tree.mask[w * kTreeMost + i] & disagree[w];
        if (!against) {                                          // kept rows are one line: a row a depth
            line[tree.depth[i]] = i;
            atomicMax(&last, i);
            atomicAdd(&count, 1);
        }
    }
    __syncthreads();
    const int kept = count;
    if (blockIdx.x == 0) {
        if (i < p.T) p.path[row0 + i] = line[i];
        if (i == 0) {
            p.new_lens[b] = n - cnt + kept;
            p.accepted[b] = kept;
            p.next[b] = kept ? p.choices[row0 + last] : -1;
        }
    }

    // Rows path[j] -> j of one (layer, head, K or V) a wave; lanes_per pieces of 16 bytes a row.
    const int lane = i & 63, lanes_per = p.row_bytes >> 4, rows = 64 / lanes_per, piece = lane % lanes_per, mine = lane / lanes_per;
    const int slab = blockIdx.x * (kThreads / 64) + (i >> 6);
    if (slab >= p.layers * p.v.H * 2) return;
    const int head = (slab >> 1) % p.v.H, layer = (slab >> 1) / p.v.H;
    char *plane = (slab & 1 ? p.v.v : p.v.k) + layer * p.layer_bytes + 16 * piece;
    for (int j0 = 0; j0 < kept; j0 += rows * kBatch) {
        uint4 x[kBatch];
        char *to[kBatch];
#pragma unroll
        for (int k = 0; k < kBatch; ++k) {
            const int j = j0 + k * rows + mine;
            to[k] = nullptr;
            if (j >= kept || line[j] == j) continue;
            const int from = line[j];
            if (block[from] < 0 || block[j] < 0) continue;
            x[k] = *reinterpret_cast<const uint4 *>(
                plane + ((static_cast<long long>(block[from]) * p.v.H + head) * p.v.R + in_block[from]) * p.row_bytes);
            to[k] = plane + ((static_cast<long long>(block[j]) * p.v.H + head) * p.v.R + in_block[j]) * p.row_bytes;
        }
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");         // a batch is read before any of it is written
#pragma unroll
        for (int k = 0; k < kBatch; ++k)
            if (to[k]) *reinterpret_cast<uint4 *>(to[k]) = x[k];
    }
}

template <int D>
void launch_append(const AppendParams &p, bool wide, dim3 grid) {
    if (wide)
        hipLaunchKernelGGL((kv_append_kernel<D, true>), grid, dim3(kThreads), 0, current_stream(), p);
    else
        hipLaunchKernelGGL((kv_append_kernel<D, false>), grid, dim3(kThreads), 0, current_stream(), p);
}

// The checks of a description; *bytes: of one of its planes.
int check_cache(const aljabr_rocm_kv_cache *c, const char *who, bool pointers, size_t *bytes) {
    ALJ_REQUIRE(c, "%s: cache must be non-null", who);
    if (pointers) ALJ_REQUIRE(c->k && c->v, "%s: the cache's planes must be device pointers", who);
    const bool paged = pointers ? c->block_table != nullptr : c->num_blocks > 0;
    ALJ_REQUIRE(c->layers > 0 && c->n_kv_heads > 0 && c->head_dim > 0 && c->rows > 0 && (c->sequences > 0 || (!pointers && paged)),
                "%s: layers, sequences, n_kv_heads, head_dim and rows must be positive", who);
    if (c->type != ALJABR_ROCM_TYPE_F32 && c->type != ALJABR_ROCM_TYPE_F16)
        return fail(ALJABR_ROCM_ERR_UNSUPPORTED, "%s: cache type %d is not F32 or F16", who, c->type);
    if (c->head_dim != 64 && c->head_dim != 128 && c->head_dim != 256)
        return fail(ALJABR_ROCM_ERR_UNSUPPORTED, "%s: head_dim %d is not 64, 128 or 256", who, c->head_dim);
    if (paged) {
        ALJ_REQUIRE(c->rows % 16 == 0, "%s: blocks of %d rows: a multiple of 16 is needed", who, c->rows);
        ALJ_REQUIRE(!pointers || (c->num_blocks > 0 && c->max_blocks > 0 &&
                                  static_cast<long long>(c->max_blocks) * c->rows <= (1LL << 30)),
                    "%s: a paged cache needs num_blocks and max_blocks, max_blocks * rows at most 2^30", who);
    } else {
        ALJ_REQUIRE(c->rows <= (1 << 30), "%s: rows = %d exceeds 2^30", who, c->rows);
        // kv_cache_bytes counts such a description's blocks: as a contiguous cache its sequences may pass the planes.
        ALJ_REQUIRE(c->num_blocks == 0 && c->max_blocks == 0, "%s: num_blocks and max_blocks without a block_table", who);
    }
    ALJ_REQUIRE(c->sequences <= 65535 && c->n_kv_heads <= 16384, "%s: more than 65535 sequences or 16384 heads", who);
    const size_t row = static_cast<size_t>(c->n_kv_heads) * c->rows;                       // below 2^62
    size_t all;
    ALJ_REQUIRE(!__builtin_mul_overflow(static_cast<size_t>(paged ? c->num_blocks : c->sequences), row, &all) &&
                    !__builtin_mul_overflow(all, static_cast<size_t>(c->layers), &all) &&
                    !__builtin_mul_overflow(all, static_cast<size_t>(c->head_dim) * (c->type == ALJABR_ROCM_TYPE_F16 ? 2 : 4), &all) &&
                    all < (size_t{1} << 62),
                "%s: a plane of this shape has 2^62 bytes or more", who);
    *bytes = all;
    if (pointers) ALJ_REQUIRE(aligned(c->k, 16) && aligned(c->v, 16), "%s: the cache's planes must be 16-byte aligned", who);
    return ALJABR_ROCM_OK;
}

}  // namespace

int kv_view(const aljabr_rocm_kv_cache *c, int layer, const char *who, KvView &v) {
    size_t bytes;
    const int rc = check_cache(c, who, true, &bytes);
    if (rc != ALJABR_ROCM_OK) return rc;
    ALJ_REQUIRE(layer >= 0 && layer < c->layers, "%s: layer %d of %d", who, layer, c->layers);
    const size_t at = bytes / c->layers * layer;
    v.k = static_cast<char *>(c->k) + at;
    v.v = static_cast<char *>(c->v) + at;
    v.table = static_cast<const int *>(c->block_table);
    v.B = c->sequences;
    v.H = c->n_kv_heads;
    v.D = c->head_dim;
    v.R = c->rows;
    v.num_blocks = v.table ? c->num_blocks : c->sequences;
    v.max_blocks = v.table ? c->max_blocks : 1;
    v.f16 = c->type == ALJABR_ROCM_TYPE_F16;
    return ALJABR_ROCM_OK;
}

int enqueue_kv_append(const KvView &v, const KvAppend &a) {
    AppendParams p{};
    p.v = v;
    p.a = a;
    const int heads = a.Hq + 2 * v.H;
    p.by_heads.set(heads);
    p.quarter = 2.0 / 3.14159265358979323846;
    p.step = a.rot ? std::log2(a.base) * -2.0 / a.rot : 0.0;
    const size_t unit = a.f16 ? 8 : 16;
    const bool wide = aligned(a.q, unit) && aligned(a.k, unit) && aligned(a.v, unit) && a.q_sb % 4 == 0 && a.q_st % 4 == 0 &&
                      a.q_sh % 4 == 0 && a.kv_sb % 4 == 0 && a.kv_st % 4 == 0 && a.kv_sh % 4 == 0;
    const int gpb = kThreads / (v.D / 8);
    const dim3 grid(static_cast<unsigned>((static_cast<long long>(a.T) * heads + gpb - 1) / gpb), v.B);
    if (v.D == 64) launch_append<64>(p, wide, grid);
    else if (v.D == 128) launch_append<128>(p, wide, grid);
    else launch_append<256>(p, wide, grid);
    return ALJABR_ROCM_OK;
}

}  // namespace aljabr

using namespace aljabr;

extern "C" {

int aljabr_rocm_kv_cache_bytes(const aljabr_rocm_kv_cache *cache, size_t *bytes) {
    ALJ_REQUIRE(bytes, "kv_cache_bytes: bytes is null");
    return check_cache(cache, "kv_cache_bytes", false, bytes);
}

int aljabr_rocm_kv_append(const aljabr_rocm_kv_cache *cache, int layer, void *q_out, const void *Q, const void *K,
                          const void *V, const int *positions, const int *counts, const int *angles, int T, int Hq,
                          long long q_stride_b, long long q_stride_t, long long q_stride_h, long long kv_stride_b,
                          long long kv_stride_t, long long kv_stride_h, int type, const aljabr_rocm_rotation *rotation) {
    KvView v;
    int rc = kv_view(cache, layer, "kv_append", v);
    if (rc != ALJABR_ROCM_OK) return rc;
    ALJ_REQUIRE(Q || K || V, "kv_append: one of Q, K and V must be a device pointer");
    ALJ_REQUIRE(!Q == !q_out, "kv_append: Q and q_out go together");
    ALJ_REQUIRE(positions, "kv_append: positions must be a device pointer");
    ALJ_REQUIRE(T > 0 && T <= (1 << 30), "kv_append: T = %d is outside [1, 2^30]", T);
    ALJ_REQUIRE(Q ? Hq > 0 && Hq <= 65536 : Hq >= 0 && Hq <= 65536, "kv_append: Hq = %d is outside [1, 65536]", Hq);
    if (type != ALJABR_ROCM_TYPE_F32 && type != ALJABR_ROCM_TYPE_F16)
        return fail(ALJABR_ROCM_ERR_UNSUPPORTED, "kv_append: Q/K/V type %d is not F32 or F16", type);
    ALJ_REQUIRE(q_stride_b >= 0 && q_stride_t >= 0 && q_stride_h >= 0 && kv_stride_b >= 0 && kv_stride_t >= 0 && kv_stride_h >= 0,
                "kv_append: strides must not be negative");
    KvAppend a{};
    if (rotation) {
        ALJ_REQUIRE(std::isfinite(rotation->base) && rotation->base > 0.0f, "kv_append: the rotation's base must be positive and finite");
        a.rot = rotation->rotary_dim ? rotation->rotary_dim : v.D;
        ALJ_REQUIRE(a.rot > 0 && a.rot <= v.D, "kv_append: rotary_dim = %d is outside [0, %d]", rotation->rotary_dim, v.D);
        if (a.rot % 8) return fail(ALJABR_ROCM_ERR_UNSUPPORTED, "kv_append: rotary_dim %d is not a multiple of 8", a.rot);
        ALJ_REQUIRE(aligned(rotation->freq_divisors, 4), "kv_append: freq_divisors must be aligned to its elements");
        a.base = rotation->base;
        a.interleaved = rotation->interleaved != 0;
        a.divisors = static_cast<const float *>(rotation->freq_divisors);
    }
    a.Hq = Q ? Hq : 0;
    if (!q_stride_b && !q_stride_t && !q_stride_h) {
        q_stride_h = v.D;
        q_stride_t = static_cast<long long>(Hq) * v.D;
        q_stride_b = T * q_stride_t;
    }
    if (!kv_stride_b && !kv_stride_t && !kv_stride_h) {
        kv_stride_h = v.D;
        kv_stride_t = static_cast<long long>(v.H) * v.D;
        kv_stride_b = T * kv_stride_t;
    }
    const size_t elem = type == ALJABR_ROCM_TYPE_F16 ? 2 : 4;
    ALJ_REQUIRE(aligned(Q, elem) && aligned(K, elem) && aligned(V, elem), "kv_append: Q, K and V must be aligned to their elements");
    ALJ_REQUIRE(aligned(q_out, 16), "kv_append: q_out must be 16-byte aligned");
    ALJ_REQUIRE(!Q || q_out != Q || (type == ALJABR_ROCM_TYPE_F32 && (Hq == 1 || q_stride_h == v.D) &&
                                     (T == 1 || q_stride_t == static_cast<long long>(Hq) * v.D) &&
                                     (v.B == 1 || q_stride_b == static_cast<long long>(T) * Hq * v.D)),
                "kv_append: q_out is a Q that is not dense fp32 rows");
    ALJ_REQUIRE(static_cast<long long>(T) * (a.Hq + 2 * v.H) * (v.D / 8) <= 0xffffff00LL,       // lanes of a launch
                "kv_append: T = %d rows of %d heads are more than one launch takes", T, a.Hq + 2 * v.H);
    ALJ_CHECK_READY();
    a.q_out = static_cast<float *>(q_out);
    a.q = Q;
    a.k = K;
    a.v = V;
    a.positions = positions;
    a.counts = counts;
    a.angles = angles;
    a.T = T;
    a.f16 = type == ALJABR_ROCM_TYPE_F16;
    a.q_sb = q_stride_b;
    a.q_st = q_stride_t;
    a.q_sh = q_stride_h;
    a.kv_sb = kv_stride_b;
    a.kv_st = kv_stride_t;
    a.kv_sh = kv_stride_h;
    rc = enqueue_kv_append(v, a);
    return rc == ALJABR_ROCM_OK ? finish_launch("kv_append") : rc;
}

int aljabr_rocm_kv_tree_accept(const aljabr_rocm_kv_cache *cache, int *new_lens, int *path, int *accepted, int *next_token,
                               const int *context_lens, const int *counts, const int *parents, const int *tokens,
                               const int *choices, int T) {
    AcceptParams p{};
    const int rc = kv_view(cache, 0, "kv_tree_accept", p.v);
    if (rc != ALJABR_ROCM_OK) return rc;
    ALJ_REQUIRE(new_lens && path && accepted && next_token && context_lens && tokens && choices,
                "kv_tree_accept: new_lens, path, accepted, next_token, context_lens, tokens and choices must be device pointers");
    // Other workgroups read the inputs while the first writes these.
    for (const int *out : {new_lens, path, accepted, next_token})
        for (const int *in : {context_lens, counts, parents, tokens, choices, static_cast<const int *>(cache->block_table)})
            ALJ_REQUIRE(out != in, "kv_tree_accept: an output is one of the inputs");
    ALJ_REQUIRE(T > 0, "kv_tree_accept: T = %d must be positive", T);
    if (T > kTreeMost) return fail(ALJABR_ROCM_ERR_UNSUPPORTED, "kv_tree_accept: T = %d exceeds a tree's %d rows", T, kTreeMost);
    p.layers = cache->layers;
    p.row_bytes = p.v.D * (p.v.f16 ? 2 : 4);
    p.layer_bytes = static_cast<long long>(p.v.num_blocks) * p.v.H * p.v.R * p.row_bytes;
    const long long slabs = 2LL * p.layers * p.v.H;
    ALJ_REQUIRE(slabs <= (1 << 24), "kv_tree_accept: layers * n_kv_heads exceeds 2^23");
    ALJ_CHECK_READY();
    p.lens = context_lens;
    p.counts = counts;
    p.parents = parents;
    p.tokens = tokens;
    p.choices = choices;
    p.new_lens = new_lens;
    p.path = path;
    p.accepted = accepted;
    p.next = next_token;
    p.T = T;
    const unsigned per = kThreads / 64;
    hipLaunchKernelGGL(kv_tree_accept_kernel, dim3(static_cast<unsigned>((slabs + per - 1) / per), p.v.B), dim3(kThreads), 0,
                       current_stream(), p);
    return finish_launch("kv_tree_accept");
}

}  // extern "C"
