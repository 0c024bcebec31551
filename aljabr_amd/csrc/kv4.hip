// kv4.hip - rows written to and read from the 4-bit KV cache (layout: kv4.hpp).
//
// Encoder, per block of 32: lo and hi are its smallest and largest values; the
// scale is -top / 8, top = lo if -lo >= hi else hi, rounded to 8 significant
// bits (ties to even; multiples of 2^-24; at most 8160), so the value of
// largest magnitude takes code 0 and every (code - 8) * scale is an fp16
// number. The code is floor(x / scale + 1/2) of the exact quotient, clamped
// to [-8, 7], plus 8. A block with an infinity or a NaN gets a NaN scale: it
// reads back as NaN instead of hiding what was written.
//
// The quotient: |scale| has 8 bits, so (k + 1/2) * scale is exact in fp32 and
// x - k * scale is exact for the two candidates k next to x / scale; an
// estimate from v_rcp_f32 is at most one off, and comparing that residual
// with scale / 2 settles it. No division.
//
// Work: one lane per code dword (8 values: 4q..4q+3 and 16+4q..+3 of a block,
// two 16-byte loads), four lanes a block (its minimum and maximum in two DPP
// steps), D/8 lanes a row. Bound by the bytes: 4 in and 0.5625 out a value.
// Measured: 4 prompts of 2048 rows of 8 x 128 written in 16 us from fp32 (4.7
// TB/s) and in 15 from fp16, 16 of 8192 in 275 (4.45 TB/s) and 185 (3.7 TB/s);
// 16 sequences of 8192 read as fp16 in 164 us (688 MB, 4.2 TB/s, near a copy's
// 4.7); one token in 3.1 us (2.4 in a trace), a launch's time.
#include "device.hpp"
#include "internal.hpp"
#include "kv4.hpp"

namespace aljabr {
namespace {

constexpr int kThreads = 256;

struct RowParams {
    const int *positions, *counts;
    int T;
    long long sb, st, sh;
    int t_tiles;             // > 0: blockIdx.x is a tile of tokens, blockIdx.y a head; 0: heads vary fastest
};

// The (token, head) of this lane's row and its dword of the row; false past the end.
template <int D>
__device__ __forceinline__ bool row_of(const RowParams &p, int H, int &t, int &h, int &w) {
    constexpr int LPR = D / 8, RPW = kThreads / LPR;
    w = threadIdx.x % LPR;
    const int r = blockIdx.x * RPW + threadIdx.x / LPR;
    if (p.t_tiles) {
        t = r;
        h = blockIdx.y >> 1;
        return t < p.T;
    }
    t = r / H;
    h = r - t * H;
    return t < p.T;
}

template <bool F16, bool WIDE>
__device__ __forceinline__ void load4(const void *base, long long at, float (&x)[4]) {
    if constexpr (F16) {
        const uint16_t *s = static_cast<const uint16_t *>(base) + at;
        if constexpr (WIDE) {
            const uint2 u = *reinterpret_cast<const uint2 *>(s);
            x[0] = f16_bits_to_f32(u.x & 0xffffu);
            x[1] = f16_bits_to_f32(u.x >> 16);
            x[2] = f16_bits_to_f32(u.y & 0xffffu);
            x[3] = f16_bits_to_f32(u.y >> 16);
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] = f16_bits_to_f32(s[i]);
        }
    } else {
        const float *s = static_cast<const float *>(base) + at;
        if constexpr (WIDE) {
            const float4 u = *reinterpret_cast<const float4 *>(s);
            x[0] = u.x; x[1] = u.y; x[2] = u.z; x[3] = u.w;
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] = s[i];
        }
    }
}

// This lane's 8 values of a block spread over four lanes -> its code dword and
// the block's scale (the same in all four).
__device__ __forceinline__ uint32_t encode8(const float (&a)[4], const float (&c)[4], uint32_t &scale_bits) {
    float lo = a[0], hi = a[0], probe = 0.0f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        lo = fminf(lo, fminf(a[i], c[i]));
        hi = fmaxf(hi, fmaxf(a[i], c[i]));
        probe = fmaf(a[i], 0.0f, fmaf(c[i], 0.0f, probe));   // NaN where a value is not finite
    }
    lo = fminf(lo, dpp_f32<0xB1>(lo));
    hi = fmaxf(hi, dpp_f32<0xB1>(hi));
    probe += dpp_f32<0xB1>(probe);
    lo = fminf(lo, dpp_f32<0x4E>(lo));
    hi = fmaxf(hi, dpp_f32<0x4E>(hi));
    probe += dpp_f32<0x4E>(probe);
    const bool neg = -lo >= hi;                              // the value of largest magnitude is negative
    float step = (neg ? -lo : hi) * 0.125f;
    if (step >= 7.62939453125e-06f) {                        // 2^-17: 8 significant bits, ties to even
        uint32_t u = __float_as_uint(step);
        u += 0x7fffu + ((u >> 16) & 1u);
        step = __uint_as_float(u & 0xffff0000u);
    } else {
        step = __fsub_rn(__fadd_rn(step, 0.75f), 0.75f);     // multiples of 2^-24, ties to even
    }
    step = fminf(step, 8160.0f);
    const float d = neg || step == 0.0f ? step : -step;
    const float inv = __builtin_amdgcn_rcpf(d), half = 0.5f * step;
    const float sgn = d < 0.0f ? -1.0f : 1.0f;
    const bool flat = step == 0.0f || probe != 0.0f;         // nothing to code: zeros, or a block that is not finite
    uint32_t word = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float x = i < 4 ? a[i] : c[i - 4];
        float q = fminf(fmaxf(rintf(x * inv), -9.0f), 8.0f);
        const float r = fmaf(-q, d, x) * sgn;
        q += r >= half ? 1.0f : r < -half ? -1.0f : 0.0f;
        q = fminf(fmaxf(q, -8.0f), 7.0f);
        const uint32_t code = flat ? 8u : static_cast<uint32_t>(static_cast<int>(q) + 8);
        word |= code << (8 * (i & 3) + 4 * (i >> 2));
    }
    scale_bits = probe != 0.0f ? 0x7e00u : __builtin_bit_cast(uint16_t, static_cast<_Float16>(d));
    return word;
}

template <int D, bool F16, bool WIDE>
__global__ __launch_bounds__(kThreads) void kv4_write_kernel(Kv4View v, RowParams p, const void *__restrict__ k,
                                                             const void *__restrict__ vv) {
    int t, h, w;
    const bool is_v = blockIdx.y & 1;
    const int b = blockIdx.z;
    const void *src = is_v ? vv : k;
    if (!row_of<D>(p, v.H, t, h, w) || !src) return;
    const int cnt = p.counts ? p.counts[b] : p.T;
    int s, row;
    if (t >= cnt || !kv4_locate(v, b, static_cast<long long>(p.positions[b]) + t, s, row)) return;
    const long long at = b * p.sb + t * p.st + h * p.sh + 32 * (w / 4) + 4 * (w % 4);
    float a[4], c[4];
    load4<F16, WIDE>(src, at, a);
    load4<F16, WIDE>(src, at + 16, c);
    uint32_t scale;
    const uint32_t word = encode8(a, c, scale);
    const long long head = static_cast<long long>(s) * v.H + h;
    reinterpret_cast<uint32_t *>((is_v ? v.vc : v.kc) + (head * v.R + row) * (D / 2))[w] = word;
    if (w % 4 == 0) (is_v ? v.vs : v.ks)[(head * (D / 32) + w / 4) * v.R + row] = static_cast<uint16_t>(scale);
}

template <bool F16, bool WIDE>
__device__ __forceinline__ void store4(void *base, long long at, const _Float16 (&x)[4]) {
    if constexpr (F16) {
        uint16_t *d = static_cast<uint16_t *>(base) + at;
        uint16_t u[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) u[i] = __builtin_bit_cast(uint16_t, x[i]);
        if constexpr (WIDE) {
            *reinterpret_cast<uint2 *>(d) = make_uint2(u[0] | static_cast<uint32_t>(u[1]) << 16,
                                                       u[2] | static_cast<uint32_t>(u[3]) << 16);
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) d[i] = u[i];
        }
    } else {
        float *d = static_cast<float *>(base) + at;
        if constexpr (WIDE) {
            *reinterpret_cast<float4 *>(d) = make_float4(x[0], x[1], x[2], x[3]);
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) d[i] = x[i];
        }
    }
}

template <int D, bool F16, bool WIDE>
__global__ __launch_bounds__(kThreads) void kv4_read_kernel(Kv4View v, RowParams p, void *__restrict__ k,
                                                            void *__restrict__ vv) {
    int t, h, w;
    const bool is_v = blockIdx.y & 1;
    const int b = blockIdx.z;
    void *dst = is_v ? vv : k;
    if (!row_of<D>(p, v.H, t, h, w) || !dst) return;
    const int cnt = p.counts ? p.counts[b] : p.T;
    if (t >= cnt) return;
    int s, row;
    _Float16 a[4] = {}, c[4] = {};                           // zeros where the cache has no such row
    if (kv4_locate(v, b, static_cast<long long>(p.positions[b]) + t, s, row)) {
        const long long head = static_cast<long long>(s) * v.H + h;
        const uint32_t word = reinterpret_cast<const uint32_t *>((is_v ? v.vc : v.kc) + (head * v.R + row) * (D / 2))[w];
        const _Float16 d =
            __builtin_bit_cast(_Float16, (is_v ? v.vs : v.ks)[(head * (D / 32) + w / 4) * v.R + row]);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            a[i] = static_cast<_Float16>(static_cast<int>(word >> (8 * i) & 15) - 8) * d;
            c[i] = static_cast<_Float16>(static_cast<int>(word >> (8 * i + 4) & 15) - 8) * d;
        }
    }
    const long long at = b * p.sb + t * p.st + h * p.sh + 32 * (w / 4) + 4 * (w % 4);
    store4<F16, WIDE>(dst, at, a);
    store4<F16, WIDE>(dst, at + 16, c);
}

// Tokens vary fastest from 16 rows on (their scales are neighbours in the
// cache), heads below.
template <int D>
dim3 row_grid(RowParams &p, const Kv4View &v) {
    constexpr int RPW = kThreads / (D / 8);
    p.t_tiles = p.T >= 16;
    const long long rows = p.t_tiles ? p.T : static_cast<long long>(p.T) * v.H;
    return dim3(static_cast<unsigned>((rows + RPW - 1) / RPW), p.t_tiles ? 2 * v.H : 2, v.B);
}

template <int D, bool F16, bool WIDE>
void launch_rows(bool write, const Kv4View &v, RowParams p, void *k, void *vv) {
    const dim3 grid = row_grid<D>(p, v);
    if (write)
        hipLaunchKernelGGL((kv4_write_kernel<D, F16, WIDE>), grid, dim3(kThreads), 0, current_stream(), v, p,
                           static_cast<const void *>(k), static_cast<const void *>(vv));
    else
        hipLaunchKernelGGL((kv4_read_kernel<D, F16, WIDE>), grid, dim3(kThreads), 0, current_stream(), v, p, k, vv);
}

template <int D>
void launch_typed(bool write, const Kv4View &v, const RowParams &p, void *k, void *vv, int type, bool wide) {
    if (type == ALJABR_ROCM_TYPE_F16)
        wide ? launch_rows<D, true, true>(write, v, p, k, vv) : launch_rows<D, true, false>(write, v, p, k, vv);
    else
        wide ? launch_rows<D, false, true>(write, v, p, k, vv) : launch_rows<D, false, false>(write, v, p, k, vv);
}

int enqueue_rows(bool write, const Kv4View &v, void *k, void *vv, const int *positions, const int *counts, int T,
                 long long sb, long long st, long long sh, int type) {
    RowParams p{positions, counts, T, sb, st, sh, 0};
    // 4 elements a load or store where every row starts on as many.
    const size_t unit = type == ALJABR_ROCM_TYPE_F16 ? 8 : 16;
    const bool wide = aligned(k, unit) && aligned(vv, unit) && sb % 4 == 0 && st % 4 == 0 && sh % 4 == 0;
    switch (v.D) {
    case 64: launch_typed<64>(write, v, p, k, vv, type, wide); break;
    case 128: launch_typed<128>(write, v, p, k, vv, type, wide); break;
    default: launch_typed<256>(write, v, p, k, vv, type, wide); break;
    }
    return ALJABR_ROCM_OK;
}

// The checks that kv4_write and kv4_read share; zero strides become [B][T][H][D].
int check_rows(const char *who, const Kv4View &v, const void *k, const void *vv, const int *positions, int T,
               long long &sb, long long &st, long long &sh, int type) {
    ALJ_REQUIRE(k || vv, "%s: K or V must be a device pointer", who);
    ALJ_REQUIRE(positions, "%s: positions must be a device pointer", who);
    ALJ_REQUIRE(T > 0 && T <= (1 << 30), "%s: T = %d is outside [1, 2^30]", who, T);
    if (type != ALJABR_ROCM_TYPE_F32 && type != ALJABR_ROCM_TYPE_F16)
        return fail(ALJABR_ROCM_ERR_UNSUPPORTED, "%s: K/V type %d is not F32 or F16", who, type);
    ALJ_REQUIRE(static_cast<long long>(T) * (v.D / 8) <= 0xffffff00LL,      // lanes of a launch, whole workgroups
                "%s: T = %d rows of %d values are more than one launch takes", who, T, v.D);
    ALJ_REQUIRE(sb >= 0 && st >= 0 && sh >= 0, "%s: strides must not be negative", who);
    if (!sb && !st && !sh) {
        sh = v.D;
        st = static_cast<long long>(v.H) * v.D;
        sb = static_cast<long long>(T) * st;
    }
    const size_t elem = type == ALJABR_ROCM_TYPE_F16 ? 2 : 4;
    ALJ_REQUIRE(aligned(k, elem) && aligned(vv, elem), "%s: K and V must be aligned to their elements", who);
    return ALJABR_ROCM_OK;
}

}  // namespace

int kv4_view(const aljabr_rocm_kv4_cache *c, const char *who, Kv4View &v) {
    ALJ_REQUIRE(c, "%s: cache must be non-null", who);
    ALJ_REQUIRE(c->k_codes && c->k_scales && c->v_codes && c->v_scales, "%s: the cache's four planes must be device pointers",
                who);
    ALJ_REQUIRE(c->sequences > 0 && c->n_kv_heads > 0 && c->head_dim > 0 && c->rows > 0,
                "%s: sequences, n_kv_heads, head_dim and rows must be positive", who);
    ALJ_REQUIRE(c->rows % 16 == 0 && c->rows <= (1 << 26), "%s: rows = %d must be a multiple of 16, at most 2^26", who, c->rows);
    if (c->block_table)
        ALJ_REQUIRE(c->num_blocks > 0 && c->max_blocks > 0 && static_cast<long long>(c->max_blocks) * c->rows <= (1LL << 30),
                    "%s: a paged cache needs num_blocks and max_blocks, max_blocks * rows at most 2^30", who);
    else
        // kv4_cache_bytes counts such a description's blocks: as a contiguous cache its sequences may pass the planes.
        ALJ_REQUIRE(c->num_blocks == 0 && c->max_blocks == 0, "%s: num_blocks and max_blocks without a block_table", who);
    ALJ_REQUIRE(c->sequences <= 65535 && c->n_kv_heads <= 16384, "%s: more than 65535 sequences or 16384 heads", who);
    ALJ_REQUIRE(aligned(c->k_codes, 16) && aligned(c->v_codes, 16) && aligned(c->k_scales, 16) && aligned(c->v_scales, 16),
                "%s: the cache's planes must be 16-byte aligned", who);
    if (c->head_dim != 64 && c->head_dim != 128 && c->head_dim != 256)
        return fail(ALJABR_ROCM_ERR_UNSUPPORTED, "%s: head_dim %d is not 64, 128 or 256", who, c->head_dim);
    v.kc = static_cast<uint8_t *>(c->k_codes);
    v.vc = static_cast<uint8_t *>(c->v_codes);
    v.ks = static_cast<uint16_t *>(c->k_scales);
    v.vs = static_cast<uint16_t *>(c->v_scales);
    v.table = static_cast<const int *>(c->block_table);
    v.B = c->sequences;
    v.H = c->n_kv_heads;
    v.D = c->head_dim;
    v.R = c->rows;
    v.num_blocks = v.table ? c->num_blocks : c->sequences;
    v.max_blocks = v.table ? c->max_blocks : 1;
    return ALJABR_ROCM_OK;
}

int enqueue_kv4_write(const Kv4View &v, const void *k, const void *vv, const int *positions, const int *counts, int T,
                      long long sb, long long st, long long sh, int type) {
    return enqueue_rows(true, v, const_cast<void *>(k), const_cast<void *>(vv), positions, counts, T, sb, st, sh, type);
}

int enqueue_kv4_read(const Kv4View &v, void *k, void *vv, const int *positions, const int *counts, int T, long long sb,
                     long long st, long long sh, int type) {
    return enqueue_rows(false, v, k, vv, positions, counts, T, sb, st, sh, type);
}

}  // namespace aljabr

using namespace aljabr;

extern "C" {

int aljabr_rocm_kv4_cache_bytes(const aljabr_rocm_kv4_cache *cache, size_t *codes_bytes, size_t *scales_bytes) {
    ALJ_REQUIRE(cache && codes_bytes && scales_bytes, "cache, codes_bytes and scales_bytes must be non-null");
    const bool paged = cache->num_blocks > 0;
    ALJ_REQUIRE((paged || cache->sequences > 0) && cache->n_kv_heads > 0 && cache->rows > 0 && cache->rows % 16 == 0,
                "sequences (or num_blocks) and n_kv_heads must be positive, rows a positive multiple of 16");
    if (cache->head_dim != 64 && cache->head_dim != 128 && cache->head_dim != 256)
        return fail(ALJABR_ROCM_ERR_UNSUPPORTED, "kv4_cache_bytes: head_dim %d is not 64, 128 or 256", cache->head_dim);
    const size_t of_each = static_cast<size_t>(cache->n_kv_heads) * cache->rows;      // below 2^62
    size_t rows, codes;
    ALJ_REQUIRE(!__builtin_mul_overflow(static_cast<size_t>(paged ? cache->num_blocks : cache->sequences), of_each, &rows) &&
                    !__builtin_mul_overflow(rows, static_cast<size_t>(cache->head_dim / 2), &codes),
                "kv4_cache_bytes: a plane of this shape has 2^64 bytes or more");
    *codes_bytes = codes;
    *scales_bytes = codes / 8;                               // 2 bytes for every 16 of codes
    return ALJABR_ROCM_OK;
}

int aljabr_rocm_kv4_write(const aljabr_rocm_kv4_cache *cache, const void *K, const void *V, const int *positions,
                          const int *counts, int T, long long stride_b, long long stride_t, long long stride_h, int type) {
    Kv4View v;
    int rc = kv4_view(cache, "kv4_write", v);
    if (rc == ALJABR_ROCM_OK) rc = check_rows("kv4_write", v, K, V, positions, T, stride_b, stride_t, stride_h, type);
    if (rc == ALJABR_ROCM_OK) rc = ensure_ready();
    if (rc == ALJABR_ROCM_OK) rc = enqueue_kv4_write(v, K, V, positions, counts, T, stride_b, stride_t, stride_h, type);
    return rc == ALJABR_ROCM_OK ? finish_launch("kv4_write") : rc;
}

int aljabr_rocm_kv4_read(void *K, void *V, const aljabr_rocm_kv4_cache *cache, const int *positions, const int *counts,
                         int T, long long stride_b, long long stride_t, long long stride_h, int type) {
    Kv4View v;
    int rc = kv4_view(cache, "kv4_read", v);
    if (rc == ALJABR_ROCM_OK) rc = check_rows("kv4_read", v, K, V, positions, T, stride_b, stride_t, stride_h, type);
    if (rc == ALJABR_ROCM_OK)      // rows read to one place: which stays would be chance
        ALJ_REQUIRE((stride_b || v.B == 1) && (stride_t || T == 1) && (stride_h || v.H == 1),
                    "kv4_read: a stride of 0 over several sequences, tokens or heads");
    if (rc == ALJABR_ROCM_OK) rc = ensure_ready();
    if (rc == ALJABR_ROCM_OK) rc = enqueue_kv4_read(v, K, V, positions, counts, T, stride_b, stride_t, stride_h, type);
    return rc == ALJABR_ROCM_OK ? finish_launch("kv4_read") : rc;
}

}  // extern "C"
