// kv4_rows.hip - attention of many stacked rows over the 4-bit cache: prompts,
// chunks of prompts, drafts of large groups (kv4_attention.hip has the
// formulas, the precision and the treatment of keys that are not finite).
//
// A workgroup takes 128 stacked rows. Two groups of four waves (one at D = 256,
// whose accumulators leave room for one wave a SIMD) take every other tile of
// 32 keys, a wave 32 rows. The group decodes its tile once for its four waves,
// into LDS as the fragments that v_mfma_f32_32x32x16_f16 takes:
//   K   [key][D + 8]: dword w of a row as the 8 halves at 8w, in decode8's
//       order, which the query's fragments follow;
//   V^T [16 x + n][36]: nibble x of dword n (D = 64: 16-bit piece n) of 32
//       keys, so that a thread that holds two keys' dword n writes a pair of
//       keys for each nibble.
// A tile is a phase of matrix products (O^T += V^T P^T of the tile before, then
// S^T = K Q^T) and a phase of vector work (the softmax, the decoding of the next
// tile), a barrier between them, and the two groups are a phase apart: on every
// SIMD one wave has the matrix cores while the other has the vector ALU. At the
// end the groups' states are joined through LDS. Rows run along the lanes: a
// row's query parts, maximum and sum stay in its two lanes.
#include "kv4_attention.hpp"

namespace aljabr {

using namespace kv4;

namespace {

typedef _Float16 half4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr int kGroup = 256;                  // threads that share a tile
constexpr int kVStride = kTile + 4;          // halves: 72-byte rows

template <int D>
struct Shape {
    static constexpr int kGroups = D == 256 ? 1 : 2;
    static constexpr int kThreads = kGroup * kGroups;
    static constexpr int kKStride = D + 8;                                 // halves
    static constexpr int kK = kTile * kKStride, kV = D * kVStride;         // halves of a tile's fragments
    static constexpr int kHalves = kK + 2 * kV;                            // a group's: V stays while the next tile is decoded
};

// A thread's share of a tile: dwords of one K row, and of two V rows.
template <int D>
struct Raw {
    uint32_t k[D / 64];
    uint32_t v[2][D == 256 ? 2 : 1];
    uint32_t ks, vs;                         // K's scale, the two V rows' scales
    bool ok;                                 // the rows' block exists (uniform)
};

template <class T>
__device__ __forceinline__ T load_at(const void *base, uint32_t off) {
    return *reinterpret_cast<const T *>(static_cast<const char *>(base) + off);
}

// `tid` is the thread's number in its group. Threads of a wave hold 8 neighbouring keys, of one 16-key half: key 8w + i / 8 of K, 8w + 2 (i / 16) of V.
template <int D, bool PAGED>
__device__ __forceinline__ void load_raw(const Params &p, int b, int kvh, int n_keys, int kt, int tid, Raw<D> &x) {
    const int u = __builtin_amdgcn_readfirstlane(tid >> 7);
    int key = kt * kTile + 16 * u;
    if (key >= n_keys) key = kt * kTile;
    int s = b, row = key;
    x.ok = true;
    if constexpr (PAGED) {
        const int blk = p.by_rows(key);
        s = p.v.table[static_cast<long long>(b) * p.v.max_blocks + blk];
        row = key - blk * p.v.R;
        x.ok = s >= 0 && s < p.v.num_blocks;
        if (!x.ok) s = 0;
    }
    const long long head = static_cast<long long>(s) * p.v.H + kvh;
    const uint8_t *kc = p.v.kc + (head * p.v.R + row) * (D / 2), *vc = p.v.vc + (head * p.v.R + row) * (D / 2);
    const uint16_t *ks = p.v.ks + head * (D / 32) * p.v.R + row, *vs = p.v.vs + head * (D / 32) * p.v.R + row;
    // K row of the half and its first dword; first V row of the half.
    const uint32_t kk = tid >> 3 & 15, kd = (tid & 7) * (D / 64), vk = 2 * (tid >> 4 & 7), n = tid & 15;
    const uint32_t kat = kk * (D / 2) + 4 * kd, vat = vk * (D / 2) + (D == 64 ? 4 * (n >> 1) : D == 128 ? 4 * n : 8 * n);
    if constexpr (D == 64) {
        x.k[0] = load_at<uint32_t>(kc, kat);
    } else if constexpr (D == 128) {
        const uint2 a = load_at<uint2>(kc, kat);
        x.k[0] = a.x; x.k[1] = a.y;
    } else {
        const uint4 a = load_at<uint4>(kc, kat);
        x.k[0] = a.x; x.k[1] = a.y; x.k[2] = a.z; x.k[3] = a.w;
    }
    x.ks = load_at<uint16_t>(ks, 2 * ((kd >> 2) * p.v.R + kk));
#pragma unroll
    for (int r = 0; r < 2; ++r) {
        if constexpr (D == 256) {
            const uint2 a = load_at<uint2>(vc, vat + r * (D / 2));
            x.v[r][0] = a.x;
            x.v[r][1] = a.y;
        } else {
            x.v[r][0] = load_at<uint32_t>(vc, vat + r * (D / 2));
        }
    }
    x.vs = load_at<uint32_t>(vs, 2 * ((D == 64 ? n >> 3 : D == 128 ? n >> 2 : n >> 1) * p.v.R + vk));
}

// Bit u: half u of a tile is on a block that exists (a half past the end counts as the first).
template <bool PAGED>
__device__ __forceinline__ uint32_t half_ok(const Params &p, int b, int n_keys, int kt) {
    uint32_t m = 0;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
        int key = kt * kTile + 16 * u;
        if (key >= n_keys) key = kt * kTile;
        const int s = PAGED ? p.v.table[static_cast<long long>(b) * p.v.max_blocks + p.by_rows(key)] : 0;
        m |= s >= 0 && s < p.v.num_blocks ? 1u << u : 0;
    }
    return m;
}
template <bool PAGED>
__device__ __forceinline__ bool both_ok(const Params &p, int b, int n_keys, int kt) {
    return !PAGED || half_ok<PAGED>(p, b, n_keys, kt) == 3;
}

// Decodes a thread's share into the tile's fragments. `edge`: some row does not see some key; scales of V rows past
// the end, or on no block, are then taken as 0, and one that is not finite too, with its key's bit set in bad[block].
template <int D>
__device__ __forceinline__ void decode_tile(const Magic &g, const Raw<D> &x, int k0, int n_keys, bool edge, int tid,
                                            _Float16 *kbuf, _Float16 *vbuf, uint32_t *bad) {
    const int key = tid >> 3, kd = (tid & 7) * (D / 64);
    const half2v kdup = as_half2(__builtin_amdgcn_perm(x.ks, x.ks, 0x01000100u));
#pragma unroll
    for (int i = 0; i < D / 64; ++i) {
        uint32_t f[4];
        decode8(g, x.k[i], kdup, f);
        *reinterpret_cast<uint4 *>(kbuf + key * Shape<D>::kKStride + 8 * (kd + i)) = make_uint4(f[0], f[1], f[2], f[3]);
    }
    const int pr = tid >> 4, n = tid & 15;                                 // pair of keys 2 pr, 2 pr + 1
    half2v vd = as_half2(x.vs);
    if (edge) {
        const int vg = D == 64 ? n >> 3 : D == 128 ? n >> 2 : n >> 1;
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            if (k0 + 2 * pr + r >= n_keys || !x.ok) vd[r] = static_cast<_Float16>(0.0f);
            if (not_finite(vd[r])) {
                vd[r] = static_cast<_Float16>(0.0f);
                atomicOr(bad + vg, 1u << (2 * pr + r));
            }
        }
    }
    _Float16 *vt = vbuf + n * kVStride + 2 * pr;
#pragma unroll
    for (int i = 0; i < (D == 256 ? 2 : 1); ++i)
#pragma unroll
        for (int half = 0; half < (D == 64 ? 1 : 2); ++half) {
            const uint32_t sel = D == 64 ? (n & 1 ? 0x07060302u : 0x05040100u) : half ? 0x07060302u : 0x05040100u;
            uint32_t f[4];
            decode8(g, __builtin_amdgcn_perm(x.v[1][i], x.v[0][i], sel), vd, f);
#pragma unroll
            for (int j = 0; j < 4; ++j) *reinterpret_cast<uint32_t *>(vt + 16 * (8 * i + 4 * half + j) * kVStride) = f[j];
        }
}

// The row group of the i-th set of items: the last, of most keys when causal, first.
__device__ __forceinline__ int group_of(const Params &p, int i) { return p.row_groups - 1 - i; }

template <int D, bool PAGED, bool CAP>
__global__ __launch_bounds__(Shape<D>::kThreads, D == 256 ? 1 : 2) void kv4_rows_kernel(Params p) {
    constexpr int STEPS = D / 16, DT = D / 32, KS = Shape<D>::kKStride, GROUPS = Shape<D>::kGroups;
    __shared__ __attribute__((aligned(16))) _Float16 lds[GROUPS * Shape<D>::kHalves];
    __shared__ uint32_t bad[GROUPS][3][8];                                 // per tile in flight and block: keys not finite
    __shared__ float joint[3][kRowsBlock];                                 // the second group's m, l and poison
    const int lane = threadIdx.x & 63, h = lane >> 5, nl = lane & 31;
    const int grp = GROUPS == 1 ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x / kGroup), tid = threadIdx.x % kGroup;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    _Float16 *kbuf = lds + grp * Shape<D>::kHalves, *vbufs = kbuf + Shape<D>::kK;
    const Magic g;

    // With p.pairs a workgroup takes a row group of many keys and then one of few, so that all have alike.
    for (int pass = 0; pass < (p.pairs ? 2 : 1); ++pass) {
    int item, w;
    work_of(p, blockIdx.x, item, w);
    if (pass) {
        const int i = p.by_heads(item), other = p.row_groups - 1 - i;
        if (other <= i) return;
        item += (other - i) * p.v.H;
        __syncthreads();                                                   // the first pass has left LDS
    }
    const int group = group_of(p, p.by_heads(item)), kvh = item - p.by_heads(item) * p.v.H;
    const int r0 = group * kRowsBlock;
    const Chunk chunk = find_chunk(p, w, r0, kRowsBlock, 4);
    if (chunk.b < 0) {
        if (p.pairs) continue;
        return;
    }
    const int b = chunk.b, t0 = chunk.t0, t1 = chunk.t1;
    if (p.quota && w == chunk.first && threadIdx.x == 0)
        p.chunks[static_cast<long long>(item) * p.v.B + b] = make_int2(chunk.first, chunk.count);
    const Seq seq = chunk.seq;
    const int r1 = min(r0 + kRowsBlock, seq.cnt * p.G);
    const int w0 = r0 + 32 * wave;
    if (tid < 24) (&bad[grp][0][0])[tid] = 0;

    Raw<D> raw;
    if (t0 + grp < t1) load_raw<D, PAGED>(p, b, kvh, seq.n, t0 + grp, tid, raw);

    // This lane's row, its keys, and the wave's and the workgroup's.
    const int r = min(w0 + nl, r1 - 1);                                    // lanes past the rows repeat the last and are not stored
    const int t = p.by_g(r);
    int lo, hi, x;
    key_range(p, seq, t, lo, hi);
    int w_lo, w_hi, full_lo, full_hi, all_lo, all_hi;                      // keys that a row of the wave sees; that all its rows see; all of the workgroup's
    key_range(p, seq, p.by_g(min(w0, r1 - 1)), w_lo, full_hi);
    key_range(p, seq, p.by_g(min(w0 + 31, r1 - 1)), full_lo, w_hi);
    key_range(p, seq, p.by_g(r0), x, all_hi);
    key_range(p, seq, p.by_g(r1 - 1), all_lo, x);
    const bool idle = w0 >= r1;                                            // a wave without rows only decodes

    // The row times scale * log2(e) as two fp16 parts: step s holds dword 2s + h, in decode8's order.
    half8 qh[STEPS], ql[STEPS];
    float unscale;
    {
        const float *qr = p.q + ((static_cast<long long>(b) * p.T + t) * p.Hq + kvh * p.G + (r - t * p.G)) * D + 4 * h;
        const float qs = p.scale * kLog2e;
        float top = 0.0f;
#pragma unroll
        for (int s = 0; s < STEPS; ++s) {
            const float4 a = *reinterpret_cast<const float4 *>(qr + 32 * (s >> 1) + 8 * (s & 1));
            const float4 c = *reinterpret_cast<const float4 *>(qr + 32 * (s >> 1) + 8 * (s & 1) + 16);
            top = fmaxf(top, fmaxf(fmaxf(fmaxf(fabsf(a.x), fabsf(a.y)), fmaxf(fabsf(a.z), fabsf(a.w))),
                                   fmaxf(fmaxf(fabsf(c.x), fabsf(c.y)), fmaxf(fabsf(c.z), fabsf(c.w)))));
        }
        top = fmaxf(top, __shfl_xor(top, 32)) * qs;
        int e = 0;
        if (top > 0.0f && top <= 3.4028235e38f) (void)frexpf(top, &e);     // top in [2^(e-1), 2^e)
        e = e < -100 ? -100 : e;
        const float up = ldexpf(1.0f, 15 - e);
        unscale = ldexpf(1.0f, e - 15);
#pragma unroll
        for (int s = 0; s < STEPS; ++s) {
            const float4 a = *reinterpret_cast<const float4 *>(qr + 32 * (s >> 1) + 8 * (s & 1));
            const float4 c = *reinterpret_cast<const float4 *>(qr + 32 * (s >> 1) + 8 * (s & 1) + 16);
            const float y[8] = {a.x, a.z, c.x, c.z, a.y, a.w, c.y, c.w};
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float v = y[i] * qs * up;
                qh[s][i] = static_cast<_Float16>(v);
                ql[s][i] = static_cast<_Float16>(v - static_cast<float>(qh[s][i]));
            }
        }
    }

    f32x16 o[DT];
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) o[dt] = f32x16{};
    float m = -INFINITY, l = 0.0f;
    uint32_t poison = 0;                                                   // blocks of 32 dims with a visible key that is not finite

    auto edge_of = [&](int kt) { return kt * kTile < all_lo || kt * kTile + kTile > all_hi || !both_ok<PAGED>(p, b, seq.n, kt); };
    auto live_of = [&](int kt) { return !idle && kt < t1 && kt * kTile < w_hi && kt * kTile + kTile > w_lo; };
    auto decode = [&](int kt, int j, int slot) __attribute__((always_inline)) {
        decode_tile<D>(g, raw, kt * kTile, seq.n, edge_of(kt), tid, kbuf, vbufs + (j & 1) * Shape<D>::kV, bad[grp][slot]);
    };
    half8 ph[2], pl[2];                                                    // the weights as two fp16 parts
    // O^T += V^T P^T: lane half h supplies contraction entries 0..3 -> key 16j + 4h + e and 4..7 -> key 16j + 8 + 4h + e - 4.
    auto add_values = [&](int j2) __attribute__((always_inline)) {
        const _Float16 *vl = vbufs + (j2 & 1) * Shape<D>::kV;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            half8 a[DT];
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) {
                const _Float16 *at = vl + (32 * dt + nl) * kVStride + 16 * j + 4 * h;
                const half4 a0 = *reinterpret_cast<const half4 *>(at), a1 = *reinterpret_cast<const half4 *>(at + 8);
                a[dt] = half8{a0[0], a0[1], a0[2], a0[3], a1[0], a1[1], a1[2], a1[3]};
            }
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) o[dt] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a[dt], pl[j], o[dt], 0, 0, 0);
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) o[dt] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a[dt], ph[j], o[dt], 0, 0, 0);
        }
    };

    const int tiles = (t1 - t0 + GROUPS - 1) / GROUPS;                     // of a group, the second's last may not exist
    __syncthreads();                                                       // `bad` is clear
    if (t0 + grp < t1) {
        decode(t0 + grp, 0, 0);
        if (t0 + grp + GROUPS < t1) load_raw<D, PAGED>(p, b, kvh, seq.n, t0 + grp + GROUPS, tid, raw);
    }
    __syncthreads();
    if (grp) __syncthreads();                                              // a phase behind the first group
    bool pending = false;                                                  // ph and pl hold weights of the tile before
    for (int j = 0, slot = 0; j < tiles; ++j, slot = slot == 2 ? 0 : slot + 1) {
        const int kt = t0 + grp + GROUPS * j, k0 = kt * kTile, slot1 = slot == 2 ? 0 : slot + 1;
        // ---- matrix products
        const bool live = live_of(kt);
        if (pending) add_values(j - 1);
        f32x16 s = {};
        if (live) {
            // S^T in two chains (a product that waits for the one before it takes twice its time): accumulator i is
            // key k0 + 8 (i / 4) + 4h + i % 4 of this lane's row.
            f32x16 s1 = {};
#pragma unroll
            for (int st = 0; st < STEPS; ++st) {
                const half8 a = *reinterpret_cast<const half8 *>(kbuf + nl * KS + 16 * st + 8 * h);
                s1 = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, ql[st], s1, 0, 0, 0);
                s = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, qh[st], s, 0, 0, 0);
            }
#pragma unroll
            for (int i = 0; i < 16; ++i) s[i] += s1[i];
        }
        __syncthreads();
        // ---- vector work
        if (tid < 8) bad[grp][slot1 == 2 ? 0 : slot1 + 1][tid] = 0;        // the tile before's
        if (kt + GROUPS < t1) {
            decode(kt + GROUPS, j + 1, slot1);
            if (kt + 2 * GROUPS < t1) load_raw<D, PAGED>(p, b, kvh, seq.n, kt + 2 * GROUPS, tid, raw);
        }
        pending = live;
        if (live) {
            const float us = CAP ? 1.0f : unscale;
            if constexpr (CAP) {
                const float cap = p.soft_cap * kLog2e, in = unscale / cap;
#pragma unroll
                for (int i = 0; i < 16; ++i) s[i] = cap * tanhf(s[i] * in);
            }
            const bool ok = both_ok<PAGED>(p, b, seq.n, kt);
            if (k0 < full_lo || k0 + kTile > full_hi || !ok) {
                const int first = lo - k0 - 4 * h, end = hi - k0 - 4 * h;
                const uint32_t there = ok ? 3 : half_ok<PAGED>(p, b, seq.n, kt);          // halves on blocks that exist
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const int c = 8 * (i >> 2) + (i & 3);
                    if (c < first || c >= end || !(there >> (i >> 3) & 1)) s[i] = -INFINITY;
                }
            }
            if (edge_of(kt)) {
                // Keys of this tile that the row sees, against the ones that are not finite.
                const int a = max(lo - k0, 0), z = min(hi - k0, kTile);
                const uint32_t see = z <= a ? 0 : (z == 32 ? 0xffffffffu : (1u << z) - 1) & ~((1u << a) - 1);
#pragma unroll
                for (int q = 0; q < DT; ++q) poison |= bad[grp][slot][q] & see ? 1u << q : 0;
            }
            float mx = s[0];
#pragma unroll
            for (int i = 1; i < 16; ++i) mx = fmaxf(mx, s[i]);
            mx *= us;
            // The row's reference m is raised only when a score exceeds it by more than 2.
            if (__any(mx > m + 2.0f)) {
                mx = fmaxf(mx, __shfl_xor(mx, 32));
                const float up = mx > m + 2.0f ? mx : m;
                const float alpha = up == m ? 1.0f : __builtin_amdgcn_exp2f(m - up);              // 0 while m is -inf
                l *= alpha;
#pragma unroll
                for (int dt = 0; dt < DT; ++dt) o[dt] *= alpha;
                m = up;
            }
            const float ref = m == -INFINITY ? 0.0f : m;
            float sum[4] = {};
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                float e[2];
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    e[c] = __builtin_amdgcn_exp2f(fmaf(s[2 * i + c], us, -ref)) * kWeightScale;
                    sum[(2 * i + c) & 3] += e[c];
                }
                const half2v first = pair(e[0], e[1]);
                const half2v rest = pair(e[0] - static_cast<float>(first[0]), e[1] - static_cast<float>(first[1]));
                ph[i >> 2][2 * (i & 3)] = first[0];
                ph[i >> 2][2 * (i & 3) + 1] = first[1];
                pl[i >> 2][2 * (i & 3)] = rest[0];
                pl[i >> 2][2 * (i & 3) + 1] = rest[1];
            }
            l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
        }
        __syncthreads();
    }
    if (pending) add_values(tiles - 1);
    if (GROUPS == 2 && !grp) __syncthreads();

    l += __shfl_xor(l, 32);
    if (m == -INFINITY && l != l) m = 0.0f;                                // a NaN score alone leaves no reference
    const bool whole = chunk.count == 1;
    const long long part = (static_cast<long long>(w) * p.v.H * p.row_groups + item) * kRowsBlock + 32 * wave;
    // The groups' states in one reference; O through LDS, so that whole lines are stored: rounds of two blocks of dims
    // (D = 64: of one), a wave's own [32 rows][block of h][32]. Accumulator j of tile dt is row
    // 32 dt + 8 (j / 4) + 4h + j % 4 of V^T: nibble 2 dt + j / 8 of piece n = 8 (j / 4 % 2) + 4h + j % 4.
    constexpr int SPAN = D == 64 ? 32 : 64, STRIDE = SPAN + 4, ROUNDS = D / SPAN, LPR = SPAN / 4;
    static_assert(sizeof(lds) >= kRowsBlock * STRIDE * sizeof(float), "room for a round");
    float *st = reinterpret_cast<float *>(lds) + wave * 32 * STRIDE;
    float f = 1.0f;
    if constexpr (GROUPS == 2) {
        const int lr = 32 * wave + nl;
        // First the second group's state, then the joint one.
        if (grp && h == 0) {
            joint[0][lr] = m;
            joint[1][lr] = l;
            joint[2][lr] = __uint_as_float(poison);
        }
        __syncthreads();
        float m2 = 0.0f, l2 = 0.0f;
        if (!grp) {
            m2 = joint[0][lr];
            l2 = joint[1][lr];
            poison |= __float_as_uint(joint[2][lr]);
        }
        __syncthreads();
        if (!grp) {
            const float M = fmaxf(m, m2);
            f = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - M);
            const float f2 = m2 == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m2 - M);
            l = fmaf(l, f, l2 * f2);
            m = M;
            const float norm = whole ? (l == 0.0f ? 0.0f : 1.0f / l) : 1.0f;
            f *= norm;
            if (h == 0) joint[0][lr] = f2 * norm;
        }
        __syncthreads();
        if (grp) f = joint[0][lr];
    } else {
        f = whole ? (l == 0.0f ? 0.0f : 1.0f / l) : 1.0f;
        __syncthreads();                                                   // every wave is done with the tiles
    }
    if (!grp && !whole && h == 0 && w0 + nl < r1) *reinterpret_cast<float2 *>(p.part_ml + (part + nl) * 2) = make_float2(m, l);
#pragma unroll
    for (int rd = 0; rd < ROUNDS; ++rd) {
        const int u = D == 256 ? rd >> 1 : rd, sub = rd & 1;               // D = 256: j % 4 / 2 == sub
        // This lane's values of the round into its places, added to what the second group left there.
        auto put = [&](bool add) __attribute__((always_inline)) {
#pragma unroll
            for (int j = 0; j < 16; ++j) {
                if ((j >> 2 & 1) != u || (D == 256 && (j >> 1 & 1) != sub)) continue;
                const int odd = j >> 3;
                if constexpr (D == 64) {
                    float2 *at = reinterpret_cast<float2 *>(st + nl * STRIDE + 16 * odd + 4 * (2 * h + (j >> 1 & 1)) + 2 * (j & 1));
                    const float2 y = add ? *at : make_float2(0.0f, 0.0f);
                    *at = make_float2(fmaf(o[0][j], f, y.x), fmaf(o[1][j], f, y.y));
                } else {
#pragma unroll
                    for (int c = 0; c < DT / 4; ++c) {
                        float4 *at = reinterpret_cast<float4 *>(st + nl * STRIDE + 32 * h + 16 * odd +
                                                                (D == 128 ? 4 * (j & 3) : 8 * (j & 1) + 4 * c));
                        const float4 y = add ? *at : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                        *at = make_float4(fmaf(o[4 * c][j], f, y.x), fmaf(o[4 * c + 1][j], f, y.y), fmaf(o[4 * c + 2][j], f, y.z),
                                          fmaf(o[4 * c + 3][j], f, y.w));
                    }
                }
            }
        };
        if constexpr (GROUPS == 2) {
            if (grp) put(false);
            __syncthreads();
            if (!grp) put(true);
        } else {
            put(false);
        }
        if (!grp) {
            if (poison && (D != 64 || h == 0)) {
                const int own = D == 64 ? u : D == 128 ? 2 * u + h : 4 * u + 2 * h + sub;
                if (poison >> own & 1)
                    for (int i = 0; i < 32; ++i) st[nl * STRIDE + (D == 64 ? 0 : 32 * h) + i] = NAN;
            }
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");             // the wave's own writes
#pragma unroll
            for (int i = 0; i < 32 * LPR / 64; ++i) {
                const int lr = (64 * i + lane) / LPR, d = 4 * ((64 * i + lane) % LPR), rr = w0 + lr;
                if (rr < r1) {
                    const float4 val = *reinterpret_cast<const float4 *>(st + lr * STRIDE + d);
                    const int block = D == 64 ? u : D == 128 ? 2 * u + (d >> 5) : 4 * u + 2 * (d >> 5) + sub;
                    const int tt = p.by_g(rr);
                    float *dst = whole ? p.out + ((static_cast<long long>(b) * p.T + tt) * p.Hq + kvh * p.G + (rr - tt * p.G)) * D
                                       : p.part_o + (part + lr) * D;
                    *reinterpret_cast<float4 *>(dst + 32 * block + (d & 31)) = val;
                }
            }
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");             // read before the next round's writes
        }
        if constexpr (GROUPS == 2) __syncthreads();
    }
    }
}

// A wave a row of a sequence with several chunks: D/4 lanes take a chunk's
// partial as float4s (64 / (D/4) chunks at once), folded in order, then across
// the lane groups.
template <int D>
__global__ __launch_bounds__(256) void kv4_merge_rows_kernel(Params p, long long rows) {
    constexpr int LPS = D / 4, SG = 64 / LPS;
    const long long row = static_cast<long long>(blockIdx.x) * 4 + (threadIdx.x >> 6);
    if (row >= rows) return;
    const int bt = static_cast<int>(row / p.Hq), hq = static_cast<int>(row - static_cast<long long>(bt) * p.Hq);
    const int b = bt / p.T, t = bt - b * p.T;
    const int kvh = p.by_g(hq), r = t * p.G + hq - kvh * p.G;
    const int item = group_of(p, r / kRowsBlock) * p.v.H + kvh;
    const int2 chunk = p.chunks[static_cast<long long>(item) * p.v.B + b];   // written for the rows that exist
    if (t >= sequence(p, b).cnt || chunk.y <= 1) return;   // no row, or its one chunk wrote it
    const long long step = static_cast<long long>(p.v.H) * p.row_groups * kRowsBlock;
    const long long first = chunk.x * step + static_cast<long long>(item) * kRowsBlock + r % kRowsBlock;
    const int lane = threadIdx.x & 63, sg = lane / LPS, j = lane % LPS;
    float m = -INFINITY, l = 0.0f;
    float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    constexpr int U = 4;                                   // chunks in flight per lane group
    for (int s0 = sg; s0 < chunk.y; s0 += U * SG) {
        float2 ml[U];
        float4 os[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const long long s = s0 + u * SG < chunk.y ? s0 + u * SG : s0;
            ml[u] = *reinterpret_cast<const float2 *>(p.part_ml + (first + s * step) * 2);
            os[u] = *reinterpret_cast<const float4 *>(p.part_o + (first + s * step) * D + 4 * j);
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (s0 + u * SG < chunk.y) fold(m, l, o, ml[u].x, ml[u].y, os[u]);
    }
#pragma unroll
    for (int off = LPS; off < 64; off <<= 1) {
        const float m2 = __shfl_xor(m, off), l2 = __shfl_xor(l, off);
        const float4 o2 = make_float4(__shfl_xor(o.x, off), __shfl_xor(o.y, off), __shfl_xor(o.z, off), __shfl_xor(o.w, off));
        fold(m, l, o, m2, l2, o2);
    }
    const float f = l == 0.0f ? 0.0f : 1.0f / l;
    if (sg == 0) *reinterpret_cast<float4 *>(p.out + row * D + 4 * j) = make_float4(o.x * f, o.y * f, o.z * f, o.w * f);
}

template <int D, bool PAGED>
void launch_typed(const Params &p, hipStream_t s) {
    const int items = p.v.H * (p.pairs ? (p.row_groups + 1) / 2 : p.row_groups);
    const dim3 grid(items * (p.quota ? p.quota + (p.v.B > 1 ? p.v.B : 0) : p.v.B)), block(Shape<D>::kThreads);
    if (p.soft_cap > 0.0f)
        hipLaunchKernelGGL((kv4_rows_kernel<D, PAGED, true>), grid, block, 0, s, p);
    else
        hipLaunchKernelGGL((kv4_rows_kernel<D, PAGED, false>), grid, block, 0, s, p);
    const long long rows = static_cast<long long>(p.v.B) * p.T * p.Hq;
    if (p.quota)
        hipLaunchKernelGGL((kv4_merge_rows_kernel<D>), dim3(static_cast<unsigned>((rows + 3) / 4)), dim3(256), 0, s, p, rows);
}

template <int D>
void launch_d(const Params &p, hipStream_t s) {
    p.v.table ? launch_typed<D, true>(p, s) : launch_typed<D, false>(p, s);
}

}  // namespace

void kv4::launch_rows(const Params &p, hipStream_t s) {
    if (p.v.D == 64) launch_d<64>(p, s);
    else if (p.v.D == 128) launch_d<128>(p, s);
    else launch_d<256>(p, s);
}

}  // namespace aljabr
