// kv4_rows.hip - attention of many stacked rows over the 4-bit cache: prompts,
// chunks of prompts, drafts of large groups (kv4_attention.hip has the
// formulas, the precision and the treatment of keys that are not finite).
//
// A workgroup takes 128 stacked rows, 32 a wave, and walks tiles of 32 keys.
// Its four waves decode a tile once for all of them, into LDS as the fp16
// fragments that v_mfma_f32_32x32x16_f16 takes:
//   K   [key][D + 8]: dword w of a row as the 8 halves at 8w, in decode8's
//       order, which the query's fragments follow;
//   V^T [16 x + n][36]: nibble x of dword n (D = 64: 16-bit piece n) of 32
//       keys, so that a thread that holds two keys' dword n writes a pair of
//       keys for each nibble.
// The next tile is decoded into the other buffer before this one is used, and
// the one after that is on its way in registers: one barrier a tile.
//   S^T = K Q^T, O^T += V^T P^T, rows along the lanes: a row's query parts,
// maximum and sum stay in its two lanes.
// Two products a score and a value, for the two fp16 parts of queries and
// weights. Measured: a causal prompt of 2048 rows of 32 heads of 128 99 us (0.35
// PFLOP/s, 0.70 with both parts; matrix cores 26 %, vector ALU 35 %), 256 rows
// over 2048 keys 36.6 us with the merge (19 %, 30 %); with heads of 64 68 and
// 31 us. The waves' products and softmax go in turn:
// what a CU's other workgroup covers is lost where the last rows of a causal
// prompt, of the most keys, run alone. The next tile's decoding is laid between
// the score products (3 % of a prompt of 4096 rows). D = 256 has one buffer and
// two barriers a tile, one workgroup a CU (512 registers; with a soft cap 24
// bytes a lane spill), and takes 212 us and 70 us.
#include "kv4_attention.hpp"

namespace aljabr {

using namespace kv4;

namespace {

typedef _Float16 half4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr int kThreads = 256;
constexpr int kVStride = kTile + 4;          // halves: 72-byte rows

template <int D>
struct Shape {
    static constexpr int kKStride = D + 8;                                 // halves
    static constexpr int kHalves = kTile * kKStride + D * kVStride;        // of a decoded tile
    static constexpr int kBuffers = D == 256 ? 1 : 2;                      // as many as fit 64 KB
    static constexpr int kPieces = D == 256 ? 2 : 1;                       // dwords of a V row a thread decodes
};

// A thread's share of a tile: dwords of one K row, and of two V rows.
template <int D>
struct Raw {
    uint32_t k[D / 64];
    uint32_t v[2][D == 256 ? 2 : 1];
    uint32_t ks, vs;                         // K's scale, the two V rows' scales
    bool ok;                                 // the rows' block exists (uniform)
};

// Threads of a wave hold 8 neighbouring keys, of one 16-key half: key 8w + i / 8 of K, 8w + 2 (i / 16) of V.
template <int D, bool PAGED>
__device__ __forceinline__ void load_raw(const Params &p, int b, int kvh, int n_keys, int kt, int tid, Raw<D> &x) {
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), u = wave >> 1;
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
    const int kk = (tid >> 3) & 15, kd = (tid & 7) * (D / 64);             // K row of the half, first dword
    const uint32_t *ksrc = reinterpret_cast<const uint32_t *>(kc + kk * (D / 2)) + kd;
    if constexpr (D == 64) {
        x.k[0] = ksrc[0];
    } else if constexpr (D == 128) {
        const uint2 a = *reinterpret_cast<const uint2 *>(ksrc);
        x.k[0] = a.x; x.k[1] = a.y;
    } else {
        const uint4 a = *reinterpret_cast<const uint4 *>(ksrc);
        x.k[0] = a.x; x.k[1] = a.y; x.k[2] = a.z; x.k[3] = a.w;
    }
    x.ks = ks[static_cast<uint32_t>(kd >> 2) * p.v.R + kk];
    const int vk = 2 * ((tid >> 4) & 7), n = tid & 15;                     // first V row of the half
#pragma unroll
    for (int r = 0; r < 2; ++r) {
        const uint32_t *vsrc = reinterpret_cast<const uint32_t *>(vc + (vk + r) * (D / 2));
        if constexpr (D == 256) {
            const uint2 a = *reinterpret_cast<const uint2 *>(vsrc + 2 * n);
            x.v[r][0] = a.x;
            x.v[r][1] = a.y;
        } else {
            x.v[r][0] = vsrc[D == 64 ? n >> 1 : n];
        }
    }
    const int vg = D == 64 ? n >> 3 : D == 128 ? n >> 2 : n >> 1;
    x.vs = *reinterpret_cast<const uint32_t *>(vs + static_cast<uint32_t>(vg) * p.v.R + vk);
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

// The scales of a thread's two V rows. `edge`: some row does not see some key; scales of V rows past the end, or on
// no block, are then taken as 0, and one that makes a value of the thread's not finite too, with its key's bit set in
// bad[block].
template <int D>
__device__ __forceinline__ half2v value_scales(const Magic &g, const Raw<D> &x, int k0, int n_keys, bool edge, int tid, uint32_t *bad) {
    const int pr = tid >> 4, n = tid & 15;                                 // pair of keys 2 pr, 2 pr + 1
    half2v vd = as_half2(x.vs);
    if (edge) {
        const int vg = D == 64 ? n >> 3 : D == 128 ? n >> 2 : n >> 1;
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            if (k0 + 2 * pr + r >= n_keys || !x.ok) vd[r] = static_cast<_Float16>(0.0f);
            if (may_overflow(vd[r])) {
                const uint32_t w = x.v[r][0];
                bool over = overflows(g, D == 64 ? __builtin_amdgcn_perm(w, w, n & 1 ? 0x03020302u : 0x01000100u) : w, vd[r]);
                if constexpr (D == 256) over |= overflows(g, x.v[r][1], vd[r]);
                if (over) {
                    vd[r] = static_cast<_Float16>(0.0f);
                    atomicOr(bad + vg, 1u << (2 * pr + r));
                }
            }
        }
    }
    return vd;
}

// Decodes a thread's share into the tile's fragments.
template <int D>
__device__ __forceinline__ void decode_tile(const Magic &g, const Raw<D> &x, half2v vd, int tid, _Float16 *buf) {
    const int key = tid >> 3, kd = (tid & 7) * (D / 64);
    const half2v kdup = as_half2(__builtin_amdgcn_perm(x.ks, x.ks, 0x01000100u));
#pragma unroll
    for (int i = 0; i < D / 64; ++i) {
        uint32_t f[4];
        decode8(g, x.k[i], kdup, f);
        *reinterpret_cast<uint4 *>(buf + key * Shape<D>::kKStride + 8 * (kd + i)) = make_uint4(f[0], f[1], f[2], f[3]);
    }
    const int pr = tid >> 4, n = tid & 15;                                 // pair of keys 2 pr, 2 pr + 1
    _Float16 *vt = buf + kTile * Shape<D>::kKStride + n * kVStride + 2 * pr;
#pragma unroll
    for (int i = 0; i < Shape<D>::kPieces; ++i)
#pragma unroll
        for (int half = 0; half < (D == 64 ? 1 : 2); ++half) {
            const uint32_t sel = D == 64 ? (n & 1 ? 0x07060302u : 0x05040100u) : half ? 0x07060302u : 0x05040100u;
            uint32_t f[4];
            decode8(g, __builtin_amdgcn_perm(x.v[1][i], x.v[0][i], sel), vd, f);
#pragma unroll
            for (int j = 0; j < 4; ++j) *reinterpret_cast<uint32_t *>(vt + 16 * (8 * i + 4 * half + j) * kVStride) = f[j];
        }
}

// The row group of the item group i, and the other way round: the last, of most keys when causal, first.
__device__ __forceinline__ int group_of(const Params &p, int i) { return p.row_groups - 1 - i; }

template <int D, bool PAGED, bool CAP>
__global__ __launch_bounds__(kThreads, D == 256 ? 1 : 2) void kv4_rows_kernel(Params p) {
    constexpr int STEPS = D / 16, DT = D / 32, KS = Shape<D>::kKStride, BUFS = Shape<D>::kBuffers;
    __shared__ __attribute__((aligned(16))) _Float16 lds[BUFS * Shape<D>::kHalves];
    __shared__ uint32_t bad[3][8];                                         // per tile in flight and block: keys not finite
    const int tid = threadIdx.x, lane = tid & 63, h = lane >> 5, nl = lane & 31;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    int item, w;
    work_of(p, blockIdx.x, item, w);
    const int group = group_of(p, p.by_heads(item)), kvh = item - p.by_heads(item) * p.v.H;
    const int r0 = group * kRowsBlock;
    const Chunk chunk = find_chunk(p, w, r0, kRowsBlock, kRowsLeast);
    if (chunk.b < 0) return;
    const int b = chunk.b, t0 = chunk.t0, t1 = chunk.t1;
    if (p.quota && w == chunk.first && tid == 0)
        p.chunks[static_cast<long long>(item) * p.v.B + b] = make_int2(chunk.slot, chunk.count);
    const Seq seq = chunk.seq;
    const int r1 = min(r0 + kRowsBlock, seq.cnt * p.G);
    const int w0 = r0 + 32 * wave;
    const Magic g;
    if (tid < 24) (&bad[0][0])[tid] = 0;

    Raw<D> raw;
    if (t0 < t1) load_raw<D, PAGED>(p, b, kvh, seq.n, t0, tid, raw);

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
        float top = 0.0f;
        float4 qa[STEPS], qc[STEPS];
#pragma unroll
        for (int s = 0; s < STEPS; ++s) {
            qa[s] = *reinterpret_cast<const float4 *>(qr + 32 * (s >> 1) + 8 * (s & 1));
            qc[s] = *reinterpret_cast<const float4 *>(qr + 32 * (s >> 1) + 8 * (s & 1) + 16);
        }
#pragma unroll
        for (int s = 0; s < STEPS; ++s) {
            const float4 a = qa[s], c = qc[s];
            top = fmaxf(top, fmaxf(fmaxf(fmaxf(fabsf(a.x), fabsf(a.y)), fmaxf(fabsf(a.z), fabsf(a.w))),
                                   fmaxf(fmaxf(fabsf(c.x), fabsf(c.y)), fmaxf(fabsf(c.z), fabsf(c.w)))));
        }
        top = fmaxf(top, __shfl_xor(top, 32)) * p.scale;
        int e = 0;
        if (top > 0.0f && top <= 3.4028235e38f) (void)frexpf(top, &e);     // top in [2^(e-1), 2^e)
        e = e < -100 ? -100 : e;
        const float up = ldexpf(1.0f, 15 - e);             // a power of two: y is the same number wherever it is used
        unscale = ldexpf(p.unscale, e - 15);
#pragma unroll
        for (int s = 0; s < STEPS; ++s) {
            const float4 a = qa[s], c = qc[s];
            const float y[8] = {a.x, a.z, c.x, c.z, a.y, a.w, c.y, c.w};
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float v = y[i] * p.scale * up;
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

    auto read_values = [&](const _Float16 *vl, int dt, int j) __attribute__((always_inline)) {
        const _Float16 *at = vl + (32 * dt + nl) * kVStride + 16 * j + 4 * h;
        const half4 a0 = *reinterpret_cast<const half4 *>(at), a1 = *reinterpret_cast<const half4 *>(at + 8);
        return half8{a0[0], a0[1], a0[2], a0[3], a1[0], a1[1], a1[2], a1[3]};
    };
    auto edge_of = [&](int kt) { return kt * kTile < all_lo || kt * kTile + kTile > all_hi; };
    bool ok = true, ok_next = true;                                        // both halves of the tile exist
    if (BUFS == 2 && t0 < t1) {
        __syncthreads();                                                   // `bad` is clear
        ok_next = both_ok<PAGED>(p, b, seq.n, t0);
        decode_tile<D>(g, raw, value_scales<D>(g, raw, t0 * kTile, seq.n, edge_of(t0) || !ok_next, tid, bad[0]), tid, lds);
        if (t0 + 1 < t1) load_raw<D, PAGED>(p, b, kvh, seq.n, t0 + 1, tid, raw);
    }
    for (int kt = t0, i = 0; kt < t1; ++kt, i = i == 2 ? 0 : i + 1) {
        const int k0 = kt * kTile, ahead = i == 2 ? 0 : i + 1;
        __syncthreads();                                                   // this tile is decoded; the other buffer is free
        const _Float16 *kl = lds + (BUFS == 2 ? ((kt - t0) & 1) * Shape<D>::kHalves : 0), *vl = kl + kTile * KS;
        ok = ok_next;
        half8 ka[STEPS];
        auto read_keys = [&]() __attribute__((always_inline)) {
#pragma unroll
            for (int st = 0; st < STEPS; ++st) ka[st] = *reinterpret_cast<const half8 *>(kl + nl * KS + 16 * st + 8 * h);
            __builtin_amdgcn_sched_barrier(0);
        };
        // S^T: accumulator j is key k0 + 8 (j / 4) + 4h + j % 4 of this lane's row.
        f32x16 s = {};
        auto scores = [&]() __attribute__((always_inline)) {
#pragma unroll
            for (int st = 0; st < STEPS; ++st) {
                s = __builtin_amdgcn_mfma_f32_32x32x16_f16(ka[st], ql[st], s, 0, 0, 0);
                s = __builtin_amdgcn_mfma_f32_32x32x16_f16(ka[st], qh[st], s, 0, 0, 0);
            }
        };
        const bool unseen = idle || k0 >= w_hi || k0 + kTile <= w_lo;      // by the wave's rows
        if constexpr (BUFS == 2) {
            read_keys();
            if (tid < 8) bad[ahead == 2 ? 0 : ahead + 1][tid] = 0;         // the tile before this one's
            half2v vd = {};
            if (kt + 1 < t1) {
                ok_next = both_ok<PAGED>(p, b, seq.n, kt + 1);
                vd = value_scales<D>(g, raw, k0 + kTile, seq.n, edge_of(kt + 1) || !ok_next, tid, bad[ahead]);
            }
            // The next tile is decoded between the products (past the last one, what it holds is not used).
            __builtin_amdgcn_sched_barrier(0);
            scores();
            decode_tile<D>(g, raw, vd, tid, lds + ((kt + 1 - t0) & 1) * Shape<D>::kHalves);
#pragma unroll
            for (int i = 0; i < 2 * STEPS; ++i) {
                __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);         // a product,
                __builtin_amdgcn_sched_group_barrier(0x002, 6, 0);         // six vector instructions (about its 32 cycles),
                __builtin_amdgcn_sched_group_barrier(0x200, 1, 0);         // a store to LDS
            }
            __builtin_amdgcn_sched_barrier(0);
            if (kt + 2 < t1) load_raw<D, PAGED>(p, b, kvh, seq.n, kt + 2, tid, raw);
            if (unseen) continue;
        } else {
            ok = both_ok<PAGED>(p, b, seq.n, kt);
            if (tid < 8) bad[ahead][tid] = 0;
            decode_tile<D>(g, raw, value_scales<D>(g, raw, k0, seq.n, edge_of(kt) || !ok, tid, bad[i]), tid, lds);
            if (kt + 1 < t1) load_raw<D, PAGED>(p, b, kvh, seq.n, kt + 1, tid, raw);
            __syncthreads();
            read_keys();
            if (unseen) continue;
            scores();
        }
        // V's fragments arrive while the weights are computed.
        half8 va[2][DT];
        if constexpr (D < 256) {
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int dt = 0; dt < DT; ++dt) va[j][dt] = read_values(vl, dt, j);
            __builtin_amdgcn_sched_barrier(0);
        }
        if constexpr (CAP) {
            const float cap = p.soft_cap * kLog2e, in = fminf(unscale / cap, 3e38f);       // finite: 0 stays 0
#pragma unroll
            for (int j = 0; j < 16; ++j) s[j] = cap * tanhf(s[j] * in);
        }
        const float us = CAP ? 1.0f : unscale;
        if (k0 < full_lo || k0 + kTile > full_hi || !ok) {
            const int first = lo - k0 - 4 * h, end = hi - k0 - 4 * h;
            uint32_t there = 0xffffffffu;                                  // keys on blocks that exist
            if (!ok) there = half_ok<PAGED>(p, b, seq.n, kt);
#pragma unroll
            for (int j = 0; j < 16; ++j) {
                const int c = 8 * (j >> 2) + (j & 3);
                if (c < first || c >= end || !(there >> (j >> 3) & 1)) s[j] = -INFINITY;
            }
        }
        if (edge_of(kt) || !ok) {
            // Keys of this tile that the row sees, against the ones that are not finite.
            const int a = max(lo - k0, 0), z = min(hi - k0, kTile);
            const uint32_t see = z <= a ? 0 : (z == 32 ? 0xffffffffu : (1u << z) - 1) & ~((1u << a) - 1);
#pragma unroll
            for (int q = 0; q < DT; ++q) poison |= bad[i][q] & see ? 1u << q : 0;
        }
        float mx = s[0];
#pragma unroll
        for (int j = 1; j < 16; ++j) mx = fmaxf(mx, s[j]);
        mx *= us;
        if (__any(mx > m + 2.0f)) {
            mx = fmaxf(mx, __shfl_xor(mx, 32));
            const float up = mx > m + 2.0f ? mx : m;
            const float alpha = up == m ? 1.0f : __builtin_amdgcn_exp2f(m - up);                  // 0 while m is -inf
            l *= alpha;
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) o[dt] *= alpha;
            m = up;
        }
        const float ref = m == -INFINITY ? 0.0f : m;
        half8 ph[2], pl[2];
        float sum[4] = {};
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            float e[2];
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                e[c] = __builtin_amdgcn_exp2f(fmaf(s[2 * j + c], us, -ref)) * kWeightScale;
                sum[(2 * j + c) & 3] += e[c];
            }
            const half2v first = pair(e[0], e[1]);
            const half2v rest = pair(e[0] - static_cast<float>(first[0]), e[1] - static_cast<float>(first[1]));
            ph[j >> 2][2 * (j & 3)] = first[0];
            ph[j >> 2][2 * (j & 3) + 1] = first[1];
            pl[j >> 2][2 * (j & 3)] = rest[0];
            pl[j >> 2][2 * (j & 3) + 1] = rest[1];
        }
        l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
        // Lane half h supplies contraction entries 0..3 -> key 16j + 4h + e and 4..7 -> key 16j + 8 + 4h + e - 4.
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            if constexpr (D == 256) {
#pragma unroll
                for (int dt = 0; dt < DT; ++dt) va[j][dt] = read_values(vl, dt, j);
            }
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) o[dt] = __builtin_amdgcn_mfma_f32_32x32x16_f16(va[j][dt], pl[j], o[dt], 0, 0, 0);
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) o[dt] = __builtin_amdgcn_mfma_f32_32x32x16_f16(va[j][dt], ph[j], o[dt], 0, 0, 0);
        }
    }

    l += __shfl_xor(l, 32);
    if (m == -INFINITY && l != l) m = 0.0f;                                // a NaN score alone leaves no reference
    const bool whole = chunk.count == 1;
    const float f = whole ? (l == 0.0f ? 0.0f : 1.0f / l) : 1.0f;
    const long long part = (static_cast<long long>(chunk.slot + w - chunk.first) * p.v.H * p.row_groups + item) * kRowsBlock + 32 * wave;
    if (!whole && h == 0 && w0 + nl < r1) *reinterpret_cast<float2 *>(p.part_ml + (part + nl) * 2) = make_float2(m, l);
    __syncthreads();                                                       // every wave is done with the tiles
    // O through LDS, so that whole lines are stored: rounds of two blocks of dims (D = 64: of one), a wave's own
    // [32 rows][block of h][32]. Accumulator j of tile dt is row 32 dt + 8 (j / 4) + 4h + j % 4 of V^T: nibble
    // 2 dt + j / 8 of piece n = 8 (j / 4 % 2) + 4h + j % 4.
    constexpr int SPAN = D == 64 ? 32 : 64, STRIDE = SPAN + 4, ROUNDS = D / SPAN, LPR = SPAN / 4;
    float *st = reinterpret_cast<float *>(lds) + wave * 32 * STRIDE;
#pragma unroll
    for (int rd = 0; rd < ROUNDS; ++rd) {
        const int u = D == 256 ? rd >> 1 : rd, sub = rd & 1;               // D = 256: j % 4 / 2 == sub
#pragma unroll
        for (int j = 0; j < 16; ++j) {
            if ((j >> 2 & 1) != u || (D == 256 && (j >> 1 & 1) != sub)) continue;
            const int odd = j >> 3;
            if constexpr (D == 64) {
                *reinterpret_cast<float2 *>(st + nl * STRIDE + 16 * odd + 4 * (2 * h + (j >> 1 & 1)) + 2 * (j & 1)) =
                    make_float2(o[0][j] * f, o[1][j] * f);
            } else {
#pragma unroll
                for (int c = 0; c < DT / 4; ++c)
                    *reinterpret_cast<float4 *>(st + nl * STRIDE + 32 * h + 16 * odd +
                                                (D == 128 ? 4 * (j & 3) : 8 * (j & 1) + 4 * c)) =
                        make_float4(o[4 * c][j] * f, o[4 * c + 1][j] * f, o[4 * c + 2][j] * f, o[4 * c + 3][j] * f);
            }
        }
        if (poison && (D != 64 || h == 0)) {
            const int own = D == 64 ? u : D == 128 ? 2 * u + h : 4 * u + 2 * h + sub;
            if (poison >> own & 1)
                for (int i = 0; i < 32; ++i) st[nl * STRIDE + (D == 64 ? 0 : 32 * h) + i] = NAN;
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");                 // the wave's own writes
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
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");                 // read before the next round's writes
    }
}

// A wave a row of a sequence with several chunks: D/4 lanes take a chunk's
// partial as float4s (64 / (D/4) chunks at once), folded in order, then across
// the lane groups.
template <int D>
__global__ __launch_bounds__(256) void kv4_merge_rows_kernel(Params p) {
    constexpr int LPS = D / 4, SG = 64 / LPS;
    const int of_seq = blockIdx.x * 4 + (threadIdx.x >> 6), b = blockIdx.y;
    const int t = of_seq / p.Hq, hq = of_seq - t * p.Hq;
    if (t >= p.T) return;
    const long long row = static_cast<long long>(b) * p.T * p.Hq + of_seq;
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
    const dim3 grid(p.v.H * p.row_groups * (p.quota ? p.quota + (p.v.B > 1 ? p.v.B : 0) : p.v.B));
    if (p.soft_cap > 0.0f)
        hipLaunchKernelGGL((kv4_rows_kernel<D, PAGED, true>), grid, dim3(kThreads), 0, s, p);
    else
        hipLaunchKernelGGL((kv4_rows_kernel<D, PAGED, false>), grid, dim3(kThreads), 0, s, p);
    if (p.quota)                                           // few row groups, so few rows of a sequence
        hipLaunchKernelGGL((kv4_merge_rows_kernel<D>), dim3((p.T * p.Hq + 3) / 4, p.v.B), dim3(256), 0, s, p);
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
