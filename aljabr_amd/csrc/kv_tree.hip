// kv_tree.hip - attention of a draft's rows over an fp16 or fp32 cache (layout
// and trees: kv_cache.hpp).
//
//   out[t, h] = sum_j w_j v_j / sum_j w_j,  w_j = exp(s_j - max s),
//   s_j = cap(scale * q[t, h] . k_j), over the keys j that row t sees.
//
// The rows of a KV head are stacked, r = t * G + g (G = Hq / Hkv), 16 or 32 a
// workgroup (65 and more over large caches: kv_tree_rows.hip). A wave walks
// tiles of 16 U keys, whose fragments come straight from the cache into
// registers, each refilled for the wave's next tile as soon as the matrix cores
// have taken it: no LDS, no barrier in the loop.
//   S[key][row]   = K Q^T: lane (n, h) holds key n, 16 bytes at every step;
//   O^T[d][row] += V^T P^T: a lane loads whole pieces of V's rows, 4 keys of
//     each 16 and 8 (4) dims, and a weight of each row it computed itself.
//     fp16: v_mfma_f32_16x16x32_f16 over the 32 keys, V transposed by a byte
//       permutation of two keys' dwords (one a dword and key pair), weights as
//       two fp16 parts;
//     fp32: v_mfma_f32_16x16x4_f32, one number a lane, which needs no
//       transposition. fp16 caches went this way first: a tree of 64 over
//       8 x 8192 keys took 433 us, with fp16 products 180 us.
// Bound by the bytes of the cache, read once a row group: 32 sequences of about
// 2100 keys, 8 KV heads of 128, 20 rows each, 57 to 68 us with the merge (4.1 to
// 4.9 TB/s); an fp32 cache of 4 x 2048 keys, 64 rows a head, 32.6 us, of which its
// products at fp32's rate are 14; short calls by the chain lengths - table - tile
// - states - merge: 8 drafted rows over 512 keys 10.7 us.
//
// Precision: an fp16 K enters as it is against a query row scaled by a power of
// two to a largest magnitude in [2^14, 2^15) and split into two fp16 parts
// (2^-22 of each element); weights of an fp16 cache are two fp16 parts as well
// (2^-22, nothing below 2^-36 of the largest); everything else is fp32.
//
// Keys a row does not see get weight 0. In a tile that not every row sees
// whole, V rows past the end are taken as 0, and values that are not finite are
// taken out of the product and added by hand for the rows that see them. The
// two fp16 parts of a query or a weight times an infinity may make a NaN where
// the sum has none: a wave whose sums are not finite walks its tiles again, with
// scores that are NaN computed in fp32 and every tile treated as above.
#include <algorithm>
#include <cmath>

#include "kv_tree.hpp"

namespace aljabr {

using namespace kvt;

namespace {

template <bool F16, int D>
struct Shape {
    static constexpr int kSize = F16 ? 2 : 4, kRow = D * kSize;
    static constexpr int U = F16 || D == 64 ? 2 : 1;       // groups of 16 keys of a tile: at most 32 KB of K and V
    static constexpr int KT = 16 * U;
    static constexpr int VE = F16 && D > 64 ? 8 : 4;       // dims of a lane's piece of a V row
    static constexpr int VP = D / 16 / VE;                 // pieces
    static constexpr int KL = D * kSize / 64;              // K's 16-byte loads of a group, a step of the contraction each
    static constexpr int OT = D / 16;                      // output tiles
    static constexpr int kQuery = KL * (F16 ? 2 : 1);      // 16-byte pieces of a lane's query
};

// A piece of a V row as loaded.
template <bool F16, int D>
struct Piece {
    static constexpr int kWords = Shape<F16, D>::VE * Shape<F16, D>::kSize / 4;
    uint32_t w[kWords];
    __device__ __forceinline__ void load(const char *at) {
        if constexpr (kWords == 4) {
            const uint4 x = *reinterpret_cast<const uint4 *>(at);
            w[0] = x.x; w[1] = x.y; w[2] = x.z; w[3] = x.w;
        } else {
            const uint2 x = *reinterpret_cast<const uint2 *>(at);
            w[0] = x.x; w[1] = x.y;
        }
    }
    __device__ __forceinline__ float get(int e) const {
        if constexpr (F16) return f16_bits_to_f32(w[e >> 1] >> (16 * (e & 1)) & 0xffffu);
        else return __uint_as_float(w[e]);
    }
    // The bits of values that are not finite have an exponent of ones.
    __device__ __forceinline__ bool finite() const {
        uint32_t bad = 0;
#pragma unroll
        for (int i = 0; i < kWords; ++i) bad |= F16 ? ((w[i] & 0x7fff7fffu) + 0x04000400u) & 0x80008000u : ((w[i] & 0x7fffffffu) + 0x00800000u) & 0x80000000u;
        return !bad;
    }
    __device__ __forceinline__ void drop() {
#pragma unroll
        for (int i = 0; i < kWords; ++i) w[i] = 0;
    }
    // Values that are not finite become 0.
    __device__ __forceinline__ void clean() {
#pragma unroll
        for (int i = 0; i < kWords; ++i) {
            if constexpr (F16) {
                if ((w[i] & 0x7c00u) == 0x7c00u) w[i] &= 0xffff0000u;
                if ((w[i] & 0x7c000000u) == 0x7c000000u) w[i] &= 0x0000ffffu;
            } else {
                if ((w[i] & 0x7f800000u) == 0x7f800000u) w[i] = 0;
            }
        }
    }
};

// The largest of x in the four lanes of a column.
__device__ __forceinline__ float group_max(float x) {
    const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    const auto c = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(c[0]), __uint_as_float(c[1]));
}

// The 8 halves of dim e of a piece, of the 8 keys that a lane holds.
template <int D, int W>
__device__ __forceinline__ half8 dim_of(const Piece<true, D> (&v)[2][4][W], int x, int e) {
    const uint32_t sel = e & 1 ? 0x07060302u : 0x05040100u;
    uint32_t f[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
        f[i] = __builtin_amdgcn_perm(v[i >> 1][2 * (i & 1) + 1][x].w[e >> 1], v[i >> 1][2 * (i & 1)][x].w[e >> 1], sel);
    return __builtin_bit_cast(half8, make_uint4(f[0], f[1], f[2], f[3]));
}

// What a lane loads of a row's query: of fp16's steps dims 32s + 8h .. + 7, of fp32's 16s + 4h .. + 3.
template <bool F16, int D>
struct Query {
    float4 x[D / 16];
    __device__ __forceinline__ void load(const float *row, int h) {
#pragma unroll
        for (int i = 0; i < D / 16; ++i) x[i] = *reinterpret_cast<const float4 *>(row + (F16 ? 32 * (i >> 1) + 8 * h + 4 * (i & 1) : 16 * i + 4 * h));
    }
    // The pieces that enter products: fp16 the two parts of each step, fp32 as it is, times scale. It was scaled by 2^(15 - e).
    __device__ __forceinline__ void pieces(const Params &p, uint4 (&q)[Shape<F16, D>::kQuery], int &e) const {
        const float scale = p.scale;
        e = 15;
        if constexpr (F16) {
            float top = 0.0f;
#pragma unroll
            for (int i = 0; i < D / 16; ++i) top = fmaxf(top, fmaxf(fmaxf(fabsf(x[i].x), fabsf(x[i].y)), fmaxf(fabsf(x[i].z), fabsf(x[i].w))));
            top = group_max(top) * scale;
            e = query_exponent(p, top);
            const float up = ldexpf(1.0f, 15 - e);
#pragma unroll
            for (int s = 0; s < D / 32; ++s) {
                const float4 a = x[2 * s], c = x[2 * s + 1];
                const float y[8] = {a.x, a.y, a.z, a.w, c.x, c.y, c.z, c.w};
                half8 first, rest;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float z = y[i] * scale * up;
                    first[i] = static_cast<_Float16>(z);
                    rest[i] = static_cast<_Float16>(z - static_cast<float>(first[i]));
                }
                q[2 * s] = __builtin_bit_cast(uint4, first);
                q[2 * s + 1] = __builtin_bit_cast(uint4, rest);
            }
        } else {
#pragma unroll
            for (int s = 0; s < D / 16; ++s)
                q[s] = make_uint4(__float_as_uint(x[s].x * scale), __float_as_uint(x[s].y * scale), __float_as_uint(x[s].z * scale),
                                  __float_as_uint(x[s].w * scale));
        }
    }
};

// Whether the queries are kept in LDS: in registers they would be D / 4 of each column tile.
constexpr bool query_in_lds(int D, int NT) { return NT * D >= 256; }

// grid: chunks of KV heads and row groups (work_at).
template <bool F16, int D, int NT>
__global__ __launch_bounds__(kThreads, D == 256 ? 1 : 2) void kv_split_kernel(Params p) {
    using S = Shape<F16, D>;
    constexpr int U = S::U, KT = S::KT, VE = S::VE, VP = S::VP, KL = S::KL, OT = S::OT, ROWS = 16 * NT, QL = S::kQuery;
    constexpr bool QLDS = query_in_lds(D, NT);
    extern __shared__ float smem[];                        // queries, states on their way, weights of odd tiles
    __shared__ Tree tree;
    // Of a row: t and what it sees (a wave's own copy); and what scales its scores back.
    __shared__ int4 row_info[kWaves][ROWS];
    __shared__ float query_scale[QLDS ? ROWS : 1];
    float *work = smem + (QLDS ? NT * QL * 256 : 0);
    const int lane = threadIdx.x & 63, n = lane & 15, h = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const Work work_item = work_at(p, blockIdx.x);
    const int kvh = work_item.kvh, group = work_item.group, w = work_item.w, item = item_of(p, kvh, group), r0 = group * ROWS;
    if (!p.quota && w >= p.v.B) return;                    // numbers past the last unit
    const Chunk chunk = find_chunk(p, w, r0, ROWS, kWaves);
    if (chunk.b < 0) return;
    const int b = chunk.b, t0 = chunk.t0, t1 = chunk.t1;
    if (p.quota && w == chunk.first && threadIdx.x == 0)
        p.chunks[static_cast<long long>(item) * p.v.B + b] = make_int2(chunk.slot, chunk.count);
    const Seq seq = chunk.seq;
    const int base = seq.base, r1 = min(r0 + ROWS, seq.cnt * p.G);

    // The first tile's places, the tree's parents, the queries and then the tile: all on their way before any is used.
    const int tile0 = t0 < t1 ? min(t0 + wave, t1 - 1) : 0;            // a wave without a tile loads one that is there
    Places<U> places{tile0, kWaves};
    const auto entry = places.fetch(p, lane, b, seq.n, 0);
    const bool filled = p.parents && (p.window > 0 || t1 * KT > base);
    int parent = -1;
    if (filled && tree_row(seq.cnt) < seq.cnt) parent = p.parents[static_cast<long long>(b) * p.T + tree_row(seq.cnt)];
    auto row_at = [&](int t, int r) __attribute__((always_inline)) {
        return p.q + ((static_cast<long long>(b) * p.T + t) * p.Hq + kvh * p.G + (r - t * p.G)) * D;
    };
    Query<F16, D> raw[QLDS ? 1 : NT];
    static_assert(!QLDS || NT <= kWaves, "a wave loads one column tile's queries");
#pragma unroll
    for (int c = 0; c < (QLDS ? 1 : NT); ++c) {
        const int r = min(r0 + 16 * (QLDS ? wave : c) + n, r1 - 1);    // columns past the rows repeat the last and are not stored
        if (!QLDS || wave < NT) raw[c].load(row_at(p.by_g(r), r), h);
    }
    uint4 kf[U][KL];
    Piece<F16, D> vf[U][4][VP];
    struct Place {
        long long at[U];                                   // of its groups of 16 keys in the planes
        uint32_t ok;                                       // bit u: the group's block exists
    } here = {}, next = {};
    auto place = [&](int i) __attribute__((always_inline)) {
        Place x;
        x.ok = places.ok(i);
#pragma unroll
        for (int u = 0; u < U; ++u) x.at[u] = places.offset(i, u);
        return x;
    };
    // The last of the 16 rows of group u of tile kt that is in the plane.
    auto last_of = [&](int kt, int u) __attribute__((always_inline)) {
        return last_row(p, kt * KT + (kt * KT + 16 * u < seq.n ? 16 * u : 0));
    };
    // Offsets from an address that the wave shares, in 32 bits.
    auto load_keys = [&](const Place &x, int kt) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const char *at = p.v.k + x.at[u];
            const uint32_t off = min(n, last_of(kt, u)) * S::kRow + 16 * h;
#pragma unroll
            for (int s = 0; s < KL; ++s) kf[u][s] = *reinterpret_cast<const uint4 *>(at + off + 64 * s);
        }
    };
    auto load_values = [&](const Place &x, int kt) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const char *at = p.v.v + x.at[u];
            const int last = last_of(kt, u);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const uint32_t off = min(4 * h + r, last) * S::kRow + n * VE * S::kSize;
#pragma unroll
                for (int c = 0; c < VP; ++c) vf[u][r][c].load(at + off + c * 16 * VE * S::kSize);
            }
        }
    };
    // By every wave, also one without a tile: loads that only some paths make would all be waited for before the first of
    // the others is used.
    places.hold(p, entry, S::kRow, kvh, 0);
    here = place(0);
    load_keys(here, tile0);
    load_values(here, tile0);
    if (filled) fill_tree(tree, parent, seq.cnt, p.window);

    // This lane's columns: the query times scale * log2(e), and in LDS what the paths that are rarely taken need of the row.
    uint4 qr[QLDS ? 1 : NT][QL];
    float unscale[NT];
    uint4 *qlds = reinterpret_cast<uint4 *>(smem) + lane;
#pragma unroll
    for (int c = 0; c < NT; ++c) {
        const int t = p.by_g(min(r0 + 16 * c + n, r1 - 1));
        const Range range = range_of(p, seq, t, tree, filled);
        row_info[wave][16 * c + n] = make_int4(t, range.lo, range.hi, 0);                      // the same of four lanes
        if (QLDS && c != wave) continue;
        int e;
        raw[QLDS ? 0 : c].pieces(p, qr[QLDS ? 0 : c], e);
        unscale[c] = ldexpf(p.unscale, e - 15);
        if constexpr (QLDS) {
#pragma unroll
            for (int i = 0; i < QL; ++i) qlds[(c * QL + i) * 64] = qr[0][i];
            if (lane < 16) query_scale[16 * c + n] = unscale[c];
        }
    }
    if constexpr (QLDS) {
        __syncthreads();
#pragma unroll
        for (int c = 0; c < NT; ++c) unscale[c] = query_scale[16 * c + n];
    }
    // For the paths that are rarely taken: the lane's number, of which the compiler keeps nothing in registers.
    auto fresh_lane = [](int mask) __attribute__((always_inline)) {
        int x = threadIdx.x;
        asm volatile("" : "+v"(x));
        return x & mask;
    };
    auto query = [&](int c, int i) __attribute__((always_inline)) { return QLDS ? qlds[(c * QL + i) * 64] : qr[QLDS ? 0 : c][i]; };
    // Keys that every row sees: a tree's rows stand at most at their places.
    const int full_lo = window_start(p, base + p.by_g(r1 - 1) + 1);
    const int full_hi = min(p.parents ? base : base + p.by_g(r0) + 1, seq.n);

    f32x4 o[NT][OT];
    float m[NT], l[NT];
    bool careful = false;
again:
#pragma unroll
    for (int c = 0; c < NT; ++c) {
        m[c] = -INFINITY;
        l[c] = 0.0f;
#pragma unroll
        for (int j = 0; j < OT; ++j) o[c][j] = f32x4{};
    }

    for (int kt = t0 + wave, i = 0; kt < t1; kt += kWaves, ++i) {
        const int k0 = kt * KT;
        const bool more = kt + kWaves < t1;
        if (more) {
            if (i + 1 == places.held + 64 / U) places.load(p, lane, S::kRow, b, kvh, seq.n, i + 1);
            next = place(i + 1);
        }
        // Every row sees every key.
        const bool whole = !careful && k0 >= full_lo && k0 + KT <= full_hi && here.ok == (1u << U) - 1;

        // S: accumulator r of group u is key k0 + 16u + 4h + r of this lane's column.
        f32x4 s[NT][U];
#pragma unroll
        for (int c = 0; c < NT; ++c)
#pragma unroll
            for (int u = 0; u < U; ++u) s[c][u] = f32x4{};
#pragma unroll
        for (int i = 0; i < KL; ++i)
#pragma unroll
            for (int c = 0; c < NT; ++c) {
                if constexpr (F16) {
                    const half8 q0 = __builtin_bit_cast(half8, query(c, 2 * i)), q1 = __builtin_bit_cast(half8, query(c, 2 * i + 1));
#pragma unroll
                    for (int u = 0; u < U; ++u) {
                        const half8 a = __builtin_bit_cast(half8, kf[u][i]);
                        s[c][u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, q1, s[c][u], 0, 0, 0);
                        s[c][u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, q0, s[c][u], 0, 0, 0);
                    }
                } else {
                    const f32x4 q = __builtin_bit_cast(f32x4, query(c, i));
#pragma unroll
                    for (int u = 0; u < U; ++u) {
                        const f32x4 a = __builtin_bit_cast(f32x4, kf[u][i]);
#pragma unroll
                        for (int e = 0; e < 4; ++e) s[c][u] = __builtin_amdgcn_mfma_f32_16x16x4f32(a[e], q[e], s[c][u], 0, 0, 0);
                    }
                }
            }
        if (more) load_keys(next, kt + kWaves);
        uint32_t see[NT];
        float pw[NT][U][4];
#pragma unroll
        for (int c = 0; c < NT; ++c) {
            see[c] = 0xffffffffu;
            if (!whole) {
                const int4 info = row_info[wave][16 * c + fresh_lane(15)];
                see[c] = seen(p, seq, Range{info.y, info.z}, info.x, k0, tree);
#pragma unroll
                for (int u = 0; u < U; ++u)
                    if (!(here.ok >> u & 1)) see[c] &= ~(0xffffu << 16 * u);
            }
#pragma unroll
            for (int i = 0; i < 4 * U; ++i) pw[c][i >> 2][i & 3] = s[c][i >> 2][i & 3];
            if (F16 && careful) {                          // scores that are NaN, in fp32
                const int lane = fresh_lane(63), h = lane >> 4, row = min(r0 + 16 * c + (lane & 15), r1 - 1);
                const float *q = row_at(row_info[wave][16 * c + (lane & 15)].x, row);
                const float up = p.unscale / unscale[c];   // powers of two
                float *mine = work + wave * (ROWS * KT) + lane;
#pragma unroll
                for (int i = 0; i < 4 * U; ++i) mine[64 * i] = pw[c][i >> 2][i & 3];
                int keys = 4 * U, dims = D;
                asm("" : "+s"(keys), "+s"(dims));          // loops that stay loops
                for (int i = 0; i < keys; ++i) {
                    const int r = 4 * h + (i & 3);
                    if (mine[64 * i] == mine[64 * i] || !(see[c] >> (16 * (i >> 2) + r) & 1)) continue;
                    const _Float16 *kr = reinterpret_cast<const _Float16 *>(p.v.k + here.at[i >= 4 ? U - 1 : 0] + r * S::kRow);
                    float sum = 0.0f;
                    for (int d = 0; d < dims; ++d) sum = fmaf(q[d] * p.scale * up, static_cast<float>(kr[d]), sum);
                    mine[64 * i] = sum;
                }
#pragma unroll
                for (int i = 0; i < 4 * U; ++i) pw[c][i >> 2][i & 3] = mine[64 * i];
            }
            if (p.soft_cap > 0.0f) {
                const float cap = p.soft_cap * kLog2e, in = fminf(unscale[c] / cap, 3e38f);    // finite: 0 stays 0
#pragma unroll
                for (int i = 0; i < 4 * U; ++i) pw[c][i >> 2][i & 3] = cap * tanhf(pw[c][i >> 2][i & 3] * in);
            }
            if (!whole) {
                const uint32_t mine = see[c] >> (4 * (fresh_lane(63) >> 4));
#pragma unroll
                for (int i = 0; i < 4 * U; ++i)
                    if (!(mine >> (16 * (i >> 2) + (i & 3)) & 1)) pw[c][i >> 2][i & 3] = -INFINITY;
            }
            float mx = pw[c][0][0];
#pragma unroll
            for (int i = 1; i < 4 * U; ++i) mx = fmaxf(mx, pw[c][i >> 2][i & 3]);
            const float us = p.soft_cap > 0.0f ? 1.0f : unscale[c];
            mx *= us;
            // The reference m of a column is raised only when a score exceeds it by more than kRaise.
            if (__any(mx > m[c] + kRaise)) {
                mx = group_max(mx);
                const float to = mx > m[c] + kRaise ? mx : m[c];
                const float alpha = to == m[c] ? 1.0f : __builtin_amdgcn_exp2f(m[c] - to);     // 0 while m is -inf
                l[c] *= alpha;
#pragma unroll
                for (int j = 0; j < OT; ++j) o[c][j] *= alpha;
                m[c] = to;
            }
            const float ref = m[c] == -INFINITY ? 0.0f : m[c];
            float sum[2] = {};
#pragma unroll
            for (int i = 0; i < 4 * U; ++i) {
                float &y = pw[c][i >> 2][i & 3];
                y = __builtin_amdgcn_exp2f(fmaf(y, us, -ref)) * kWeightScale<F16>;
                sum[i & 1] += y;
            }
            l[c] += sum[0] + sum[1];
        }
        if (!whole) {
            const int lane = fresh_lane(63), n = lane & 15, h = lane >> 4;
            bool odd = false;
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int r = 0; r < 4; ++r)
#pragma unroll
                    for (int c = 0; c < VP; ++c) {
                        if (k0 + 16 * u + 4 * h + r >= seq.n || !(here.ok >> u & 1)) vf[u][r][c].drop();
                        odd |= !vf[u][r][c].finite();
                    }
            if (__any(odd)) {
                float *pl = work + wave * (ROWS * KT);     // the wave's weights, [column tile][key][row]
#pragma unroll
                for (int c = 0; c < NT; ++c)
#pragma unroll
                    for (int i = 0; i < 4 * U; ++i) pl[(c * KT + 16 * (i >> 2) + 4 * h + (i & 3)) * 16 + n] = pw[c][i >> 2][i & 3];
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");     // the wave's own writes
                int keys = KT;
                asm("" : "+s"(keys));                      // a loop that stays one
                for (int i = 0; i < keys; ++i) {
                    if (k0 + i >= seq.n || !(here.ok >> (i >> 4) & 1)) continue;
                    const char *vr = p.v.v + here.at[U == 2 && i >= 16 ? U - 1 : 0] + (i & 15) * S::kRow;
#pragma unroll
                    for (int x = 0; x < VP; ++x)
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            Piece<F16, D> v;
                            v.load(vr + (x * 16 + 4 * h + r) * VE * S::kSize);
                            if (!__any(!v.finite())) continue;
#pragma unroll
                            for (int e = 0; e < VE; ++e) {
                                const float val = v.get(e);
#pragma unroll
                                for (int c = 0; c < NT; ++c)
                                    o[c][x * VE + e][r] += val - val != 0.0f && (see[c] >> i & 1) ? pl[(c * KT + i) * 16 + n] * val : 0.0f;
                            }
                        }
                }
#pragma unroll
                for (int u = 0; u < U; ++u)
#pragma unroll
                    for (int r = 0; r < 4; ++r)
#pragma unroll
                        for (int c = 0; c < VP; ++c) vf[u][r][c].clean();
            }
        }
        if constexpr (F16) {
            half8 p0[NT], p1[NT];
#pragma unroll
            for (int c = 0; c < NT; ++c)
#pragma unroll
                for (int i = 0; i < 4 * U; ++i) {
                    const float y = pw[c][i >> 2][i & 3];
                    p0[c][i] = static_cast<_Float16>(y);
                    p1[c][i] = static_cast<_Float16>(fmaf(static_cast<float>(p0[c][i]), -1.0f, y));
                }
#pragma unroll
            for (int x = 0; x < VP; ++x)
#pragma unroll
                for (int e = 0; e < VE; ++e) {
                    const half8 a = dim_of<D, VP>(vf, x, e);
#pragma unroll
                    for (int c = 0; c < NT; ++c) {
                        f32x4 &acc = o[c][x * VE + e];
                        acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, p1[c], acc, 0, 0, 0);
                        acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, p0[c], acc, 0, 0, 0);
                    }
                }
        } else {
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int r = 0; r < 4; ++r)
#pragma unroll
                    for (int x = 0; x < VP; ++x)
#pragma unroll
                        for (int e = 0; e < VE; ++e) {
                            const float a = vf[u][r][x].get(e);
#pragma unroll
                            for (int c = 0; c < NT; ++c)
                                o[c][x * VE + e] = __builtin_amdgcn_mfma_f32_16x16x4f32(a, pw[c][u][r], o[c][x * VE + e], 0, 0, 0);
                        }
        }
        if (more) load_values(next, kt + kWaves);
        here = next;
    }
    if (F16 && !careful) {
        // Sums that are not finite are made again, carefully.
        float probe = 0.0f;
#pragma unroll
        for (int c = 0; c < NT; ++c)
#pragma unroll
            for (int j = 0; j < OT; ++j)
#pragma unroll
                for (int r = 0; r < 4; ++r) probe = fmaf(o[c][j][r], 0.0f, probe);
        if (__any(probe != probe)) {
            careful = true;
            places.load(p, lane, S::kRow, b, kvh, seq.n, 0);     // the wave had a tile: its sums are not zeros
            here = place(0);
            load_keys(here, t0 + wave);
            load_values(here, t0 + wave);
            goto again;
        }
    }

    // The four waves' states through LDS as rows, then a thread takes four dims of a row from all of them. O^T tile x VE + e,
    // accumulator i: dim 16 VE x + VE (4h + i) + e of the row.
    constexpr int kStride = D + 4;
    float2 *ml = reinterpret_cast<float2 *>(smem + kWaves * ROWS * kStride);               // [wave][row]
    __syncthreads();                                       // the queries and weights are done with
#pragma unroll
    for (int c = 0; c < NT; ++c) {
        l[c] += __shfl_xor(l[c], 16);
        l[c] += __shfl_xor(l[c], 32);
        if (m[c] == -INFINITY && l[c] != l[c]) m[c] = 0.0f;            // a NaN score alone leaves no reference: any finite one carries it
        float *row = smem + (wave * ROWS + 16 * c + n) * kStride + VE * 4 * h;
#pragma unroll
        for (int x = 0; x < VP; ++x)
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int e = 0; e < VE; e += 4)
                    *reinterpret_cast<float4 *>(row + 16 * VE * x + VE * i + e) =
                        make_float4(o[c][x * VE + e][i], o[c][x * VE + e + 1][i], o[c][x * VE + e + 2][i], o[c][x * VE + e + 3][i]);
        if (h == 0) ml[wave * ROWS + 16 * c + n] = make_float2(m[c], l[c]);
    }
    __syncthreads();
    const bool all = chunk.count == 1;
    const long long part = (static_cast<long long>(chunk.slot + w - chunk.first) * p.v.H * p.row_groups + item) * ROWS;
    constexpr int LPR = D / 4;
#pragma unroll
    for (int i = 0; i < ROWS * LPR / kThreads; ++i) {
        const int lr = (kThreads * i + static_cast<int>(threadIdx.x)) / LPR, d = 4 * (threadIdx.x % LPR), r = r0 + lr;
        if (r >= r1) continue;
        float2 of[kWaves];
        float top = -INFINITY, sum = 0.0f;
#pragma unroll
        for (int k = 0; k < kWaves; ++k) {
            of[k] = ml[k * ROWS + lr];
            top = fmaxf(top, of[k].x);
        }
        float4 y = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
        for (int k = 0; k < kWaves; ++k) {
            const float e = of[k].x == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(of[k].x - top);
            const float4 x = *reinterpret_cast<const float4 *>(smem + (k * ROWS + lr) * kStride + d);
            sum = fmaf(of[k].y, e, sum);
            y.x = fmaf(x.x, e, y.x);
            y.y = fmaf(x.y, e, y.y);
            y.z = fmaf(x.z, e, y.z);
            y.w = fmaf(x.w, e, y.w);
        }
        if (all) {
            const int t = p.by_g(r);
            const float f = sum == 0.0f ? 0.0f : 1.0f / sum;
            *reinterpret_cast<float4 *>(p.out + ((static_cast<long long>(b) * p.T + t) * p.Hq + kvh * p.G + (r - t * p.G)) * D + d) =
                make_float4(y.x * f, y.y * f, y.z * f, y.w * f);
        } else {
            *reinterpret_cast<float4 *>(p.part_o + (part + lr) * D + d) = y;
            if (d == 0) *reinterpret_cast<float2 *>(p.part_ml + (part + lr) * 2) = make_float2(top, sum);
        }
    }
}

template <bool F16, int D, int NT>
void launch_split(const Params &p, hipStream_t s) {
    using S = Shape<F16, D>;
    constexpr size_t states = kWaves * 16 * NT * (D + 6) * 4, weights = kWaves * 16 * NT * S::KT * 4;
    constexpr size_t loop = weights + (query_in_lds(D, NT) ? NT * S::kQuery * 1024 : 0), lds = states > loop ? states : loop;
    static_assert(lds + sizeof(Tree) + NT * 1088 <= 160 * 1024, "LDS of a workgroup");
    if (lds + sizeof(Tree) + NT * 1088 > 65536)
        (void)hipFuncSetAttribute(reinterpret_cast<const void *>(kv_split_kernel<F16, D, NT>), hipFuncAttributeMaxDynamicSharedMemorySize,
                                  static_cast<int>(lds));
    hipLaunchKernelGGL((kv_split_kernel<F16, D, NT>), dim3(workgroups(p)), dim3(kThreads), lds, s, p);
    if (p.quota) launch_merge<D, 16 * NT>(p, kWaves << p.tile_shift, s);
}

template <bool F16, int D>
void launch_d(const Params &p, int rows, hipStream_t s) {
    if (rows == 16) return launch_split<F16, D, 1>(p, s);
    launch_split<F16, D, 2>(p, s);
}

template <bool F16>
void launch(const Params &p, int rows, hipStream_t s) {
    if (p.v.D == 64) launch_d<F16, 64>(p, rows, s);
    else if (p.v.D == 128) launch_d<F16, 128>(p, rows, s);
    else launch_d<F16, 256>(p, rows, s);
}

// How a call's work is laid out: stacked rows of a workgroup, row groups, keys of a tile, and the chunks that the keys
// are cut into (all sequences together, per KV head and row group).
struct Plan {
    int rows, groups, tile, quota;
};

// The plan with this many rows a workgroup, where the cache may hold so many bytes of visible keys.
Plan plan_of(const KvView &v, int T, int Hq, int rows, double bytes) {
    Plan s;
    s.rows = rows;
    s.tile = v.f16 || v.D == 64 ? 32 : 16;
    s.groups = static_cast<int>((static_cast<long long>(T) * (Hq / v.H) + rows - 1) / rows);
    const long long items = static_cast<long long>(v.H) * s.groups;
    const long long cus = device_cu_count() > 0 ? device_cu_count() : 256;
    const int least = s.tile * kWaves;                     // keys of the smallest chunk (kRowsLeast tiles as well)
    const long long most = (static_cast<long long>(kv_capacity(v)) + least - 1) / least;   // chunks of a sequence
    // Workgroups a CU: with a second one the chunks are finer and one's waits are covered by the other, which is worth its
    // partials where the bytes are many and either lengths may differ or row groups share the keys. Of 8 KV heads of 128,
    // one and two a CU: 20 rows over 32 fp16 sequences of about 2100 keys 80 and 66 us, fp32 178 and 126 (of 4096 keys each
    // 99 and 104); 48 rows over one of 131072 132 and 121, 20 rows 98 and 106; 64 rows over one of 8192 19.0 and 20.1; the
    // rows kernel, 128 rows over 32 of 4096, 202 and 181. Heads of 256 fill a CU's registers with one.
    const int per_cu = s.rows == kRowsBlock || (v.D < 256 && bytes >= 0x1p27 && (v.B > 1 || s.groups > 1)) ? 2 : 1;
    s.quota = static_cast<int>(std::min(per_cu * cus / items, v.B * most));
    if (s.quota <= 1 || most == 1) s.quota = 0;            // heads and row groups fill the chip, or no sequence is cut
    return s;
}

// Bytes of the keys that the rows of a call may see.
double seen_bytes(const KvView &v, int T, int window) {
    const long long seen = window > 0 ? std::min<long long>(kv_capacity(v), static_cast<long long>(window) + T) : kv_capacity(v);
    return static_cast<double>(v.B) * seen * v.H * v.D * (v.f16 ? 4 : 8);
}

Plan make_plan(const KvView &v, int T, int Hq, int window) {
    const long long rows = static_cast<long long>(T) * (Hq / v.H);
    // The lengths are on the device: rules go by what the cache may hold of visible keys. More rows a workgroup read a key
    // less often and start later. In us, 8 KV heads of 128 in fp16 filled to the end, in brackets w below:
    //   rows a KV head, cache                16 a workgroup    32   128 (the rows kernel)
    //   20, one of 1024 keys      (2^22)                11.4  12.7  16.0
    //   32, four of 4096          (2^26)                19.6  21.5  27.0
    //   20, one of 32768          (2^27)                34.7  32.3  38.0
    //   20, 32 of 4096            (2^29)               107.3 104.1 111.4
    //   64, one of 4096           (2^30 with the rows)  15.5  16.7  21.4
    //   64, one of 8192           (2^31)                19.5  19.4  25.4
    //   48, four of 4096          (2^31.6)              27.4  25.3  31.5
    //   64, 32 of 1024            (2^33)                56.4  40.9  48.0
    //   256, one of 8192          (2^33)                44.2  35.7  37.0
    //   96, one of 32768          (2^33.6)              76.7  51.3  49.4
    //   256, four of 4096         (2^34)                80.3  58.8  54.3
    //   256, 32 of 4096           (2^37)               608.8 362.4 288.6
    // fp32 and heads of 64 and 256 turn at the same w (of 259 shapes the rule is 0.3 % from the better choice, at most 8 %).
    // Heads of 256 in a rows kernel (a ring of 96 KB, one workgroup a CU) took longer throughout: 256 rows over 8192 keys 109
    // us, with 32 rows a workgroup 59.
    const double bytes = seen_bytes(v, T, window), w = bytes / (v.D * (v.f16 ? 4 : 8)) * std::max(v.D, 128) * 4;
    if (v.f16 && v.D < 256 && rows > 64 && rows * w > 0x1p33) return plan_of(v, T, Hq, kRowsBlock, bytes);
    if (rows > 32 ? rows * w > 0x1p31 : rows > 16 && w >= 0x1p27) return plan_of(v, T, Hq, 32, bytes);
    return plan_of(v, T, Hq, 16, bytes);
}

// Slots of partials that so many chunks need at the most: sequence b of x_b > 1 chunk sizes takes ceil(x_b), fewer
// than 2 x_b and than x_b + 1, and the x_b add up to at most the quota.
size_t partial_slots(const KvView &v, int quota) {
    return quota ? static_cast<size_t>(std::min<long long>(2LL * quota - 1, static_cast<long long>(quota) + v.B - 1)) : 0;
}
// Bytes of partials with this many chunks.
size_t partial_bytes(const KvView &v, const Plan &s, int quota) {
    return static_cast<size_t>(v.H) * s.groups *
           (partial_slots(v, quota) * s.rows * (v.D + 2) * sizeof(float) + v.B * sizeof(int2));
}

}  // namespace

size_t kv_tree_attention_scratch_bytes(const KvView &v, int T, int Hq) {
    // Of the call without a window, or, as a window makes the visible keys fewer, of any plan for fewer: with fewer rows a
    // workgroup there are more row groups, whose chunk table (and, in sequences of many chunks, slots) may be larger.
    const double bytes = seen_bytes(v, T, 0);
    size_t most = 0;
    for (int rows : {16, 32, kRowsBlock}) {
        if (rows > make_plan(v, T, Hq, 0).rows) break;
        const Plan s = plan_of(v, T, Hq, rows, bytes);
        if (s.quota) most = std::max(most, partial_bytes(v, s, s.quota));
    }
    return most;
}

int enqueue_kv_tree_attention(const KvView &v, const KvTreeAttention &a) {
    Params p{};
    p.v = v;
    p.out = a.out;
    p.q = a.q;
    p.lens = a.lens;
    p.counts = a.counts;
    p.parents = a.T > 1 ? a.parents : nullptr;             // one row is its own line
    p.T = a.T;
    p.Hq = a.Hq;
    p.G = a.Hq / v.H;
    // scale * log2(e) as p.scale p.unscale, the first between 2^-61 and 2^100: where scores are in fp32's range, so is a
    // query element times it.
    int k;
    const double m = std::frexp(static_cast<double>(a.scale) * 1.4426950408889634, &k);
    const int in = std::min(std::max(k, -60), 100);
    p.scale = static_cast<float>(std::ldexp(m, in));
    p.unscale = static_cast<float>(std::ldexp(1.0, k - in));           // at least 2^-88
    p.least_exp = std::max(-100, 15 - 126 - (k - in));
    // Within fp32's range with the scores' scaling, and to fp32 the same: past 2^64 a cap is none for every score that
    // softmax tells from its neighbours, below 2^-30 all weights are equal.
    p.soft_cap = a.soft_cap > 0.0f ? std::min(std::max(a.soft_cap, 0x1p-30f), 0x1p64f) : 0.0f;
    p.window = a.window;
    const Plan plan = make_plan(v, a.T, a.Hq, p.window);
    if ((static_cast<double>(v.H) * (plan.quota + static_cast<double>(v.B)) + 7.0) * plan.groups > 0x7fffff)
        return fail(ALJABR_ROCM_ERR_UNSUPPORTED, "kv_tree_attention: T = %d rows of %d heads are more than one launch takes", a.T, a.Hq);
    p.row_groups = plan.groups;
    p.quota = plan.quota;
    p.tile_shift = log2_exact(plan.tile);
    p.by_g.set(p.G);
    p.by_rows.set(v.R);
    p.by_groups.set(plan.groups);
    p.by_heads.set(v.H);
    float *part = a.scratch;
    if (p.quota) {
        if (a.scratch) {
            // As many chunks as the caller's workspace holds the partials of.
            const size_t none = partial_bytes(v, plan, 0), slot = partial_bytes(v, plan, 1) - none;
            const size_t fit = a.scratch_bytes < none ? 0 : (a.scratch_bytes - none) / slot;
            if (fit < partial_slots(v, p.quota)) {
                const size_t most = std::max((fit + 1) / 2, fit + 1 > static_cast<size_t>(v.B) ? fit + 1 - v.B : 0);
                p.quota = most < 2 ? 0 : static_cast<int>(most);
            }
        } else {
            part = static_cast<float *>(stream_scratch(partial_bytes(v, plan, p.quota)));
            if (!part) {
                hipStreamCaptureStatus cs = hipStreamCaptureStatusNone;
                if (hipStreamIsCapturing(current_stream(), &cs) != hipSuccess || cs != hipStreamCaptureStatusNone)
                    return ALJABR_ROCM_ERR_BUFFER;
                (void)hipGetLastError();                   // no memory: one chunk a sequence needs none
                p.quota = 0;
            }
        }
    }
    if (p.quota) {
        p.part_o = part;
        const size_t all = partial_slots(v, p.quota) * v.H * plan.groups * plan.rows;
        p.part_ml = part + all * v.D;
        p.chunks = reinterpret_cast<int2 *>(p.part_ml + 2 * all);
    }
    p.by_chunks.set(p.quota ? p.quota : v.B);
    const int units = v.H * (p.quota ? p.quota : v.B);     // in eights, or enough that a last part of eight is little
    p.span_shift = units % 8 == 0 || units >= 64 ? 3 : 0;
    hipStream_t s = current_stream();
    if (plan.rows == kRowsBlock) launch_rows(p, s);
    else v.f16 ? launch<true>(p, plan.rows, s) : launch<false>(p, plan.rows, s);
    return ALJABR_ROCM_OK;
}

}  // namespace aljabr

using namespace aljabr;

namespace {

int check_attention(const aljabr_rocm_kv_cache *cache, int layer, int T, int Hq, KvView &v) {
    const int rc = kv_view(cache, layer, "kv_tree_attention", v);
    if (rc != ALJABR_ROCM_OK) return rc;
    ALJ_REQUIRE(T > 0 && Hq > 0 && Hq % v.H == 0, "kv_tree_attention: T = %d must be positive and Hq = %d a multiple of %d KV heads",
                T, Hq, v.H);
    ALJ_REQUIRE(static_cast<long long>(T) * Hq <= (1 << 30), "kv_tree_attention: T * Hq exceeds 2^30");
    ALJ_REQUIRE(static_cast<long long>(v.B) * kv_capacity(v) <= (1LL << 34),
                "kv_tree_attention: sequences * the positions of each exceeds 2^34");   // find_chunk adds up tiles, of 16 keys and more
    return ALJABR_ROCM_OK;
}

}  // namespace

extern "C" {

int aljabr_rocm_kv_tree_attention_workspace(const aljabr_rocm_kv_cache *cache, int T, int Hq, size_t *bytes) {
    ALJ_REQUIRE(bytes, "kv_tree_attention_workspace: bytes is null");
    KvView v;
    const int rc = check_attention(cache, 0, T, Hq, v);
    if (rc != ALJABR_ROCM_OK) return rc;
    ALJ_CHECK_READY();
    *bytes = kv_tree_attention_scratch_bytes(v, T, Hq);
    return ALJABR_ROCM_OK;
}

int aljabr_rocm_kv_tree_attention(void *out, const void *Q, const aljabr_rocm_kv_cache *cache, int layer,
                                  const int *context_lens, const int *counts, const int *parents, int T, int Hq, float scale,
                                  int window, float soft_cap, void *workspace, size_t workspace_bytes) {
    KvView v;
    int rc = check_attention(cache, layer, T, Hq, v);
    if (rc != ALJABR_ROCM_OK) return rc;
    ALJ_REQUIRE(out && Q && context_lens, "kv_tree_attention: out, Q and context_lens must be device pointers");
    ALJ_REQUIRE(aligned(out, 16) && aligned(Q, 16) && aligned(workspace, 16),
                "kv_tree_attention: out, Q and workspace must be 16-byte aligned");
    ALJ_REQUIRE(std::isfinite(scale) && std::isfinite(soft_cap), "kv_tree_attention: scale and soft_cap must be finite");
    if (parents && T > kTreeMost)
        return fail(ALJABR_ROCM_ERR_UNSUPPORTED, "kv_tree_attention: a tree of T = %d rows exceeds %d", T, kTreeMost);
    ALJ_CHECK_READY();
    KvTreeAttention a{};
    a.out = static_cast<float *>(out);
    a.q = static_cast<const float *>(Q);
    a.lens = context_lens;
    a.counts = counts;
    a.parents = parents;
    a.T = T;
    a.Hq = Hq;
    a.scale = scale > 0.0f ? scale : static_cast<float>(1.0 / std::sqrt(static_cast<double>(v.D)));
    a.window = window;
    a.soft_cap = soft_cap;
    a.scratch = static_cast<float *>(workspace);
    a.scratch_bytes = workspace ? workspace_bytes : 0;
    rc = enqueue_kv_tree_attention(v, a);
    return rc == ALJABR_ROCM_OK ? finish_launch("kv_tree_attention") : rc;
}

}  // extern "C"
