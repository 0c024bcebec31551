// kv4_attention.hip - attention over the 4-bit KV cache (layout: kv4.hpp).
//
//   out[t, h] = sum_j w_j v_j / sum_j w_j,  w_j = exp(s_j - max s),
//   s_j = cap(scale * q[t, h] . k_j), over the keys j that row t sees.
//
// The rows of a KV head are stacked, r = t * G + g (G = Hq / Hkv). A wave walks
// tiles of 32 keys and keeps 8 rows as the 16 columns of
// v_mfma_f32_16x16x32_f16: columns c and c + 8 carry row c's two fp16 parts,
// so the matrix cores' idle columns buy fp32 accuracy. Both products take the
// decoded codes as their other operand, straight from the cache:
//   S[key][row]  = K Q^T: lane (n, h) of a 16-key half holds key n, dwords
//     [h D/32, (h+1) D/32) of its row: one 16-byte load at D = 128;
//   O^T[d][row] += V^T P^T: lane (n, h) holds the codes of 8 dims (dword n of
//     a row) for the 8 keys whose weights its lane group computed, so V is
//     transposed in registers by taking nibble j of 8 dwords.
// Any order of the contraction will do as long as both operands agree on it,
// and the order of the dims in O is undone when it is stored.
//
// Decoding: a nibble under an exponent is 1024 + q or 64 + q; subtracting 1032
// or 72 is exact, times the scale is the value (kv4.hpp): three instructions a
// pair of values, and a shift for every other one.
//
// Precision: K and V enter as the fp16 numbers they stand for. A query row is
// scaled by a power of two to a largest magnitude in [2^14, 2^15) and split
// into two fp16 parts (2^-22 of each element), a weight, scaled to at most
// 2^15, likewise (what it has below 2^-38 of the largest is lost); sums are
// fp32. The sum of the weights is one more row of the V product, of ones, so
// numerator and denominator hold the same weights.
//
// Keys a row does not see get weight 0, and V rows past a sequence's end may
// hold anything: their scales are taken as 0. In a tile with keys that not every
// row sees, a scale that makes one of a lane's values not finite is taken as 0
// too and remembered for the rows that see the key: their values of these dims
// are made NaN at the end.
//
// Most of the time goes into the vector ALU (55 to 59 % of the issue slots):
// about 364 instructions a tile of 32 keys and 8 rows at D = 128, most of them
// decoding, against 17 matrix products that run beside them. The rest is waits
// (22 to 30 % of the waves' cycles) that 1.6 to 1.7 waves a SIMD do not cover:
// make_plan cuts the keys for two workgroups a CU, of which registers (120 to
// 125 at D = 128, 90 to 93 at D = 64) and the rings would let four run; more
// chunks have not been measured. Measured with the merge: one sequence of
// 131072 keys 39.6 us (151 MB, 3.8 TB/s), 16 of 4096 23.8 us (D = 64 18.5 us,
// D = 256 48 us), 512 keys 8.9 us.
#include <algorithm>
#include <cmath>

#include "kv4_attention.hpp"

namespace aljabr {

using namespace kv4;

namespace {

// One lane's share of a tile as loaded.
template <int D>
struct Keys {
    uint32_t k[2][D / 32];       // per half: this lane's dwords of key n
    uint32_t s[2][D == 256 ? 2 : 1];
};
template <int D>
struct Values {
    uint32_t v[2][4][D == 256 ? 2 : 1];   // per half and key 4h + r: dword(s) of its dims
    uint2 s[2];                  // scales of keys 4h .. 4h + 3
};

// A tile on its way: copied to LDS as it is (16 bytes a lane, whole lines: the
// fragments' own order would touch a line for every 16 bytes), two tiles ahead
// in a ring that is the wave's own. Per half of 16 keys: K and V codes as
// 16-byte chunks, then the scales of both.
//   K: row r's chunk c at 16 (CPR r + (c ^ swizzle(r))): the 16-byte reads of
//      eight neighbouring rows take eight different bank groups;
//   V: rows rotated by r / 4 within their four: the four rows that a read
//      takes are in different banks;
//   scales: [K, V][D/32][16].
template <int D>
struct Ring {
    static constexpr int CPR = D / 32;                     // chunks of a row
    static constexpr int kHalf = 16 * 16 * CPR;            // bytes of K's codes (and of V's) of a half
    static constexpr int kLoads = 2 * kHalf / 1024;        // wave-wide copies of both
    static constexpr int kScaleLoads = D == 256 ? 2 : 1;
    static constexpr int kScales = 256 * kScaleLoads;
    static constexpr int kSlot = 2 * (2 * kHalf + kScales);
    static constexpr int kTileLoads = 2 * (kLoads + kScaleLoads);
    static constexpr int kBytes = 2 * kSlot;               // of a wave
    __device__ static __forceinline__ int swizzle(int r) { return D == 256 ? r & 7 : D == 128 ? r >> 1 & 3 : r >> 2 & 1; }

    const uint8_t *codes[kLoads];                          // this lane's source in row 0 of the planes
    const uint8_t *scales[kScaleLoads];
    uint32_t base;                                         // LDS address of the ring

    __device__ __forceinline__ Ring(const Kv4View &v, int lane, uint32_t lds) : base(lds) {
#pragma unroll
        for (int j = 0; j < kLoads; ++j) {
            const int i = 64 * j + lane, c = i % (16 * CPR);
            const bool is_v = i >= 16 * CPR;
            const int at = c / CPR;
            const int row = is_v ? (at & ~3) | ((at - (at >> 2)) & 3) : at;
            const int chunk = is_v ? c % CPR : c % CPR ^ swizzle(at);
            codes[j] = (is_v ? v.vc : v.kc) + row * (D / 2) + 16 * chunk;
        }
#pragma unroll
        for (int j = 0; j < kScaleLoads; ++j) {
            const int i = (64 * j + lane) % (16 * CPR), g = i % (8 * CPR) >> 3;
            const uint16_t *s = i >= 8 * CPR ? v.vs : v.ks;
            scales[j] = reinterpret_cast<const uint8_t *>(s + static_cast<long long>(g) * v.R + 2 * (i & 7));
        }
    }
    // The copies of a tile into slot `slot` of the ring.
    __device__ __forceinline__ void fetch(const Place &w, int slot) const {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const uint32_t dst = base + slot * kSlot + u * (kSlot / 2);
#pragma unroll
            for (int j = 0; j < kLoads; ++j) dma16(codes[j] + w.row[u] * (D / 2), dst + 1024 * j);
#pragma unroll
            for (int j = 0; j < kScaleLoads; ++j) dma4(scales[j] + w.scale[u] * 2, dst + 2 * kHalf + 256 * j);
        }
    }
};

template <int N>
__device__ __forceinline__ void wait_copies() {
    static_assert(N < 64, "vmcnt range");
    asm volatile("s_waitcnt vmcnt(%0)" ::"i"(N) : "memory");
}

template <class T>
__device__ __forceinline__ T lds_at(const char *slot, int off) {
    return *reinterpret_cast<const T *>(slot + off);
}

// A tile from its slot of the ring.
template <int D>
__device__ __forceinline__ void read_tile(const char *slot, int n, int h, Keys<D> &xk, Values<D> &xv) {
    using R = Ring<D>;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
        const char *half = slot + u * (R::kSlot / 2), *sc = half + 2 * R::kHalf;
        if constexpr (D == 64) {
            const uint2 a = lds_at<uint2>(half, 32 * n + 16 * (h >> 1 ^ R::swizzle(n)) + 8 * (h & 1));
            xk.k[u][0] = a.x;
            xk.k[u][1] = a.y;
            xk.s[u][0] = lds_at<uint16_t>(sc, 32 * (h >> 1) + 2 * n);
        } else {
#pragma unroll
            for (int i = 0; i < D / 128; ++i) {
                const int c = D / 128 * h + i;
                const uint4 a = lds_at<uint4>(half, 16 * (R::CPR * n + (c ^ R::swizzle(n))));
                xk.k[u][4 * i] = a.x; xk.k[u][4 * i + 1] = a.y; xk.k[u][4 * i + 2] = a.z; xk.k[u][4 * i + 3] = a.w;
                xk.s[u][i] = lds_at<uint16_t>(sc, 32 * c + 2 * n);
            }
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int at = R::kHalf + (4 * h + (r + h & 3)) * (D / 2);
            if constexpr (D == 256) {
                const uint2 a = lds_at<uint2>(half, at + 8 * n);
                xv.v[u][r][0] = a.x;
                xv.v[u][r][1] = a.y;
            } else {
                xv.v[u][r][0] = lds_at<uint32_t>(half, at + (D == 64 ? 4 * (n >> 1) : 4 * n));
            }
        }
        xv.s[u] = lds_at<uint2>(sc, 32 * (R::CPR + (D == 64 ? n >> 3 : D == 128 ? n >> 2 : n >> 1)) + 8 * h);
    }
}

// O += V^T P^T of a tile: NT column tiles, output tile j holds nibble j of the
// lanes' dwords (D = 256: j / 8 picks the dword). vd: scales of key pairs.
template <int D, int NT>
__device__ __forceinline__ void add_values(const Magic &g, const Values<D> &x, const half2v (&vd)[4], const half8 (&pw)[NT],
                                           uint32_t vsel, f32x4 (&o)[NT][D / 16]) {
#pragma unroll
    for (int i = 0; i < (D == 256 ? 2 : 1); ++i) {
#pragma unroll
        for (int half = 0; half < (D == 64 ? 1 : 2); ++half) {
            uint32_t f[4][4];                              // [key pair][nibble]
#pragma unroll
            for (int pr = 0; pr < 4; ++pr) {
                const uint32_t w0 = x.v[pr >> 1][2 * (pr & 1)][i], w1 = x.v[pr >> 1][2 * (pr & 1) + 1][i];
                const uint32_t sel = D == 64 ? vsel : half ? 0x07060302u : 0x05040100u;
                decode8(g, __builtin_amdgcn_perm(w1, w0, sel), vd[pr], f[pr]);
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const half8 a = frag(f[0][j], f[1][j], f[2][j], f[3][j]);
#pragma unroll
                for (int c = 0; c < NT; ++c) {
                    f32x4 &acc = o[c][8 * i + 4 * half + j];
                    acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, pw[c], acc, 0, 0, 0);
                }
            }
        }
    }
}

// grid: chunks of KV heads and row groups (work_of).
template <int D, int NT, bool PAGED, bool CAP>
__global__ __launch_bounds__(waves(D) * 64, D == 256 ? 2 : NT == 1 || D == 64 ? 3 : 2) void kv4_split_kernel(Params p) {
    constexpr int ND = D / 32, ROWS = 8 * NT, OT = D / 16, kWaves = waves(D);
    extern __shared__ float smem[];                        // the waves' rings, then their states [kWaves][ROWS][D + 2]
    const int lane = threadIdx.x & 63, n = lane & 15, h = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    int item, w;
    work_of(p, blockIdx.x, item, w);
    const int kvh = p.by_groups(item), r0 = (item - kvh * p.row_groups) * ROWS;
    const Chunk chunk = find_chunk(p, w, r0, ROWS, kWaves);
    if (chunk.b < 0) return;
    const int b = chunk.b, t0 = chunk.t0, t1 = chunk.t1;
    if (p.quota && w == chunk.first && threadIdx.x == 0)
        p.chunks[static_cast<long long>(item) * p.v.B + b] = make_int2(chunk.slot, chunk.count);
    const Seq seq = chunk.seq;
    const int r1 = min(r0 + ROWS, seq.cnt * p.G);

    // The first two tiles go out before anything else is read.
    const Ring<D> ring(p.v, lane, lds_address(smem) + wave * Ring<D>::kBytes);
    const char *slots = reinterpret_cast<const char *>(smem) + wave * Ring<D>::kBytes;
    Place here, next;
    if (t0 + wave < t1) {
        here = place<D, PAGED>(p, b, kvh, seq.n, t0 + wave);
        ring.fetch(here, 0);
    }
    if (t0 + wave + kWaves < t1) {
        next = place<D, PAGED>(p, b, kvh, seq.n, t0 + wave + kWaves);
        ring.fetch(next, 1);
    }

    // This lane's columns: row, visible keys, query parts (dword i of the lane's share of a row).
    int lo[NT], hi[NT];
    half8 qf[NT][ND];
    float unscale[NT];
    int full_lo = 0, full_hi = 0x7fffffff;                 // keys that every row sees
#pragma unroll
    for (int c = 0; c < NT; ++c) {
        const int r = min(r0 + 8 * c + (n & 7), r1 - 1);   // columns past the rows repeat the last and are not stored
        const int t = p.by_g(r), g = r - t * p.G;
        key_range(p, seq, t, lo[c], hi[c]);
        const float *qr = p.q + ((static_cast<long long>(b) * p.T + t) * p.Hq + kvh * p.G + g) * D;
        float x[ND][8], top = 0.0f;
#pragma unroll
        for (int i = 0; i < ND; ++i) {
            const int w = h * ND + i;
            const float4 a = *reinterpret_cast<const float4 *>(qr + 32 * (w >> 2) + 4 * (w & 3));
            const float4 e = *reinterpret_cast<const float4 *>(qr + 32 * (w >> 2) + 4 * (w & 3) + 16);
            // decode8's order: nibbles 0 4 1 5 2 6 3 7; even nibbles are dims 0..3 of the dword, odd ones 16..19.
            x[i][0] = a.x; x[i][1] = a.z; x[i][2] = e.x; x[i][3] = e.z;
            x[i][4] = a.y; x[i][5] = a.w; x[i][6] = e.y; x[i][7] = e.w;
#pragma unroll
            for (int j = 0; j < 8; ++j) top = fmaxf(top, fabsf(x[i][j]));
        }
        top = fmaxf(top, __shfl_xor(top, 16));
        top = fmaxf(top, __shfl_xor(top, 32)) * p.scale;
        int e = 0;
        if (top > 0.0f && top <= 3.4028235e38f) (void)frexpf(top, &e);     // top in [2^(e-1), 2^e)
        e = e < -100 ? -100 : e;
        const float up = ldexpf(1.0f, 15 - e);             // a power of two: y is the same number wherever it is used
        unscale[c] = ldexpf(p.unscale, e - 15);
#pragma unroll
        for (int i = 0; i < ND; ++i)
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float y = x[i][j] * p.scale * up;
                const _Float16 first = static_cast<_Float16>(y);
                qf[c][i][j] = n < 8 ? first : static_cast<_Float16>(y - static_cast<float>(first));
            }
    }
    {
        int first_lo, first_hi, last_lo, last_hi;
        key_range(p, seq, p.by_g(r0), first_lo, first_hi);
        key_range(p, seq, p.by_g(r1 - 1), last_lo, last_hi);
        full_lo = last_lo;
        full_hi = first_hi;
    }
    const float lo_part = n < 8 ? 0.0f : 1.0f;
    const uint32_t vsel = n & 1 ? 0x07060302u : 0x05040100u;

    f32x4 o[NT][OT], l[NT];                                // l: the sum of the weights, in every accumulator
    float m[NT];
    uint32_t poison[NT];                                   // per lane n: a value of its dims, of a key this column sees, is not finite
#pragma unroll
    for (int c = 0; c < NT; ++c) {
        m[c] = -INFINITY;
        poison[c] = 0;
        l[c] = f32x4{};
#pragma unroll
        for (int j = 0; j < OT; ++j) o[c][j] = f32x4{};
    }
    const Magic g;
    const half8 ones = frag(0x3c003c00u, 0x3c003c00u, 0x3c003c00u, 0x3c003c00u);

    int slot = 0;
    for (int kt = t0 + wave; kt < t1; kt += kWaves, slot ^= 1) {
        const int k0 = kt * kTile;
        Keys<D> xk;
        Values<D> xv;
        if (kt + kWaves < t1) wait_copies<Ring<D>::kTileLoads>();
        else wait_copies<0>();
        read_tile<D>(slots + slot * Ring<D>::kSlot, n, h, xk, xv);
        Place after;
        if (kt + 2 * kWaves < t1) {
            after = place<D, PAGED>(p, b, kvh, seq.n, kt + 2 * kWaves);
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");     // the slot has been read
            ring.fetch(after, slot);
        }
        const bool whole = k0 >= full_lo && k0 + kTile <= full_hi && here.ok[0] && here.ok[1];   // every row sees every key

        // S of the two halves: accumulator r is key k0 + 16u + 4h + r of this lane's column.
        f32x4 s[NT][2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
#pragma unroll
            for (int c = 0; c < NT; ++c) s[c][u] = f32x4{};
            half2v kd[D == 256 ? 2 : 1];
#pragma unroll
            for (int i = 0; i < (D == 256 ? 2 : 1); ++i) kd[i] = as_half2(__builtin_amdgcn_perm(xk.s[u][i], xk.s[u][i], 0x01000100u));
#pragma unroll
            for (int i = 0; i < ND; ++i) {
                uint32_t f[4];
                decode8(g, xk.k[u][i], kd[D == 256 ? i / 4 : 0], f);
                const half8 a = frag(f[0], f[1], f[2], f[3]);
#pragma unroll
                for (int c = 0; c < NT; ++c) s[c][u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, qf[c][i], s[c][u], 0, 0, 0);
            }
        }
        half8 pw[NT];
#pragma unroll
        for (int c = 0; c < NT; ++c) {
            float y[8], mx = -INFINITY;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float raw = s[c][i >> 2][i & 3];
                y[i] = raw + other_part(raw);
            }
            if constexpr (CAP) {
                const float cap = p.soft_cap * kLog2e, in = fminf(unscale[c] / cap, 3e38f);    // finite: 0 stays 0
#pragma unroll
                for (int i = 0; i < 8; ++i) y[i] = cap * tanhf(y[i] * in);
            }
            const float us = CAP ? 1.0f : unscale[c];
            if (!whole) {
                const int first = lo[c] - k0 - 4 * h, end = hi[c] - k0 - 4 * h;
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (16 * (i >> 2) + (i & 3) < first || 16 * (i >> 2) + (i & 3) >= end || !here.ok[i >> 2]) y[i] = -INFINITY;
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) mx = fmaxf(mx, y[i]);
            mx *= us;
            // The reference m of a column is raised only when a score exceeds it by more than 2.
            if (__any(mx > m[c] + 2.0f)) {
                mx = fmaxf(mx, __shfl_xor(mx, 16));
                mx = fmaxf(mx, __shfl_xor(mx, 32));
                const float up = mx > m[c] + 2.0f ? mx : m[c];
                const float alpha = up == m[c] ? 1.0f : __builtin_amdgcn_exp2f(m[c] - up);     // 0 while m is -inf
                l[c] *= alpha;
#pragma unroll
                for (int j = 0; j < OT; ++j) o[c][j] *= alpha;
                m[c] = up;
            }
            const float ref = m[c] == -INFINITY ? 0.0f : m[c];
            uint32_t w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float e[2];
#pragma unroll
                for (int k = 0; k < 2; ++k) e[k] = __builtin_amdgcn_exp2f(fmaf(y[2 * i + k], us, -ref)) * kWeightScale;
                const half2v first = pair(e[0], e[1]);
                w[i] = as_u32(pair(fmaf(static_cast<float>(first[0]), -lo_part, e[0]),
                                   fmaf(static_cast<float>(first[1]), -lo_part, e[1])));
            }
            pw[c] = frag(w[0], w[1], w[2], w[3]);
            l[c] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ones, pw[c], l[c], 0, 0, 0);
        }
        half2v vd[4] = {as_half2(xv.s[0].x), as_half2(xv.s[0].y), as_half2(xv.s[1].x), as_half2(xv.s[1].y)};
        if (!whole) {
            bool odd = false;
            const int end = seq.n - k0 - 4 * h;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                if (16 * (i >> 2) + (i & 3) >= end || !here.ok[i >> 2]) vd[i >> 1][i & 1] = static_cast<_Float16>(0.0f);
                odd |= may_overflow(vd[i >> 1][i & 1]);
            }
            if (__any(odd)) {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const _Float16 d = vd[i >> 1][i & 1];
                    const uint32_t w = xv.v[i >> 2][i & 3][0];
                    bool over = overflows(g, D == 64 ? __builtin_amdgcn_perm(w, w, vsel) : w, d);
                    if constexpr (D == 256) over |= overflows(g, xv.v[i >> 2][i & 3][1], d);
                    const uint64_t bad = __ballot(over);
#pragma unroll 1
                    for (int hh = 0; hh < 4; ++hh) {
                        const int key = k0 + 16 * (i >> 2) + 4 * hh + (i & 3);
#pragma unroll
                        for (int c = 0; c < NT; ++c)
                            if (key >= lo[c] && key < hi[c]) poison[c] |= static_cast<uint32_t>(bad >> (16 * hh)) & 0xffffu;
                    }
                    if (over) vd[i >> 1][i & 1] = static_cast<_Float16>(0.0f);
                }
            }
        }
        add_values<D, NT>(g, xv, vd, pw, vsel, o);
        here = next;
        next = after;
    }
    __syncthreads();                                       // every wave has left its ring (its last copies were waited for)

    // The wave's state to LDS: O^T tile j, accumulator r: nibble j of dword 4h + r (D = 64: of 16-bit piece 4h + r;
    // D = 256: of dword 2 (4h + r) + j / 8).
#pragma unroll
    for (int c = 0; c < NT; ++c) {
        const float sum = l[c][0] + other_part(l[c][0]);
        if (m[c] == -INFINITY && sum != sum) m[c] = 0.0f;  // a NaN score alone leaves no reference: any finite one carries it
        float *st = smem + (wave * ROWS + 8 * c + (n & 7)) * (D + 2);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int piece = 4 * h + r;                   // the lane n whose V codes these are
            const float bad = poison[c] >> piece & 1 ? NAN : 0.0f;
#pragma unroll
            for (int j = 0; j < OT; ++j) {
                const float val = o[c][j][r] + other_part(o[c][j][r]) + bad;
                const int w = D == 128 ? piece : D == 64 ? piece >> 1 : 2 * piece + (j >> 3);
                const int x = D == 64 ? 4 * (piece & 1) + j : j & 7;           // nibble of dword w
                if (n < 8) st[32 * (w >> 2) + 16 * (x & 1) + 4 * (w & 3) + (x >> 1)] = val;
            }
        }
        if (lane < 8) {
            st[D] = m[c];
            st[D + 1] = sum;
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < ROWS * D; i += kWaves * 64) {
        const int r = r0 + i / D, dd = i % D;
        if (r >= r1) break;
        float M = -INFINITY, mw[kWaves];
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            mw[w] = smem[(w * ROWS + i / D) * (D + 2) + D];
            M = fmaxf(M, mw[w]);
        }
        float L = 0.0f, O = 0.0f;
        if (M != -INFINITY) {
#pragma unroll
            for (int w = 0; w < kWaves; ++w) {
                const float *st = smem + (w * ROWS + i / D) * (D + 2);
                const float f = mw[w] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(mw[w] - M);
                L = fmaf(st[D + 1], f, L);
                O = fmaf(st[dd], f, O);
            }
        }
        if (chunk.count == 1) {
            const int t = p.by_g(r), g = r - t * p.G;
            p.out[((static_cast<long long>(b) * p.T + t) * p.Hq + kvh * p.G + g) * D + dd] = L == 0.0f ? 0.0f : O / L;
        } else {
            const long long row = (static_cast<long long>(chunk.slot + w - chunk.first) * p.v.H * p.row_groups + item) * ROWS + i / D;
            p.part_o[row * D + dd] = O;
            if (dd == 0) *reinterpret_cast<float2 *>(p.part_ml + row * 2) = make_float2(M, L);
        }
    }
}

// Rows a workgroup stacks: 8 or 16 in the split kernel, kRowsBlock in the rows
// kernel, which decodes a tile once for all its rows but leaves waves idle
// below 128. It is taken from 33 rows a KV head on. Rows kernel / split kernel,
// us, 8 KV heads:
//   rows               20       32       40       48       64       80       96
//   D = 64
//   4 x 2048 keys  16.5/15.8 17.1/17.0 17.8/19.2 18.3/19.3 19.2/19.8 20.6/23.1 21.4/29.9
//   16 x 4096        62/38     63/39     65/66     66/67     67/58     70/77     71/79
//   D = 128
//   1 x 4096       18.9/18.1 19.8/19.0 20.7/21.9 21.3/22.1 22.4/21.7 23.7/24.3 24.8/26.4
//   4 x 2048       21.2/21.9 22.4/23.5 23.5/26.5 24.3/27.1 25.7/28.0 26.7/32.4 26.6/40.4
//   16 x 4096        82/52     84/53     86/100    87/101    88/82     92/116    94/119
//   D = 256
//   1 x 4096       33.1/23.9 35.0/26.4 36.5/30.1 37.4/30.0 39.5/34.2 39.9/40.1 40.3/40.4
//   4 x 2048       36.8/29.6 39.1/35.7 40.3/41.3 41.0/41.9 42.4/48.4 43.7/61.5 45.3/61.7
//   16 x 4096       168/100   173/131   177/200   179/176   183/193   187/266   191/345
// So it loses at 49 to 64 rows of many long sequences at D <= 128 (four full
// row groups of 16; 7 to 14 %), at D = 256 over one sequence up to 64 rows
// (16 to 25 %), and below the threshold 4 % in one of the rows above.
constexpr int kManyRows = 33;
int stacked_rows(long long rows, int D) { return rows >= kManyRows ? kRowsBlock : rows > 8 && D < 256 ? 16 : 8; }

template <int D, int NT, bool PAGED>
void launch_split(const Params &p, hipStream_t s) {
    constexpr int kWaves = waves(D), states = kWaves * 8 * NT * (D + 2) * 4, rings = kWaves * Ring<D>::kBytes;
    constexpr size_t lds = states > rings ? states : rings;
    static_assert(lds <= 65536, "LDS of a workgroup");
    const dim3 grid(p.v.H * p.row_groups * (p.quota ? p.quota + (p.v.B > 1 ? p.v.B : 0) : p.v.B));
    if (p.soft_cap > 0.0f)
        hipLaunchKernelGGL((kv4_split_kernel<D, NT, PAGED, true>), grid, dim3(kWaves * 64), lds, s, p);
    else
        hipLaunchKernelGGL((kv4_split_kernel<D, NT, PAGED, false>), grid, dim3(kWaves * 64), lds, s, p);
    if (p.quota) hipLaunchKernelGGL((kv4_merge_kernel<D, 8 * NT>), dim3(p.Hq, p.T, p.v.B), dim3(256), 0, s, p);
}

template <int D, int NT>
void launch(const Params &p, hipStream_t s) {
    p.v.table ? launch_split<D, NT, true>(p, s) : launch_split<D, NT, false>(p, s);
}

// How a call's work is laid out: stacked rows of a workgroup, row groups, and
// the chunks that the keys are cut into (all sequences together, per KV head
// and row group): two workgroups a CU, of 128 rows one (256 rows of a 2048-key
// chunk: 38.3 us against 40.0 with two), of D = 256 three, whose workgroups have
// two waves (16 sequences of 4096 keys: 47.8 us against 54.5; a draft of 5 over a
// window of 1024 in 8 sequences: 26.8 against 31.9, with four 28.3).
struct Plan {
    int rows, groups, quota;
};
Plan make_plan(const Kv4View &v, int T, int Hq) {
    Plan s;
    const long long rows = static_cast<long long>(T) * (Hq / v.H);
    s.rows = stacked_rows(rows, v.D);
    s.groups = static_cast<int>((rows + s.rows - 1) / s.rows);
    const long long items = static_cast<long long>(v.H) * s.groups;
    const long long cus = device_cu_count() > 0 ? device_cu_count() : 256;
    const int least = kTile * (s.rows == kRowsBlock ? kRowsLeast : waves(v.D));          // keys of the smallest chunk
    const long long most = (static_cast<long long>(kv4_capacity(v)) + least - 1) / least;   // chunks of a sequence
    s.quota = static_cast<int>(std::min((s.rows == kRowsBlock ? 1 : v.D == 256 ? 3 : 2) * cus / items, v.B * most));
    if (s.quota <= 1 || most == 1) s.quota = 0;            // heads and row groups fill the chip, or no sequence is cut
    return s;
}

// Slots of partials that so many chunks need at the most: sequence b of x_b > 1 chunk sizes takes ceil(x_b), fewer
// than 2 x_b and than x_b + 1, and the x_b add up to at most the quota.
size_t partial_slots(const Kv4View &v, int quota) {
    return quota ? static_cast<size_t>(std::min<long long>(2LL * quota - 1, static_cast<long long>(quota) + v.B - 1)) : 0;
}
// Bytes of partials with this many chunks.
size_t partial_bytes(const Kv4View &v, const Plan &s, int quota) {
    return static_cast<size_t>(v.H) * s.groups *
           (partial_slots(v, quota) * s.rows * (v.D + 2) * sizeof(float) + v.B * sizeof(int2));
}

}  // namespace

size_t kv4_attention_scratch_bytes(const Kv4View &v, int T, int Hq) {
    const Plan s = make_plan(v, T, Hq);
    return s.quota ? partial_bytes(v, s, s.quota) : 0;
}

int enqueue_kv4_attention(const Kv4View &v, const Kv4Attention &a) {
    Params p{};
    p.v = v;
    p.out = a.out;
    p.q = a.q;
    p.lens = a.lens;
    p.counts = a.counts;
    p.T = a.T;
    p.Hq = a.Hq;
    p.G = a.Hq / v.H;
    // scale * log2(e) as p.scale p.unscale, the first between 2^-61 and 2^100: where scores are in fp32's range, so is a
    // query element times it.
    int k;
    const double m = std::frexp(static_cast<double>(a.scale) * 1.4426950408889634, &k);
    const int in = std::min(std::max(k, -60), 100);
    p.scale = static_cast<float>(std::ldexp(m, in));
    p.unscale = static_cast<float>(std::ldexp(1.0, k - in));
    // Within fp32's range with the scores' scaling, and to fp32 the same: past 2^64 a cap is none for every score that
    // softmax tells from its neighbours, below 2^-30 all weights are equal.
    p.soft_cap = a.soft_cap > 0.0f ? std::min(std::max(a.soft_cap, 0x1p-30f), 0x1p64f) : 0.0f;
    p.causal = a.causal;
    p.window = std::min(a.window, 1 << 30);                // past every key; pos - window stays in 32 bits
    const Plan plan = make_plan(v, a.T, a.Hq);
    if (static_cast<double>(v.H) * plan.groups * (plan.quota + static_cast<double>(v.B)) > 0x7fffff)
        return fail(ALJABR_ROCM_ERR_UNSUPPORTED, "kv4_attention: T = %d rows of %d heads are more than one launch takes", a.T, a.Hq);
    p.row_groups = plan.groups;
    p.quota = plan.quota;
    p.by_g.set(p.G);
    p.by_groups.set(plan.groups);
    p.by_rows.set(v.R);
    p.by_items.set(v.H * plan.groups);
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
    const int per = plan.rows;
    hipStream_t s = current_stream();
    if (per == kRowsBlock) launch_rows(p, s);
    else if (v.D == 64) per == 8 ? launch<64, 1>(p, s) : launch<64, 2>(p, s);
    else if (v.D == 128) per == 8 ? launch<128, 1>(p, s) : launch<128, 2>(p, s);
    else launch<256, 1>(p, s);
    return ALJABR_ROCM_OK;
}

}  // namespace aljabr

using namespace aljabr;

namespace {

int check_attention(const aljabr_rocm_kv4_cache *cache, int T, int Hq, Kv4View &v) {
    const int rc = kv4_view(cache, "kv4_attention", v);
    if (rc != ALJABR_ROCM_OK) return rc;
    ALJ_REQUIRE(T > 0 && Hq > 0 && Hq % v.H == 0, "kv4_attention: T = %d must be positive and Hq = %d a multiple of %d KV heads",
                T, Hq, v.H);
    ALJ_REQUIRE(static_cast<long long>(T) * Hq <= (1 << 30), "kv4_attention: T * Hq exceeds 2^30");
    ALJ_REQUIRE(static_cast<long long>(v.B) * kv4_capacity(v) <= (1LL << 35),
                "kv4_attention: sequences * the positions of each exceeds 2^35");   // find_chunk adds up their tiles
    return ALJABR_ROCM_OK;
}

}  // namespace

extern "C" {

int aljabr_rocm_kv4_attention_workspace(const aljabr_rocm_kv4_cache *cache, int T, int Hq, size_t *bytes) {
    ALJ_REQUIRE(bytes, "kv4_attention_workspace: bytes is null");
    Kv4View v;
    const int rc = check_attention(cache, T, Hq, v);
    if (rc != ALJABR_ROCM_OK) return rc;
    ALJ_CHECK_READY();
    *bytes = kv4_attention_scratch_bytes(v, T, Hq);
    return ALJABR_ROCM_OK;
}

int aljabr_rocm_kv4_attention(void *out, const void *Q, const aljabr_rocm_kv4_cache *cache, const int *context_lens,
                              const int *counts, int T, int Hq, float scale, int is_causal, int window, float soft_cap,
                              void *workspace, size_t workspace_bytes) {
    Kv4View v;
    int rc = check_attention(cache, T, Hq, v);
    if (rc != ALJABR_ROCM_OK) return rc;
    ALJ_REQUIRE(out && Q && context_lens, "kv4_attention: out, Q and context_lens must be device pointers");
    ALJ_REQUIRE(aligned(out, 16) && aligned(Q, 16) && aligned(workspace, 16),
                "kv4_attention: out, Q and workspace must be 16-byte aligned");
    ALJ_REQUIRE(std::isfinite(scale) && std::isfinite(soft_cap), "kv4_attention: scale and soft_cap must be finite");
    ALJ_CHECK_READY();
    Kv4Attention a{};
    a.out = static_cast<float *>(out);
    a.q = static_cast<const float *>(Q);
    a.lens = context_lens;
    a.counts = counts;
    a.T = T;
    a.Hq = Hq;
    a.scale = scale > 0.0f ? scale : static_cast<float>(1.0 / std::sqrt(static_cast<double>(v.D)));
    a.causal = is_causal != 0;
    a.window = window;
    a.soft_cap = soft_cap;
    a.scratch = static_cast<float *>(workspace);
    a.scratch_bytes = workspace ? workspace_bytes : 0;
    rc = enqueue_kv4_attention(v, a);
    return rc == ALJABR_ROCM_OK ? finish_launch("kv4_attention") : rc;
}

}  // extern "C"
