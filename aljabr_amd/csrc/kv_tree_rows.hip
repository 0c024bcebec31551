// kv_tree_rows.hip - attention of many stacked rows over an fp16 cache: trees
// of large groups, chunks of prompts, prompts (kv_tree.hip has the formulas and
// the precision).
//
// A workgroup takes 128 stacked rows, 32 a wave, and walks tiles of 32 keys,
// which its waves copy to LDS as they lie in the cache, two tiles ahead, with
// one barrier a tile. K's rows are read from there as the fragments of
// v_mfma_f32_32x32x16_f16, V's transposed by the LDS itself (ds_read_b64_tr_b16
// gives a lane four keys of one dim):
//   S^T = K Q^T, O^T += V^T P^T, rows along the lanes: a row's query parts,
// maximum and sum stay in its two lanes. Two products a score and a value, for
// the two fp16 parts of queries and weights.
//
// The 16-byte chunks of a row are swapped around on the way, so that the rows
// that one LDS access takes lie in different banks: chunk c of K's row n at
// c ^ (n & 15) (D = 64: c ^ (n / 2 & 7)), of V's, of which an access takes 32
// bytes of four neighbouring rows for two groups of 16 dims, at c ^ 4 (n & 3)
// (D = 64: c ^ 4 (n / 2 & 1)).
//
// Values that are not finite: a tile that not every row sees whole is cleaned
// of them in LDS first, and they are added by hand for the rows that see them.
// In any other tile, and in keys, they make sums that are not finite; the
// workgroup then walks its keys again with every tile treated so, and scores
// that are NaN computed in fp32.
#include "kv_tree.hpp"

namespace aljabr {

using namespace kvt;

namespace {

typedef _Float16 half4 __attribute__((ext_vector_type(4)));
typedef _Float16 half2v __attribute__((ext_vector_type(2)));
typedef __fp16 fp16x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr int kTile = 32;

template <int D>
struct Rows {
    static constexpr int kRow = 2 * D;                     // bytes
    static constexpr int kPlane = kTile * kRow;            // of K's (or V's) tile
    static constexpr int kBuffer = 2 * kPlane;
    static constexpr int kBuffers = 3;
    static constexpr int CPR = kRow / 16;                  // chunks of a row
    static constexpr int RPL = 64 / CPR;                   // rows of a wave-wide copy
    static constexpr int kCopies = 8 / RPL;                // of a wave's 8 rows of K (and of V)
    static constexpr int kSpan = D == 64 ? 32 : 64, kStride = kSpan + 4;   // dims of a round of the output, and its rows in LDS
    static constexpr int kOut = kWaves * 32 * kStride * 4;
    static constexpr int kBytes = kBuffers * kBuffer > kOut ? kBuffers * kBuffer : kOut;
    __device__ static __forceinline__ int k_swap(int row) { return D == 64 ? row >> 1 & 7 : row & 15; }
    __device__ static __forceinline__ int v_swap(int row) { return D == 64 ? 4 * (row >> 1 & 1) : 4 * (row & 3); }
};

__device__ __forceinline__ uint32_t lds_address(const void *p) {
    return static_cast<uint32_t>(reinterpret_cast<uintptr_t>((const __attribute__((address_space(3))) void *)p));
}

template <int N>
__device__ __forceinline__ void wait_copies() {
    static_assert(N < 64, "vmcnt range");
    asm volatile("s_waitcnt vmcnt(%0)" ::"i"(N) : "memory");
}

__device__ __forceinline__ half2v pair(float a, float b) { return half2v{static_cast<_Float16>(a), static_cast<_Float16>(b)}; }

// A dword of two fp16 numbers: bits of those whose exponent is all ones.
__device__ __forceinline__ uint32_t not_finite(uint32_t w) { return ((w & 0x7fff7fffu) + 0x04000400u) & 0x80008000u; }
__device__ __forceinline__ uint32_t clean(uint32_t w) {
    const uint32_t bad = not_finite(w);
    return w & ~((bad >> 15) * 0xffffu);
}

template <int D>
__global__ __launch_bounds__(kThreads, D == 256 ? 1 : 2) void kv_rows_kernel(Params p) {
    using R = Rows<D>;
    constexpr int STEPS = D / 16, DT = D / 32;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    __shared__ Tree tree;
    __shared__ int odd_tile;                               // the last tile that held values which are not finite, plus 1
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
    const int base = seq.n - seq.cnt, r1 = min(r0 + kRowsBlock, seq.cnt * p.G), w0 = r0 + 32 * wave;
    const bool idle = w0 >= r1;                            // a wave without rows only copies

    // This wave copies rows 8 wave .. + 7 of a tile, of its half wave / 2. A lane's chunk and row of each copy:
    const int own = lane / R::CPR, slot = lane % R::CPR;
    const uint32_t ring = lds_address(lds);
    uint32_t ok = 0, ok_next = 0;                          // of the tile at hand and the next: halves whose block exists
    Places<2> places{t0, 1};
    auto copy = [&](int kt, int buffer) __attribute__((always_inline)) {
        const int i = kt - t0, u = wave >> 1, first = 8 * (wave & 1);
        if (i == places.held + 32) places.load(p, R::kRow, b, kvh, seq.n, i);
        const long long at = places.offset(i, u);
        const int last = last_row(p, kt * kTile + (kt * kTile + 16 * u < seq.n ? 16 * u : 0));
        const uint32_t dst = ring + buffer * R::kBuffer + (16 * u + first) * R::kRow;
#pragma unroll
        for (int j = 0; j < R::kCopies; ++j) {
            const int row = first + j * R::RPL + own, in = min(row, last) * R::kRow;
            dma16(p.v.k + at + (in + 16 * (slot ^ R::k_swap(row))), dst + 1024 * j);
            dma16(p.v.v + at + (in + 16 * (slot ^ R::v_swap(row))), dst + R::kPlane + 1024 * j);
        }
        return places.ok(i);
    };
    auto start = [&]() __attribute__((always_inline)) {
        places.load(p, R::kRow, b, kvh, seq.n, 0);
        if (t0 < t1) ok = copy(t0, 0);
        if (t0 + 1 < t1) ok_next = copy(t0 + 1, 1);
    };
    // A tile's rows by hand, for the paths that are rarely taken.
    auto row_of = [&](int kt, int key, bool of_v) __attribute__((always_inline)) {
        int at = min(kt * kTile + key, seq.n - 1), s = b;
        if (p.v.table) {
            const int blk = p.by_rows(at);
            s = p.v.table[static_cast<long long>(b) * p.v.max_blocks + blk];
            at -= blk * p.v.R;
            if (s < 0 || s >= p.v.num_blocks) s = 0;
        }
        return (of_v ? p.v.v : p.v.k) + ((static_cast<long long>(s) * p.v.H + kvh) * p.v.R + at) * R::kRow;
    };
    start();
    const bool filled = p.parents && (p.window > 0 || t1 * kTile > base);
    if (tid == 0) odd_tile = 0;
    if (filled) fill_tree(tree, p.parents + static_cast<long long>(b) * p.T, seq.cnt, p.window);
    else __syncthreads();

    // This lane's row, what it sees; the wave's keys, and those that all rows of the wave and of the workgroup see.
    const int r = min(w0 + nl, r1 - 1);                    // lanes past the rows repeat the last and are not stored
    const int t = p.by_g(r);
    const Range range = range_of(p, seq, t, tree, filled);
    const int t_first = p.by_g(min(w0, r1 - 1)), t_last = p.by_g(min(w0 + 31, r1 - 1));
    const int w_lo = p.window > 0 ? base + (p.parents ? 0 : t_first) - p.window + 1 : 0, w_hi = base + t_last + 1;
    const int full_lo = p.window > 0 ? base + t_last - p.window + 1 : 0, full_hi = p.parents ? base : base + t_first + 1;
    const int all_lo = p.window > 0 ? base + p.by_g(r1 - 1) - p.window + 1 : 0, all_hi = p.parents ? base : base + p.by_g(r0) + 1;

    // The row times scale * log2(e) as two fp16 parts: step s holds dims 16s + 8h .. + 7.
    half8 qh[STEPS], ql[STEPS];
    float unscale, up;
    const float *qrow = p.q + ((static_cast<long long>(b) * p.T + t) * p.Hq + kvh * p.G + (r - t * p.G)) * D;
    {
        float top = 0.0f;
        float4 qa[STEPS], qc[STEPS];
#pragma unroll
        for (int s = 0; s < STEPS; ++s) {
            qa[s] = *reinterpret_cast<const float4 *>(qrow + 16 * s + 8 * h);
            qc[s] = *reinterpret_cast<const float4 *>(qrow + 16 * s + 8 * h + 4);
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
        up = ldexpf(1.0f, 15 - e);
        unscale = ldexpf(p.unscale, e - 15);
#pragma unroll
        for (int s = 0; s < STEPS; ++s) {
            const float4 a = qa[s], c = qc[s];
            const float y[8] = {a.x, a.y, a.z, a.w, c.x, c.y, c.z, c.w};
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float v = y[i] * p.scale * up;
                qh[s][i] = static_cast<_Float16>(v);
                ql[s][i] = static_cast<_Float16>(v - static_cast<float>(qh[s][i]));
            }
        }
    }

    f32x16 o[DT];
    float m, l;
    // A lane's share of V's transposed reads: of 16 lanes, row i / 4 and dims 4 (i % 4) .. + 3 of 16.
    const int vrow = 4 * h + (lane >> 2 & 3), vchunk = 2 * (lane >> 4 & 1) + (lane >> 1 & 1), vbyte = 8 * (lane & 1);
    for (bool careful = false;; careful = true) {
        m = -INFINITY;
        l = 0.0f;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) o[dt] = f32x16{};
        for (int kt = t0, cur = 0; kt < t1; ++kt, cur = cur == 2 ? 0 : cur + 1) {
            const int k0 = kt * kTile;
            if (kt + 1 < t1) wait_copies<2 * R::kCopies>();
            else wait_copies<0>();
            lds_barrier();                                 // the tile is there; the buffer after the next is free
            char *kl = lds + cur * R::kBuffer, *vl = kl + R::kPlane;
            const bool seen_here = !(idle || k0 >= w_hi || k0 + kTile <= w_lo);
            half8 ka[STEPS];
#pragma unroll
            for (int st = 0; st < STEPS; ++st) ka[st] = *reinterpret_cast<const half8 *>(kl + nl * R::kRow + 16 * (2 * st + h ^ R::k_swap(nl)));
            __builtin_amdgcn_sched_barrier(0);
            uint32_t ok_after = 0;
            if (kt + 2 < t1) ok_after = copy(kt + 2, cur == 0 ? 2 : cur - 1);
            const bool edge = careful || k0 < all_lo || k0 + kTile > all_hi || ok != 3;
            bool odd = false;
            if (edge) {
                bool found = false;
#pragma unroll
                for (int j = 0; j < R::kPlane / 4096; ++j) {
                    const int at = 16 * (tid + kThreads * j), row = at / R::kRow;
                    uint4 x = *reinterpret_cast<const uint4 *>(vl + at);
                    const bool gone = k0 + row >= seq.n || !(ok >> (row >> 4) & 1);
                    const bool bad = not_finite(x.x) | not_finite(x.y) | not_finite(x.z) | not_finite(x.w);
                    if (gone || bad) {
                        found |= !gone;
                        x = gone ? make_uint4(0, 0, 0, 0) : make_uint4(clean(x.x), clean(x.y), clean(x.z), clean(x.w));
                        *reinterpret_cast<uint4 *>(vl + at) = x;
                    }
                }
                if (found) odd_tile = kt + 1;
                lds_barrier();
                odd = odd_tile == kt + 1;
            }
            half8 ph[2], pl[2];
            uint32_t see = 0xffffffffu;
            if (seen_here) {
                // S^T: accumulator j is key k0 + 8 (j / 4) + 4h + j % 4 of this lane's row.
                f32x16 s = {};
#pragma unroll
                for (int st = 0; st < STEPS; ++st) {
                    s = __builtin_amdgcn_mfma_f32_32x32x16_f16(ka[st], ql[st], s, 0, 0, 0);
                    s = __builtin_amdgcn_mfma_f32_32x32x16_f16(ka[st], qh[st], s, 0, 0, 0);
                }
                // V's fragments arrive while the weights are computed (D = 256 has no registers for them).
                auto read_values = [&](int dt, int j) __attribute__((always_inline)) {
                    fp16x4 a[2];
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const int row = 16 * j + 8 * i + vrow;
                        a[i] = __builtin_amdgcn_ds_read_tr16_b64_v4f16((__attribute__((address_space(3))) fp16x4 *)(
                            vl + row * R::kRow + 16 * (4 * dt + vchunk ^ R::v_swap(row)) + vbyte));
                    }
                    return __builtin_bit_cast(half8, __builtin_shufflevector(a[0], a[1], 0, 1, 2, 3, 4, 5, 6, 7));
                };
                half8 va[DT][2];
                if constexpr (D < 256) {
                    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                        for (int j = 0; j < 2; ++j) va[dt][j] = read_values(dt, j);
                    __builtin_amdgcn_sched_barrier(0);
                }
                if (k0 < full_lo || k0 + kTile > full_hi || ok != 3) {
                    see = seen(p, seq, range, t, k0, tree);
                    if (!(ok & 1)) see &= 0xffff0000u;
                    if (!(ok & 2)) see &= 0x0000ffffu;
                }
                if (careful) {                             // scores that are NaN, in fp32
                    int dims = D;
                    asm("" : "+s"(dims));                  // a loop that stays one
#pragma unroll
                    for (int j = 0; j < 16; ++j) {
                        const int key = 8 * (j >> 2) + 4 * h + (j & 3);
                        if (s[j] != s[j] && (see >> key & 1)) {
                            const _Float16 *kr = reinterpret_cast<const _Float16 *>(row_of(kt, key, false));
                            float sum = 0.0f;
                            for (int d = 0; d < dims; ++d) sum = fmaf(qrow[d] * p.scale * up, static_cast<float>(kr[d]), sum);
                            s[j] = sum;
                        }
                    }
                }
                if (p.soft_cap > 0.0f) {
                    const float cap = p.soft_cap * kLog2e, in = fminf(unscale / cap, 3e38f);       // finite: 0 stays 0
#pragma unroll
                    for (int j = 0; j < 16; ++j) s[j] = cap * tanhf(s[j] * in);
                }
                const float us = p.soft_cap > 0.0f ? 1.0f : unscale;
                if (see != 0xffffffffu) {
                    const uint32_t mine = see >> (4 * h);
#pragma unroll
                    for (int j = 0; j < 16; ++j)
                        if (!(mine >> (8 * (j >> 2) + (j & 3)) & 1)) s[j] = -INFINITY;
                }
                float mx = s[0];
#pragma unroll
                for (int j = 1; j < 16; ++j) mx = fmaxf(mx, s[j]);
                mx *= us;
                // The reference m of a row is raised only when a score exceeds it by more than 2.
                if (__any(mx > m + 2.0f)) {
                    mx = fmaxf(mx, __shfl_xor(mx, 32));
                    const float to = mx > m + 2.0f ? mx : m;
                    const float alpha = to == m ? 1.0f : __builtin_amdgcn_exp2f(m - to);           // 0 while m is -inf
                    l *= alpha;
#pragma unroll
                    for (int dt = 0; dt < DT; ++dt) o[dt] *= alpha;
                    m = to;
                }
                const float ref = m == -INFINITY ? 0.0f : m;
                float sum[4] = {};
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    float e[2];
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        e[c] = __builtin_amdgcn_exp2f(fmaf(s[2 * j + c], us, -ref)) * kWeightScale<true>;
                        sum[(2 * j + c) & 3] += e[c];
                    }
                    const half2v first = pair(e[0], e[1]);
                    const half2v rest = pair(fmaf(static_cast<float>(first[0]), -1.0f, e[0]), fmaf(static_cast<float>(first[1]), -1.0f, e[1]));
                    ph[j >> 2][2 * (j & 3)] = first[0];
                    ph[j >> 2][2 * (j & 3) + 1] = first[1];
                    pl[j >> 2][2 * (j & 3)] = rest[0];
                    pl[j >> 2][2 * (j & 3) + 1] = rest[1];
                }
                l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
                // Lane half h supplies contraction entries 0..3 -> key 16j + 4h + e and 4..7 -> key 16j + 8 + 4h + e - 4.
#pragma unroll
                for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        if constexpr (D == 256) va[dt][j] = read_values(dt, j);
                        o[dt] = __builtin_amdgcn_mfma_f32_32x32x16_f16(va[dt][j], pl[j], o[dt], 0, 0, 0);
                        o[dt] = __builtin_amdgcn_mfma_f32_32x32x16_f16(va[dt][j], ph[j], o[dt], 0, 0, 0);
                    }
            }
            if (odd) {
                // The values that were taken out, times the rows' weights, which go through the tile's LDS.
                float *wt = reinterpret_cast<float *>(kl) + wave * 512;
                for (int u = 0; u < 2; ++u) {
                    lds_barrier();                         // every wave has left the tile, or the other half's weights
                    if (!seen_here) continue;
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        wt[(8 * (j >> 2) + 4 * h + (j & 3)) * 32 + nl] =
                            u ? static_cast<float>(ph[1][j]) + static_cast<float>(pl[1][j]) : static_cast<float>(ph[0][j]) + static_cast<float>(pl[0][j]);
                    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");     // the wave's own writes
                    int keys = 16;
                    asm("" : "+s"(keys));                  // a loop that stays one
                    for (int i = 0; i < keys; ++i) {
                        if (k0 + 16 * u + i >= seq.n || !(ok >> u & 1)) continue;
                        const char *vr = row_of(kt, 16 * u + i, true) + 8 * h;
#pragma unroll
                        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                            for (int q = 0; q < 4; ++q) {
                                const uint2 v = *reinterpret_cast<const uint2 *>(vr + 64 * dt + 16 * q);
                                if (!__any((not_finite(v.x) | not_finite(v.y)) != 0)) continue;
#pragma unroll
                                for (int e = 0; e < 4; ++e) {
                                    const float val = f16_bits_to_f32((e < 2 ? v.x : v.y) >> (16 * (e & 1)) & 0xffffu);
                                    o[dt][4 * q + e] += val - val != 0.0f && (see >> (16 * u + i) & 1) ? wt[i * 32 + nl] * val : 0.0f;
                                }
                            }
                    }
                }
                lds_barrier();
            }
            ok = ok_next;
            ok_next = ok_after;
        }
        if (careful) break;
        float probe = 0.0f;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
            for (int j = 0; j < 16; ++j) probe = fmaf(o[dt][j], 0.0f, probe);
        if (!__syncthreads_or(probe != probe)) break;      // every wave is done with the tiles
        start();
    }

    l += __shfl_xor(l, 32);
    if (m == -INFINITY && l != l) m = 0.0f;                // a NaN score alone leaves no reference
    const bool whole = chunk.count == 1;
    const float f = (whole ? (l == 0.0f ? 0.0f : 1.0f / l) : 1.0f);
    const long long part = (static_cast<long long>(chunk.slot + w - chunk.first) * p.v.H * p.row_groups + item) * kRowsBlock + 32 * wave;
    if (!whole && h == 0 && w0 + nl < r1) *reinterpret_cast<float2 *>(p.part_ml + (part + nl) * 2) = make_float2(m, l);
    // O through LDS, so that whole lines are stored: rounds of kSpan dims. Accumulator j of tile dt is dim 32 dt +
    // 8 (j / 4) + 4h + j % 4.
    __syncthreads();
    float *st = reinterpret_cast<float *>(lds) + wave * 32 * R::kStride;
    constexpr int LPR = R::kSpan / 4;
#pragma unroll
    for (int rd = 0; rd < D / R::kSpan; ++rd) {
#pragma unroll
        for (int c = 0; c < R::kSpan / 32; ++c)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const f32x16 &x = o[rd * (R::kSpan / 32) + c];
                *reinterpret_cast<float4 *>(st + nl * R::kStride + 32 * c + 8 * q + 4 * h) =
                    make_float4(x[4 * q] * f, x[4 * q + 1] * f, x[4 * q + 2] * f, x[4 * q + 3] * f);
            }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");                 // the wave's own writes
#pragma unroll
        for (int i = 0; i < 32 * LPR / 64; ++i) {
            const int lr = (64 * i + lane) / LPR, d = 4 * ((64 * i + lane) % LPR), rr = w0 + lr;
            if (rr < r1) {
                const float4 val = *reinterpret_cast<const float4 *>(st + lr * R::kStride + d);
                const int tt = p.by_g(rr);
                float *dst = whole ? p.out + ((static_cast<long long>(b) * p.T + tt) * p.Hq + kvh * p.G + (rr - tt * p.G)) * D
                                   : p.part_o + (part + lr) * D;
                *reinterpret_cast<float4 *>(dst + rd * R::kSpan + d) = val;
            }
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");                 // read before the next round's writes
    }
}

template <int D>
void launch(const Params &p, hipStream_t s) {
    using R = Rows<D>;
    const dim3 grid(p.v.H * p.row_groups * (p.quota ? p.quota + (p.v.B > 1 ? p.v.B : 0) : p.v.B));
    if (R::kBytes + sizeof(Tree) + 16 > 65536)
        (void)hipFuncSetAttribute(reinterpret_cast<const void *>(kv_rows_kernel<D>), hipFuncAttributeMaxDynamicSharedMemorySize, R::kBytes);
    hipLaunchKernelGGL((kv_rows_kernel<D>), grid, dim3(kThreads), R::kBytes, s, p);
    if (p.quota)                                           // few row groups, so few rows of a sequence
        hipLaunchKernelGGL((merge_rows_kernel<Params, D, kRowsBlock>), dim3((p.T * p.Hq + 3) / 4, p.v.B), dim3(256), 0, s, p);
}

}  // namespace

void kvt::launch_rows(const Params &p, hipStream_t s) {
    if (p.v.D == 64) launch<64>(p, s);
    else if (p.v.D == 128) launch<128>(p, s);
    else launch<256>(p, s);
}

}  // namespace aljabr
