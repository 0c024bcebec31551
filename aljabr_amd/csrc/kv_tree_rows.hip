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
// the two fp16 parts of queries and weights. The next tile's scores are laid
// between this one's weights, so that matrix cores and vector ALU work at once.
//
// Bound by the products: 256 rows of 8 KV heads of 128 over 8 x 8192 keys 157
// us, 104 rows over 131072 keys 163 us, chunks of 512 rows of 32 heads over
// 2 x 4096 keys 145 us, with the merges: of the rows that are there 0.88, 0.68
// (104 of the 128 rows computed) and 0.95 PFLOP/s with both parts, where the
// library's product of 8192^3 reaches 1.2. Matrix cores 44 % of the cycles, vector
// ALU 42 %, both at once 20 %; under this load the clock falls to 2.0 GHz. Tiles
// of both operands shared in LDS by 128 rows took 157 us of the chunks where the
// waves of 32 rows loaded their own (kv_tree.hip) 422; addresses of tiles held by
// the lanes made that 149, the pipeline 143.
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
    static constexpr int kValues = 3 * kPlane;             // three tiles of K, then three of V
    static constexpr int CPR = kRow / 16;                  // chunks of a row
    static constexpr int RPL = 64 / CPR;                   // rows of a wave-wide copy
    static constexpr int kCopies = 8 / RPL;                // of a wave's 8 rows of K (and of V)
    static constexpr int kSpan = D == 64 ? 32 : 64, kStride = kSpan + 4;   // dims of a round of the output, and its rows in LDS
    static constexpr int kOut = kWaves * 32 * kStride * 4;
    static constexpr int kBytes = 6 * kPlane > kOut ? 6 * kPlane : kOut;
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

// The larger of x in this lane and in the one 32 lanes away.
__device__ __forceinline__ float half_max(float x) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

// 16 bytes a lane from base + offset to LDS at dst + 16 * lane (dma16 of device.hpp with a base that the wave shares).
__device__ __forceinline__ void dma16(const char *base, uint32_t offset, uint32_t dst) {
    uint32_t save;
    asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %2, %3\n\ts_mov_b32 m0, %0"
                 : "=&s"(save)
                 : "s"(dst), "v"(offset), "s"(base)
                 : "memory");
}

// A dword of two fp16 numbers: bits of those whose exponent is all ones.
__device__ __forceinline__ uint32_t not_finite(uint32_t w) { return ((w & 0x7fff7fffu) + 0x04000400u) & 0x80008000u; }
__device__ __forceinline__ uint32_t clean(uint32_t w) {
    const uint32_t bad = not_finite(w);
    return w & ~((bad >> 15) * 0xffffu);
}

template <int D>
__global__ __launch_bounds__(kThreads, 2) void kv_rows_kernel(Params p) {
    using R = Rows<D>;
    constexpr int STEPS = D / 16, DT = D / 32;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    __shared__ Tree tree;
    __shared__ int4 row_info[kThreads];                    // of a lane's row: t, its range, the power of two it was scaled by
    __shared__ int odd_tile;                               // the last tile that held values which are not finite, plus 1
    __shared__ uint32_t weighs[kThreads];                  // in such a tile, bits of a lane's 16 keys whose weight is not 0 in fp32
    const int tid = threadIdx.x, lane = tid & 63, h = lane >> 5, nl = lane & 31;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    // For the paths that are rarely taken: the thread's number, of which the compiler keeps nothing in registers.
    auto fresh_tid = []() __attribute__((always_inline)) {
        int x = threadIdx.x;
        asm volatile("" : "+v"(x));
        return x;
    };
    const Work work_item = work_at(p, blockIdx.x);
    const int kvh = work_item.kvh, w = work_item.w, group = group_of(p, work_item.group), item = item_of(p, kvh, group);
    if (!p.quota && w >= p.v.B) return;                    // numbers past the last unit
    const int r0 = group * kRowsBlock;
    const Chunk chunk = find_chunk(p, w, r0, kRowsBlock, kRowsLeast);
    if (chunk.b < 0) return;
    const int b = chunk.b, t0 = chunk.t0, t1 = chunk.t1;
    if (p.quota && w == chunk.first && tid == 0)
        p.chunks[static_cast<long long>(item) * p.v.B + b] = make_int2(chunk.slot, chunk.count);
    const Seq seq = chunk.seq;
    const int base = seq.base, r1 = min(r0 + kRowsBlock, seq.cnt * p.G), w0 = r0 + 32 * wave;
    const bool idle = w0 >= r1;                            // a wave without rows only copies

    const uint32_t ring = lds_address(lds);
    Places<2> places{t0, 1};
    // This wave copies rows 8 wave .. + 7 of a tile, of its half wave / 2. A lane's part of the half's rows, copy j:
    const int u = wave >> 1, first = 8 * (wave & 1);
    auto share = [&](int lane, int j, int last, bool of_v) __attribute__((always_inline)) {
        const int row = first + j * R::RPL + lane / R::CPR, slot = lane % R::CPR;
        return min(row, last) * R::kRow + 16 * (slot ^ (of_v ? R::v_swap(row) : R::k_swap(row)));
    };
    int k_from[R::kCopies], v_from[R::kCopies];
#pragma unroll
    for (int j = 0; j < R::kCopies; ++j) {
        k_from[j] = share(lane, j, 15, false);
        v_from[j] = share(lane, j, 15, true);
    }
    // Tile i of the chunk's K, or V, into its third of the ring.
    auto copy = [&](int i, int third, bool of_v) __attribute__((always_inline)) {
        const int key = (t0 + i) * kTile;
        if (i == places.held + 32) places.load(p, fresh_tid() & 63, R::kRow, b, kvh, seq.n, i - 16);
        const char *at = (of_v ? p.v.v : p.v.k) + places.offset(i, u);
        const int last = last_row(p, key + 16 * u < seq.n ? key + 16 * u : key);
        const uint32_t dst = ring + (of_v ? R::kValues : 0) + third * R::kPlane + (16 * u + first) * R::kRow;
        if (last < 15) {                                   // the end of a contiguous plane
            const int lane = fresh_tid() & 63;
#pragma unroll
            for (int j = 0; j < R::kCopies; ++j) dma16(at, share(lane, j, last, of_v), __builtin_amdgcn_readfirstlane(dst + 1024 * j));
        } else {
#pragma unroll
            for (int j = 0; j < R::kCopies; ++j) dma16(at, of_v ? v_from[j] : k_from[j], __builtin_amdgcn_readfirstlane(dst + 1024 * j));
        }
    };
    const int tiles = t1 - t0;
    // The first tiles: two of K, then a third of K with the first of V.
    auto start = [&]() __attribute__((always_inline)) {
        places.load(p, fresh_tid() & 63, R::kRow, b, kvh, seq.n, 0);
        if (tiles > 0) copy(0, 0, false);
        if (tiles > 1) copy(1, 1, false);
        if (tiles > 2) copy(2, 2, false);
        if (tiles > 0) copy(0, 0, true);
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
    const bool filled = p.parents && (p.window > 0 || t1 * kTile > base);
    start();
    if (tid == 0) odd_tile = 0;
    if (filled) {
        const int row = tree_row(seq.cnt);
        fill_tree(tree, row < seq.cnt ? p.parents[static_cast<long long>(b) * p.T + row] : -1, seq.cnt, p.window);
    }
    __syncthreads();

    // This lane's row, what it sees; the keys that all rows of the wave, and of the workgroup, see.
    const int r = min(w0 + nl, r1 - 1);                    // lanes past the rows repeat the last and are not stored
    const int t = p.by_g(r);
    const Range seen_range = range_of(p, seq, t, tree, filled);
    const int t_first = p.by_g(min(w0, r1 - 1)), t_last = p.by_g(min(w0 + 31, r1 - 1));
    const int full_lo = window_start(p, base + t_last + 1), full_hi = min(p.parents ? base : base + t_first + 1, seq.n);
    const int all_lo = window_start(p, base + p.by_g(r1 - 1) + 1), all_hi = min(p.parents ? base : base + p.by_g(r0) + 1, seq.n);

    // The row times scale * log2(e) as two fp16 parts: step s holds dims 16s + 8h .. + 7.
    half8 qh[STEPS], ql[STEPS];
    float unscale;
    {
        const float *qrow = p.q + ((static_cast<long long>(b) * p.T + t) * p.Hq + kvh * p.G + (r - t * p.G)) * D;
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
        const int e = query_exponent(p, top);
        const float up = ldexpf(1.0f, 15 - e);
        row_info[tid] = make_int4(t, seen_range.lo, seen_range.hi, __float_as_int(up));        // read by this thread alone
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
    // A lane's part of K's fragment 0, its row's chunk h, and of V's transposed reads: of 16 lanes, row i / 4 and dims
    // 4 (i % 4) .. + 3 of 16. Further chunks of the row are an exclusive or away.
    const int vrow = 4 * h + (lane >> 2 & 3);
    const int k_part = nl * R::kRow + 16 * (h ^ R::k_swap(nl));
    const int v_part = vrow * R::kRow + 16 * (2 * (lane >> 4 & 1) + (lane >> 1 & 1) ^ R::v_swap(vrow)) + 8 * (lane & 1);
    for (bool careful = false;; careful = true) {
        m = -INFINITY;
        l = 0.0f;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) o[dt] = f32x16{};
        half8 ka[STEPS];
        f32x16 s = {};
        int k_at = 0;
        auto read_key = [&](int st) __attribute__((always_inline)) { ka[st] = *reinterpret_cast<const half8 *>(lds + (k_at ^ 32 * st)); };
        auto keys_at = [&](int third) __attribute__((always_inline)) {
            k_at = third * R::kPlane + k_part;
            asm("" : "+v"(k_at));                          // one register, not one for each fragment
        };
        // S^T: accumulator j is key k0 + 8 (j / 4) + 4h + j % 4 of this lane's row.
        auto scores = [&]() __attribute__((always_inline)) {
            f32x16 x = {};
#pragma unroll
            for (int st = 0; st < STEPS; ++st) {
                x = __builtin_amdgcn_mfma_f32_32x32x16_f16(ka[st], ql[st], x, 0, 0, 0);
                x = __builtin_amdgcn_mfma_f32_32x32x16_f16(ka[st], qh[st], x, 0, 0, 0);
            }
            return x;
        };
        if (tiles > 0) {
            if (tiles > 2) wait_copies<2 * R::kCopies>();
            else wait_copies<0>();
            lds_barrier();                                 // the first two tiles of K are there
            if (!idle) {
                keys_at(0);
#pragma unroll
                for (int st = 0; st < STEPS; ++st) read_key(st);
                s = scores();
                keys_at(1);
#pragma unroll
                for (int st = 0; st < STEPS; ++st) read_key(st);
            }
            lds_barrier();                                 // every wave has read the first
            if (tiles > 3) copy(3, 0, false);
            if (tiles > 1) copy(1, 1, true);
        }
        // Tile i: its scores are in s, the next one's K in registers. Behind it lie V of i and K of i + 2, copied two trips
        // ago, and in flight V of i + 1 and K of i + 3; V of i + 2 and K of i + 4 go where those of i - 1 and i + 1 lay.
        for (int i = 0, cur = 0; i < tiles; ++i, cur = cur == 2 ? 0 : cur + 1) {
            const int k0 = (t0 + i) * kTile;
            if (i + 3 < tiles) wait_copies<2 * R::kCopies>();
            else if (i + 1 < tiles) wait_copies<R::kCopies>();
            else wait_copies<0>();
            lds_barrier();                                 // ... and every wave has left V of i - 1 and K of i + 1
            const uint32_t ok = places.ok(i);
            const int before = cur == 0 ? 2 : cur - 1, after = cur == 2 ? 0 : cur + 1;
            if (i + 4 < tiles) copy(i + 4, after, false);
            if (i + 2 < tiles) copy(i + 2, before, true);
            char *vl = lds + R::kValues + cur * R::kPlane;
            const bool edge = careful || k0 < all_lo || k0 + kTile > all_hi || ok != 3;
            bool odd = false;
            if (edge) {
                bool found = false;
                const int thread = fresh_tid();
#pragma unroll
                for (int j = 0; j < R::kPlane / 4096; ++j) {
                    const int at = 16 * (thread + kThreads * j), row = at / R::kRow;
                    uint4 x = *reinterpret_cast<const uint4 *>(vl + at);
                    const bool gone = k0 + row >= seq.n || !(ok >> (row >> 4) & 1);
                    const bool bad = not_finite(x.x) | not_finite(x.y) | not_finite(x.z) | not_finite(x.w);
                    if (gone || bad) {
                        found |= !gone;
                        x = gone ? make_uint4(0, 0, 0, 0) : make_uint4(clean(x.x), clean(x.y), clean(x.z), clean(x.w));
                        *reinterpret_cast<uint4 *>(vl + at) = x;
                    }
                }
                if (found) odd_tile = i + 1;
                lds_barrier();
                odd = odd_tile == i + 1;
            }
            half8 ph[2], pl[2];
            uint32_t see = 0xffffffffu;
            if (!idle) {
                int v_at = R::kValues + cur * R::kPlane + v_part;
                asm("" : "+v"(v_at));
                auto read_values = [&](int dt, half8 (&v)[2]) __attribute__((always_inline)) {
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        fp16x4 a[2];
#pragma unroll
                        for (int c = 0; c < 2; ++c)
                            a[c] = __builtin_amdgcn_ds_read_tr16_b64_v4f16((__attribute__((address_space(3))) fp16x4 *)(
                                lds + (v_at ^ 64 * dt) + (16 * j + 8 * c) * R::kRow));
                        v[j] = __builtin_bit_cast(half8, __builtin_shufflevector(a[0], a[1], 0, 1, 2, 3, 4, 5, 6, 7));
                    }
                };
                if (k0 < full_lo || k0 + kTile > full_hi || ok != 3) {
                    const int4 info = row_info[fresh_tid()];
                    see = seen(p, seq, Range{info.y, info.z}, info.x, k0, tree);
                    if (!(ok & 1)) see &= 0xffff0000u;
                    if (!(ok & 2)) see &= 0x0000ffffu;
                }
                if (careful) {                             // scores that are NaN, in fp32
                    int dims = D;
                    asm("" : "+s"(dims));                  // a loop that stays one
                    const int thread = fresh_tid(), h = thread >> 5 & 1;
                    const int4 info = row_info[thread];
                    const int r = min(w0 + (thread & 31), r1 - 1), t = info.x;
                    const float *qrow = p.q + ((static_cast<long long>(b) * p.T + t) * p.Hq + kvh * p.G + (r - t * p.G)) * D;
                    const float up = __int_as_float(info.w);
#pragma unroll
                    for (int j = 0; j < 16; ++j) {
                        const int key = 8 * (j >> 2) + 4 * h + (j & 3);
                        if (s[j] != s[j] && (see >> key & 1)) {
                            const _Float16 *kr = reinterpret_cast<const _Float16 *>(row_of(t0 + i, key, false));
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
                    const uint32_t mine = see >> (4 * (fresh_tid() >> 5 & 1));
#pragma unroll
                    for (int j = 0; j < 16; ++j)
                        if (!(mine >> (8 * (j >> 2) + (j & 3)) & 1)) s[j] = -INFINITY;
                }
                float mx = s[0];
#pragma unroll
                for (int j = 1; j < 16; ++j) mx = fmaxf(mx, s[j]);
                mx *= us;
                // The reference m of a row is raised only when a score exceeds it by more than kRaise.
                if (__any(mx > m + kRaise)) {
                    mx = half_max(mx);
                    const float to = mx > m + kRaise ? mx : m;
                    const float alpha = to == m ? 1.0f : __builtin_amdgcn_exp2f(m - to);           // 0 while m is -inf
                    l *= alpha;
#pragma unroll
                    for (int dt = 0; dt < DT; ++dt) o[dt] *= alpha;
                    m = to;
                }
                const float ref = m == -INFINITY ? 0.0f : m;
                if (odd) {
                    uint32_t bits = 0;
#pragma unroll
                    for (int j = 0; j < 16; ++j) bits |= __builtin_amdgcn_exp2f(fmaf(s[j], us, -ref)) > 0.0f ? 1u << j : 0;
                    weighs[fresh_tid()] = bits;            // read by this thread alone
                }
                half8 va[2][2];
                read_values(0, va[0]);
                // The next tile's scores on the matrix cores, between them this one's weights.
                __builtin_amdgcn_sched_barrier(0);
                const f32x16 after_s = scores();
                float sum[4] = {};
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    float e[2];
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        e[c] = __builtin_amdgcn_exp2f(fmaf(s[2 * j + c], us, -ref));
                        sum[(2 * j + c) & 3] += e[c];
                    }
                    constexpr float up = kWeightScale<true>;
                    const half2v first = pair(e[0] * up, e[1] * up);
                    const half2v rest = pair(fmaf(e[0], up, -static_cast<float>(first[0])), fmaf(e[1], up, -static_cast<float>(first[1])));
                    ph[j >> 2][2 * (j & 3)] = first[0];
                    ph[j >> 2][2 * (j & 3) + 1] = first[1];
                    pl[j >> 2][2 * (j & 3)] = rest[0];
                    pl[j >> 2][2 * (j & 3) + 1] = rest[1];
                }
                l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
#pragma unroll
                for (int j = 0; j < 2 * STEPS; ++j) {
                    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);                 // a product,
                    __builtin_amdgcn_sched_group_barrier(0x402, 104 / (2 * STEPS), 0); // vector instructions for its 32 cycles
                }
                __builtin_amdgcn_sched_barrier(0);
                s = after_s;
                // Lane half h supplies contraction entries 0..3 -> key 16j + 4h + e and 4..7 -> key 16j + 8 + 4h + e - 4. Behind
                // the products go the reads of the next dims and of K of i + 2.
                keys_at(before);
#pragma unroll
                for (int dt = 0; dt < DT; ++dt) {
                    if (dt + 1 < DT) read_values(dt + 1, va[(dt + 1) & 1]);
                    read_key(2 * dt);
                    read_key(2 * dt + 1);
                    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        o[dt] = __builtin_amdgcn_mfma_f32_32x32x16_f16(va[dt & 1][j], pl[j], o[dt], 0, 0, 0);
                        o[dt] = __builtin_amdgcn_mfma_f32_32x32x16_f16(va[dt & 1][j], ph[j], o[dt], 0, 0, 0);
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
            if (odd) {
                // The values that were taken out, times the rows' weights, which go through the tile's LDS, 8 keys at once. A
                // weight that its two parts have lost is still not 0: an infinity times it is one.
                float *wt = reinterpret_cast<float *>(vl) + wave * 256;
                const int thread = fresh_tid(), h = thread >> 5 & 1, nl = thread & 31;
                for (int q = 0; q < 4; ++q) {
                    lds_barrier();                         // every wave has left the tile, or the last weights
                    if (idle) continue;
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const float w0 = static_cast<float>(ph[0][j]) + static_cast<float>(pl[0][j]);
                        const float w1 = static_cast<float>(ph[0][4 + j]) + static_cast<float>(pl[0][4 + j]);
                        const float w2 = static_cast<float>(ph[1][j]) + static_cast<float>(pl[1][j]);
                        const float w3 = static_cast<float>(ph[1][4 + j]) + static_cast<float>(pl[1][4 + j]);
                        const float w = q & 2 ? (q & 1 ? w3 : w2) : (q & 1 ? w1 : w0);
                        wt[(4 * h + j) * 32 + nl] = w == 0.0f && (weighs[thread] >> (4 * q + j) & 1) ? 0x1p-126f : w;
                    }
                    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");     // the wave's own writes
                    int keys = 8;
                    asm("" : "+s"(keys));                  // a loop that stays one
                    for (int c = 0; c < keys; ++c) {
                        const int key = 8 * q + c;
                        if (k0 + key >= seq.n || !(ok >> (q >> 1) & 1)) continue;
                        const char *vr = row_of(t0 + i, key, true) + 8 * h;
#pragma unroll
                        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                            for (int x = 0; x < 4; ++x) {
                                const uint2 v = *reinterpret_cast<const uint2 *>(vr + 64 * dt + 16 * x);
                                if (!__any((not_finite(v.x) | not_finite(v.y)) != 0)) continue;
#pragma unroll
                                for (int e = 0; e < 4; ++e) {
                                    const float val = f16_bits_to_f32((e < 2 ? v.x : v.y) >> (16 * (e & 1)) & 0xffffu);
                                    o[dt][4 * x + e] += val - val != 0.0f && (see >> key & 1) ? wt[c * 32 + nl] * val : 0.0f;
                                }
                            }
                    }
                }
                lds_barrier();
            }
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

    l = (l + __shfl_xor(l, 32)) * kWeightScale<true>;
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
    if (R::kBytes + sizeof(Tree) + kThreads * (sizeof(int4) + sizeof(uint32_t)) + 16 > 65536)
        (void)hipFuncSetAttribute(reinterpret_cast<const void *>(kv_rows_kernel<D>), hipFuncAttributeMaxDynamicSharedMemorySize, R::kBytes);
    hipLaunchKernelGGL((kv_rows_kernel<D>), dim3(workgroups(p)), dim3(kThreads), R::kBytes, s, p);
    if (p.quota) launch_merge<D, kRowsBlock>(p, kRowsLeast * kTile, s);
}

}  // namespace

void kvt::launch_rows(const Params &p, hipStream_t s) {
    p.v.D == 64 ? launch<64>(p, s) : launch<128>(p, s);
}

}  // namespace aljabr
