// A tile of a product A B^T, A^T B or A B on the matrix instructions: operands through LDS by direct loads, in slabs of the summed
// dimension and a ring of them.  An operand either lies with the summed dimension along its rows or across them; the second kind goes into
// LDS as it lies and is transposed by the LDS reads.  16-byte pieces are XOR-ed by their row against bank conflicts, on the side of the
// global address.
#pragma once
#include "common.h"

#include <math.h>

namespace vtdge {

__device__ __forceinline__ int wave_uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }

// 16 bytes on any boundary of their elements' type
typedef u32x4 u32x4_on2 __attribute__((aligned(2)));
typedef u32x4 u32x4_on4 __attribute__((aligned(4)));
template <typename T> struct Loose { typedef u32x4_on4 vector; };
template <> struct Loose<bf16_t> { typedef u32x4_on2 vector; };

// ------------------------------------------------------------------------------------------------ the product of a tile
// A bf16 matrix, or the three parts of an fp32 one `plane` elements apart.
struct Operand {
    const bf16_t *p;
    int64_t pitch, plane;
};

// A shape of the product: WM x WN waves, each with IM x JN blocks of 32 x 32; slabs of SLAB of the summed dimension in a ring of
// SLOTS; PARTS 3 for fp32 operands.
template <int IM_, int JN_, int WM_, int WN_, int SLAB_, int SLOTS_, int PARTS_> struct Shape {
    static constexpr int IM = IM_, JN = JN_, WM = WM_, WN = WN_, SLAB = SLAB_, SLOTS = SLOTS_, PARTS = PARTS_;
    static constexpr int ROWS = 32 * IM * WM, COLS = 32 * JN * WN, WAVES = WM * WN, THREADS = 64 * WAVES;
    static constexpr int STAGE = PARTS * (ROWS + COLS) * SLAB * 2, RING = SLOTS * STAGE;
    static constexpr int LDS = RING + COLS * 4;                          // and the bias of the tile's classes
    using Half = Shape<IM / 2, JN, WM, WN, SLAB, SLOTS, PARTS>;
    static constexpr bool HALVES = WAVES == 8 && IM == 2;               // the last tiles of a launch may be cut in two, see halved()
    static constexpr bool FLAT = IM == 1 && JN == 2;                    // few rows
    static constexpr bool WHOLE_LINES = IM == 1 && JN == 1;             // gradients leave by way of LDS
    static constexpr int PER_SIMD = WAVES / 4 * (2 * LDS <= 160 * 1024 ? 2 : 1);
    static_assert(LDS <= 160 * 1024 && 6 * ROWS * 4 <= RING, "LDS");
};

// Direct loads of one operand of a tile.  T = rows of the tile on its side.
// ALONG: the summed dimension lies along the rows of memory: tile rows are rows of memory, `limit` of them from the first on.
// Across: the summed dimension counts the rows of memory, `limit` of them, and tile rows are elements of a row, which has a multiple
// of 8 of them, `span`.  No stage begins behind `limit`: a sum of n rows of memory has ceil(n / SLAB) stages.
// LDS rows are 2 SLAB bytes (ALONG) or 2 T bytes (across) without gaps; their 16-byte pieces are XOR-ed by the row, so that the lanes
// that read together (half a wave of transposed reads, whose four rows take sixteen pieces) meet each of the 64 banks once.
template <bool ALONG, int T, int SLAB, int WAVES, bool MAY_STREAM = false> struct Loader {
    static constexpr int ROW = ALONG ? 2 * SLAB : 2 * T, STAGE = 2 * SLAB * T;
    static constexpr int LPR = ROW / 16, RPI = 64 / LPR;                  // lanes a row, rows an instruction
    static constexpr int PIECES = STAGE / 1024 / WAVES;                   // instructions of a wave
    static_assert(PIECES * WAVES * 1024 == STAGE && LPR <= 64, "whole instructions");
    const unsigned char *base;
    int64_t plane, pitch;                                                 // bytes
    int limit, lane, row0, last;
    bool stream = false;                                                  // past the caches

    __device__ __forceinline__ Loader(const Operand &o, int64_t first, int64_t lim, int64_t span)
        : base(reinterpret_cast<const unsigned char *>(o.p) + (ALONG ? first * o.pitch * 2 : first * 2)), plane(o.plane * 2), pitch(o.pitch * 2), lane(threadIdx.x & 63)
    {
        const int wid = wave_uniform(threadIdx.x >> 6);
        row0 = wid * RPI + lane / LPR;
        if constexpr (ALONG) limit = (int)(lim - first < T ? lim - first : T);
        else limit = (int)lim;
        last = ALONG ? 0 : (int)(span - first < T ? span - first : T) * 2 - 16;
    }
    static __device__ __forceinline__ int swizzle(int r)
    {
        if constexpr (ALONG) return SLAB == 64 ? (r >> 1) & 7 : SLAB == 32 ? (r >> 2) & 3 : (r >> 3) & 1;
        else return LPR == 8 ? ((r >> 1) & 3) << 1 : (r & 3) << 2;
    }
    // stage `kt` of part `part` to LDS byte `lds`
    __device__ __forceinline__ void load(int part, int kt, uint32_t lds) const
    {
        const void *const from = uniform_ptr(base + part * plane + (ALONG ? (int64_t)kt * (2 * SLAB) : (int64_t)kt * SLAB * pitch));
        const int wid = wave_uniform(threadIdx.x >> 6);
#pragma unroll
        for (int d = 0; d < PIECES; d++) {
            const int r = d * WAVES * RPI + row0;
            const int at = ((lane % LPR) ^ swizzle(r)) * 16;
            const int row = ALONG ? min(r, limit - 1) : min(r, limit - 1 - kt * SLAB);
            const int col = ALONG ? at : min(at, last);
            const uint32_t off = (uint32_t)row * (uint32_t)pitch + col, to = wave_uniform(lds + (d * WAVES + wid) * 1024);
            if (MAY_STREAM && stream) dma16_nt(from, off, to);
            else dma16(from, off, to);
        }
    }
    // the 8 values of step s (16 of the summed dimension) of tile row `block` * 32 + lane % 32
    static __device__ __forceinline__ u32x4 fragment(const unsigned char *stage, int block, int s)
    {
        const int lane = threadIdx.x & 63, lr = lane & 31, lg = lane >> 5;
        if constexpr (ALONG) {
            return *reinterpret_cast<const u32x4 *>(stage + (block * 32 + lr) * ROW + (((2 * s + lg) ^ swizzle(lr)) * 16));
        } else {
            const int k = 16 * s + 8 * lg + ((lane & 15) >> 2);
            const int at = block * 64 + ((lane >> 4) & 1) * 32 + (lane & 3) * 8;       // byte of the row
            const u32x2 lo = lds_read_tr16(stage + k * ROW + (((at >> 4) ^ swizzle(k)) << 4) + (at & 15));
            const u32x2 hi = lds_read_tr16(stage + (k + 4) * ROW + (((at >> 4) ^ swizzle(k + 4)) << 4) + (at & 15));
            return u32x4{lo.x, lo.y, hi.x, hi.y};
        }
    }
};

// acc[i][j][v] += A[row i*32 + lane%32 of the wave] . B[row j*32 + 8*(v/4) + 4*(lane/32) + v%4], stages t0 .. t1 - 1.  SUMS: also the sums of
// A's rows (of this half of the lanes' values), for what `sums_wanted` says.  ENDS: the sum has `live` terms, and what A holds in a slab behind
// them is taken for zeros.
template <class S, bool SUMS, bool ENDS = false, class LA, class LB>
__device__ __forceinline__ void multiply_tile(const LA &a, const LB &b, int t0, int t1, unsigned char *smem, f32x16 (&acc)[S::IM][S::JN],
                                              bool sums_wanted, float (&sums)[S::IM], int live = 0)
{
    constexpr int IM = S::IM, JN = S::JN, PARTS = S::PARTS, SLOTS = S::SLOTS, A_BYTES = PARTS * LA::STAGE;
    constexpr int LOADS = PARTS * (LA::PIECES + LB::PIECES);
    static_assert(LOADS * (SLOTS - 2) < 64, "the counter of outstanding loads");
    const int wid = wave_uniform(threadIdx.x >> 6), wm = wid / S::WN, wn = wid % S::WN;
    const uint32_t lds0 = (uint32_t)(uintptr_t)smem;
    auto issue = [&](int t, int slot) {
        const uint32_t at = lds0 + slot * S::STAGE;
#pragma unroll
        for (int p = 0; p < PARTS; p++) {
            a.load(p, t, at + p * LA::STAGE);
            b.load(p, t, at + A_BYTES + p * LB::STAGE);
        }
    };
    int in = 0, out = 0;                            // slots
#pragma unroll
    for (int d = 0; d < SLOTS - 1; d++)
        if (t0 + d < t1) {
            issue(t0 + d, in);
            in++;
        }
    for (int t = t0; t < t1; t++) {
        // this wave's loads of the stage have landed when only those of the stages behind it are outstanding
        const int behind = min(t1 - 1 - t, SLOTS - 2);
        static_for<SLOTS - 1>([&](auto X) {
            constexpr int x = decltype(X)::value;
            if (behind == x) wait_vmcnt<x * LOADS>();
        });
        lds_barrier();                              // everybody's have, and the slot before this one is read no more
        const unsigned char *sa = smem + out * S::STAGE, *sb = sa + A_BYTES;
        out = out == SLOTS - 1 ? 0 : out + 1;
        // fragments a step ahead of their products, the direct loads behind the first of them
        constexpr int STEPS = S::SLAB / 16;
        u32x4 fa[2][PARTS][IM], fb[2][PARTS][JN];
        auto fetch = [&](int s) {
#pragma unroll
            for (int p = 0; p < PARTS; p++) {
#pragma unroll
                for (int i = 0; i < IM; i++) fa[s & 1][p][i] = LA::fragment(sa + p * LA::STAGE, wm * IM + i, s);
#pragma unroll
                for (int j = 0; j < JN; j++) fb[s & 1][p][j] = LB::fragment(sb + p * LB::STAGE, wn * JN + j, s);
            }
        };
        fetch(0);
        __builtin_amdgcn_sched_barrier(0);
        if (t + SLOTS - 1 < t1) {
            issue(t + SLOTS - 1, in);
            in = in == SLOTS - 1 ? 0 : in + 1;
        }
#pragma unroll
        for (int s = 0; s < STEPS; s++) {
            __builtin_amdgcn_sched_barrier(0);
            if (s + 1 < STEPS) fetch(s + 1);
            __builtin_amdgcn_sched_barrier(0);
            if constexpr (ENDS) {
                const int left = live - t * S::SLAB - 16 * s - 8 * ((threadIdx.x & 63) >> 5);
                if ((t + 1) * S::SLAB > live) {
#pragma unroll
                    for (int p = 0; p < PARTS; p++)
#pragma unroll
                        for (int i = 0; i < IM; i++)
#pragma unroll
                            for (int w = 0; w < 4; w++) {
                                const uint32_t keep = (left > 2 * w ? 0xffffu : 0u) | (left > 2 * w + 1 ? 0xffff0000u : 0u);
                                fa[s & 1][p][i][w] &= keep;
                            }
                }
            }
            // smallest products first: parts whose numbers add up to 2, to 1, to 0
#pragma unroll
            for (int order = PARTS - 1; order >= 0; order--)
#pragma unroll
                for (int p = 0; p <= order; p++)
#pragma unroll
                    for (int i = 0; i < IM; i++)
#pragma unroll
                        for (int j = 0; j < JN; j++) Slab<bf16_t>::mma(fb[s & 1][order - p][j], fa[s & 1][p][i], acc[i][j]);
            if constexpr (SUMS) {
                if (sums_wanted) {
#pragma unroll
                    for (int p = PARTS - 1; p >= 0; p--)
#pragma unroll
                        for (int i = 0; i < IM; i++) {
                            const u32x4 &f = fa[s & 1][p][i];
                            sums[i] = bf16_pair_sum(f.x, bf16_pair_sum(f.y, bf16_pair_sum(f.z, bf16_pair_sum(f.w, sums[i]))));
                        }
                }
            }
        }
    }
    lds_barrier();                                  // the ring is free for the epilogue
}

// A tile's results to memory, [rows, cols] dense: by way of LDS (the ring, behind its last reader), a wave 32 rows at a time, so that whole
// lines leave at once.  finish(j, q, v) has the last word on four of a row, columns (wn JN + j) 32 + 8 q + 4 (lane / 32) .. of the tile;
// `stream`: past the caches.  In runs without branches where the tile is whole: with them the stores of a piece wait for one another (an 8-bit
// product of 65536 x 1024 x 4096 in bf16: 470 us in pieces of 32 bytes, 400 in whole lines, 385 without branches).
template <class S, typename T, class F>
__device__ __forceinline__ void put_tile(unsigned char *smem, const f32x16 (&acc)[S::IM][S::JN], F &&finish, T *out, int64_t rows, int64_t cols, int64_t r0, int64_t c0,
                                         bool stream)
{
    constexpr int JN = S::JN, JP = sizeof(T) == 2 || JN == 1 ? JN : JN / 2, ROW = JP * 32 * sizeof(T), PITCH = ROW + 16, VEC = Elem<T>::VEC, LANES = ROW / 16;
    static_assert(S::WAVES * 32 * PITCH <= S::RING, "LDS");
    const int lane = threadIdx.x & 63, lr = lane & 31, lg = lane >> 5;
    const int wid = wave_uniform(threadIdx.x >> 6), wm = wid / S::WN, wn = wid % S::WN;
    using V = typename Loose<T>::vector;             // (rows of any length)
    unsigned char *const mine = smem + wid * 32 * PITCH;
    auto leave = [&](auto WHOLE, auto STREAM) {
        constexpr bool whole = decltype(WHOLE)::value, past = decltype(STREAM)::value;
#pragma unroll
        for (int i = 0; i < S::IM; i++) {
#pragma unroll
            for (int j0 = 0; j0 < JN; j0 += JP) {
#pragma unroll
                for (int j = j0; j < j0 + JP; j++) {
                    f32x4 v[4];
#pragma unroll
                    for (int q = 0; q < 4; q++) {
                        v[q] = f32x4{acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]};
                        finish(j, q, v[q]);
                    }
                    unsigned char *const at = mine + lr * PITCH + (j - j0) * 32 * sizeof(T);
                    if constexpr (sizeof(T) == 2) {
                        // half-wave swaps leave a lane 8 consecutive columns
#pragma unroll
                        for (int q = 0; q < 2; q++) {
                            const uint32_t o[4] = {pack_bf16x2(v[2 * q][0], v[2 * q][1]), pack_bf16x2(v[2 * q][2], v[2 * q][3]),
                                                   pack_bf16x2(v[2 * q + 1][0], v[2 * q + 1][1]), pack_bf16x2(v[2 * q + 1][2], v[2 * q + 1][3])};
                            const auto s0 = __builtin_amdgcn_permlane32_swap(o[0], o[2], false, false), s1 = __builtin_amdgcn_permlane32_swap(o[1], o[3], false, false);
                            *reinterpret_cast<u32x4 *>(at + 32 * q + 16 * lg) = u32x4{s0[0], s1[0], s0[1], s1[1]};
                        }
                    } else {
#pragma unroll
                        for (int q = 0; q < 4; q++) *reinterpret_cast<f32x4 *>(at + 32 * q + 16 * lg) = v[q];
                    }
                }
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");        // (the wave's own)
                const int64_t first = r0 + (wm * S::IM + i) * 32, column = c0 + (wn * JN + j0) * 32;
                T *const to = out + first * cols + column;
                if constexpr (whole) {
                    constexpr int TIMES = 32 * LANES / 64;
                    const int row = lane / LANES, c = lane % LANES;
                    T *const from = to + (int64_t)row * cols + c * VEC;
#pragma unroll
                    for (int k = 0; k < TIMES; k++) {
                        const u32x4 o = *reinterpret_cast<const u32x4 *>(mine + (row + k * (64 / LANES)) * PITCH + c * 16);
                        T *const at = from + (int64_t)k * (64 / LANES) * cols;
                        if constexpr (past) __builtin_nontemporal_store(o, reinterpret_cast<u32x4 *>(at));
                        else *reinterpret_cast<V *>(at) = o;
                    }
                } else {
                    const int live = (int)(rows - first < 32 ? rows - first : 32), left = (int)(cols - column < JP * 32 ? cols - column : JP * 32);
#pragma unroll 8
                    for (int k = lane; k < 32 * LANES; k += 64) {
                        const int row = k / LANES, c = k % LANES * VEC;
                        const u32x4 o = *reinterpret_cast<const u32x4 *>(mine + row * PITCH + c * sizeof(T));
                        if (row >= live || c >= left) continue;
                        T *const at = to + (int64_t)row * cols + c;
                        if (c + VEC <= left) *reinterpret_cast<V *>(at) = o;
                        else
                            for (int e = 0; e < left - c; e++) at[e] = *reinterpret_cast<const T *>(mine + row * PITCH + (c + e) * sizeof(T));
                    }
                }
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            }
        }
    };
    if (r0 + S::ROWS > rows || c0 + S::COLS > cols) leave(std::false_type{}, std::false_type{});
    else if (stream && cols % VEC == 0) leave(std::true_type{}, std::true_type{});
    else leave(std::true_type{}, std::false_type{});
}

// Workgroup id of `count` -> place in the list of all: an XCD (every eighth id) takes a contiguous run of it.
__device__ __forceinline__ int place_of(int id, int count)
{
    const int xcd = id & 7, whole = count >> 3, rest = count & 7;
    return xcd * whole + (xcd < rest ? xcd : rest) + (id >> 3);
}
// The list of tiles goes through eight row tiles for each column tile, so that what an XCD's L2 holds is used again.
__device__ __forceinline__ void tile_at(int place, int tm, int tn, int &m, int &n)
{
    const int group = 8 * tn, g = place / group, first = g * 8, size = min(8, tm - first);
    const int in = place - g * group;
    m = first + in % size;
    n = in / size;
}
// the same over all parts of a sum -> part
__device__ __forceinline__ int tile_of(int id, int parts, int tm, int tn, int &m, int &n)
{
    const int tiles = tm * tn, place = place_of(id, tiles * parts), part = place / tiles;
    tile_at(place - part * tiles, tm, tn, m, n);
    return part;
}

}  // namespace vtdge
