// Softmax cross entropy of a Linear's outputs over many classes, with the gradients of its input, weight and bias (gfx950).
//
//   z = x W^T + b,   loss_r = log sum_v exp z_rv - (1 - eps) z_rt - eps mean_v z_rv
//   d_rv = g_r (exp(z_rv) / sum - (1 - eps) [v = t_r] - eps / classes),   dx = d W,   dW = d^T x,   db = sum_r d_r
//
// z is not in memory (for fp32 gradients, see keeps_logits).  Forward, every workgroup multiplies a tile of rows by a tile of classes and keeps of it each row's largest
// z and the sum of exp(z - largest); a second kernel joins the tiles of a row.  Backward, the classes are taken in pieces: the
// tiles of a piece are multiplied again, d is rounded to bf16 (an error of half a step on each of many terms, as on any bf16
// operand; the sums over it are fp32) and kept for this piece only, and two products take it to dx and dW.  Four products of
// rows x classes x width in place of three, and no more than rows x piece values of scratch.
//
// One product routine does all of it: tiles through LDS by direct loads, in slabs of 32 or 64 of the summed dimension and a ring of two
// to six of them.  An operand either lies with the summed dimension along its rows (x and W for z, d for dx) or across them (W for dx, d and x for
// dW); the second kind goes into LDS as it lies and is transposed by the LDS reads.  16-byte pieces are XOR-ed by their row against
// bank conflicts, on the side of the global address.
// fp32 operands are split into three bf16 parts each (24 bits), and the six products of parts down to 2^-24 are a six times longer
// sum, smallest first, in the same fp32 sums: the same kernels at a sixth of their rate, which is above that of the fp32 matrix
// instructions.  Bits below 2^-133 are lost, which only values below 2^-110 have, and an infinity meets parts of either sign and may
// become NaN.  (Two fp16 parts and three products would be 22 bits of a row's largest value and fewer of its small ones.)
//
// Bound by the matrix units in long products: 8192 rows x 65536 classes x 1024 in bf16, tiles 0.98 ms (1.12 PFLOP/s), d 4 x 0.30 (0.93,
// with the writing of d), gradients 4 x 0.52 (1.06); in fp32 2048 x 21841 x 384, tiles with the logits kept 0.21 ms (166 TFLOP/s of fp32, 1.0
// PFLOP/s issued), d 0.07 from those, gradients 0.38.  Their units are busy for 56 to 58 percent (d 44) at the 1.7 - 2.0 GHz that the clock
// falls to, waves wait for a third of their cycles.  By the reading of W where rows are few (1 row x 65536 x 1024 in 21.6 us, 6.2 TB/s), by launches where all is small (256 x 1000 x
// 384: four kernels of 6 - 9 us).
#include "common.h"

#include <math.h>

namespace vtdge {

constexpr float LOG2E = 1.44269504f, LN2 = 0.69314718f;
__device__ __forceinline__ int wave_uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }
// What the first bf16 part of an fp32 value is rounded from: the largest finite numbers would become infinite, and are cut to bf16's
// largest; the next part has the rest.  (Infinity and NaN go on to the next part.)
constexpr float BF16_MOST = 0x1.fep127f;
__device__ __forceinline__ float first_part(float f) { return __builtin_amdgcn_fmed3f(f, -BF16_MOST, BF16_MOST); }

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
// LDS rows are 2 SLAB bytes (ALONG) or 2 T bytes (across) without gaps; their 16-byte pieces are XOR-ed by the row, so that the
// sixteen lanes that read together meet every bank once.
template <bool ALONG, int T, int SLAB, int WAVES, bool MAY_STREAM = false> struct Loader {
    static constexpr int ROW = ALONG ? 2 * SLAB : 2 * T, STAGE = 2 * SLAB * T;
    static constexpr int LPR = ROW / 16, RPI = 64 / LPR;                  // lanes a row, rows an instruction
    static constexpr int PIECES = STAGE / 1024 / WAVES;                   // instructions of a wave
    static_assert(PIECES * WAVES * 1024 == STAGE && LPR <= 64, "whole instructions");
    const unsigned char *base;
    int64_t plane, pitch;                                                 // bytes
    int limit, row0, last;
    bool stream = false;                                                  // past the caches

    __device__ __forceinline__ Loader(const Operand &o, int64_t first, int64_t lim, int64_t span)
        : base(reinterpret_cast<const unsigned char *>(o.p) + (ALONG ? first * o.pitch * 2 : first * 2)), plane(o.plane * 2), pitch(o.pitch * 2)
    {
        const int lane = threadIdx.x & 63, wid = wave_uniform(threadIdx.x >> 6);
        row0 = wid * RPI + lane / LPR;
        if constexpr (ALONG) limit = (int)(lim - first < T ? lim - first : T);
        else limit = (int)lim;
        last = ALONG ? 0 : (int)(span - first < T ? span - first : T) * 2 - 16;
    }
    static __device__ __forceinline__ int swizzle(int r)
    {
        if constexpr (ALONG) return SLAB == 64 ? (r >> 1) & 7 : SLAB == 32 ? (r >> 2) & 3 : (r >> 3) & 1;
        else return LPR == 8 ? ((r >> 1) & 3) << 1 : (r & 7) << 1;
    }
    // stage `kt` of part `part` to LDS byte `lds`
    __device__ __forceinline__ void load(int part, int kt, uint32_t lds) const
    {
        const int lane = threadIdx.x & 63, wid = wave_uniform(threadIdx.x >> 6);
        const void *from = uniform_ptr(base + part * plane + (ALONG ? (int64_t)kt * (2 * SLAB) : (int64_t)kt * SLAB * pitch));
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
// A's rows (of this half of the lanes' values), for what `sums_wanted` says.
template <class S, bool SUMS, class LA, class LB>
__device__ __forceinline__ void multiply_tile(const LA &a, const LB &b, int t0, int t1, unsigned char *smem, f32x16 (&acc)[S::IM][S::JN],
                                              bool sums_wanted, float (&sums)[S::IM])
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

struct CeArgs {
    Operand x, w;
    const void *bias; const int64_t *target; int64_t rows, classes; int64_t ignore; float smoothing; int stages;
    int64_t v0, v1;                                 // classes of this piece
    int bias_f32;
    bool stream_w;                                  // forward, few rows: W past the caches
    // forward: [class tiles][rows] each
    float *tile_max, *tile_sum, *tile_total, *target_z;
    float *z; int64_t z_pitch;                      // nullable: the logits times log2 e, kept for the gradients; -inf behind the last class
    // backward
    const float *row_max, *row_inv, *row_scale; bf16_t *d; int64_t d_pitch, d_plane;
    bf16_t *x_copy; int width;                      // nullable: x with zeros for the rows that are left out
};

__device__ __forceinline__ bool counts(int64_t target, int64_t ignore, int64_t classes) { return target != ignore && target >= 0 && target < classes; }

// the bias of the tile's classes times log2 e, -inf behind the last class
template <class S> __device__ __forceinline__ void read_bias(const CeArgs &p, int64_t c0, float *bias)
{
    for (int c = threadIdx.x; c < S::COLS; c += S::THREADS) {
        float b = -INFINITY;
        if (c0 + c < p.v1) {
            b = 0.f;
            if (p.bias != nullptr)
                b = LOG2E * (p.bias_f32 ? static_cast<const float *>(p.bias)[c0 + c] : bf16_to_f32(static_cast<const bf16_t *>(p.bias)[c0 + c]));
        }
        bias[c] = b;
    }
}
// z of a tile, times log2 e, in place of acc; `bias` of the wave's first class
template <class S> __device__ __forceinline__ void logits(const float *bias, f32x16 (&acc)[S::IM][S::JN])
{
    const int lg = (threadIdx.x & 63) >> 5;
#pragma unroll
    for (int j = 0; j < S::JN; j++)
#pragma unroll
        for (int q = 0; q < 4; q++) {
            const f32x4 b = *reinterpret_cast<const f32x4 *>(bias + j * 32 + 8 * q + 4 * lg);
#pragma unroll
            for (int e = 0; e < 4; e++)
#pragma unroll
                for (int i = 0; i < S::IM; i++) acc[i][j][4 * q + e] = __builtin_fmaf(acc[i][j][4 * q + e], LOG2E, b[e]);
        }
}

// ------------------------------------------------------------------------------------------------ forward
template <class S, bool TOTAL> __device__ __forceinline__ void logits_tile(const CeArgs &p, int64_t r0, int n, unsigned char *smem)
{
    constexpr int IM = S::IM, JN = S::JN, ROWS = S::ROWS;
    const int64_t c0 = (int64_t)n * S::COLS;
    float *const bias = reinterpret_cast<float *>(smem + S::RING);
    read_bias<S>(p, c0, bias);
    const int lane = threadIdx.x & 63, lr = lane & 31, lg = lane >> 5;
    const int wid = wave_uniform(threadIdx.x >> 6), wm = wid / S::WN, wn = wid % S::WN;
    const int64_t cw = c0 + wn * 32 * JN;
    // the rows' own classes, asked for before the product: which of the wave's classes, or less than 0
    int own[IM];
#pragma unroll
    for (int i = 0; i < IM; i++) {
        const int64_t r = r0 + (wm * IM + i) * 32 + lr, t = r < p.rows ? p.target[r] : -1;
        own[i] = r < p.rows && counts(t, p.ignore, p.classes) && t >= cw && t < cw + 32 * JN ? (int)(t - cw) : -1;
    }
    f32x16 acc[IM][JN] = {};
    float none[IM];
    const Loader<true, ROWS, S::SLAB, S::WAVES> a(p.x, r0, p.rows, 0);
    Loader<true, S::COLS, S::SLAB, S::WAVES, S::FLAT> b(p.w, c0, p.classes, 0);
    b.stream = p.stream_w;
    multiply_tile<S, false>(a, b, 0, p.stages, smem, acc, false, none);
    logits<S>(bias + wn * 32 * JN, acc);
    if (S::PARTS > 1 && p.z != nullptr) {
#pragma unroll
        for (int i = 0; i < IM; i++) {
            const int64_t r = r0 + (wm * IM + i) * 32 + lr;
            if (r >= p.rows) continue;
#pragma unroll
            for (int j = 0; j < JN; j++)
#pragma unroll
                for (int q = 0; q < 4; q++) {
                    const int64_t c = cw + j * 32 + 8 * q + 4 * lg;
                    if (c < p.z_pitch)
                        *reinterpret_cast<f32x4 *>(p.z + r * p.z_pitch + c) = f32x4{acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]};
                }
        }
    }
    float *const shared = reinterpret_cast<float *>(smem);          // [waves along the classes][largest, sum, total][rows]
#pragma unroll
    for (int i = 0; i < IM; i++) {
        const int row = (wm * IM + i) * 32 + lr;
        float top = -INFINITY, total = 0.f;
#pragma unroll
        for (int j = 0; j < JN; j++)
#pragma unroll
            for (int v = 0; v < 16; v++) top = fmaxf(top, acc[i][j][v]);
        top = fmaxf(top, __shfl_xor(top, 32, WAVE));
        const float from = top == -INFINITY ? 0.f : top;            // nothing in sight: exp2(-inf) = 0, and NaN stays NaN
        float sum = 0.f;
#pragma unroll
        for (int j = 0; j < JN; j++)
#pragma unroll
            for (int v = 0; v < 16; v++) {
                sum += __builtin_amdgcn_exp2f(acc[i][j][v] - from);
                if constexpr (TOTAL) total += cw + j * 32 + 8 * (v / 4) + 4 * lg + v % 4 < p.classes ? acc[i][j][v] : 0.f;
            }
        sum += __shfl_xor(sum, 32, WAVE);
        if constexpr (TOTAL) total += __shfl_xor(total, 32, WAVE);
        if (lg == 0) {
            shared[(wn * 3 + 0) * ROWS + row] = top;
            shared[(wn * 3 + 1) * ROWS + row] = sum;
            if constexpr (TOTAL) shared[(wn * 3 + 2) * ROWS + row] = total;
        }
        // the z of the row's own class
        const int at = own[i];
        const bool mine = at >= 0 && ((at >> 2) & 1) == lg;
        if (__ballot(mine) != 0) {
            const int reg = (at >> 5) * 16 + ((at & 31) >> 3) * 4 + (at & 3);
            float z = 0.f;
#pragma unroll
            for (int j = 0; j < JN; j++)
#pragma unroll
                for (int v = 0; v < 16; v++) z = reg == j * 16 + v ? acc[i][j][v] : z;
            if (mine) p.target_z[r0 + row] = z;
        }
    }
    __syncthreads();
    for (int row = threadIdx.x; row < ROWS && r0 + row < p.rows; row += S::THREADS) {
        static_assert(S::WN == 2, "two waves along the classes");
        const float t0 = shared[row], t1 = shared[3 * ROWS + row], top = fmaxf(t0, t1);
        const float from = top == -INFINITY ? 0.f : top;
        const float sum = shared[ROWS + row] * __builtin_amdgcn_exp2f((t0 == -INFINITY ? from : t0) - from) +
                          shared[4 * ROWS + row] * __builtin_amdgcn_exp2f((t1 == -INFINITY ? from : t1) - from);
        const int64_t at = (int64_t)n * p.rows + r0 + row;
        p.tile_max[at] = top;
        p.tile_sum[at] = sum;
        if constexpr (TOTAL) p.tile_total[at] = shared[2 * ROWS + row] + shared[5 * ROWS + row];
    }
}
// Workgroups from `whole` on have half a tile each.
template <class S, bool TOTAL> __global__ __launch_bounds__(S::THREADS, S::PER_SIMD) void cross_entropy_tiles_kernel(CeArgs p, int tm, int tn, int whole)
{
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    int m, n;
    const int id = blockIdx.x;
    if (!S::HALVES || id < whole) {
        tile_at(place_of(id, whole), tm, tn, m, n);
        logits_tile<S, TOTAL>(p, (int64_t)m * S::ROWS, n, smem);
    } else if constexpr (S::HALVES) {
        tile_at(whole + (id - whole) / 2, tm, tn, m, n);
        const int64_t r0 = (int64_t)m * S::ROWS + (id - whole) % 2 * S::Half::ROWS;
        if (r0 < p.rows) logits_tile<typename S::Half, TOTAL>(p, r0, n, smem);
    }
}

// A row's tiles joined, by the waves of a workgroup side by side (64 rows, one a lane).  `mean`: the only workgroup goes through
// all rows and on to their mean or sum.
constexpr int JOIN_WAVES = 16;
struct JoinArgs {
    const float *tile_max, *tile_sum, *tile_total, *target_z; const int64_t *target; int64_t rows, classes, ignore; float smoothing; int tn;
    float *loss_rows, *row_max, *row_inv, *loss, *inv_count;
};
__device__ __forceinline__ float scaled(float sum, float top, float to) { return sum * __builtin_amdgcn_exp2f((top == -INFINITY ? to : top) - to); }

__device__ void mean_of(double sum, int64_t n, const JoinArgs &p)
{
    __shared__ double sums[JOIN_WAVES];
    __shared__ int64_t ns[JOIN_WAVES];
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        sum += __shfl_xor(sum, o, WAVE);
        n += __shfl_xor(n, o, WAVE);
    }
    if ((threadIdx.x & 63) == 0) sums[threadIdx.x >> 6] = sum, ns[threadIdx.x >> 6] = n;
    __syncthreads();
    if (threadIdx.x != 0) return;
    sum = 0.0, n = 0;
    for (int w = 0; w < JOIN_WAVES; w++) sum += sums[w], n += ns[w];
    if (p.inv_count == nullptr) {
        *p.loss = (float)sum;
    } else {
        *p.loss = n > 0 ? (float)(sum / (double)n) : 0.f;
        *p.inv_count = n > 0 ? (float)(1.0 / (double)n) : 0.f;
    }
}
__device__ __forceinline__ float loss_of(const JoinArgs &p, int64_t r, float top, float sum, float total, bool &live)
{
    const int64_t t = p.target[r];
    live = counts(t, p.ignore, p.classes);
    if (!live) return 0.f;
    // log2 sum + (1 - eps) (largest - z_t) + eps (largest - mean): differences of like size, not of large sums
    float loss = __builtin_amdgcn_logf(sum) + (1.f - p.smoothing) * (top - p.target_z[r]);
    if (p.smoothing != 0.f) loss += p.smoothing * (top - total / (float)p.classes);
    return loss * LN2;
}
__device__ __forceinline__ void join_tiles(const JoinArgs &p, int64_t r, int first, int step, float &top, float &sum, float &total)
{
#pragma unroll 8
    for (int n = first; n < p.tn; n += step) {
        const int64_t at = (int64_t)n * p.rows + r;
        const float t = p.tile_max[at], s = p.tile_sum[at], next = fmaxf(top, t), to = next == -INFINITY ? 0.f : next;
        sum = scaled(sum, top, to) + scaled(s, t, to);
        top = next;
        if (p.smoothing != 0.f) total += p.tile_total[at];
    }
}

__global__ __launch_bounds__(64 * JOIN_WAVES) void cross_entropy_join_kernel(JoinArgs p)
{
    __shared__ float tops[JOIN_WAVES][64], sums[JOIN_WAVES][64], totals[JOIN_WAVES][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t r = (int64_t)blockIdx.x * 64 + lane;
    const bool in = r < p.rows;
    float top = -INFINITY, sum = 0.f, total = 0.f;
    if (in) join_tiles(p, r, wave, JOIN_WAVES, top, sum, total);
    tops[wave][lane] = top;
    sums[wave][lane] = sum;
    totals[wave][lane] = total;
    __syncthreads();
    if (wave != 0 || !in) return;
    top = -INFINITY;
    for (int w = 0; w < JOIN_WAVES; w++) top = fmaxf(top, tops[w][lane]);
    const float to = top == -INFINITY ? 0.f : top;
    sum = total = 0.f;
    for (int w = 0; w < JOIN_WAVES; w++) {
        sum += scaled(sums[w][lane], tops[w][lane], to);
        total += totals[w][lane];
    }
    bool live;
    p.loss_rows[r] = loss_of(p, r, top, sum, total, live);
    p.row_max[r] = top;
    p.row_inv[r] = 1.0f / sum;
}
// few rows of many tiles: a workgroup takes one row, its threads the tiles
__global__ __launch_bounds__(64 * JOIN_WAVES) void cross_entropy_join_row_kernel(JoinArgs p)
{
    __shared__ float tops[JOIN_WAVES], sums[JOIN_WAVES], totals[JOIN_WAVES];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t r = blockIdx.x;
    float top = -INFINITY, sum = 0.f, total = 0.f;
    join_tiles(p, r, threadIdx.x, 64 * JOIN_WAVES, top, sum, total);
    const float all = wave_max(top), to = all == -INFINITY ? 0.f : all;
    sum = wave_sum(scaled(sum, top, to));
    total = wave_sum(total);
    if (lane == 0) tops[wave] = all, sums[wave] = sum, totals[wave] = total;
    __syncthreads();
    if (threadIdx.x != 0) return;
    top = -INFINITY;
    for (int w = 0; w < JOIN_WAVES; w++) top = fmaxf(top, tops[w]);
    const float base = top == -INFINITY ? 0.f : top;
    sum = total = 0.f;
    for (int w = 0; w < JOIN_WAVES; w++) {
        sum += scaled(sums[w], tops[w], base);
        total += totals[w];
    }
    bool live;
    p.loss_rows[r] = loss_of(p, r, top, sum, total, live);
    p.row_max[r] = top;
    p.row_inv[r] = 1.0f / sum;
}
// few rows of few tiles: one workgroup does all of it, a row a thread
__global__ __launch_bounds__(64 * JOIN_WAVES) void cross_entropy_join_mean_kernel(JoinArgs p)
{
    double all = 0.0;
    int64_t n = 0;
    for (int64_t r = threadIdx.x; r < p.rows; r += 64 * JOIN_WAVES) {
        float top = -INFINITY, sum = 0.f, total = 0.f;
        join_tiles(p, r, 0, 1, top, sum, total);
        bool live;
        const float loss = loss_of(p, r, top, sum, total, live);
        p.loss_rows[r] = loss;
        p.row_max[r] = top;
        p.row_inv[r] = 1.0f / sum;
        all += loss;
        n += live ? 1 : 0;
    }
    if (p.loss != nullptr) mean_of(all, n, p);
}
__global__ __launch_bounds__(64 * JOIN_WAVES) void cross_entropy_mean_kernel(JoinArgs p)
{
    double sum = 0.0;
    int64_t n = 0;
    for (int64_t r = threadIdx.x; r < p.rows; r += 64 * JOIN_WAVES) {
        sum += p.loss_rows[r];
        n += counts(p.target[r], p.ignore, p.classes) ? 1 : 0;
    }
    mean_of(sum, n, p);
}

// ------------------------------------------------------------------------------------------------ backward
// d of a piece of the classes; rows and classes behind the last are written as zeros, so that slabs may run over them
// (rows `from` on of a tile of `of`, which is this one or twice as high)
template <class S> __device__ __forceinline__ void d_tile(const CeArgs &p, int64_t r0, int n, int tn, int from, int of, unsigned char *smem)
{
    constexpr int IM = S::IM, JN = S::JN;
    const int64_t c0 = p.v0 + (int64_t)n * S::COLS;
    float *const bias = reinterpret_cast<float *>(smem + S::RING);
    read_bias<S>(p, c0, bias);
    if (p.x_copy != nullptr) {
        // this tile's share of the rows: all class tiles together copy them
        const int vecs = p.width / 8, share = (of + tn - 1) / tn;
        for (int i = threadIdx.x; i < share * vecs; i += S::THREADS) {
            const int k = n * share + i / vecs - from, c = (i % vecs) * 8;
            const int64_t r = r0 + k;
            if (k < 0) continue;
            if (k >= S::ROWS || r >= p.rows) break;
            u32x4 v = *reinterpret_cast<const u32x4 *>(p.x.p + r * p.x.pitch + c);
            if (!counts(p.target[r], p.ignore, p.classes)) v = u32x4{0u, 0u, 0u, 0u};
            *reinterpret_cast<u32x4 *>(p.x_copy + r * p.width + c) = v;
        }
    }
    const int lane = threadIdx.x & 63, lr = lane & 31, lg = lane >> 5;
    const int wid = wave_uniform(threadIdx.x >> 6), wm = wid / S::WN, wn = wid % S::WN;
    const int64_t cw = c0 + wn * 32 * JN;
    const bool edge = cw + 32 * JN > p.v1;
    // what the rows bring, asked for before the product
    const float even = p.smoothing / (float)p.classes;
    int own[IM];
    bool lives[IM];
    float tops[IM], invs[IM], scales[IM];
#pragma unroll
    for (int i = 0; i < IM; i++) {
        const int64_t r = r0 + (wm * IM + i) * 32 + lr, at = r < p.rows ? r : p.rows - 1, t = p.target[at];
        lives[i] = r < p.rows && counts(t, p.ignore, p.classes);
        own[i] = lives[i] && t >= cw && t < cw + 32 * JN && t < p.v1 ? (int)(t - cw) : -1;
        const float top = p.row_max[at], inv = p.row_inv[at], g = p.row_scale != nullptr ? p.row_scale[at] : 1.f;
        tops[i] = lives[i] ? top : 0.f;
        scales[i] = lives[i] ? g : 0.f;
        invs[i] = lives[i] ? inv * g : 0.f;
    }
    f32x16 acc[IM][JN] = {};
    float none[IM];
    const Loader<true, S::ROWS, S::SLAB, S::WAVES> a(p.x, r0, p.rows, 0);
    const Loader<true, S::COLS, S::SLAB, S::WAVES> b(p.w, c0, p.classes, 0);
    multiply_tile<S, false>(a, b, 0, p.stages, smem, acc, false, none);
    logits<S>(bias + wn * 32 * JN, acc);
    // To memory: half-wave swaps leave a lane 8 consecutive classes.  bf16: as they are, 32 bytes of a row side by side, while the other
    // workgroup of the compute unit multiplies (8192 x 1024 x 65536: 313 us a piece, by way of LDS 328).  fp32, where a workgroup
    // is alone: part by part through LDS, rows in whole lines (2048 x 384 x 21841: 290 us without, 251 so).
    constexpr int PITCH = S::COLS * 2 + 16, VECS = S::COLS / 8;
    static_assert(S::PARTS == 1 || S::ROWS * PITCH <= S::RING, "LDS");
    auto put = [&](int i, bool first, bool rest) {  // and what is left of the values for the next part
        bf16_t *const row = p.d + (r0 + (wm * IM + i) * 32 + lr) * p.d_pitch + (cw - p.v0) + 8 * lg;
        unsigned char *const at = smem + ((wm * IM + i) * 32 + lr) * PITCH + wn * 64 * JN + 16 * lg;
#pragma unroll
        for (int j = 0; j < JN; j++)
#pragma unroll
            for (int q = 0; q < 2; q++) {
                uint32_t o[4];
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const float a = acc[i][j][8 * q + 2 * e], b = acc[i][j][8 * q + 2 * e + 1];
                    o[e] = first ? pack_bf16x2(first_part(a), first_part(b)) : pack_bf16x2(a, b);
                    if (rest) acc[i][j][8 * q + 2 * e] -= bf16lo(o[e]), acc[i][j][8 * q + 2 * e + 1] -= bf16hi(o[e]);
                }
                const auto s0 = __builtin_amdgcn_permlane32_swap(o[0], o[2], false, false), s1 = __builtin_amdgcn_permlane32_swap(o[1], o[3], false, false);
                const u32x4 v = {s0[0], s1[0], s0[1], s1[1]};
                if constexpr (S::PARTS == 1) *reinterpret_cast<u32x4 *>(row + j * 32 + 16 * q) = v;
                else *reinterpret_cast<u32x4 *>(at + j * 64 + 32 * q) = v;
            }
    };
#pragma unroll
    for (int i = 0; i < IM; i++) {
        const bool live = lives[i];
        const float top = tops[i], inv = invs[i], minus = -even * scales[i];
#pragma unroll
        for (int j = 0; j < JN; j++)
#pragma unroll
            for (int v = 0; v < 16; v++) acc[i][j][v] = __builtin_fmaf(__builtin_amdgcn_exp2f(acc[i][j][v] - top), inv, minus);
        const int at = own[i];
        const bool mine = at >= 0 && ((at >> 2) & 1) == lg;
        if (__ballot(mine) != 0) {
            const int reg = mine ? (at >> 5) * 16 + ((at & 31) >> 3) * 4 + (at & 3) : -1;
            const float one = (1.f - p.smoothing) * scales[i];
#pragma unroll
            for (int j = 0; j < JN; j++)
#pragma unroll
                for (int v = 0; v < 16; v++) acc[i][j][v] -= reg == j * 16 + v ? one : 0.f;
        }
        if (edge || __ballot(!live) != 0) {
#pragma unroll
            for (int j = 0; j < JN; j++)
#pragma unroll
                for (int v = 0; v < 16; v++) acc[i][j][v] = live && cw + j * 32 + 8 * (v / 4) + 4 * lg + v % 4 < p.v1 ? acc[i][j][v] : 0.f;
        }
        put(i, S::PARTS > 1, S::PARTS > 1);
    }
    if constexpr (S::PARTS > 1) {
        for (int part = 0; part < S::PARTS; part++) {
            if (part > 0) {
                __syncthreads();
#pragma unroll
                for (int i = 0; i < IM; i++) put(i, false, part + 1 < S::PARTS);
            }
            __syncthreads();
            bf16_t *const to = p.d + part * p.d_plane + r0 * p.d_pitch + (c0 - p.v0);
#pragma unroll 4
            for (int k = threadIdx.x; k < S::ROWS * VECS; k += S::THREADS)
                *reinterpret_cast<u32x4 *>(to + (int64_t)(k / VECS) * p.d_pitch + (k % VECS) * 8) =
                    *reinterpret_cast<const u32x4 *>(smem + (k / VECS) * PITCH + (k % VECS) * 16);
        }
    }
}

template <class S> __global__ __launch_bounds__(S::THREADS, S::PER_SIMD) void cross_entropy_d_kernel(CeArgs p, int tm, int tn, int whole)
{
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    int m, n;
    const int id = blockIdx.x;
    if (!S::HALVES || id < whole) {
        tile_at(place_of(id, whole), tm, tn, m, n);
        d_tile<S>(p, (int64_t)m * S::ROWS, n, tn, 0, S::ROWS, smem);
    } else if constexpr (S::HALVES) {
        tile_at(whole + (id - whole) / 2, tm, tn, m, n);
        const int from = (id - whole) % 2 * S::Half::ROWS;
        const int64_t r0 = (int64_t)m * S::ROWS + from;
        // (a half without a row lies behind the slabs that are read)
        if (r0 < p.rows) d_tile<typename S::Half>(p, r0, n, tn, from, S::ROWS, smem);
    }
}

// The same from kept logits, in three parts: a lane has eight classes of a row, `vecs` of them side by side and `rows` rows to be written.
__global__ __launch_bounds__(256) void cross_entropy_d_kept_kernel(CeArgs p, int vecs, int64_t rows)
{
    const uint32_t id = blockIdx.x * 256 + threadIdx.x, row = id / (uint32_t)vecs;
    const int64_t r = row;
    if (r >= rows) return;
    const int64_t c = (int64_t)(id - row * (uint32_t)vecs) * 8, v = p.v0 + c, at = r < p.rows ? r : p.rows - 1, t = p.target[at];
    const bool live = r < p.rows && counts(t, p.ignore, p.classes);
    float f[8];
#pragma unroll
    for (int e = 0; e < 8; e++) f[e] = 0.f;
    if (live && v < p.v1) {
        const float g = p.row_scale != nullptr ? p.row_scale[at] : 1.f, top = p.row_max[at], inv = p.row_inv[at] * g;
        const float minus = -(p.smoothing / (float)p.classes) * g, one = (1.f - p.smoothing) * g;
        const f32x4 a = *reinterpret_cast<const f32x4 *>(p.z + r * p.z_pitch + v), b = *reinterpret_cast<const f32x4 *>(p.z + r * p.z_pitch + v + 4);
#pragma unroll
        for (int e = 0; e < 8; e++) {
            f[e] = __builtin_fmaf(__builtin_amdgcn_exp2f((e < 4 ? a[e & 3] : b[e & 3]) - top), inv, minus);
            if (v + e == t) f[e] -= one;
            if (v + e >= p.v1) f[e] = 0.f;
        }
    }
    bf16_t *const to = p.d + r * p.d_pitch + c;
#pragma unroll
    for (int part = 0; part < 3; part++) {
        u32x4 o;
#pragma unroll
        for (int e = 0; e < 4; e++) {
            o[e] = part == 0 ? pack_bf16x2(first_part(f[2 * e]), first_part(f[2 * e + 1])) : pack_bf16x2(f[2 * e], f[2 * e + 1]);
            f[2 * e] -= bf16lo(o[e]), f[2 * e + 1] -= bf16hi(o[e]);
        }
        *reinterpret_cast<u32x4 *>(to + part * p.d_plane) = o;
    }
}

// ---- out = A B, dx = d W or dW = d^T x, over a dimension that may be cut into several parts, which leave sums of their own
struct GradArgs {
    Operand a, b;
    int64_t rows, cols, span_a, span_b, sum_a, sum_b;      // of the result; elements of a row of memory; rows of memory that may be read
    int tm, tn, stages, splits;
    float *part; int64_t part_stride; int accumulate;       // [splits], [rows][cols] fp32 each
    void *out;                                              // without `part`: the result, scaled; neither: only the sums
    float *sums_part; int64_t sums_stride; void *sums;     // nullable: the sums of A's rows, in the same way
};
struct GradPair {
    GradArgs dx, dw;
    int first_dw;                                           // workgroups before are dx's
    const float *scale, *scale2; int f32;
};

// four values of row r from column c on, to a part or to the result
__device__ __forceinline__ void put_four(const GradArgs &p, const GradPair &all, int z, int64_t r, int64_t c, f32x4 v, float scale)
{
    const int left = (int)(p.cols - c);
    const bool whole = left >= 4 && p.cols % 4 == 0;
    if (p.part != nullptr) {
        float *const to = p.part + z * p.part_stride + r * p.cols + c;
        if (whole) {
            if (p.accumulate) v += *reinterpret_cast<const f32x4 *>(to);
            *reinterpret_cast<f32x4 *>(to) = v;
        } else {
#pragma unroll
            for (int e = 0; e < 4; e++)
                if (e < left) to[e] = v[e] + (p.accumulate ? to[e] : 0.f);
        }
    } else if (p.out != nullptr) {
        v *= scale;
        if (all.f32) {
            float *const to = static_cast<float *>(p.out) + r * p.cols + c;
            if (whole) {
                *reinterpret_cast<f32x4 *>(to) = v;
            } else {
#pragma unroll
                for (int e = 0; e < 4; e++)
                    if (e < left) to[e] = v[e];
            }
        } else {
            bf16_t *const to = static_cast<bf16_t *>(p.out) + r * p.cols + c;
            if (whole) {
                *reinterpret_cast<u32x2 *>(to) = u32x2{pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3])};
            } else {
#pragma unroll
                for (int e = 0; e < 4; e++)
                    if (e < left) to[e] = f32_to_bf16(v[e]);
            }
        }
    }
}
template <class S, bool A_ALONG> __device__ __forceinline__ void gradient_tile(const GradArgs &p, const GradPair &all, int id, unsigned char *smem)
{
    constexpr int IM = S::IM, JN = S::JN;
    int m, n;
    const int z = tile_of(id, p.splits, p.tm, p.tn, m, n);
    const int64_t r0 = (int64_t)m * S::ROWS, c0 = (int64_t)n * S::COLS;
    const int t0 = (int)((int64_t)p.stages * z / p.splits), t1 = (int)((int64_t)p.stages * (z + 1) / p.splits);
    f32x16 acc[IM][JN] = {};
    float sums[IM] = {};
    const Loader<A_ALONG, S::ROWS, S::SLAB, S::WAVES> a(p.a, r0, A_ALONG ? p.rows : p.sum_a, p.span_a);
    const Loader<false, S::COLS, S::SLAB, S::WAVES> b(p.b, c0, p.sum_b, p.span_b);
    const int lane = threadIdx.x & 63, lr = lane & 31, lg = lane >> 5;
    const int wid = wave_uniform(threadIdx.x >> 6), wm = wid / S::WN, wn = wid % S::WN;
    const bool with_sums = !A_ALONG && n == 0 && wn == 0 && (p.sums_part != nullptr || p.sums != nullptr);
    float scale = 1.f;
    if (all.scale != nullptr) scale = *all.scale;
    if (all.scale2 != nullptr) scale *= *all.scale2;
    multiply_tile<S, !A_ALONG>(a, b, t0, t1, smem, acc, with_sums, sums);
#pragma unroll
    for (int i = 0; i < IM; i++) {
        const int64_t r = r0 + (wm * IM + i) * 32 + lr;
        if constexpr (!A_ALONG) {
            if (with_sums) {
                const float sum = sums[i] + __shfl_xor(sums[i], 32, WAVE);
                if (lg == 0 && r < p.rows) {
                    if (p.sums_part != nullptr) p.sums_part[z * p.sums_stride + r] = sum;
                    else if (all.f32) static_cast<float *>(p.sums)[r] = sum * scale;
                    else static_cast<bf16_t *>(p.sums)[r] = f32_to_bf16(sum * scale);
                }
            }
        }
        if (S::WHOLE_LINES || r >= p.rows) continue;
#pragma unroll
        for (int j = 0; j < JN; j++)
#pragma unroll
            for (int q = 0; q < 4; q++) {
                const f32x4 v = {acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]};
                put_four(p, all, z, r, c0 + (wn * JN + j) * 32 + 8 * q + 4 * lg, v, scale);
            }
    }
    if constexpr (S::WHOLE_LINES) {
        // by way of LDS, lanes side by side in a row (bf16 1 x 363 x 25766: 40 us without, 22 so)
        constexpr int PITCH = S::COLS + 4;
        static_assert(S::ROWS * PITCH * 4 <= S::RING && IM == 1, "LDS");
        if (p.part == nullptr && p.out == nullptr) return;
        float *const tile = reinterpret_cast<float *>(smem);
#pragma unroll
        for (int j = 0; j < JN; j++)
#pragma unroll
            for (int q = 0; q < 4; q++)
                *reinterpret_cast<f32x4 *>(tile + (wm * 32 + lr) * PITCH + (wn * JN + j) * 32 + 8 * q + 4 * lg) =
                    f32x4{acc[0][j][4 * q], acc[0][j][4 * q + 1], acc[0][j][4 * q + 2], acc[0][j][4 * q + 3]};
        __syncthreads();
        const int rows = (int)(p.rows - r0 < S::ROWS ? p.rows - r0 : S::ROWS);
        if (p.cols % 4 == 0) {
#pragma unroll 4
            for (int k = threadIdx.x; k < rows * (S::COLS / 4); k += S::THREADS) {
                const int row = k / (S::COLS / 4), c = k % (S::COLS / 4) * 4;
                if (c0 + c < p.cols) put_four(p, all, z, r0 + row, c0 + c, *reinterpret_cast<const f32x4 *>(tile + row * PITCH + c), scale);
            }
        } else {
#pragma unroll 4
            for (int k = threadIdx.x; k < rows * S::COLS; k += S::THREADS) {
                const int row = k / S::COLS, c = k % S::COLS;
                if (c0 + c >= p.cols) continue;
                const int64_t at = (r0 + row) * p.cols + c0 + c;
                const float v = tile[row * PITCH + c];
                if (p.part != nullptr) p.part[z * p.part_stride + at] = v + (p.accumulate ? p.part[z * p.part_stride + at] : 0.f);
                else if (all.f32) static_cast<float *>(p.out)[at] = v * scale;
                else static_cast<bf16_t *>(p.out)[at] = f32_to_bf16(v * scale);
            }
        }
    }
}
template <class S> __global__ __launch_bounds__(S::THREADS, S::PER_SIMD) void cross_entropy_grad_kernel(GradPair p)
{
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    if ((int)blockIdx.x < p.first_dw) gradient_tile<S, true>(p.dx, p, blockIdx.x, smem);
    else gradient_tile<S, false>(p.dw, p, blockIdx.x - p.first_dw, smem);
}

// out = scale * (sum over the parts), for up to three results in one launch
struct SumJob {
    const float *part; void *out; int64_t n, stride; int parts;
};
struct SumArgs {
    SumJob job[3];
    int64_t first[4];                               // workgroups
    const float *scale, *scale2; int f32;
};
__global__ __launch_bounds__(256) void cross_entropy_sum_kernel(SumArgs p)
{
    int j = 0;
    while (j < 2 && (int64_t)blockIdx.x >= p.first[j + 1]) j++;
    const SumJob &job = p.job[j];
    const int64_t i = (((int64_t)blockIdx.x - p.first[j]) * 256 + threadIdx.x) * 4;
    if (i >= job.n) return;
    float scale = p.scale != nullptr ? *p.scale : 1.f;
    if (p.scale2 != nullptr) scale *= *p.scale2;
    // (parts lie on 16-byte boundaries and are filled up to whole pieces)
    f32x4 sum = {0.f, 0.f, 0.f, 0.f};
    for (int k = 0; k < job.parts; k++) sum += *reinterpret_cast<const f32x4 *>(job.part + k * job.stride + i);
    sum *= scale;
    const int live = job.n - i < 4 ? (int)(job.n - i) : 4;
    if (p.f32) {
        float *const to = static_cast<float *>(job.out) + i;
        for (int e = 0; e < live; e++) to[e] = sum[e];
    } else {
        bf16_t *const to = static_cast<bf16_t *>(job.out) + i;
        for (int e = 0; e < live; e++) to[e] = f32_to_bf16(sum[e]);
    }
}

// Rows as the product routine reads them: `width` filled up with zeros to whole slabs, fp32 in three parts; rows that are left out
// (target given) as zeros, so that what they hold reaches no gradient.  Up to two operands in one launch.
struct PackJob {
    const void *from; int64_t ld, rows; const int64_t *target; bf16_t *to;
};
struct PackArgs {
    PackJob job[2];
    int64_t first;                                  // workgroups of the first
    int width, padded; int64_t ignore, classes;
};
template <typename T> __global__ __launch_bounds__(256) void cross_entropy_pack_kernel(PackArgs p)
{
    const bool second = (int64_t)blockIdx.x >= p.first;
    const PackJob &job = p.job[second ? 1 : 0];
    const int per_row = p.padded / 8;
    const int64_t i = ((int64_t)blockIdx.x - (second ? p.first : 0)) * 256 + threadIdx.x, r = i / per_row;
    if (r >= job.rows) return;
    const int c = (int)(i - r * per_row) * 8;
    const bool live = job.target == nullptr || counts(job.target[r], p.ignore, p.classes);
    const T *const from = static_cast<const T *>(job.from) + r * job.ld + c;
    float f[8];
    if (live && c + 8 <= p.width && ((uintptr_t)from & 15) == 0) {
#pragma unroll
        for (int e = 0; e < 8; e += Elem<T>::VEC) Elem<T>::unpack(*reinterpret_cast<const u32x4 *>(from + e), f + e);
    } else {
#pragma unroll
        for (int e = 0; e < 8; e++) f[e] = live && c + e < p.width ? Elem<T>::load(from + e) : 0.f;
    }
    bf16_t *const at = job.to + r * p.padded + c;
    if constexpr (sizeof(T) == 2) {
        *reinterpret_cast<u32x4 *>(at) = Elem<bf16_t>::pack(f);
    } else {
#pragma unroll
        for (int part = 0; part < 3; part++) {
            float v[8];
#pragma unroll
            for (int e = 0; e < 8; e++) {
                // (infinity and NaN have no rest)
                v[e] = part == 0 && fabsf(f[e]) < INFINITY ? first_part(f[e]) : f[e];
                const float rest = f[e] - Elem<bf16_t>::round(v[e]);
                f[e] = fabsf(rest) < INFINITY ? rest : 0.f;
            }
            *reinterpret_cast<u32x4 *>(at + part * job.rows * p.padded) = Elem<bf16_t>::pack(v);
        }
    }
}

// ------------------------------------------------------------------------------------------------ on the host
// Shapes.  What bounds the large ones is how fast a compute unit takes its operands in: a slab of a 256 x 256 tile by eight waves is 64 KB
// for 2048 clocks of products, of 128 x 256 96 KB, and direct loads of whole lines (slabs of 64) pass faster than of half ones.  The
// matrix units of the first are busy for about 60 percent of a long product at the 1.8 GHz that remain, 1.1 PFLOP/s (8192 x 1024 x
// 65536, with its epilogue); tiles of 128 x 256, two workgroups a compute unit, 0.97, but one's epilogue runs beside the other's
// products, which makes up for it in short sums.  Tiles of 64 x 64 with a deep ring where a call waits for memory and not for products,
// 64 rows by 128 classes for few rows of many classes, which wait for W.
using LogitsLarge = Shape<2, 4, 4, 2, 64, 2, 1>;
using LogitsMiddle = Shape<2, 4, 2, 2, 32, 3, 1>;
using LogitsFlat = Shape<1, 2, 2, 2, 64, 3, 1>;
using LogitsSmall = Shape<1, 1, 2, 2, 64, 6, 1>;
using GradLarge = Shape<2, 4, 4, 2, 64, 2, 1>;
using GradMiddle = Shape<2, 2, 4, 2, 64, 3, 1>;
// (short sums of many tiles: three on a compute unit, fp32 two, rather than a deep ring for one; bf16 1 row x 363 x 25766 classes 43 -> 22 us,
// 256 x 384 x 1000 10.2 -> 9.7)
using GradSmall = Shape<1, 1, 2, 2, 64, 3, 1>;
using SplitLarge = Shape<2, 2, 4, 2, 32, 2, 3>;
using SplitFlat = Shape<1, 2, 2, 2, 32, 3, 3>;
using SplitSmall = Shape<1, 1, 2, 2, 32, 4, 3>;
using SplitGradSmall = Shape<1, 1, 2, 2, 32, 3, 3>;

constexpr int CE_PAD = 64;                          // rows of operands are filled up to whole slabs of any shape
constexpr int64_t CE_PIECE_BYTES = 320ll << 20;     // of d
constexpr int64_t CE_KEPT_BYTES = 256ll << 20;      // of logits
enum { CE_LARGE, CE_MIDDLE, CE_FLAT, CE_SMALL };

// Everything a call lays out, the same for the size and the call.
struct CePlan {
    int64_t rows, classes; int width, padded, parts;
    bool backward, split;
    int logits, grads;                              // shapes
    int lm, ln, gm, gn, slab_l, slab_g;             // their tiles and slabs
    int64_t tm, tn;                                 // row and class tiles of all classes
    int64_t piece, d_rows;                          // classes of a piece, rows of d
    int dx_splits, dw_splits;
    // bytes of the workspace
    int64_t x_at, w_at, kept_at, max_at, sum_at, total_at, z_at, d_at, dx_at, dw_at, db_at, bytes;
};

static int64_t part_of(int64_t n) { return (n + 63) / 64 * 64; }      // elements from one part of a sum to the next
static int64_t take(int64_t &at, int64_t bytes)
{
    const int64_t here = at;
    at += (bytes + 255) / 256 * 256;
    return here;
}
template <class S> static void use(int &m, int &n, int &slab) { m = S::ROWS, n = S::COLS, slab = S::SLAB; }

// When `slots` workers are done with n1 jobs of l1 and then n2 of l2, each taken by whoever is free first.
static int64_t makespan(int64_t slots, int64_t n1, int64_t l1, int64_t n2, int64_t l2)
{
    int64_t at[8] = {0}, count[8] = {slots};        // workers by the time they are free, soonest first
    int groups = 1;
    auto work = [&](int64_t n, int64_t l) {
        while (n > 0) {
            const int64_t now = n < count[0] ? n : count[0], t = at[0] + l;
            n -= now;
            count[0] -= now;
            int from = 0;
            if (count[0] == 0) from = 1;            // the group is gone; else it stays (and n is 0)
            int to = groups;
            while (to > from && at[to - 1] > t) at[to] = at[to - 1], count[to] = count[to - 1], to--;
            at[to] = t, count[to] = now;
            groups++;
            if (from == 1) {
                for (int g = 1; g < groups; g++) at[g - 1] = at[g], count[g - 1] = count[g];
                groups--;
            }
        }
    };
    work(n1, l1);                                   // (a group is split only by the last jobs of a kind: four at most)
    work(n2, l2);
    return at[groups - 1];
}

// Shape and cuts of both gradients of a piece.  Large tiles where their work is 16 slabs for each compute unit; then the tiles and as
// many parts of each sum as end first: a compute unit takes one tile after the other, a tile as long as its slabs (measured in long
// products) and an epilogue, and parts are written and read again at 4 TB/s.  us of a backward call, uncut / as chosen: bf16 2999 x
// 768 x 21841 555 / 360, 300 x 768 x 21841 389 / 83, 8192 x 384 x 1000 116 / 82; fp32 2048 x 384 x 21841 1715 / 640, 128 x 768 x
// 21841 1338 / 166.
struct GradShape {
    int grads, m, n, slab;
    double us, tile_us;                             // of a slab, of an epilogue
};
static double cuts(CePlan &p, const GradShape &s, int64_t of_piece, bool choose)
{
    const int64_t cu = compute_units(), across = ceil_div(p.width, s.n);
    const int64_t tx = ceil_div(p.rows, s.m) * across, tw = ceil_div(of_piece, s.m) * across, sx = ceil_div(of_piece, s.slab), sw = ceil_div(p.rows, s.slab);
    const int64_t extra = (int64_t)(s.tile_us / s.us + 0.5);
    double best = 1e30;
    for (int64_t x = 1; x <= 32 && (x == 1 || sx / x >= 8); x++)
        for (int64_t w = 1; w <= 32 && (w == 1 || sw / w >= 8); w++) {
            if ((x > 1 && tx * x > 8 * cu) || (w > 1 && tw * w > 8 * cu)) continue;
            const double bytes = ((x > 1 ? 8.0 * x * p.rows : 0.0) + (w > 1 ? 8.0 * w * of_piece : 0.0)) * p.width;
            const double t = s.us * makespan(cu, tx * x, ceil_div(sx, x) + extra, tw * w, ceil_div(sw, w) + extra) + bytes / 4e6 + (x > 1 || w > 1 ? 5.0 : 0.0);
            if (t >= best) continue;
            best = t;
            if (choose) p.dx_splits = (int)x, p.dw_splits = (int)w;
        }
    if (choose) p.grads = s.grads, p.gm = s.m, p.gn = s.n, p.slab_g = s.slab;
    return best;
}
template <class S> static GradShape grad_shape(int grads, double us, double tile_us) { return GradShape{grads, S::ROWS, S::COLS, S::SLAB, us, tile_us}; }

static void plan_gradients(CePlan &p, int64_t of_piece)
{
    const GradShape large = p.split ? grad_shape<SplitLarge>(CE_LARGE, 3.0, 12.0) : grad_shape<GradLarge>(CE_LARGE, 2.0, 6.0);
    const GradShape middle = grad_shape<GradMiddle>(CE_MIDDLE, 1.3, 4.0);
    const GradShape small = p.split ? grad_shape<SplitGradSmall>(CE_SMALL, 0.6, 2.4) : grad_shape<GradSmall>(CE_SMALL, 0.35, 1.4);
    // slabs of 32 of 256 x 128 tiles
    const int64_t work = ceil_div(p.width, 128) * (ceil_div(p.rows, 256) * ceil_div(of_piece, 32) + ceil_div(of_piece, 256) * ceil_div(p.rows, 32));
    if (work < 16 * compute_units() * (p.split ? 1 : 2)) cuts(p, small, of_piece, true);
    else if (p.split || cuts(p, large, of_piece, false) <= cuts(p, middle, of_piece, false)) cuts(p, large, of_piece, true);
    else cuts(p, middle, of_piece, true);
}

// us of the tiles of the logits: rounds of large tiles, the last perhaps of halves, or of middle ones two on a compute unit, a last one of
// which may have it alone
static bool large_logits(int64_t rows, int64_t classes, int padded)
{
    const int64_t cu = compute_units(), slabs = padded / 64;
    const int64_t large = ceil_div(rows, LogitsLarge::ROWS) * ceil_div(classes, LogitsLarge::COLS);
    const int64_t middle = ceil_div(rows, LogitsMiddle::ROWS) * ceil_div(classes, LogitsMiddle::COLS), rest = middle % (2 * cu);
    const double t = (double)(middle / (2 * cu)) + (rest == 0 ? 0.0 : rest <= cu ? 0.6 : 1.0);
    const double rounds = (double)(large / cu) + (large % cu == 0 ? 0.0 : large > cu && 2 * (large % cu) <= cu ? 0.7 : 1.0);
    return rounds * (1.57 * slabs + 6.0) <= t * (1.98 * slabs + 3.5);
}

// Logits of fp32 operands stay for the gradients where they are no more than 256 MB: six products of parts cost more than their way to
// memory and back (2048 x 384 x 21841, 179 MB: d 70 us from them and 246 from products, 35 us more for the forward call's writing;
// 2000 x 64 x 20000 64 and 79, 22 more).  bf16: one product, which costs as
// much (2999 x 768 x 21841, 262 MB: tiles 145 us and 190 with the writing, d 150 and 77; a call 460 and 464).
static int64_t z_pitch(int64_t classes) { return (classes + 7) / 8 * 8; }
static bool keeps_logits(int64_t rows, int64_t classes, int dtype) { return dtype == VTDGE_F32 && rows * z_pitch(classes) * 4 <= CE_KEPT_BYTES; }

// (x_lies, w_lies: read where they lie, see lies_well; the gradients want room for x with zeros all the same.  keeps: of a forward
// call, room for the logits too; of the gradients, what it laid out is at hand and needs no room)
static CePlan plan_of(int64_t rows, int64_t classes, int width, int dtype, bool backward, bool x_lies, bool w_lies, bool keeps)
{
    CePlan p{};
    p.rows = rows, p.classes = classes, p.width = width, p.backward = backward;
    p.padded = (int)ceil_div(width, CE_PAD) * CE_PAD;
    p.split = dtype == VTDGE_F32;
    p.parts = p.split ? 3 : 1;
    const int cu = compute_units();
    const int64_t tiles = p.split ? ceil_div(rows, SplitLarge::ROWS) * ceil_div(classes, SplitLarge::COLS)
                                  : ceil_div(rows, LogitsMiddle::ROWS) * ceil_div(classes, LogitsMiddle::COLS);
    p.logits = rows <= 64 && classes >= 64 * cu ? CE_FLAT : tiles < cu ? CE_SMALL : p.split || large_logits(rows, classes, p.padded) ? CE_LARGE : CE_MIDDLE;
    auto shape = [&](auto large, auto middle, auto flat, auto small) {
        if (p.logits == CE_LARGE) use<decltype(large)>(p.lm, p.ln, p.slab_l);
        else if (p.logits == CE_MIDDLE) use<decltype(middle)>(p.lm, p.ln, p.slab_l);
        else if (p.logits == CE_FLAT) use<decltype(flat)>(p.lm, p.ln, p.slab_l);
        else use<decltype(small)>(p.lm, p.ln, p.slab_l);
    };
    if (p.split) shape(SplitLarge{}, SplitLarge{}, SplitFlat{}, SplitSmall{});
    else shape(LogitsLarge{}, LogitsMiddle{}, LogitsFlat{}, LogitsSmall{});
    p.tm = ceil_div(rows, p.lm), p.tn = ceil_div(classes, p.ln);
    int64_t at = 0;
    const bool at_hand = backward && keeps;
    p.x_at = take(at, (x_lies && !backward) || (!x_lies && at_hand) ? 0 : rows * p.padded * 2 * p.parts);
    p.w_at = take(at, w_lies || at_hand ? 0 : classes * p.padded * 2 * p.parts);
    p.kept_at = take(at, !backward && keeps && keeps_logits(rows, classes, dtype) ? rows * z_pitch(classes) * 4 : 0);
    if (!backward) {
        p.max_at = take(at, p.tn * rows * 4);
        p.sum_at = take(at, p.tn * rows * 4);
        p.total_at = take(at, p.tn * rows * 4);
        p.z_at = take(at, rows * 4);
    } else {
        p.d_rows = ceil_div(rows, 256) * 256;
        int64_t piece = CE_PIECE_BYTES / (p.d_rows * 2 * p.parts) / 256 * 256;
        if (piece < 1024) piece = 1024;
        const int64_t pieces = ceil_div(classes, piece);                      // of equal size
        p.piece = ceil_div(ceil_div(classes, pieces), 256) * 256;
        const int64_t of_piece = p.piece < classes ? p.piece : classes;
        plan_gradients(p, p.piece < classes ? p.piece : classes);
        p.d_at = take(at, p.d_rows * p.piece * 2 * p.parts);
        p.dx_at = take(at, part_of(rows * width) * 4 * p.dx_splits);
        p.dw_at = take(at, part_of(p.piece * width) * 4 * p.dw_splits);
        p.db_at = take(at, part_of(p.piece) * 4 * p.dw_splits);
    }
    p.bytes = at;
    return p;
}

static int check_sizes(const char *what, int64_t rows, int64_t classes, int width, int dtype)
{
    VT_REQUIRE(dtype == VTDGE_F32 || dtype == VTDGE_BF16, VTDGE_ERR_ARG, "%s: dtype %d", what, dtype);
    VT_REQUIRE(rows > 0 && classes > 0 && width > 0, VTDGE_ERR_ARG, "%s: %lld rows, %lld classes of %d", what, (long long)rows, (long long)classes, width);
    VT_REQUIRE(rows < (1 << 24) && classes < (1 << 24) && width <= (1 << 16) && rows * (int64_t)width < (1ll << 31) &&
                   classes * (int64_t)width < (1ll << 31) && ceil_div(rows, 64) * ceil_div(classes, 64) < (1 << 23),
               VTDGE_ERR_UNSUPPORTED, "%s: %lld rows, %lld classes of %d", what, (long long)rows, (long long)classes, width);
    return VTDGE_OK;
}

#define VT_STEP(call)                        \
    do {                                     \
        const int vt_rc = (call);            \
        if (vt_rc != VTDGE_OK) return vt_rc; \
    } while (0)

// whether the product routine can read an operand where it lies
static bool lies_well(const void *src, int64_t ld, int width, int dtype)
{
    return dtype == VTDGE_BF16 && width % CE_PAD == 0 && ld % 8 == 0 && ld < (1 << 22) && ((uintptr_t)src & 15) == 0;
}
static bool lies_well(const void *src, int64_t ld, const CePlan &p) { return lies_well(src, ld, p.width, p.split ? VTDGE_F32 : VTDGE_BF16); }
// x and W as they lie, else packed in the workspace; rows of x that are left out as zeros there
static int operands_of(CeArgs &a, const void *x, int64_t ldx, const void *w, int64_t ldw, const CePlan &p, unsigned char *ws, hipStream_t st)
{
    PackArgs g{};
    int n = 0;
    int64_t blocks = 0;
    auto take = [&](Operand &o, const void *src, int64_t ld, int64_t rows, const int64_t *target, int64_t at) {
        if (lies_well(src, ld, p)) {
            o = Operand{(const bf16_t *)src, ld, 0};
            return;
        }
        bf16_t *const to = (bf16_t *)(ws + at);
        o = Operand{to, p.padded, rows * p.padded};
        g.job[n++] = PackJob{src, ld, rows, target, to};
        blocks += ceil_div(rows * (p.padded / 8), 256);
        if (n == 1) g.first = blocks;
    };
    take(a.x, x, ldx, p.rows, a.target, p.x_at);
    take(a.w, w, ldw, p.classes, nullptr, p.w_at);
    if (n == 0) return VTDGE_OK;
    g.width = p.width, g.padded = p.padded, g.ignore = a.ignore, g.classes = p.classes;
    VT_REQUIRE(blocks < (1 << 24), VTDGE_ERR_UNSUPPORTED, "cross_entropy: %lld blocks to lay out", (long long)blocks);
    auto kern = p.split ? cross_entropy_pack_kernel<float> : cross_entropy_pack_kernel<bf16_t>;
    note_kernel(reinterpret_cast<const void *>(kern));
    kern<<<(unsigned)blocks, 256, 0, st>>>(g);
    return check_launch("cross_entropy");
}

// Tiles of a launch that stay whole: where each has a compute unit to itself and the last round would be half empty or more, its tiles are
// cut in two (2999 x 768 x 21841, 1032 tiles on 256 compute units: loss and gradients 497 us without, 485 so).
template <class S> static int halved(int64_t tiles)
{
    const int64_t cu = compute_units(), rest = tiles % cu;
    return (int)(S::HALVES && tiles > cu && 2 * rest <= cu ? tiles - rest : tiles);
}
template <class S> static int go_tiles(const CeArgs &a, const CePlan &p, hipStream_t st)
{
    auto kern = a.smoothing != 0.f ? cross_entropy_tiles_kernel<S, true> : cross_entropy_tiles_kernel<S, false>;
    VT_RESERVE_LDS((cross_entropy_tiles_kernel<S, true>), S::LDS, "cross_entropy");
    VT_RESERVE_LDS((cross_entropy_tiles_kernel<S, false>), S::LDS, "cross_entropy");
    note_kernel(reinterpret_cast<const void *>(kern));
    const int whole = halved<S>(p.tm * p.tn);
    kern<<<(unsigned)(2 * p.tm * p.tn - whole), S::THREADS, S::LDS, st>>>(a, (int)p.tm, (int)p.tn, whole);
    return check_launch("cross_entropy");
}
template <class S> static int go_d(const CeArgs &a, const CePlan &p, hipStream_t st)
{
    auto kern = cross_entropy_d_kernel<S>;
    VT_RESERVE_LDS(kern, S::LDS, "cross_entropy_backward");
    note_kernel(reinterpret_cast<const void *>(kern));
    const int tn = (int)ceil_div(a.v1 - a.v0, S::COLS);
    const int whole = halved<S>(p.tm * tn);
    kern<<<(unsigned)(2 * p.tm * tn - whole), S::THREADS, S::LDS, st>>>(a, (int)p.tm, tn, whole);
    return check_launch("cross_entropy_backward");
}
static int go_d_kept(const CeArgs &a, hipStream_t st)
{
    // slabs run over the classes of a piece and the rows behind the last, 64 at most
    const int64_t vecs = ceil_div(a.v1 - a.v0, 256) * 32, rows = ceil_div(a.rows, CE_PAD) * CE_PAD, blocks = ceil_div(rows * vecs, 256);
    VT_REQUIRE(blocks < (1 << 24) && vecs * 8 <= a.d_pitch, VTDGE_ERR_UNSUPPORTED, "cross_entropy_backward: d of %lld blocks", (long long)blocks);
    note_kernel(reinterpret_cast<const void *>(cross_entropy_d_kept_kernel));
    cross_entropy_d_kept_kernel<<<(unsigned)blocks, 256, 0, st>>>(a, (int)vecs, rows);
    return check_launch("cross_entropy_backward");
}
template <class S> static int go_grad(GradPair &g, hipStream_t st)
{
    int64_t blocks = 0;
    for (GradArgs *a : {&g.dx, &g.dw}) {
        const bool along = a == &g.dx;
        if (!along) g.first_dw = (int)blocks;
        if (a->rows == 0) continue;
        a->tm = (int)ceil_div(a->rows, S::ROWS), a->tn = (int)ceil_div(a->cols, S::COLS);
        if (a->out == nullptr && a->part == nullptr) a->tn = 1;                // the sums alone
        VT_REQUIRE(a->stages <= ceil_div(a->sum_b, S::SLAB) && (along || a->stages <= ceil_div(a->sum_a, S::SLAB)) && a->splits >= 1 && a->splits <= a->stages,
                   VTDGE_ERR_ARG, "cross_entropy_backward: %d stages over %lld rows in %d parts", a->stages, (long long)a->sum_b, a->splits);
        blocks += (int64_t)a->tm * a->tn * a->splits;
    }
    VT_REQUIRE(blocks < (1 << 23), VTDGE_ERR_UNSUPPORTED, "cross_entropy_backward: %lld tiles", (long long)blocks);
    if (blocks == 0) return VTDGE_OK;
    auto kern = cross_entropy_grad_kernel<S>;
    VT_RESERVE_LDS(kern, S::LDS, "cross_entropy_backward");
    note_kernel(reinterpret_cast<const void *>(kern));
    kern<<<(unsigned)blocks, S::THREADS, S::LDS, st>>>(g);
    return check_launch("cross_entropy_backward");
}

static int sum_up(const SumJob *jobs, int count, const float *scale, const float *scale2, bool f32, hipStream_t st)
{
    SumArgs a{};
    int n = 0;
    for (int i = 0; i < count; i++) {
        if (jobs[i].out == nullptr || jobs[i].part == nullptr) continue;
        a.job[n] = jobs[i];
        a.first[n + 1] = a.first[n] + ceil_div(jobs[i].n, 1024);
        n++;
    }
    if (n == 0) return VTDGE_OK;
    const int64_t blocks = a.first[n];
    for (int i = n; i < 3; i++) a.first[i + 1] = blocks;
    VT_REQUIRE(blocks < (1 << 24), VTDGE_ERR_UNSUPPORTED, "cross_entropy_backward: a gradient of %lld blocks", (long long)blocks);
    a.scale = scale, a.scale2 = scale2, a.f32 = f32;
    note_kernel(reinterpret_cast<const void *>(cross_entropy_sum_kernel));
    cross_entropy_sum_kernel<<<(unsigned)blocks, 256, 0, st>>>(a);
    return check_launch("cross_entropy_backward");
}

}  // namespace vtdge

using namespace vtdge;

extern "C" int64_t vtdge_cross_entropy_laid_out(int64_t rows, int64_t classes, int width, int dtype)
{
    if (check_sizes("cross_entropy_laid_out", rows, classes, width, dtype) != VTDGE_OK) return -1;
    return plan_of(rows, classes, width, dtype, false, false, false, true).max_at;
}

extern "C" int64_t vtdge_cross_entropy_workspace(int64_t rows, int64_t classes, int width, int dtype, int how)
{
    if (check_sizes("cross_entropy_workspace", rows, classes, width, dtype) != VTDGE_OK) return -1;
    return plan_of(rows, classes, width, dtype, how & VTDGE_CE_BACKWARD, how & VTDGE_CE_X_LIES, how & VTDGE_CE_WEIGHT_LIES, how & VTDGE_CE_KEEPS).bytes;
}

extern "C" int vtdge_cross_entropy(const void *x, int64_t ldx, const void *weight, int64_t ldw, const void *bias, const int64_t *target,
                                   int64_t rows, int64_t classes, int width, int64_t ignore_index, float smoothing, void *workspace,
                                   int64_t workspace_bytes, int keeps, float *loss_rows, float *row_max, float *row_inv, float *loss,
                                   float *inv_count, int dtype, void *stream)
{
    VT_STEP(check_sizes("cross_entropy", rows, classes, width, dtype));
    VT_REQUIRE(x && weight && target && loss_rows && row_max && row_inv && workspace, VTDGE_ERR_ARG, "cross_entropy: NULL operand");
    VT_REQUIRE(loss != nullptr || inv_count == nullptr, VTDGE_ERR_ARG, "cross_entropy: inv_count without loss");
    VT_REQUIRE(ldx >= width && ldw >= width, VTDGE_ERR_ARG, "cross_entropy: rows of %d, %lld and %lld apart", width, (long long)ldx, (long long)ldw);
    VT_REQUIRE(smoothing >= 0.f && smoothing <= 1.f, VTDGE_ERR_ARG, "cross_entropy: smoothing %g", (double)smoothing);
    const CePlan p = plan_of(rows, classes, width, dtype, false, lies_well(x, ldx, width, dtype), lies_well(weight, ldw, width, dtype), keeps != 0);
    VT_REQUIRE(workspace_bytes >= p.bytes && ((uintptr_t)workspace & 255) == 0, VTDGE_ERR_ARG, "cross_entropy: workspace of %lld bytes, %lld needed",
               (long long)workspace_bytes, (long long)p.bytes);
    unsigned char *const ws = (unsigned char *)workspace;
    const hipStream_t st = (hipStream_t)stream;
    CeArgs a{};
    a.target = target, a.ignore = ignore_index;
    VT_STEP(operands_of(a, x, ldx, weight, ldw, p, ws, st));
    a.bias = bias, a.bias_f32 = p.split, a.rows = rows, a.classes = classes;
    a.smoothing = smoothing, a.stages = (int)ceil_div(p.padded, p.slab_l), a.v0 = 0, a.v1 = classes;
    a.tile_max = (float *)(ws + p.max_at), a.tile_sum = (float *)(ws + p.sum_at), a.tile_total = (float *)(ws + p.total_at);
    a.target_z = (float *)(ws + p.z_at);
    if (keeps != 0 && keeps_logits(rows, classes, dtype)) a.z = (float *)(ws + p.kept_at), a.z_pitch = z_pitch(classes);
    // W is read once where it lies.  From a quarter of the last cache's 256 MB on, what a program does between two calls leaves little of
    // it there (1 x 1024 x 65536, 134 MB: out of memory 27.4 us through the caches, 24.7 past them; still in the cache 25.5 and 27.1)
    a.stream_w = p.logits == CE_FLAT && a.w.p == weight && classes * p.padded * 2 >= (64 << 20);
    if (p.split) VT_STEP(p.logits == CE_LARGE ? go_tiles<SplitLarge>(a, p, st) : p.logits == CE_FLAT ? go_tiles<SplitFlat>(a, p, st) : go_tiles<SplitSmall>(a, p, st));
    else VT_STEP(p.logits == CE_LARGE ? go_tiles<LogitsLarge>(a, p, st) : p.logits == CE_MIDDLE ? go_tiles<LogitsMiddle>(a, p, st) : p.logits == CE_FLAT ? go_tiles<LogitsFlat>(a, p, st) : go_tiles<LogitsSmall>(a, p, st));
    const JoinArgs j{a.tile_max, a.tile_sum, a.tile_total, a.target_z, target, rows, classes, ignore_index, smoothing, (int)p.tn,
                     loss_rows, row_max, row_inv, loss, inv_count};
    // one workgroup is done with some 20000 values before a second launch would have begun (by sizes alone: the same bits for each reduction)
    if (rows <= 2048 && rows * p.tn <= 20480 && p.tn <= 32) {
        note_kernel(reinterpret_cast<const void *>(cross_entropy_join_mean_kernel));
        cross_entropy_join_mean_kernel<<<1, 64 * JOIN_WAVES, 0, st>>>(j);
        return check_launch("cross_entropy");
    }
    auto join = rows <= 256 && p.tn > 128 ? cross_entropy_join_row_kernel : cross_entropy_join_kernel;
    note_kernel(reinterpret_cast<const void *>(join));
    join<<<(unsigned)(join == cross_entropy_join_kernel ? ceil_div(rows, 64) : rows), 64 * JOIN_WAVES, 0, st>>>(j);
    VT_STEP(check_launch("cross_entropy"));
    if (loss == nullptr) return VTDGE_OK;
    note_kernel(reinterpret_cast<const void *>(cross_entropy_mean_kernel));
    cross_entropy_mean_kernel<<<1, 64 * JOIN_WAVES, 0, st>>>(j);
    return check_launch("cross_entropy");
}

extern "C" int vtdge_cross_entropy_backward(const void *x, int64_t ldx, const void *weight, int64_t ldw, const void *bias, const int64_t *target,
                                            const float *row_max, const float *row_inv, const float *grad, int grad_stride,
                                            const float *inv_count, int64_t rows, int64_t classes, int width, int64_t ignore_index,
                                            float smoothing, const void *laid_out, void *workspace, int64_t workspace_bytes, void *dx,
                                            void *dweight, void *dbias, int dtype, void *stream)
{
    VT_STEP(check_sizes("cross_entropy_backward", rows, classes, width, dtype));
    VT_REQUIRE(x && weight && target && row_max && row_inv && grad && workspace, VTDGE_ERR_ARG, "cross_entropy_backward: NULL operand");
    VT_REQUIRE(ldx >= width && ldw >= width, VTDGE_ERR_ARG, "cross_entropy_backward: rows of %d, %lld and %lld apart", width, (long long)ldx, (long long)ldw);
    VT_REQUIRE(((uintptr_t)laid_out & 255) == 0, VTDGE_ERR_ARG, "cross_entropy_backward: laid_out off its boundary");
    VT_REQUIRE(grad_stride == 0 || (grad_stride == 1 && inv_count == nullptr), VTDGE_ERR_ARG, "cross_entropy_backward: grad_stride %d", grad_stride);
    VT_REQUIRE(smoothing >= 0.f && smoothing <= 1.f, VTDGE_ERR_ARG, "cross_entropy_backward: smoothing %g", (double)smoothing);
    const bool x_lies = lies_well(x, ldx, width, dtype), w_lies = lies_well(weight, ldw, width, dtype);
    const CePlan p = plan_of(rows, classes, width, dtype, true, x_lies, w_lies, laid_out != nullptr);
    VT_REQUIRE(workspace_bytes >= p.bytes && ((uintptr_t)workspace & 255) == 0, VTDGE_ERR_ARG,
               "cross_entropy_backward: workspace of %lld bytes, %lld needed", (long long)workspace_bytes, (long long)p.bytes);
    if (dx == nullptr && dweight == nullptr && dbias == nullptr) return VTDGE_OK;
    unsigned char *const ws = (unsigned char *)workspace;
    const hipStream_t st = (hipStream_t)stream;
    CeArgs a{};
    a.target = target, a.ignore = ignore_index;
    if (laid_out != nullptr) {
        // as the forward call left them
        unsigned char *const from = (unsigned char *)const_cast<void *>(laid_out);
        const CePlan f = plan_of(rows, classes, width, dtype, false, x_lies, w_lies, true);
        if (keeps_logits(rows, classes, dtype)) a.z = (float *)(from + f.kept_at), a.z_pitch = z_pitch(classes);
        a.x = x_lies ? Operand{(const bf16_t *)x, ldx, 0} : Operand{(const bf16_t *)(from + f.x_at), p.padded, rows * p.padded};
        a.w = w_lies ? Operand{(const bf16_t *)weight, ldw, 0} : Operand{(const bf16_t *)(from + f.w_at), p.padded, classes * p.padded};
    } else {
        VT_STEP(operands_of(a, x, ldx, weight, ldw, p, ws, st));
    }
    Operand clean = a.x;                            // x with zeros for the rows that are left out, so that what they hold reaches no gradient
    const bool copy = x_lies && (dweight != nullptr || dbias != nullptr);
    if (copy) clean = Operand{(const bf16_t *)(ws + p.x_at), p.padded, 0};
    a.bias = bias, a.bias_f32 = p.split, a.rows = rows, a.classes = classes;
    a.smoothing = smoothing, a.stages = (int)ceil_div(p.padded, p.slab_l), a.width = p.padded;
    a.row_max = row_max, a.row_inv = row_inv, a.row_scale = grad_stride == 1 ? grad : nullptr;
    a.d = (bf16_t *)(ws + p.d_at), a.d_pitch = p.piece, a.d_plane = p.d_rows * p.piece;
    const float *const scale = grad_stride == 1 ? nullptr : grad;
    const bool one_piece = p.piece >= classes;
    float *const dx_part = one_piece && p.dx_splits == 1 ? nullptr : (float *)(ws + p.dx_at);
    float *const dw_part = p.dw_splits == 1 ? nullptr : (float *)(ws + p.dw_at), *const db_part = p.dw_splits == 1 ? nullptr : (float *)(ws + p.db_at);
    const int64_t elem = p.split ? 4 : 2;
    for (int64_t v0 = 0; v0 < classes; v0 += p.piece) {
        a.v0 = v0, a.v1 = v0 + p.piece < classes ? v0 + p.piece : classes;
        a.x_copy = copy && v0 == 0 ? (bf16_t *)(ws + p.x_at) : nullptr;
        const int64_t live = a.v1 - a.v0;
        if (a.z != nullptr) VT_STEP(go_d_kept(a, st));
        else if (p.split) VT_STEP(p.logits == CE_LARGE ? go_d<SplitLarge>(a, p, st) : p.logits == CE_FLAT ? go_d<SplitFlat>(a, p, st) : go_d<SplitSmall>(a, p, st));
        else VT_STEP(p.logits == CE_LARGE ? go_d<LogitsLarge>(a, p, st) : p.logits == CE_MIDDLE ? go_d<LogitsMiddle>(a, p, st) : p.logits == CE_FLAT ? go_d<LogitsFlat>(a, p, st) : go_d<LogitsSmall>(a, p, st));
        GradPair g{};
        g.scale = scale, g.scale2 = inv_count, g.f32 = p.split;
        if (dx != nullptr) {
            g.dx.a = Operand{a.d, a.d_pitch, a.d_plane}, g.dx.b = Operand{a.w.p + v0 * a.w.pitch, a.w.pitch, a.w.plane};
            g.dx.rows = rows, g.dx.cols = width, g.dx.sum_b = live, g.dx.span_b = p.padded;
            g.dx.stages = (int)ceil_div(live, p.slab_g), g.dx.splits = p.dx_splits < g.dx.stages ? p.dx_splits : g.dx.stages;
            g.dx.part = dx_part, g.dx.part_stride = part_of(rows * width), g.dx.accumulate = v0 > 0, g.dx.out = dx;
        }
        if (dweight != nullptr || dbias != nullptr) {
            g.dw.a = Operand{a.d, a.d_pitch, a.d_plane}, g.dw.b = clean;
            g.dw.rows = live, g.dw.cols = width, g.dw.sum_a = p.d_rows, g.dw.span_a = p.piece, g.dw.sum_b = rows, g.dw.span_b = p.padded;
            g.dw.stages = (int)ceil_div(rows, p.slab_g), g.dw.splits = p.dw_splits;
            g.dw.part = dweight != nullptr ? dw_part : nullptr, g.dw.part_stride = part_of(p.piece * width);
            g.dw.out = dweight != nullptr ? (unsigned char *)dweight + v0 * width * elem : nullptr;
            g.dw.sums_part = dbias != nullptr ? db_part : nullptr, g.dw.sums_stride = part_of(p.piece);
            g.dw.sums = dbias != nullptr ? (unsigned char *)dbias + v0 * elem : nullptr;
        }
        if (p.split) VT_STEP(p.grads == CE_LARGE ? go_grad<SplitLarge>(g, st) : go_grad<SplitGradSmall>(g, st));
        else VT_STEP(p.grads == CE_LARGE ? go_grad<GradLarge>(g, st) : p.grads == CE_MIDDLE ? go_grad<GradMiddle>(g, st) : go_grad<GradSmall>(g, st));
        // parts of this piece's dW and db, and of dx behind the last piece
        const bool last = a.v1 == classes;
        const SumJob jobs[3] = {{dx_part, last ? dx : nullptr, rows * width, part_of(rows * width), p.dx_splits},
                                {g.dw.part, g.dw.out, live * width, g.dw.part_stride, p.dw_splits},
                                {g.dw.sums_part, g.dw.sums, live, g.dw.sums_stride, p.dw_splits}};
        VT_STEP(sum_up(jobs, 3, scale, inv_count, p.split, st));
    }
    return VTDGE_OK;
}
