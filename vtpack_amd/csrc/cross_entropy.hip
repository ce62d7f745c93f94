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
#include "gradient_product.h"

namespace vtdge {

constexpr float LOG2E = 1.44269504f, LN2 = 0.69314718f;
// What the first bf16 part of an fp32 value is rounded from: the largest finite numbers would become infinite, and are cut to bf16's
// largest; the next part has the rest.  (Infinity and NaN go on to the next part.)
constexpr float BF16_MOST = 0x1.fep127f;
__device__ __forceinline__ float first_part(float f) { return __builtin_amdgcn_fmed3f(f, -BF16_MOST, BF16_MOST); }

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
using SplitLarge = Shape<2, 2, 4, 2, 32, 2, 3>;
using SplitFlat = Shape<1, 2, 2, 2, 32, 3, 3>;
using SplitSmall = Shape<1, 1, 2, 2, 32, 4, 3>;

constexpr int CE_PAD = 64;                          // rows of operands are filled up to whole slabs of any shape
constexpr int64_t CE_PIECE_BYTES = 320ll << 20;     // of d
constexpr int64_t CE_KEPT_BYTES = 256ll << 20;      // of logits
enum { CE_LARGE, CE_MIDDLE, CE_FLAT, CE_SMALL };

// Everything a call lays out, the same for the size and the call.
struct CePlan : GradPlan {
    int64_t rows, classes; int width, padded, parts;
    bool backward, split;
    int logits;                                     // shape
    int lm, ln, slab_l;                             // its tile and slab
    int64_t tm, tn;                                 // row and class tiles of all classes
    int64_t piece, d_rows;                          // classes of a piece, rows of d
    // bytes of the workspace
    int64_t x_at, w_at, kept_at, max_at, sum_at, total_at, z_at, d_at, dx_at, dw_at, db_at, bytes;
};

static int64_t take(int64_t &at, int64_t bytes)
{
    const int64_t here = at;
    at += (bytes + 255) / 256 * 256;
    return here;
}
template <class S> static void use(int &m, int &n, int &slab) { m = S::ROWS, n = S::COLS, slab = S::SLAB; }

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
        plan_gradients(p, rows, of_piece, width, p.split, false);
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
        g.scale = scale, g.scale2 = inv_count, g.f32 = p.split, g.f32_parts = p.split;
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
        VT_STEP(launch_gradients(p, g, "cross_entropy_backward", st));
        // parts of this piece's dW and db, and of dx behind the last piece
        const bool last = a.v1 == classes;
        const SumJob jobs[3] = {{dx_part, last ? dx : nullptr, rows * width, part_of(rows * width), p.dx_splits},
                                {g.dw.part, g.dw.out, live * width, g.dw.part_stride, p.dw_splits},
                                {g.dw.sums_part, g.dw.sums, live, g.dw.sums_stride, p.dw_splits}};
        VT_STEP(sum_parts(jobs, 3, scale, inv_count, p.split, "cross_entropy_backward", st));
    }
    return VTDGE_OK;
}
