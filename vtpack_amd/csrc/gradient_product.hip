// The products of a backward pass, see gradient_product.h (gfx950).  Bound by the matrix units in long sums (bf16 8192 rows x 65536 classes x
// 1024: 1.06 PFLOP/s), by launches and the parts' way to memory and back in short ones.
#include "gradient_product.h"

namespace vtdge {

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
template <class S, bool A_ALONG, bool ENDS> __device__ __forceinline__ void gradient_tile(const GradArgs &p, const GradPair &all, int id, unsigned char *smem)
{
    constexpr int IM = S::IM, JN = S::JN;
    int m, n;
    const int z = tile_of(id, p.splits, p.tm, p.tn, m, n);
    const int64_t r0 = (int64_t)m * S::ROWS, c0 = (int64_t)n * S::COLS;
    const int t0 = (int)((int64_t)p.stages * z / p.splits), t1 = (int)((int64_t)p.stages * (z + 1) / p.splits);
    f32x16 acc[IM][JN] = {};
    float sums[IM] = {};
    const Loader<A_ALONG, S::ROWS, S::SLAB, S::WAVES> a(p.a, r0, A_ALONG ? p.rows : p.sum_a, p.span_a);
    const Loader<ENDS, S::COLS, S::SLAB, S::WAVES> b(p.b, c0, ENDS ? p.cols : p.sum_b, p.span_b);
    const int lane = threadIdx.x & 63, lr = lane & 31, lg = lane >> 5;
    const int wid = wave_uniform(threadIdx.x >> 6), wm = wid / S::WN, wn = wid % S::WN;
    const bool with_sums = !A_ALONG && n == 0 && wn == 0 && (p.sums_part != nullptr || p.sums != nullptr);
    float scale = 1.f;
    if (all.scale != nullptr) scale = *all.scale;
    if (all.scale2 != nullptr) scale *= *all.scale2;
    multiply_tile<S, !A_ALONG, ENDS && !A_ALONG>(a, b, t0, t1, smem, acc, with_sums, sums, (int)p.sum_a);
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
        if (ENDS || S::WHOLE_LINES || r >= p.rows) continue;
#pragma unroll
        for (int j = 0; j < JN; j++)
#pragma unroll
            for (int q = 0; q < 4; q++) {
                const f32x4 v = {acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]};
                put_four(p, all, z, r, c0 + (wn * JN + j) * 32 + 8 * q + 4 * lg, v, scale);
            }
    }
    if constexpr (ENDS) {
        auto as_it_is = [](int, int, f32x4 &) {};
        if (p.part != nullptr) put_tile<S>(smem, acc, as_it_is, p.part + z * p.part_stride, p.rows, p.cols, r0, c0, false);
        else if (p.out != nullptr && all.f32) put_tile<S>(smem, acc, as_it_is, static_cast<float *>(p.out), p.rows, p.cols, r0, c0, false);
        else if (p.out != nullptr) put_tile<S>(smem, acc, as_it_is, static_cast<bf16_t *>(p.out), p.rows, p.cols, r0, c0, false);
    } else if constexpr (S::WHOLE_LINES) {
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
template <class S, bool ENDS> __device__ __forceinline__ void gradients(const GradPair &p, unsigned char *smem)
{
    if ((int)blockIdx.x < p.first_dw) gradient_tile<S, true, ENDS>(p.dx, p, blockIdx.x, smem);
    else gradient_tile<S, false, ENDS>(p.dw, p, blockIdx.x - p.first_dw, smem);
}
template <class S> __global__ __launch_bounds__(S::THREADS, S::PER_SIMD) void cross_entropy_grad_kernel(GradPair p)
{
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    gradients<S, false>(p, smem);
}
template <class S> __global__ __launch_bounds__(S::THREADS, S::PER_SIMD) void linear_grad_kernel(GradPair p)
{
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    gradients<S, true>(p, smem);
}

struct SumArgs {
    SumJob job[3];
    int64_t first[4];                               // workgroups
    const float *scale, *scale2; int f32;
};
__global__ __launch_bounds__(256) void gradient_sum_kernel(SumArgs p)
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

// ------------------------------------------------------------------------------------------------ on the host
using GradLarge = Shape<2, 4, 4, 2, 64, 2, 1>;
using GradSquare = Shape<2, 2, 2, 2, 64, 2, 1>;
using GradMiddle = Shape<2, 2, 4, 2, 64, 3, 1>;
// (short sums of many tiles: three on a compute unit, fp32 two, rather than a deep ring for one; bf16 1 row x 363 x 25766 classes 43 -> 22 us,
// 256 x 384 x 1000 10.2 -> 9.7)
using GradSmall = Shape<1, 1, 2, 2, 64, 3, 1>;
using SplitGradLarge = Shape<2, 2, 4, 2, 32, 2, 3>;
using SplitGradSmall = Shape<1, 1, 2, 2, 32, 3, 3>;
enum { GRAD_LARGE, GRAD_MIDDLE, GRAD_SMALL, GRAD_SQUARE };

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
    int per_cu;                                     // tiles side by side on a compute unit, `us` for all of them there
    double us_alone;
};
static double cuts(GradPlan &p, int64_t rows, int64_t of_piece, int width, const GradShape &s, bool choose)
{
    const int64_t cu = compute_units(), across = ceil_div(width, s.n);
    const int64_t tx = ceil_div(rows, s.m) * across, tw = ceil_div(of_piece, s.m) * across, sx = ceil_div(of_piece, s.slab), sw = ceil_div(rows, s.slab);
    double best = 1e30;
    for (int64_t x = 1; x <= 32 && (x == 1 || sx / x >= 8); x++)
        for (int64_t w = 1; w <= 32 && (w == 1 || sw / w >= 8); w++) {
            if ((x > 1 && tx * x > 8 * cu) || (w > 1 && tw * w > 8 * cu)) continue;
            const double bytes = ((x > 1 ? 8.0 * x * rows : 0.0) + (w > 1 ? 8.0 * w * of_piece : 0.0)) * width;
            double us = s.us;
            if (s.per_cu > 1) {                     // few tiles have a compute unit, or more of one, to themselves
                const double beside = (double)(tx * x + tw * w) / (double)cu - 1.0;
                us = s.us_alone + (s.us - s.us_alone) * (beside < 0.0 ? 0.0 : beside > s.per_cu - 1 ? 1.0 : beside / (s.per_cu - 1));
            }
            const int64_t extra = (int64_t)(s.tile_us / us + 0.5);
            const double t = us * makespan(cu * s.per_cu, tx * x, ceil_div(sx, x) + extra, tw * w, ceil_div(sw, w) + extra) + bytes / 4e6 + (x > 1 || w > 1 ? 5.0 : 0.0);
            if (t >= best) continue;
            best = t;
            if (choose) p.dx_splits = (int)x, p.dw_splits = (int)w;
        }
    if (choose) p.grads = s.grads, p.gm = s.m, p.gn = s.n, p.slab_g = s.slab;
    return best;
}
template <class S> static GradShape grad_shape(int grads, double us, double tile_us, int per_cu = 1, double us_alone = 0.0)
{
    return GradShape{grads, S::ROWS, S::COLS, S::SLAB, us, tile_us, per_cu, us_alone};
}

void plan_gradients(GradPlan &p, int64_t rows, int64_t of_piece, int width, bool split, bool ends)
{
    if (ends) {
        // The shape that ends first by the same count.  us of a backward call in bf16 (256 x 256, 128 x 128, 64 x 64), rows x width x outputs: 300
        // x 200 x 130 17.6, 11.9, 10.9; 1021 x 192 x 768 27.3, 19.1, 15.5; 1500 x 3000 x 1000 52, 37.5, 45; 2999 x 777 x 1301 47, 42, 45; 65536 x
        // 384 x 384 110, 84, 93; 8192 x 768 x 768 41.7, 42.1, 48; 6000 x 2000 x 2000 127, 131, 180; 32768 x 1024 x 4096 505, 594, 994.  (256 x
        // 128, one on a compute unit, was first in 5 of 28 sizes, by 8 % at most.)
        const GradShape shapes[3] = {grad_shape<GradLarge>(GRAD_LARGE, 2.0, 5.0), grad_shape<GradSquare>(GRAD_SQUARE, 1.15, 2.0, 2, 0.75),
                                     grad_shape<GradSmall>(GRAD_SMALL, 0.9, 1.0, 3, 0.65)};
        int best = 0;
        double least = 1e30;
        for (int k = 0; k < 3; k++) {
            const double t = cuts(p, rows, of_piece, width, shapes[k], false);
            if (t < least) least = t, best = k;
        }
        cuts(p, rows, of_piece, width, shapes[best], true);
        return;
    }
    const GradShape large = split ? grad_shape<SplitGradLarge>(GRAD_LARGE, 3.0, 12.0) : grad_shape<GradLarge>(GRAD_LARGE, 2.0, 6.0);
    const GradShape middle = grad_shape<GradMiddle>(GRAD_MIDDLE, 1.3, 4.0);
    const GradShape small = split ? grad_shape<SplitGradSmall>(GRAD_SMALL, 0.6, 2.4) : grad_shape<GradSmall>(GRAD_SMALL, 0.35, 1.4);
    // slabs of 32 of 256 x 128 tiles
    const int64_t work = ceil_div(width, 128) * (ceil_div(rows, 256) * ceil_div(of_piece, 32) + ceil_div(of_piece, 256) * ceil_div(rows, 32));
    if (work < 16 * compute_units() * (split ? 1 : 2)) cuts(p, rows, of_piece, width, small, true);
    else if (split || cuts(p, rows, of_piece, width, large, false) <= cuts(p, rows, of_piece, width, middle, false)) cuts(p, rows, of_piece, width, large, true);
    else cuts(p, rows, of_piece, width, middle, true);
}

template <class S, bool ENDS> static int go_grad(GradPair &g, const char *what, hipStream_t st)
{
    int64_t blocks = 0;
    for (GradArgs *a : {&g.dx, &g.dw}) {
        const bool along = a == &g.dx;
        if (!along) g.first_dw = (int)blocks;
        if (a->rows == 0) continue;
        a->tm = (int)ceil_div(a->rows, S::ROWS), a->tn = (int)ceil_div(a->cols, S::COLS);
        if (a->out == nullptr && a->part == nullptr) a->tn = 1;                // the sums alone
        VT_REQUIRE(a->stages <= ceil_div(a->sum_b, S::SLAB) && (along || a->stages <= ceil_div(a->sum_a, S::SLAB)) && a->splits >= 1 && a->splits <= a->stages,
                   VTDGE_ERR_ARG, "%s: %d stages over %lld rows in %d parts", what, a->stages, (long long)a->sum_b, a->splits);
        blocks += (int64_t)a->tm * a->tn * a->splits;
    }
    VT_REQUIRE(blocks < (1 << 23), VTDGE_ERR_UNSUPPORTED, "%s: %lld tiles", what, (long long)blocks);
    if (blocks == 0) return VTDGE_OK;
    void (*kern)(GradPair);
    if constexpr (ENDS) kern = linear_grad_kernel<S>;
    else kern = cross_entropy_grad_kernel<S>;
    VT_RESERVE_LDS(kern, S::LDS, what);
    note_kernel(reinterpret_cast<const void *>(kern));
    kern<<<(unsigned)blocks, S::THREADS, S::LDS, st>>>(g);
    return check_launch(what);
}

int sum_parts(const SumJob *jobs, int count, const float *scale, const float *scale2, bool f32, const char *what, hipStream_t st)
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
    VT_REQUIRE(blocks < (1 << 24), VTDGE_ERR_UNSUPPORTED, "%s: a gradient of %lld blocks", what, (long long)blocks);
    a.scale = scale, a.scale2 = scale2, a.f32 = f32;
    note_kernel(reinterpret_cast<const void *>(gradient_sum_kernel));
    gradient_sum_kernel<<<(unsigned)blocks, 256, 0, st>>>(a);
    return check_launch(what);
}

int launch_gradients(const GradPlan &p, GradPair &g, const char *what, hipStream_t st)
{
    if (g.f32_parts) return p.grads == GRAD_LARGE ? go_grad<SplitGradLarge, false>(g, what, st) : go_grad<SplitGradSmall, false>(g, what, st);
    if (g.ends)
        return p.grads == GRAD_LARGE ? go_grad<GradLarge, true>(g, what, st)
               : p.grads == GRAD_SQUARE ? go_grad<GradSquare, true>(g, what, st) : go_grad<GradSmall, true>(g, what, st);
    return p.grads == GRAD_LARGE ? go_grad<GradLarge, false>(g, what, st)
           : p.grads == GRAD_MIDDLE ? go_grad<GradMiddle, false>(g, what, st) : go_grad<GradSmall, false>(g, what, st);
}

}  // namespace vtdge
