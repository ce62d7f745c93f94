// Softmax cross entropy of a Linear's outputs over many classes, with the gradients of its input, weight and bias (gfx950).
//
//   z = x W^T + b,   loss_r = log sum_v exp z_rv - (1 - eps) z_rt - eps mean_v z_rv
//   d_rv = g_r (exp(z_rv) / sum - (1 - eps) [v = t_r] - eps / classes),   dx = d W,   dW = d^T x,   db = sum_r d_r
//
// z is never in memory.  Forward, every workgroup multiplies a tile of rows by a tile of classes and keeps of it each row's largest
// z and the sum of exp(z - largest); a second kernel joins the tiles of a row.  Backward, the classes are taken in pieces: the
// tiles of a piece are multiplied again, d is rounded to bf16 (an error of half a step on each of many terms, as on any bf16
// operand; the sums over it are fp32) and kept for this piece only, and two products take it to dx and dW.  Four products of
// rows x classes x width in place of three, and no more than rows x piece values of scratch.
//
// One product routine does all of it: tiles through LDS by direct loads in slabs of 64 of the summed dimension, two in turn.  An
// operand either lies with the summed dimension along its rows (x and W for z, d for dx) or across them (W for dx, d and x for
// dW); the second kind goes into LDS as it lies and is transposed by the LDS reads.  16-byte pieces are XOR-ed by their row against
// bank conflicts, on the side of the global address.
// fp32 operands are split into three bf16 parts each (24 bits), and the six products of parts down to 2^-24 are a six times longer
// sum, smallest first, in the same fp32 sums: the same kernels at a sixth of their rate, which is above that of the fp32 matrix
// instructions.
#include "common.h"

#include <math.h>

namespace vtdge {

constexpr float LOG2E = 1.44269504f, LN2 = 0.69314718f;
constexpr int CE_SLAB = 64;                        // of the summed dimension a stage
constexpr int CE_TILE = 128;                       // rows and columns of a tile

__device__ __forceinline__ int wave_uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }

// ------------------------------------------------------------------------------------------------ operands
// A bf16 matrix, or the three parts of an fp32 one `plane` elements apart.
struct Operand {
    const bf16_t *p;
    int64_t pitch, plane;
};
// parts of the two operands that are multiplied, smallest products first
__device__ __forceinline__ void parts_of(int segs, int seg, int &pa, int &pb)
{
    if (segs == 1) {
        pa = pb = 0;
    } else {
        // (2,0) (0,2) (1,1) (1,0) (0,1) (0,0), two bits each
        pa = (0x0052 >> (2 * seg)) & 3;
        pb = (0x0118 >> (2 * seg)) & 3;
    }
}

// ------------------------------------------------------------------------------------------------ the product of a tile
// ALONG: the summed dimension lies along the rows of memory: tile rows are rows of memory, `limit` of them.
// Across: the summed dimension counts the rows of memory, `limit` of them, and tile rows are elements of a row, which has a multiple
// of 8 of them, `span`.  No stage begins behind `limit`: a sum of n rows of memory has ceil(n / 64) stages.
// R: tile rows / 32 of a wave; a tile has 64 R.
template <bool ALONG, int R> struct Loader {
    static constexpr int PIECES = 2 * R;            // direct loads of a wave and stage
    static constexpr int ROW = ALONG ? 128 : 128 * R, STAGE = 8192 * R;
    const unsigned char *base;
    int64_t plane, pitch;                           // bytes
    int limit, row0, col;

    __device__ __forceinline__ Loader(const Operand &o, int64_t first, int64_t lim, int64_t span)
        : base(reinterpret_cast<const unsigned char *>(o.p)), plane(o.plane * 2), pitch(o.pitch * 2)
    {
        const int lane = threadIdx.x & 63, wid = wave_uniform(threadIdx.x >> 6);
        if constexpr (ALONG) {
            base += first * pitch;
            limit = (int)(lim - first < 64 * R ? lim - first : 64 * R);
            row0 = wid * 8 + (lane >> 3);
            col = ((lane & 7) ^ ((row0 >> 1) & 7)) * 16;
        } else {
            constexpr int LPR = 8 * R, RPI = 64 / LPR;      // lanes a row, rows an instruction
            base += first * 2;
            limit = (int)lim;
            row0 = wid * RPI + lane / LPR;
            // (the rows of an instruction's successors are 4 RPI apart: the swizzle follows in load())
            col = (lane % LPR) * 16;
            row_span = (int)(span - first < 64 * R ? span - first : 64 * R) * 2 - 16;
        }
    }
    int row_span;
    static __device__ __forceinline__ int swizzle(int k) { return R == 1 ? ((k >> 1) & 3) << 1 : (k & 7) << 1; }

    // stage `kt` of part `part` to LDS byte `lds`
    __device__ __forceinline__ void load(int part, int kt, uint32_t lds) const
    {
        const int wid = wave_uniform(threadIdx.x >> 6);
        const unsigned char *at = base + part * plane + (ALONG ? (int64_t)kt * 128 : (int64_t)kt * CE_SLAB * pitch);
        const void *from = uniform_ptr(at);
        const int p32 = (int)pitch;
#pragma unroll
        for (int d = 0; d < PIECES; d++) {
            uint32_t off, to;
            if constexpr (ALONG) {
                const int r = min(d * 32 + row0, limit - 1);
                off = (uint32_t)r * (uint32_t)p32 + col;
                to = lds + (d * 32 + wid * 8) * 128;
            } else {
                constexpr int RPI = 64 / (8 * R);
                const int k = d * 4 * RPI + row0;
                const int r = min(k, limit - 1 - kt * CE_SLAB);
                const int c = min(col ^ (swizzle(k) * 16), row_span);
                off = (uint32_t)r * (uint32_t)p32 + c;
                to = lds + (d * 4 * RPI + wid * RPI) * ROW;
            }
            dma16(from, off, wave_uniform(to));
        }
    }
    // the 8 values of step s (16 of the summed dimension) of tile row `block` * 32 + lane % 32
    static __device__ __forceinline__ u32x4 fragment(const unsigned char *stage, int block, int s)
    {
        const int lane = threadIdx.x & 63, lr = lane & 31, lg = lane >> 5;
        if constexpr (ALONG) {
            return *reinterpret_cast<const u32x4 *>(stage + (block * 32 + lr) * 128 + (((2 * s + lg) ^ ((lr >> 1) & 7)) * 16));
        } else {
            const int k = 16 * s + 8 * lg + ((lane & 15) >> 2);
            const int at = block * 64 + ((lane >> 4) & 1) * 32 + (lane & 3) * 8;       // byte of the row
            const u32x2 lo = lds_read_tr16(stage + k * ROW + (((at >> 4) ^ swizzle(k)) << 4) + (at & 15));
            const u32x2 hi = lds_read_tr16(stage + (k + 4) * ROW + (((at >> 4) ^ swizzle(k + 4)) << 4) + (at & 15));
            return u32x4{lo.x, lo.y, hi.x, hi.y};
        }
    }
};

// acc[i][j][v] += A[row i*32 + lane%32 of the wave] . B[row j*32 + 8*(v/4) + 4*(lane/32) + v%4], stages t0 .. t1 - 1 of nk a segment
template <class LA, class LB, int IM, int JN>
__device__ __forceinline__ void multiply_tile(const LA &a, const LB &b, int nk, int segs, int t0, int t1, unsigned char *smem, f32x16 (&acc)[IM][JN])
{
    const int wid = wave_uniform(threadIdx.x >> 6), wm = wid >> 1, wn = wid & 1;
    constexpr int STAGE = LA::STAGE + LB::STAGE;
    const uint32_t lds0 = (uint32_t)(uintptr_t)smem;
    int seg = t0 / nk, kt = t0 - seg * nk;
    auto issue = [&](int slot) {
        int pa, pb;
        parts_of(segs, seg, pa, pb);
        a.load(pa, kt, lds0 + slot * STAGE);
        b.load(pb, kt, lds0 + slot * STAGE + LA::STAGE);
        if (++kt == nk) kt = 0, seg++;
    };
    issue(0);
    for (int t = t0; t < t1; t++) {
        const int slot = (t - t0) & 1;
        // this stage's loads have landed, for all waves; the other slot is read no more
        wait_vmcnt<0>();
        lds_barrier();
        if (t + 1 < t1) issue(slot ^ 1);
        const unsigned char *sa = smem + slot * STAGE, *sb = sa + LA::STAGE;
#pragma unroll
        for (int s = 0; s < CE_SLAB / 16; s++) {
            u32x4 fa[IM], fb[JN];
#pragma unroll
            for (int i = 0; i < IM; i++) fa[i] = LA::fragment(sa, wm * IM + i, s);
#pragma unroll
            for (int j = 0; j < JN; j++) fb[j] = LB::fragment(sb, wn * JN + j, s);
#pragma unroll
            for (int i = 0; i < IM; i++)
#pragma unroll
                for (int j = 0; j < JN; j++) Slab<bf16_t>::mma(fb[j], fa[i], acc[i][j]);
        }
    }
    lds_barrier();                                  // the slots are free for the epilogue
}

// Workgroup id -> tile: an XCD (every eighth id) takes a contiguous run of the list, which goes through eight row tiles for each
// column tile, so that what its L2 holds is used again.
__device__ __forceinline__ void tile_of(int id, int count, int tm, int tn, int &m, int &n)
{
    const int xcd = id & 7, at = id >> 3, whole = count >> 3, rest = count & 7;
    id = xcd * whole + (xcd < rest ? xcd : rest) + at;
    const int group = 8 * tn, g = id / group, first = g * 8, size = min(8, tm - first);
    const int in = id - g * group;
    m = first + in % size;
    n = in / size;
}

struct CeArgs {
    Operand x, w;
    const void *bias; const int64_t *target; int64_t rows, classes; int64_t ignore; float smoothing; int nk, segs;
    int64_t v0, v1;                                 // classes of this piece
    // forward: [class tiles][rows] each
    float *tile_max, *tile_sum, *tile_total, *target_z;
    // backward
    const float *row_max, *row_inv, *row_scale; bf16_t *d; int64_t d_pitch, d_plane; float *bias_part; int64_t bias_stride;
    int bias_f32;
};

__device__ __forceinline__ bool counts(int64_t target, int64_t ignore, int64_t classes) { return target != ignore && target >= 0 && target < classes; }

// the sums over lane % 32 of 32 values a lane: lane r ends with the sum of value index_of(r)
template <int O> __device__ __forceinline__ float from_lane_xor(float v)
{
    if constexpr (O == 1) return dpp_move<0xB1>(v);
    else if constexpr (O == 2) return dpp_move<0x4E>(v);
    else if constexpr (O == 4) return dpp_move<0x141>(dpp_move<0x1B>(v));
    else if constexpr (O == 8) return dpp_move<0x128>(v);
    else return __shfl_xor(v, O, WAVE);
}
__device__ __forceinline__ float sum_by_halves(float (&f)[32], int lr)
{
    static_for<5>([&](auto S) {
        constexpr int o = 1 << decltype(S)::value, half = 16 >> decltype(S)::value;
        const bool up = (lr & o) != 0;
#pragma unroll
        for (int i = 0; i < half; i++) {
            const float keep = up ? f[half + i] : f[i], send = up ? f[i] : f[half + i];
            f[i] = keep + from_lane_xor<o>(send);
        }
    });
    return f[0];
}

// z of a tile, times log2 e, in place of acc; -inf behind the last class
template <int IM, int JN> __device__ __forceinline__ void logits(const CeArgs &p, int64_t c0, f32x16 (&acc)[IM][JN])
{
    const int lg = (threadIdx.x & 63) >> 5;
#pragma unroll
    for (int j = 0; j < JN; j++)
#pragma unroll
        for (int q = 0; q < 4; q++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const int64_t c = c0 + j * 32 + 8 * q + 4 * lg + e;
                const bool in = c < p.v1;
                float b = 0.f;
                if (p.bias != nullptr && in)
                    b = p.bias_f32 ? static_cast<const float *>(p.bias)[c] : bf16_to_f32(static_cast<const bf16_t *>(p.bias)[c]);
                b *= LOG2E;
#pragma unroll
                for (int i = 0; i < IM; i++) acc[i][j][4 * q + e] = in ? __builtin_fmaf(acc[i][j][4 * q + e], LOG2E, b) : -INFINITY;
            }
}

// ------------------------------------------------------------------------------------------------ forward
template <bool TOTAL> __global__ __launch_bounds__(256, 2) void cross_entropy_tiles_kernel(CeArgs p, int tm, int tn)
{
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    int m, n;
    tile_of(blockIdx.x, gridDim.x, tm, tn, m, n);
    const int64_t r0 = (int64_t)m * CE_TILE, c0 = (int64_t)n * CE_TILE;
    f32x16 acc[2][2] = {};
    const Loader<true, 2> a(p.x, r0, p.rows, 0), b(p.w, c0, p.classes, 0);
    multiply_tile(a, b, p.nk, p.segs, 0, p.nk * p.segs, smem, acc);
    const int lane = threadIdx.x & 63, lr = lane & 31, lg = lane >> 5;
    const int wid = wave_uniform(threadIdx.x >> 6), wm = wid >> 1, wn = wid & 1;
    const int64_t cw = c0 + wn * 64;
    logits<2, 2>(p, cw, acc);
    float *const shared = reinterpret_cast<float *>(smem);          // [2 halves of the classes][largest, sum, total][128 rows]
#pragma unroll
    for (int i = 0; i < 2; i++) {
        const int row = wm * 64 + i * 32 + lr;
        const int64_t r = r0 + row;
        float top = -INFINITY, total = 0.f;
#pragma unroll
        for (int j = 0; j < 2; j++)
#pragma unroll
            for (int v = 0; v < 16; v++) top = fmaxf(top, acc[i][j][v]);
        top = fmaxf(top, __shfl_xor(top, 32, WAVE));
        const float from = top == -INFINITY ? 0.f : top;            // nothing in sight: exp2(-inf) = 0, and NaN stays NaN
        float sum = 0.f;
#pragma unroll
        for (int j = 0; j < 2; j++)
#pragma unroll
            for (int v = 0; v < 16; v++) {
                sum += __builtin_amdgcn_exp2f(acc[i][j][v] - from);
                if constexpr (TOTAL) total += cw + j * 32 + 8 * (v / 4) + 4 * lg + v % 4 < p.classes ? acc[i][j][v] : 0.f;
            }
        sum += __shfl_xor(sum, 32, WAVE);
        if constexpr (TOTAL) total += __shfl_xor(total, 32, WAVE);
        if (lg == 0) {
            shared[(wn * 3 + 0) * CE_TILE + row] = top;
            shared[(wn * 3 + 1) * CE_TILE + row] = sum;
            if constexpr (TOTAL) shared[(wn * 3 + 2) * CE_TILE + row] = total;
        }
        // the z of the row's own class
        const int64_t t = r < p.rows ? p.target[r] : -1;
        const bool mine = counts(t, p.ignore, p.classes) && t >= cw && t < cw + 64 && (((int)(t - cw) >> 2) & 1) == lg;
        if (__ballot(mine) != 0) {
            const int at = (int)(t - cw), reg = (at >> 5) * 16 + ((at & 31) >> 3) * 4 + (at & 3);
            float z = 0.f;
#pragma unroll
            for (int j = 0; j < 2; j++)
#pragma unroll
                for (int v = 0; v < 16; v++) z = reg == j * 16 + v ? acc[i][j][v] : z;
            if (mine) p.target_z[r] = z;
        }
    }
    __syncthreads();
    const int row = threadIdx.x;
    if (row < CE_TILE && r0 + row < p.rows) {
        const float t0 = shared[row], t1 = shared[3 * CE_TILE + row], top = fmaxf(t0, t1);
        const float from = top == -INFINITY ? 0.f : top;
        const float sum = shared[CE_TILE + row] * __builtin_amdgcn_exp2f((t0 == -INFINITY ? from : t0) - from) +
                          shared[4 * CE_TILE + row] * __builtin_amdgcn_exp2f((t1 == -INFINITY ? from : t1) - from);
        const int64_t at = (int64_t)n * p.rows + r0 + row;
        p.tile_max[at] = top;
        p.tile_sum[at] = sum;
        if constexpr (TOTAL) p.tile_total[at] = shared[2 * CE_TILE + row] + shared[5 * CE_TILE + row];
    }
}

// joins the class tiles of each row; with `mean` given a single workgroup goes on to the mean of the losses
__global__ __launch_bounds__(256) void cross_entropy_join_kernel(CeArgs p, int tn, float *loss_rows, float *row_max, float *row_inv)
{
    // 64 rows a workgroup, four waves along the tiles
    __shared__ float tops[4][64], sums[4][64], totals[4][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t r = (int64_t)blockIdx.x * 64 + lane;
    const bool in = r < p.rows;
    float top = -INFINITY, sum = 0.f, total = 0.f;
    if (in) {
        for (int n = wave; n < tn; n += 4) {
            const int64_t at = (int64_t)n * p.rows + r;
            const float t = p.tile_max[at], s = p.tile_sum[at], next = fmaxf(top, t);
            const float from = next == -INFINITY ? 0.f : next;
            sum = sum * __builtin_amdgcn_exp2f((top == -INFINITY ? from : top) - from) + s * __builtin_amdgcn_exp2f((t == -INFINITY ? from : t) - from);
            top = next;
            if (p.smoothing != 0.f) total += p.tile_total[at];
        }
    }
    tops[wave][lane] = top;
    sums[wave][lane] = sum;
    totals[wave][lane] = total;
    __syncthreads();
    if (wave != 0 || !in) return;
    top = fmaxf(fmaxf(tops[0][lane], tops[1][lane]), fmaxf(tops[2][lane], tops[3][lane]));
    const float from = top == -INFINITY ? 0.f : top;
    sum = total = 0.f;
#pragma unroll
    for (int w = 0; w < 4; w++) {
        const float t = tops[w][lane];
        sum += sums[w][lane] * __builtin_amdgcn_exp2f((t == -INFINITY ? from : t) - from);
        total += totals[w][lane];
    }
    const int64_t t = p.target[r];
    float loss = 0.f;
    if (counts(t, p.ignore, p.classes)) {
        // log2 sum + (1 - eps) (largest - z_t) + eps (largest - mean): differences of like size, not of large sums
        loss = __builtin_amdgcn_logf(sum) + (1.f - p.smoothing) * (top - p.target_z[r]);
        if (p.smoothing != 0.f) loss += p.smoothing * (top - total / (float)p.classes);
        loss *= LN2;
    }
    loss_rows[r] = loss;
    row_max[r] = top;
    row_inv[r] = 1.0f / sum;
}

__global__ __launch_bounds__(1024) void cross_entropy_mean_kernel(const float *loss_rows, const int64_t *target, int64_t rows, int64_t classes,
                                                                  int64_t ignore, float *loss, float *inv_count)
{
    __shared__ double sums[16];
    __shared__ int64_t ns[16];
    double sum = 0.0;
    int64_t n = 0;
    for (int64_t r = threadIdx.x; r < rows; r += 1024) {
        sum += loss_rows[r];
        n += counts(target[r], ignore, classes) ? 1 : 0;
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        sum += __shfl_xor(sum, o, WAVE);
        n += __shfl_xor(n, o, WAVE);
    }
    if ((threadIdx.x & 63) == 0) sums[threadIdx.x >> 6] = sum, ns[threadIdx.x >> 6] = n;
    __syncthreads();
    if (threadIdx.x == 0) {
        sum = 0.0, n = 0;
        for (int w = 0; w < 16; w++) sum += sums[w], n += ns[w];
        if (inv_count == nullptr) {
            *loss = (float)sum;
        } else {
            *loss = n > 0 ? (float)(sum / (double)n) : 0.f;
            *inv_count = n > 0 ? (float)(1.0 / (double)n) : 0.f;
        }
    }
}

// ------------------------------------------------------------------------------------------------ backward
// d of a piece of the classes; rows and classes behind the last are written as zeros up to whole slabs
template <bool SPLIT> __global__ __launch_bounds__(256, 2) void cross_entropy_d_kernel(CeArgs p, int tm, int tn)
{
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    int m, n;
    tile_of(blockIdx.x, gridDim.x, tm, tn, m, n);
    const int64_t r0 = (int64_t)m * CE_TILE, c0 = p.v0 + (int64_t)n * CE_TILE;
    f32x16 acc[2][2] = {};
    const Loader<true, 2> a(p.x, r0, p.rows, 0), b(p.w, c0, p.classes, 0);
    multiply_tile(a, b, p.nk, p.segs, 0, p.nk * p.segs, smem, acc);
    const int lane = threadIdx.x & 63, lr = lane & 31, lg = lane >> 5;
    const int wid = wave_uniform(threadIdx.x >> 6), wm = wid >> 1, wn = wid & 1;
    const int64_t cw = c0 + wn * 64;
    logits<2, 2>(p, cw, acc);
    const float even = p.smoothing / (float)p.classes;
#pragma unroll
    for (int i = 0; i < 2; i++) {
        const int64_t r = r0 + wm * 64 + i * 32 + lr;
        const int64_t t = r < p.rows ? p.target[r] : -1;
        const bool live = r < p.rows && counts(t, p.ignore, p.classes);
        const float top = live ? p.row_max[r] : 0.f, inv = live ? p.row_inv[r] : 0.f;
        const float g = live ? (p.row_scale != nullptr ? p.row_scale[r] : 1.f) : 0.f;
#pragma unroll
        for (int j = 0; j < 2; j++)
#pragma unroll
            for (int v = 0; v < 16; v++) {
                const bool in = cw + j * 32 + 8 * (v / 4) + 4 * lg + v % 4 < p.v1;
                const float d = __builtin_fmaf(__builtin_amdgcn_exp2f(acc[i][j][v] - top), inv, -even);
                acc[i][j][v] = live && in ? d : 0.f;
            }
        const bool mine = live && t >= cw && t < cw + 64 && t < p.v1 && (((int)(t - cw) >> 2) & 1) == lg;
        if (__ballot(mine) != 0) {
            const int at = (int)(t - cw), reg = mine ? (at >> 5) * 16 + ((at & 31) >> 3) * 4 + (at & 3) : -1;
#pragma unroll
            for (int j = 0; j < 2; j++)
#pragma unroll
                for (int v = 0; v < 16; v++) acc[i][j][v] -= reg == j * 16 + v ? 1.f - p.smoothing : 0.f;
        }
        if (p.row_scale != nullptr) {
#pragma unroll
            for (int j = 0; j < 2; j++)
#pragma unroll
                for (int v = 0; v < 16; v++) acc[i][j][v] = live ? acc[i][j][v] * g : 0.f;
        }
    }
    if (p.bias_part != nullptr) {
        float *const shared = reinterpret_cast<float *>(smem);      // [2 halves of the rows][128 classes]
        float f[32];
#pragma unroll
        for (int c = 0; c < 32; c++) f[c] = acc[0][c >> 4][c & 15] + acc[1][c >> 4][c & 15];
        const float sum = sum_by_halves(f, lr);
        // lane bit b chose bit 4 - b of the value's number
        const int c = ((lr & 1) << 4) | ((lr & 2) << 2) | (lr & 4) | ((lr & 8) >> 2) | ((lr & 16) >> 4);
        shared[wm * CE_TILE + wn * 64 + (c >> 4) * 32 + 8 * ((c & 15) >> 2) + 4 * lg + (c & 3)] = sum;
        __syncthreads();
        const int at = threadIdx.x;
        if (at < CE_TILE && c0 + at < p.v1) p.bias_part[m * p.bias_stride + c0 + at] = shared[at] + shared[CE_TILE + at];
    }
    // to memory: 4 consecutive classes a lane
#pragma unroll
    for (int i = 0; i < 2; i++) {
        const int64_t r = r0 + wm * 64 + i * 32 + lr;
        bf16_t *const row = p.d + r * p.d_pitch + (cw - p.v0) + 4 * lg;
#pragma unroll
        for (int j = 0; j < 2; j++)
#pragma unroll
            for (int q = 0; q < 4; q++) {
                float f[4];
#pragma unroll
                for (int e = 0; e < 4; e++) f[e] = acc[i][j][4 * q + e];
#pragma unroll
                for (int part = 0; part < (SPLIT ? 3 : 1); part++) {
                    const u32x2 o = {pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3])};
                    *reinterpret_cast<u32x2 *>(row + part * p.d_plane + j * 32 + 8 * q) = o;
                    if constexpr (SPLIT) f[0] -= bf16lo(o.x), f[1] -= bf16hi(o.x), f[2] -= bf16lo(o.y), f[3] -= bf16hi(o.y);
                }
            }
    }
}

// ---- out = A B over a dimension that may be cut into several parts, which leave sums of their own
struct GradArgs {
    Operand a, b;
    int64_t rows, cols, span_a, span_b, sum_a, sum_b;      // of the result; elements of a row of memory; rows of memory that may be read
    int nk, segs, splits;
    float *part; int64_t part_stride; int accumulate;       // [splits], [rows][cols] fp32 each
    void *out; int f32; const float *scale, *scale2;       // without `part`: the result, times what they point to
};

template <bool A_ALONG> __global__ __launch_bounds__(256, 2) void cross_entropy_grad_kernel(GradArgs p, int tm, int tn)
{
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    const int tiles = tm * tn, z = blockIdx.x / tiles;
    int m, n;
    tile_of(blockIdx.x - z * tiles, tiles, tm, tn, m, n);
    const int64_t r0 = (int64_t)m * CE_TILE, c0 = (int64_t)n * CE_TILE;
    const int stages = p.nk * p.segs;
    const int t0 = (int)((int64_t)stages * z / p.splits), t1 = (int)((int64_t)stages * (z + 1) / p.splits);
    f32x16 acc[2][2] = {};
    const Loader<A_ALONG, 2> a(p.a, r0, A_ALONG ? p.rows : p.sum_a, p.span_a);
    const Loader<false, 2> b(p.b, c0, p.sum_b, p.span_b);
    multiply_tile(a, b, p.nk, p.segs, t0, t1, smem, acc);
    const int lane = threadIdx.x & 63, lr = lane & 31, lg = lane >> 5;
    const int wid = wave_uniform(threadIdx.x >> 6), wm = wid >> 1, wn = wid & 1;
    float scale = 1.f;
    if (p.part == nullptr) {
        if (p.scale != nullptr) scale = *p.scale;
        if (p.scale2 != nullptr) scale *= *p.scale2;
    }
#pragma unroll
    for (int i = 0; i < 2; i++) {
        const int64_t r = r0 + wm * 64 + i * 32 + lr;
        if (r >= p.rows) continue;
#pragma unroll
        for (int j = 0; j < 2; j++)
#pragma unroll
            for (int q = 0; q < 4; q++) {
                const int64_t c = c0 + wn * 64 + j * 32 + 8 * q + 4 * lg;
                if (p.part != nullptr) {
                    float *const to = p.part + z * p.part_stride + r * p.cols + c;
#pragma unroll
                    for (int e = 0; e < 4; e++)
                        if (c + e < p.cols) to[e] = acc[i][j][4 * q + e] + (p.accumulate ? to[e] : 0.f);
                } else if (p.f32) {
                    float *const to = static_cast<float *>(p.out) + r * p.cols + c;
#pragma unroll
                    for (int e = 0; e < 4; e++)
                        if (c + e < p.cols) to[e] = acc[i][j][4 * q + e] * scale;
                } else {
                    bf16_t *const to = static_cast<bf16_t *>(p.out) + r * p.cols + c;
#pragma unroll
                    for (int e = 0; e < 4; e++)
                        if (c + e < p.cols) to[e] = f32_to_bf16(acc[i][j][4 * q + e] * scale);
                }
            }
    }
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
// (target given) as zeros, so that what they hold reaches no gradient.
template <typename T> __global__ __launch_bounds__(256) void cross_entropy_pack_kernel(const T *__restrict__ from, int64_t ld, int64_t rows, int width, int padded,
                                                                                       const int64_t *__restrict__ target, int64_t ignore, int64_t classes,
                                                                                       bf16_t *__restrict__ to, int64_t plane)
{
    const int per_row = padded / 8;
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, r = i / per_row;
    if (r >= rows) return;
    const int c = (int)(i - r * per_row) * 8;
    const bool live = target == nullptr || counts(target[r], ignore, classes);
    float f[8];
#pragma unroll
    for (int e = 0; e < 8; e++) f[e] = live && c + e < width ? Elem<T>::load(from + r * ld + c + e) : 0.f;
    bf16_t *const at = to + r * padded + c;
    *reinterpret_cast<u32x4 *>(at) = Elem<bf16_t>::pack(f);
    if constexpr (sizeof(T) == 4) {
        // (infinity and NaN have no rest)
#pragma unroll
        for (int part = 1; part < 3; part++) {
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const float rest = f[e] - Elem<bf16_t>::round(f[e]);
                f[e] = fabsf(rest) < INFINITY ? rest : 0.f;
            }
            *reinterpret_cast<u32x4 *>(at + part * plane) = Elem<bf16_t>::pack(f);
        }
    }
}

// ------------------------------------------------------------------------------------------------ on the host
// Everything a call lays out, the same for the size and the call.
struct CePlan {
    int64_t rows, classes; int width, padded, parts, segs, nk;
    bool backward;
    int64_t tm, tn;                                 // row and class tiles of all classes
    int64_t piece, d_rows;                          // classes of a piece, rows of d
    int dx_splits, dw_splits;
    // bytes of the workspace
    int64_t x_at, w_at, xz_at, max_at, sum_at, total_at, z_at, d_at, dx_at, dw_at, db_at, bytes;
};
constexpr int64_t CE_PIECE_BYTES = 128ll << 20;     // of d

static int64_t part_of(int64_t n) { return (n + 63) / 64 * 64; }      // elements from one part of a sum to the next
static int64_t take(int64_t &at, int64_t bytes)
{
    const int64_t here = at;
    at += (bytes + 255) / 256 * 256;
    return here;
}
// into how many parts a sum of `stages` is cut so that `tiles` of it fill the chip twice, none shorter than 4 stages
static int splits_for(int64_t tiles, int64_t stages)
{
    const int64_t wanted = 2 * (int64_t)compute_units() / tiles, most = stages / 4;
    const int64_t s = wanted < most ? wanted : most;
    return (int)(s < 1 ? 1 : s);
}
static CePlan plan_of(int64_t rows, int64_t classes, int width, int dtype, bool backward)
{
    CePlan p{};
    p.rows = rows, p.classes = classes, p.width = width, p.backward = backward;
    p.padded = (int)ceil_div(width, CE_SLAB) * CE_SLAB;
    p.parts = dtype == VTDGE_F32 ? 3 : 1;
    p.segs = dtype == VTDGE_F32 ? 6 : 1;
    p.nk = p.padded / CE_SLAB;
    p.tm = ceil_div(rows, CE_TILE), p.tn = ceil_div(classes, CE_TILE);
    int64_t at = 0;
    p.x_at = take(at, rows * p.padded * 2 * p.parts);
    p.w_at = take(at, classes * p.padded * 2 * p.parts);
    if (!backward) {
        p.max_at = take(at, p.tn * rows * 4);
        p.sum_at = take(at, p.tn * rows * 4);
        p.total_at = take(at, p.tn * rows * 4);
        p.z_at = take(at, rows * 4);
    } else {
        p.xz_at = take(at, rows * p.padded * 2 * p.parts);
        p.d_rows = p.tm * CE_TILE;
        int64_t piece = CE_PIECE_BYTES / (p.d_rows * 2 * p.parts) / CE_TILE * CE_TILE;
        if (piece < 8 * CE_TILE) piece = 8 * CE_TILE;
        // pieces of equal size
        const int64_t pieces = ceil_div(classes, piece);
        p.piece = ceil_div(ceil_div(classes, pieces), CE_TILE) * CE_TILE;
        const int64_t cols = ceil_div(width, CE_TILE);
        p.dx_splits = splits_for(p.tm * cols, ceil_div(p.piece, CE_SLAB) * p.segs);
        p.dw_splits = splits_for(p.piece / CE_TILE * cols, ceil_div(rows, CE_SLAB) * p.segs);
        p.d_at = take(at, p.d_rows * p.piece * 2 * p.parts);
        p.dx_at = take(at, part_of(rows * width) * 4 * p.dx_splits);
        p.dw_at = take(at, part_of(p.piece * width) * 4 * p.dw_splits);
        p.db_at = take(at, p.tm * part_of(classes) * 4);
    }
    p.bytes = at;
    return p;
}

static int check_sizes(const char *what, int64_t rows, int64_t classes, int width, int dtype)
{
    VT_REQUIRE(dtype == VTDGE_F32 || dtype == VTDGE_BF16, VTDGE_ERR_ARG, "%s: dtype %d", what, dtype);
    VT_REQUIRE(rows > 0 && classes > 0 && width > 0, VTDGE_ERR_ARG, "%s: %lld rows, %lld classes of %d", what, (long long)rows, (long long)classes, width);
    VT_REQUIRE(rows < (1 << 24) && classes < (1 << 24) && width <= (1 << 16), VTDGE_ERR_UNSUPPORTED, "%s: %lld rows, %lld classes of %d", what,
               (long long)rows, (long long)classes, width);
    VT_REQUIRE(rows * (int64_t)width < (1ll << 31) && classes * (int64_t)width < (1ll << 31), VTDGE_ERR_UNSUPPORTED,
               "%s: %lld rows, %lld classes of %d", what, (long long)rows, (long long)classes, width);
    return VTDGE_OK;
}

// an operand as it lies, where the product routine can read it so, else packed at `at`
static int operand_of(Operand &o, const void *src, int64_t ld, int64_t rows, const CePlan &p, int dtype, const int64_t *target, int64_t ignore,
                      unsigned char *at, hipStream_t st)
{
    if (dtype == VTDGE_BF16 && target == nullptr && p.width == p.padded && ld % 8 == 0 && ld < (1 << 22) && ((uintptr_t)src & 15) == 0) {
        o = Operand{(const bf16_t *)src, ld, 0};
        return VTDGE_OK;
    }
    o = Operand{(const bf16_t *)at, p.padded, rows * p.padded};
    const int64_t blocks = ceil_div(rows * (p.padded / 8), 256);
    VT_REQUIRE(blocks < (1 << 24), VTDGE_ERR_UNSUPPORTED, "cross_entropy: %lld rows of %d", (long long)rows, p.width);
    if (dtype == VTDGE_F32) {
        note_kernel(reinterpret_cast<const void *>(cross_entropy_pack_kernel<float>));
        cross_entropy_pack_kernel<float><<<(unsigned)blocks, 256, 0, st>>>((const float *)src, ld, rows, p.width, p.padded, target, ignore, p.classes,
                                                                           (bf16_t *)at, o.plane);
    } else {
        note_kernel(reinterpret_cast<const void *>(cross_entropy_pack_kernel<bf16_t>));
        cross_entropy_pack_kernel<bf16_t><<<(unsigned)blocks, 256, 0, st>>>((const bf16_t *)src, ld, rows, p.width, p.padded, target, ignore, p.classes,
                                                                            (bf16_t *)at, o.plane);
    }
    return check_launch("cross_entropy");
}

constexpr int CE_LDS = 2 * 2 * 16384;

#define VT_STEP(call)                      \
    do {                                   \
        const int vt_rc = (call);          \
        if (vt_rc != VTDGE_OK) return vt_rc; \
    } while (0)

template <bool A_ALONG> static int go_grad(const GradArgs &g, hipStream_t st)
{
    const int tm = (int)ceil_div(g.rows, CE_TILE), tn = (int)ceil_div(g.cols, CE_TILE);
    VT_REQUIRE(g.nk <= ceil_div(g.sum_b, CE_SLAB) && (A_ALONG || g.nk <= ceil_div(g.sum_a, CE_SLAB)) && g.splits >= 1 && g.splits <= g.nk * g.segs,
               VTDGE_ERR_ARG, "cross_entropy_backward: %d stages over %lld rows", g.nk, (long long)g.sum_b);
    auto kern = cross_entropy_grad_kernel<A_ALONG>;
    VT_RESERVE_LDS(kern, CE_LDS, "cross_entropy_backward");
    note_kernel(reinterpret_cast<const void *>(kern));
    kern<<<(unsigned)(tm * tn * g.splits), 256, CE_LDS, st>>>(g, tm, tn);
    return check_launch("cross_entropy_backward");
}

static int sum_up(const SumJob *jobs, int count, const float *scale, const float *scale2, bool f32, hipStream_t st)
{
    SumArgs a{};
    int n = 0;
    for (int i = 0; i < count; i++) {
        if (jobs[i].out == nullptr) continue;
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

extern "C" int64_t vtdge_cross_entropy_workspace(int64_t rows, int64_t classes, int width, int dtype, int backward)
{
    if (check_sizes("cross_entropy_workspace", rows, classes, width, dtype) != VTDGE_OK) return -1;
    return plan_of(rows, classes, width, dtype, backward != 0).bytes;
}

extern "C" int vtdge_cross_entropy(const void *x, int64_t ldx, const void *weight, int64_t ldw, const void *bias, const int64_t *target,
                                   int64_t rows, int64_t classes, int width, int64_t ignore_index, float smoothing, void *workspace,
                                   int64_t workspace_bytes, float *loss_rows, float *row_max, float *row_inv, float *loss, float *inv_count,
                                   int dtype, void *stream)
{
    VT_STEP(check_sizes("cross_entropy", rows, classes, width, dtype));
    VT_REQUIRE(x && weight && target && loss_rows && row_max && row_inv && workspace, VTDGE_ERR_ARG, "cross_entropy: NULL operand");
    VT_REQUIRE(loss != nullptr || inv_count == nullptr, VTDGE_ERR_ARG, "cross_entropy: inv_count without loss");
    VT_REQUIRE(ldx >= width && ldw >= width, VTDGE_ERR_ARG, "cross_entropy: rows of %d, %lld and %lld apart", width, (long long)ldx, (long long)ldw);
    VT_REQUIRE(smoothing >= 0.f && smoothing <= 1.f, VTDGE_ERR_ARG, "cross_entropy: smoothing %g", (double)smoothing);
    const CePlan p = plan_of(rows, classes, width, dtype, false);
    VT_REQUIRE(workspace_bytes >= p.bytes && ((uintptr_t)workspace & 255) == 0, VTDGE_ERR_ARG, "cross_entropy: workspace of %lld bytes, %lld needed",
               (long long)workspace_bytes, (long long)p.bytes);
    VT_REQUIRE(p.tm * p.tn < (1 << 24), VTDGE_ERR_UNSUPPORTED, "cross_entropy: %lld tiles", (long long)(p.tm * p.tn));
    unsigned char *const ws = (unsigned char *)workspace;
    const hipStream_t st = (hipStream_t)stream;
    CeArgs a{};
    VT_STEP(operand_of(a.x, x, ldx, rows, p, dtype, nullptr, ignore_index, ws + p.x_at, st));
    VT_STEP(operand_of(a.w, weight, ldw, classes, p, dtype, nullptr, ignore_index, ws + p.w_at, st));
    a.bias = bias, a.bias_f32 = dtype == VTDGE_F32, a.target = target, a.rows = rows, a.classes = classes, a.ignore = ignore_index;
    a.smoothing = smoothing, a.nk = p.nk, a.segs = p.segs, a.v0 = 0, a.v1 = classes;
    a.tile_max = (float *)(ws + p.max_at), a.tile_sum = (float *)(ws + p.sum_at), a.tile_total = (float *)(ws + p.total_at);
    a.target_z = (float *)(ws + p.z_at);
    auto kern = smoothing != 0.f ? cross_entropy_tiles_kernel<true> : cross_entropy_tiles_kernel<false>;
    VT_RESERVE_LDS(cross_entropy_tiles_kernel<true>, CE_LDS, "cross_entropy");
    VT_RESERVE_LDS(cross_entropy_tiles_kernel<false>, CE_LDS, "cross_entropy");
    note_kernel(reinterpret_cast<const void *>(kern));
    kern<<<(unsigned)(p.tm * p.tn), 256, CE_LDS, st>>>(a, (int)p.tm, (int)p.tn);
    VT_STEP(check_launch("cross_entropy"));
    note_kernel(reinterpret_cast<const void *>(cross_entropy_join_kernel));
    cross_entropy_join_kernel<<<(unsigned)ceil_div(rows, 64), 256, 0, st>>>(a, (int)p.tn, loss_rows, row_max, row_inv);
    VT_STEP(check_launch("cross_entropy"));
    if (loss != nullptr) {
        note_kernel(reinterpret_cast<const void *>(cross_entropy_mean_kernel));
        cross_entropy_mean_kernel<<<1, 1024, 0, st>>>(loss_rows, target, rows, classes, ignore_index, loss, inv_count);
        VT_STEP(check_launch("cross_entropy"));
    }
    return VTDGE_OK;
}

extern "C" int vtdge_cross_entropy_backward(const void *x, int64_t ldx, const void *weight, int64_t ldw, const void *bias, const int64_t *target,
                                            const float *row_max, const float *row_inv, const float *grad, int grad_stride,
                                            const float *inv_count, int64_t rows, int64_t classes, int width, int64_t ignore_index,
                                            float smoothing, void *workspace, int64_t workspace_bytes, void *dx, void *dweight, void *dbias,
                                            int dtype, void *stream)
{
    VT_STEP(check_sizes("cross_entropy_backward", rows, classes, width, dtype));
    VT_REQUIRE(x && weight && target && row_max && row_inv && grad && workspace, VTDGE_ERR_ARG, "cross_entropy_backward: NULL operand");
    VT_REQUIRE(ldx >= width && ldw >= width, VTDGE_ERR_ARG, "cross_entropy_backward: rows of %d, %lld and %lld apart", width, (long long)ldx, (long long)ldw);
    VT_REQUIRE(grad_stride == 0 || (grad_stride == 1 && inv_count == nullptr), VTDGE_ERR_ARG, "cross_entropy_backward: grad_stride %d", grad_stride);
    VT_REQUIRE(smoothing >= 0.f && smoothing <= 1.f, VTDGE_ERR_ARG, "cross_entropy_backward: smoothing %g", (double)smoothing);
    const CePlan p = plan_of(rows, classes, width, dtype, true);
    VT_REQUIRE(workspace_bytes >= p.bytes && ((uintptr_t)workspace & 255) == 0, VTDGE_ERR_ARG,
               "cross_entropy_backward: workspace of %lld bytes, %lld needed", (long long)workspace_bytes, (long long)p.bytes);
    const int64_t cols = ceil_div(width, CE_TILE), piece_tiles = p.piece / CE_TILE;
    VT_REQUIRE(p.tm * piece_tiles < (1 << 24) && p.tm * cols * p.dx_splits < (1 << 24) && piece_tiles * cols * p.dw_splits < (1 << 24), VTDGE_ERR_UNSUPPORTED,
               "cross_entropy_backward: %lld x %lld tiles", (long long)p.tm, (long long)p.tn);
    if (dx == nullptr && dweight == nullptr && dbias == nullptr) return VTDGE_OK;
    unsigned char *const ws = (unsigned char *)workspace;
    const hipStream_t st = (hipStream_t)stream;
    const bool f32 = dtype == VTDGE_F32;
    CeArgs a{};
    Operand xz{};                                   // x with the rows that are left out as zeros
    VT_STEP(operand_of(a.w, weight, ldw, classes, p, dtype, nullptr, ignore_index, ws + p.w_at, st));
    VT_STEP(operand_of(xz, x, ldx, rows, p, dtype, target, ignore_index, ws + p.xz_at, st));
    a.x = xz;
    a.bias = bias, a.bias_f32 = f32, a.target = target, a.rows = rows, a.classes = classes, a.ignore = ignore_index;
    a.smoothing = smoothing, a.nk = p.nk, a.segs = p.segs;
    a.row_max = row_max, a.row_inv = row_inv, a.row_scale = grad_stride == 1 ? grad : nullptr;
    a.d = (bf16_t *)(ws + p.d_at), a.d_pitch = p.piece, a.d_plane = p.d_rows * p.piece;
    a.bias_part = dbias != nullptr ? (float *)(ws + p.db_at) : nullptr, a.bias_stride = part_of(classes);
    const float *const scale = grad_stride == 1 ? nullptr : grad;
    const bool one_piece = p.piece >= classes;
    float *const dx_part = one_piece && p.dx_splits == 1 ? nullptr : (float *)(ws + p.dx_at);
    float *const dw_part = p.dw_splits == 1 ? nullptr : (float *)(ws + p.dw_at);
    auto kern = f32 ? cross_entropy_d_kernel<true> : cross_entropy_d_kernel<false>;
    VT_RESERVE_LDS(cross_entropy_d_kernel<true>, CE_LDS, "cross_entropy_backward");
    VT_RESERVE_LDS(cross_entropy_d_kernel<false>, CE_LDS, "cross_entropy_backward");
    const size_t elem = f32 ? 4 : 2;
    for (int64_t v0 = 0; v0 < classes; v0 += p.piece) {
        a.v0 = v0, a.v1 = v0 + p.piece < classes ? v0 + p.piece : classes;
        const int64_t live = a.v1 - a.v0;
        const int tn = (int)ceil_div(live, CE_TILE);
        note_kernel(reinterpret_cast<const void *>(kern));
        kern<<<(unsigned)(p.tm * tn), 256, CE_LDS, st>>>(a, (int)p.tm, tn);
        VT_STEP(check_launch("cross_entropy_backward"));
        const Operand d{a.d, a.d_pitch, a.d_plane};
        if (dx != nullptr) {
            GradArgs g{};
            g.a = d, g.b = Operand{a.w.p + v0 * a.w.pitch, a.w.pitch, a.w.plane};
            g.rows = rows, g.cols = width, g.sum_b = live, g.span_b = p.padded;
            g.nk = (int)ceil_div(live, CE_SLAB), g.segs = p.segs;
            g.splits = p.dx_splits < g.nk * g.segs ? p.dx_splits : g.nk * g.segs;
            g.part = dx_part, g.part_stride = part_of(rows * width), g.accumulate = v0 > 0, g.out = dx, g.f32 = f32, g.scale = scale, g.scale2 = inv_count;
            VT_STEP(go_grad<true>(g, st));
        }
        if (dweight != nullptr) {
            GradArgs g{};
            g.a = d, g.b = xz;
            g.rows = live, g.cols = width, g.sum_a = p.d_rows, g.span_a = p.piece, g.sum_b = rows, g.span_b = p.padded;
            g.nk = (int)ceil_div(rows, CE_SLAB), g.segs = p.segs, g.splits = p.dw_splits;
            g.part = dw_part, g.part_stride = part_of(p.piece * width), g.out = (unsigned char *)dweight + v0 * width * elem, g.f32 = f32, g.scale = scale, g.scale2 = inv_count;
            VT_STEP(go_grad<false>(g, st));
            if (dw_part != nullptr && !one_piece) {
                const SumJob job{dw_part, g.out, live * width, g.part_stride, p.dw_splits};
                VT_STEP(sum_up(&job, 1, scale, inv_count, f32, st));
            }
        }
    }
    SumJob jobs[3] = {{dx_part, dx_part != nullptr ? dx : nullptr, rows * width, part_of(rows * width), p.dx_splits},
                      {dw_part, dw_part != nullptr && one_piece ? dweight : nullptr, classes * width, part_of(p.piece * width), p.dw_splits},
                      {a.bias_part, dbias, classes, part_of(classes), (int)p.tm}};
    return sum_up(jobs, 3, scale, inv_count, f32, st);
}
