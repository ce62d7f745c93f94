// Rows of 8-bit numbers with a power of two for every 128 of them ("blocks"), and what a training step keeps in them (gfx950): activations,
// the input of GELU, the centred input of LayerNorm.  The Linear over blocks is in linear_8bit.hip.
//
//   e = the smallest whole number with max |x| 2^-e <= 448, -110 at least;   value = e4m3(x 2^-e), nearest, ties to even
//
// A power of two makes x 2^-e exact, so that a value is rounded once; every number of a block is a bf16 number (4 bits), and from -110 on no
// denormal one.  The scale is the byte e + 127.  Infinities and NaN become NaN and do not count in the maximum; a block without a finite
// number has the least scale.  The largest fp32 numbers would be rounded beyond fp32 and stop at 240 2^120.
//
// All of these read and write each number once and are bound by memory, GELU in bf16 nearly as much by its instructions.  A lane has eight consecutive numbers (16 bytes of bf16, 32 of
// fp32), sixteen lanes a block, so that maxima are taken with four lane moves and blocks leave in whole lines of 128 bytes.  TB/s of what they
// read and write, bf16: quantize 65536 x 1024 41 us 4.9, dequantize 33 us 6.2 (from the last cache in part), GELU 65536 x 4096 235 us 5.7, its
// gradient 269 us 5.0 (both at a clock that has come up, 280 and 320 before), LayerNorm 65536 x 1024 64 us 5.2, its gradients 74 + 6 us 4.2; a large
// copy reaches 5.2.  Small ones are a launch: 4112 x 384 in fp32 6 to 10 us.
#include "eight_bit.h"

namespace vtdge {

// ------------------------------------------------------------------------------------------------ blocks
template <typename T> __global__ __launch_bounds__(256) void quantize_kernel(QuantizeArgs p)
{
    const bool second = blockIdx.x >= p.first;
    const QuantizeJob &job = p.job[second ? 1 : 0];
    const uint32_t id = (blockIdx.x - (second ? p.first : 0)) * 16 + (threadIdx.x >> 4), row = id / job.per_row, block = id - row * job.per_row;
    const int part = threadIdx.x & 15, c = (int)block * BLOCK + part * 8;
    const bool in = row < job.rows;
    Rounded q;
    if (job.from == nullptr) {                      // blocks that are there
        if (!in) return;
        q.bytes = *reinterpret_cast<const u32x2 *>(job.values + (int64_t)row * job.value_pitch + c);
        q.scale = job.scales[(int64_t)row * job.scale_pitch + block];
    } else {
        float f[8];
        load8<T>(static_cast<const T *>(job.from) + (int64_t)row * job.ld + c, in ? job.n - c : 0, f);
        q = round8(f);
        if (!in) return;
    }
    if (job.from != nullptr && job.values != nullptr) {
        *reinterpret_cast<u32x2 *>(job.values + (int64_t)row * job.value_pitch + c) = q.bytes;
        if (part == 0) put_scale(job.scales + (int64_t)row * job.scale_pitch, (int)block, (int)job.per_row, job.scale_pitch, q.scale);
    }
    if (job.expanded != nullptr && c < job.expanded_pitch) *reinterpret_cast<u32x4 *>(job.expanded + (int64_t)row * job.expanded_pitch + c) = expand8(q.bytes, q.scale);
}

// blocks -> numbers
template <typename T> __global__ __launch_bounds__(256) void dequantize_kernel(DequantizeArgs p)
{
    const uint32_t id = blockIdx.x * 256 + threadIdx.x, row = id / p.per_row, c = (id - row * p.per_row) * 8;
    if (row >= p.rows) return;
    const u32x2 bytes = *reinterpret_cast<const u32x2 *>(p.values + (int64_t)row * p.value_pitch + c);
    const int scale = p.scales[(int64_t)row * p.scale_pitch + c / BLOCK];
    float f[8];
    stands_for8(bytes, scale, f);
    store8<T>(static_cast<T *>(p.to) + (int64_t)row * p.n + c, p.n - (int)c, f);
}

// ------------------------------------------------------------------------------------------------ GELU
template <typename T> __global__ __launch_bounds__(256) void gelu_keep_kernel(GeluArgs p)
{
    const uint32_t id = blockIdx.x * 16 + (threadIdx.x >> 4), row = id / p.per_row, block = id - row * p.per_row;
    const int part = threadIdx.x & 15, c = (int)block * BLOCK + part * 8;
    const bool in = row < p.rows;
    float f[8], y[8];
    load8<T>(static_cast<const T *>(p.x) + (int64_t)row * p.ld + c, in ? p.n - c : 0, f);
#pragma unroll
    for (int e = 0; e < 8; e++) y[e] = gelu_value<T>(f[e]);
    const Rounded q = round8(f);
    if (!in) return;
    store8<T>(static_cast<T *>(p.y) + (int64_t)row * p.n + c, p.n - c, y);
    if (p.values == nullptr) return;
    *reinterpret_cast<u32x2 *>(p.values + (int64_t)row * p.value_pitch + c) = q.bytes;
    if (part == 0) put_scale(p.scales + (int64_t)row * p.scale_pitch, (int)block, (int)p.per_row, p.scale_pitch, q.scale);
}

// Phi(x) + x phi(x).  With a = |x| and e = exp(-a^2 / 2) the slope of -a is S = e (R(a) - a / sqrt(2 pi)), that of a 1 - S; R = erfcx(a / sqrt 2) / 2 falls
// like 1 / a, a polynomial in t = 1 / (1 + k a) without a constant term.  fp32: gelu_fn's, of degree 9, 6.4e-8 off over unit normals (2-norm), 1.4e-7 at most.
// bf16: of degree 4, 3.8e-5 (|S| + 0.05 e) off on [0, 13.5], a fiftieth of half a bf16 step at its smallest, and no nearer to the
// formula's zero than 2e-6; two transcendental instructions hide behind memory.  (1/2 and an odd polynomial of degree 17 on a clamped argument, 1.4e-4
// off, takes 11 instructions and leaves -1.1e-4 in place of nothing to every number below -4.2.)
template <typename T> __device__ __forceinline__ float gelu_slope(float v);
template <> __device__ __forceinline__ float gelu_slope<float>(float v)
{
    const float a = fminf(fabsf(v), 16.0f);
    const float t = __builtin_amdgcn_rcpf(__builtin_fmaf(0.35f, a, 1.0f));
    float q = -0.02912587f;
    q = __builtin_fmaf(q, t, 0.14387225f);
    q = __builtin_fmaf(q, t, -0.25550460f);
    q = __builtin_fmaf(q, t, 0.15892934f);
    q = __builtin_fmaf(q, t, -0.02293717f);
    q = __builtin_fmaf(q, t, 0.10543295f);
    q = __builtin_fmaf(q, t, 0.11985243f);
    q = __builtin_fmaf(q, t, 0.13985908f);
    q = __builtin_fmaf(q, t, 0.13962157f);
    const float e = __builtin_amdgcn_exp2f(a * (a * -0.72134752f)), neg = q * t * e;
    return __builtin_fmaf(v * 0.39894228f, e, v < 0.f ? neg : 1.f - neg);
}
template <> __device__ __forceinline__ float gelu_slope<bf16_t>(float v)
{
    const float a = fabsf(v), t = __builtin_amdgcn_rcpf(__builtin_fmaf(0.45f, a, 1.0f));
    float q = -0.11780614f;
    q = __builtin_fmaf(q, t, 0.30781589f);
    q = __builtin_fmaf(q, t, 0.12395127f);
    q = __builtin_fmaf(q, t, 0.18605228f);
    const float s = __builtin_fmaf(a, -0.39894228f, q * t) * __builtin_amdgcn_exp2f(a * (a * -0.72134752f));
    return v < 0.f ? s : 1.f - s;
}
template <typename T> __global__ __launch_bounds__(256) void gelu_slope_kernel(GeluArgs p)
{
    const uint32_t id = blockIdx.x * 256 + threadIdx.x, row = id / p.per_row, c = (id - row * p.per_row) * 8;
    if (row >= p.rows) return;
    float g[8], x[8];
    load8<T>(static_cast<const T *>(p.x) + (int64_t)row * p.ld + c, p.n - (int)c, g);
    const u32x2 bytes = *reinterpret_cast<const u32x2 *>(p.values + (int64_t)row * p.value_pitch + c);
    const int scale = p.scales[(int64_t)row * p.scale_pitch + c / BLOCK];
    stands_for8(bytes, scale, x);
#pragma unroll
    for (int e = 0; e < 8; e++) g[e] *= gelu_slope<T>(x[e]);
    store8<T>(static_cast<T *>(p.y) + (int64_t)row * p.n + c, p.n - (int)c, g);
}

// ------------------------------------------------------------------------------------------------ LayerNorm
// A row by WAVES waves, a lane CH times eight numbers, WAVES * 512 apart.
template <int WAVES> __device__ __forceinline__ int norm_column(int ch) { return (ch * WAVES * 64 + (int)(threadIdx.x & (WAVES * 64 - 1))) * 8; }

// the sums of a row's waves, in each of them; `shared` a place of its own for each call
template <int WAVES, int NV, typename V> __device__ __forceinline__ void row_sums(V (&v)[NV], V (*shared)[NV])
{
#pragma unroll
    for (int i = 0; i < NV; i++) v[i] = wave_total(v[i]);
    if constexpr (WAVES > 1) {
        const int wave = threadIdx.x >> 6 & (WAVES - 1);
        if ((threadIdx.x & 63) == 0)
#pragma unroll
            for (int i = 0; i < NV; i++) shared[wave][i] = v[i];
        __syncthreads();
#pragma unroll
        for (int i = 0; i < NV; i++) {
            v[i] = shared[0][i];
#pragma unroll
            for (int w = 1; w < WAVES; w++) v[i] += shared[w][i];
        }
    }
}

// The mean is the fp32 number next to the exact one, so that what is rounded to 8 bits behind it does not hang on the order of a sum:
// the sum is taken in 64 bits.
template <typename T, int WAVES, int CH> __global__ __launch_bounds__(256) void norm_keep_kernel(NormArgs p)
{
    __shared__ double sums64[WAVES][1];
    __shared__ float sums32[WAVES][1];
    const int64_t row = (int64_t)blockIdx.x * (4 / WAVES) + (WAVES == 1 ? threadIdx.x >> 6 : 0);
    const bool in = row < p.rows;
    if (WAVES == 1 && !in) return;                  // (a whole wave)
    float f[CH][8];
    double sum[1] = {0.0};
#pragma unroll
    for (int k = 0; k < CH; k++) {
        const int c = norm_column<WAVES>(k);
        load8<T>(static_cast<const T *>(p.x) + row * p.ld + c, p.n - c, f[k]);
#pragma unroll
        for (int e = 0; e < 8; e++) sum[0] += (double)f[k][e];
    }
    row_sums<WAVES>(sum, sums64);
    const float mean = (float)(sum[0] / (double)p.n);
    float square[1] = {0.f};
#pragma unroll
    for (int k = 0; k < CH; k++) {
        const int left = p.n - norm_column<WAVES>(k);
#pragma unroll
        for (int e = 0; e < 8; e++) {
            f[k][e] = e < left ? f[k][e] - mean : 0.f;
            square[0] = __builtin_fmaf(f[k][e], f[k][e], square[0]);
        }
    }
    row_sums<WAVES>(square, sums32);
    const float r = __builtin_amdgcn_rsqf(square[0] / (float)p.n + p.eps);
    if (p.rstd != nullptr && norm_column<WAVES>(0) == 0) p.rstd[row] = r;
#pragma unroll
    for (int k = 0; k < CH; k++) {
        const int c = norm_column<WAVES>(k), left = p.n - c;
        const Rounded q = round8(f[k]);
        if (c < p.value_pitch && p.values != nullptr) {
            *reinterpret_cast<u32x2 *>(p.values + row * p.value_pitch + c) = q.bytes;
            if (c % BLOCK == 0) put_scale(p.scales + row * p.scale_pitch, c / BLOCK, p.blocks, p.scale_pitch, q.scale);
        }
        if (left <= 0) continue;
        float w[8], b[8];
        load8<T>(static_cast<const T *>(p.weight) + c, left, w);
        load8<T>(static_cast<const T *>(p.bias) + c, left, b);
#pragma unroll
        for (int e = 0; e < 8; e++) f[k][e] = __builtin_fmaf(f[k][e] * r, w[e], b[e]);
        store8<T>(static_cast<T *>(p.y) + row * p.n + c, left, f[k]);
    }
}

// h = c r;  dx = r (g - mean g - h mean(g h)), g = dy w;  dw = sum dy h, db = sum dy over the rows: a workgroup's rows in registers, those that
// it has side by side joined in LDS, workgroups by norm_join_kernel.  A lane has eight numbers of a row, which leaves room for the next
// row's to be on their way (65536 x 1024 in bf16, two waves a row: 74 us; one wave with sixteen numbers a lane 108, with the next row's
// 110, at three waves a SIMD).
template <int WAVES> struct NormSlope {
    static constexpr int THREADS = WAVES < 4 ? 256 : WAVES * 64, ROWS = THREADS / 64 / WAVES;      // rows at once
};
template <typename T, int WAVES> __global__ __launch_bounds__(NormSlope<WAVES>::THREADS) void norm_slope_kernel(NormArgs p)
{
    using S = NormSlope<WAVES>;
    constexpr int ROWS = S::ROWS;
    __shared__ float sums32[2][ROWS][WAVES][2];
    extern __shared__ __attribute__((aligned(16))) float columns[];        // [2][n], joining ROWS > 1
    const int c = (threadIdx.x & (WAVES * 64 - 1)) * 8, left = p.n - c, group = threadIdx.x / (WAVES * 64);
    float w[8], dw[8], db[8];
    load8<T>(static_cast<const T *>(p.weight) + c, left, w);
#pragma unroll
    for (int e = 0; e < 8; e++) dw[e] = db[e] = 0.f;
    const float inv_n = 1.0f / (float)p.n;
    struct Row {
        Raw8<T> g;
        u32x2 bytes;
        int scale;
        float r;
    };
    auto load = [&](Row &o, int64_t row) {
        const bool in = row < p.rows;
        o.g.load(static_cast<const T *>(p.x) + row * p.ld + c, in ? left : 0);
        o.bytes = u32x2{0u, 0u}, o.scale = 127, o.r = 0.f;
        if (in) o.r = p.rstd[row];
        if (in && left > 0) {
            o.bytes = *reinterpret_cast<const u32x2 *>(p.values + row * p.value_pitch + c);
            o.scale = p.scales[row * p.scale_pitch + c / BLOCK];
        }
    };
    const int64_t step = (int64_t)gridDim.x * ROWS;
    int turn = 0;
    Row next;
    load(next, (int64_t)blockIdx.x * ROWS + group);
    for (int64_t first = (int64_t)blockIdx.x * ROWS; first < p.rows; first += step) {      // the same for all of the workgroup
        const int64_t row = first + group;
        const Row now = next;
        load(next, row + step);
        float g[8], h[8], s[2] = {0.f, 0.f};
        stands_for8(now.bytes, now.scale, h);
        now.g.unpack(g);
#pragma unroll
        for (int e = 0; e < 8; e++) {
            h[e] *= now.r;
            dw[e] = __builtin_fmaf(g[e], h[e], dw[e]);
            db[e] += g[e];
            g[e] *= w[e];
            s[0] += g[e];
            s[1] = __builtin_fmaf(g[e], h[e], s[1]);
        }
        if (p.y == nullptr) continue;
        row_sums<WAVES>(s, sums32[turn][group]);
        turn ^= 1;                                  // the next row's sums do not wait for the readers of these
        const float m0 = s[0] * inv_n, m1 = s[1] * inv_n;
#pragma unroll
        for (int e = 0; e < 8; e++) g[e] = now.r * (g[e] - m0 - h[e] * m1);
        if (row < p.rows) store8<T>(static_cast<T *>(p.y) + row * p.n + c, left, g);
    }
    if (p.part == nullptr) return;
    float *const part = p.part + (int64_t)blockIdx.x * 2 * p.n;
    if constexpr (ROWS > 1) {
        for (int k = 0; k < ROWS; k++) {
            if (group == k)
#pragma unroll
                for (int e = 0; e < 8; e++)
                    if (e < left) {
                        columns[c + e] = dw[e] + (k > 0 ? columns[c + e] : 0.f);
                        columns[p.n + c + e] = db[e] + (k > 0 ? columns[p.n + c + e] : 0.f);
                    }
            __syncthreads();
        }
        for (int i = threadIdx.x; i < 2 * p.n; i += S::THREADS) part[i] = columns[i];
    } else {
#pragma unroll
        for (int e = 0; e < 8; e++)
            if (e < left) part[c + e] = dw[e], part[p.n + c + e] = db[e];
    }
}
// the workgroups' sums of 64 columns, by sixteen waves
template <typename T> __global__ __launch_bounds__(1024) void norm_join_kernel(const float *part, int parts, int n, T *dw, T *db)
{
    __shared__ float sums[16][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, i = blockIdx.x * 64 + lane;
    float sum = 0.f;
    if (i < 2 * n)
#pragma unroll 8
        for (int k = wave; k < parts; k += 16) sum += part[(int64_t)k * 2 * n + i];
    sums[wave][lane] = sum;
    __syncthreads();
    if (wave != 0 || i >= 2 * n) return;
    sum = 0.f;
    for (int w = 0; w < 16; w++) sum += sums[w][lane];
    T *const to = i < n ? dw : db;
    if (to != nullptr) Elem<T>::store(to + (i < n ? i : i - n), sum);
}

// ------------------------------------------------------------------------------------------------ on the host
int check_blocks(const char *what, int64_t rows, int64_t n)
{
    VT_REQUIRE(rows > 0 && n > 0, VTDGE_ERR_ARG, "%s: %lld rows of %lld", what, (long long)rows, (long long)n);
    // sixteen threads of a launch each, of which there may be 2^32
    VT_REQUIRE(rows < (1ll << 28) && n <= (1 << 20) && rows * ceil_div(n, BLOCK) <= VTDGE_MAX_BLOCKS, VTDGE_ERR_UNSUPPORTED, "%s: %lld rows of %lld", what,
               (long long)rows, (long long)n);
    return VTDGE_OK;
}
QuantizeJob quantize_job(const void *from, int64_t ld, int64_t rows, int64_t n, void *blocks, bf16_t *expanded, int64_t expanded_pitch)
{
    QuantizeJob j{};
    j.from = from, j.ld = from != nullptr ? ld : 0, j.rows = (uint32_t)rows, j.n = (int)n, j.per_row = (uint32_t)ceil_div(n, BLOCK);
    if (blocks != nullptr) j.values = values_of(blocks), j.scales = scales_of(blocks, rows, n);
    j.value_pitch = value_pitch(n), j.scale_pitch = (int)scale_pitch(n);
    j.expanded = expanded, j.expanded_pitch = expanded_pitch;
    return j;
}
int launch_quantize(QuantizeArgs &a, int jobs, int dtype, const char *what, hipStream_t st)
{
    int64_t blocks = 0;
    for (int i = 0; i < jobs; i++) {
        blocks += ceil_div((int64_t)a.job[i].rows * a.job[i].per_row, 16);
        if (i == 0) a.first = (uint32_t)blocks;
    }
    VT_REQUIRE(blocks < (1 << 24), VTDGE_ERR_UNSUPPORTED, "%s: %lld workgroups", what, (long long)blocks);
    auto kern = dtype == VTDGE_F32 ? quantize_kernel<float> : quantize_kernel<bf16_t>;
    note_kernel(reinterpret_cast<const void *>(kern));
    kern<<<(unsigned)blocks, 256, 0, st>>>(a);
    return check_launch(what);
}

static int check_dtype(const char *what, int dtype)
{
    VT_REQUIRE(dtype == VTDGE_F32 || dtype == VTDGE_BF16, VTDGE_ERR_ARG, "%s: dtype %d", what, dtype);
    return VTDGE_OK;
}

// Waves of a row and chunks of a lane: one wave up to 16 numbers a lane, which needs no barrier (us, one wave / four: bf16 65536 x 1024 62 / 95,
// 4112 x 768 6.5 / 8.1; fp32 65536 x 768 90 / 100, 65536 x 1024 115 / 111), four beyond.
static void norm_shape(int n, int &waves, int &ch)
{
    waves = n <= 1024 ? 1 : 4;
    ch = (int)ceil_div(n, waves * 512);
    if (ch == 3) ch = 4;
}
// The same backward, a lane with eight numbers, see norm_slope_kernel.
static int slope_waves(int n)
{
    int waves = 1;
    while (waves * 512 < n) waves *= 2;
    return waves;
}
static int64_t norm_parts(int64_t rows, int n)
{
    const int waves = slope_waves(n);
    const int64_t at_once = waves < 4 ? 4 / waves : 1, most = (waves < 4 ? 4 : 16 / waves) * compute_units(), all = ceil_div(rows, at_once);
    return all < most ? all : most;
}

#define VT_NORM_CASE(T)                                                                                         \
    (waves == 1 ? (ch == 1 ? norm_keep_kernel<T, 1, 1> : norm_keep_kernel<T, 1, 2>)                             \
                : (ch == 1 ? norm_keep_kernel<T, 4, 1> : ch == 2 ? norm_keep_kernel<T, 4, 2> : norm_keep_kernel<T, 4, 4>))
#define VT_SLOPE_CASE(T)                                                                                        \
    (waves == 1 ? norm_slope_kernel<T, 1> : waves == 2 ? norm_slope_kernel<T, 2>                                \
     : waves == 4 ? norm_slope_kernel<T, 4> : waves == 8 ? norm_slope_kernel<T, 8> : norm_slope_kernel<T, 16>)

static int check_norm(const char *what, int64_t rows, int64_t n, int dtype)
{
    VT_STEP(check_dtype(what, dtype));
    VT_STEP(check_blocks(what, rows, n));
    VT_REQUIRE(n <= VTDGE_MAX_NORM_8BIT, VTDGE_ERR_UNSUPPORTED, "%s: rows of %lld, %d at most", what, (long long)n, VTDGE_MAX_NORM_8BIT);
    VT_REQUIRE(rows < (1 << 24), VTDGE_ERR_UNSUPPORTED, "%s: %lld rows, fewer than 2^24 are supported", what, (long long)rows);
    return VTDGE_OK;
}

}  // namespace vtdge

using namespace vtdge;

extern "C" int64_t vtdge_blocks_bytes(int64_t rows, int64_t n)
{
    if (check_blocks("blocks_bytes", rows, n) != VTDGE_OK) return -1;
    return blocks_bytes(rows, n);
}

extern "C" int vtdge_quantize_blocks(const void *x, int64_t ldx, int64_t rows, int64_t n, void *blocks, int dtype, void *stream)
{
    VT_STEP(check_dtype("quantize_blocks", dtype));
    VT_STEP(check_blocks("quantize_blocks", rows, n));
    VT_REQUIRE(x && blocks, VTDGE_ERR_ARG, "quantize_blocks: NULL operand");
    VT_REQUIRE(ldx >= n || rows == 1, VTDGE_ERR_ARG, "quantize_blocks: rows of %lld, %lld apart", (long long)n, (long long)ldx);
    VT_REQUIRE(((uintptr_t)blocks & 127) == 0, VTDGE_ERR_ARG, "quantize_blocks: blocks off their boundary");
    QuantizeArgs a{};
    a.job[0] = quantize_job(x, ldx, rows, n, blocks, nullptr, 0);
    return launch_quantize(a, 1, dtype, "quantize_blocks", (hipStream_t)stream);
}

extern "C" int vtdge_dequantize_blocks(const void *blocks, int64_t rows, int64_t n, void *out, int dtype, void *stream)
{
    VT_STEP(check_dtype("dequantize_blocks", dtype));
    VT_STEP(check_blocks("dequantize_blocks", rows, n));
    VT_REQUIRE(out && blocks, VTDGE_ERR_ARG, "dequantize_blocks: NULL operand");
    VT_REQUIRE(((uintptr_t)blocks & 127) == 0, VTDGE_ERR_ARG, "dequantize_blocks: blocks off their boundary");
    DequantizeArgs a{};
    a.values = values_of(blocks), a.scales = scales_of(blocks, rows, n), a.rows = (uint32_t)rows, a.per_row = (uint32_t)ceil_div(n, 8);
    a.n = (int)n, a.value_pitch = value_pitch(n), a.scale_pitch = (int)scale_pitch(n), a.to = out;
    auto kern = dtype == VTDGE_F32 ? dequantize_kernel<float> : dequantize_kernel<bf16_t>;
    note_kernel(reinterpret_cast<const void *>(kern));
    kern<<<(unsigned)ceil_div(rows * a.per_row, 256), 256, 0, (hipStream_t)stream>>>(a);
    return check_launch("dequantize_blocks");
}

static int gelu_args(const char *what, GeluArgs &a, const void *x, int64_t ldx, int64_t rows, int64_t n, const void *blocks, void *y, int dtype)
{
    VT_STEP(check_dtype(what, dtype));
    VT_STEP(check_blocks(what, rows, n));
    VT_REQUIRE(x && y, VTDGE_ERR_ARG, "%s: NULL operand", what);
    VT_REQUIRE(ldx >= n || rows == 1, VTDGE_ERR_ARG, "%s: rows of %lld, %lld apart", what, (long long)n, (long long)ldx);
    VT_REQUIRE(((uintptr_t)blocks & 127) == 0, VTDGE_ERR_ARG, "%s: blocks off their boundary", what);
    a.x = x, a.ld = ldx, a.rows = (uint32_t)rows, a.n = (int)n, a.y = y;
    if (blocks != nullptr) a.values = values_of(blocks), a.scales = scales_of(blocks, rows, n);
    a.value_pitch = value_pitch(n), a.scale_pitch = (int)scale_pitch(n);
    return VTDGE_OK;
}

extern "C" int vtdge_gelu_8bit(const void *x, int64_t ldx, int64_t rows, int64_t n, void *y, void *blocks, int dtype, void *stream)
{
    GeluArgs a{};
    VT_STEP(gelu_args("gelu_8bit", a, x, ldx, rows, n, blocks, y, dtype));
    a.per_row = (uint32_t)ceil_div(n, BLOCK);
    auto kern = dtype == VTDGE_F32 ? gelu_keep_kernel<float> : gelu_keep_kernel<bf16_t>;
    note_kernel(reinterpret_cast<const void *>(kern));
    kern<<<(unsigned)ceil_div(rows * a.per_row, 16), 256, 0, (hipStream_t)stream>>>(a);
    return check_launch("gelu_8bit");
}

extern "C" int vtdge_gelu_8bit_backward(const void *grad, int64_t ldg, int64_t rows, int64_t n, const void *blocks, void *dx, int dtype, void *stream)
{
    GeluArgs a{};
    VT_STEP(gelu_args("gelu_8bit_backward", a, grad, ldg, rows, n, blocks, dx, dtype));
    VT_REQUIRE(blocks, VTDGE_ERR_ARG, "gelu_8bit_backward: NULL operand");
    a.per_row = (uint32_t)ceil_div(n, 8);
    auto kern = dtype == VTDGE_F32 ? gelu_slope_kernel<float> : gelu_slope_kernel<bf16_t>;
    note_kernel(reinterpret_cast<const void *>(kern));
    kern<<<(unsigned)ceil_div(rows * a.per_row, 256), 256, 0, (hipStream_t)stream>>>(a);
    return check_launch("gelu_8bit_backward");
}

extern "C" int vtdge_layernorm_8bit(const void *x, int64_t ldx, const void *weight, const void *bias, float eps, int64_t rows, int64_t n, void *y,
                                    void *blocks, float *rstd, int dtype, void *stream)
{
    VT_STEP(check_norm("layernorm_8bit", rows, n, dtype));
    VT_REQUIRE(x && weight && bias && y && (blocks != nullptr) == (rstd != nullptr), VTDGE_ERR_ARG, "layernorm_8bit: NULL operand");
    VT_REQUIRE(ldx >= n || rows == 1, VTDGE_ERR_ARG, "layernorm_8bit: rows of %lld, %lld apart", (long long)n, (long long)ldx);
    VT_REQUIRE(((uintptr_t)blocks & 127) == 0, VTDGE_ERR_ARG, "layernorm_8bit: blocks off their boundary");
    NormArgs a{};
    a.x = x, a.ld = ldx, a.weight = weight, a.bias = bias, a.eps = eps, a.rows = rows, a.n = (int)n, a.y = y, a.rstd = rstd;
    if (blocks != nullptr) a.values = values_of(blocks), a.scales = scales_of(blocks, rows, n);
    a.value_pitch = (int)value_pitch(n), a.scale_pitch = (int)scale_pitch(n);
    a.blocks = (int)ceil_div(n, BLOCK);
    int waves, ch;
    norm_shape((int)n, waves, ch);
    auto kern = dtype == VTDGE_F32 ? VT_NORM_CASE(float) : VT_NORM_CASE(bf16_t);
    note_kernel(reinterpret_cast<const void *>(kern));
    kern<<<(unsigned)ceil_div(rows, 4 / waves), 256, 0, (hipStream_t)stream>>>(a);
    return check_launch("layernorm_8bit");
}

extern "C" int64_t vtdge_layernorm_8bit_backward_workspace(int64_t rows, int64_t n)
{
    if (check_norm("layernorm_8bit_backward_workspace", rows, n, VTDGE_F32) != VTDGE_OK) return -1;
    return norm_parts(rows, (int)n) * 2 * n * 4;
}

extern "C" int vtdge_layernorm_8bit_backward(const void *grad, int64_t ldg, const void *weight, const void *blocks, const float *rstd, int64_t rows,
                                             int64_t n, void *workspace, int64_t workspace_bytes, void *dx, void *dweight, void *dbias, int dtype,
                                             void *stream)
{
    VT_STEP(check_norm("layernorm_8bit_backward", rows, n, dtype));
    VT_REQUIRE(grad && weight && blocks && rstd && workspace, VTDGE_ERR_ARG, "layernorm_8bit_backward: NULL operand");
    VT_REQUIRE(ldg >= n || rows == 1, VTDGE_ERR_ARG, "layernorm_8bit_backward: rows of %lld, %lld apart", (long long)n, (long long)ldg);
    VT_REQUIRE(((uintptr_t)blocks & 127) == 0, VTDGE_ERR_ARG, "layernorm_8bit_backward: blocks off their boundary");
    const int64_t parts = norm_parts(rows, (int)n), bytes = parts * 2 * n * 4;
    VT_REQUIRE(workspace_bytes >= bytes && ((uintptr_t)workspace & 15) == 0, VTDGE_ERR_ARG, "layernorm_8bit_backward: workspace of %lld bytes, %lld needed",
               (long long)workspace_bytes, (long long)bytes);
    const bool columns = dweight != nullptr || dbias != nullptr;
    if (dx == nullptr && !columns) return VTDGE_OK;
    NormArgs a{};
    a.x = grad, a.ld = ldg, a.weight = weight, a.rows = rows, a.n = (int)n, a.y = dx, a.rstd = const_cast<float *>(rstd);
    a.values = values_of(blocks), a.scales = scales_of(blocks, rows, n), a.value_pitch = (int)value_pitch(n), a.scale_pitch = (int)scale_pitch(n);
    a.part = columns ? static_cast<float *>(workspace) : nullptr;
    const int waves = slope_waves((int)n);
    auto kern = dtype == VTDGE_F32 ? VT_SLOPE_CASE(float) : VT_SLOPE_CASE(bf16_t);
    note_kernel(reinterpret_cast<const void *>(kern));
    kern<<<(unsigned)parts, waves < 4 ? 256 : waves * 64, waves < 4 ? 2 * n * 4 : 0, (hipStream_t)stream>>>(a);
    VT_STEP(check_launch("layernorm_8bit_backward"));
    if (!columns) return VTDGE_OK;
    const unsigned blocks64 = (unsigned)ceil_div(2 * n, 64);
    if (dtype == VTDGE_F32) {
        note_kernel(reinterpret_cast<const void *>(norm_join_kernel<float>));
        norm_join_kernel<float><<<blocks64, 1024, 0, (hipStream_t)stream>>>(a.part, (int)parts, (int)n, (float *)dweight, (float *)dbias);
    } else {
        note_kernel(reinterpret_cast<const void *>(norm_join_kernel<bf16_t>));
        norm_join_kernel<bf16_t><<<blocks64, 1024, 0, (hipStream_t)stream>>>(a.part, (int)parts, (int)n, (bf16_t *)dweight, (bf16_t *)dbias);
    }
    return check_launch("layernorm_8bit_backward");
}
