// Blocks of 128 8-bit numbers with a power of two, shared by the kernels that make and read them.
#pragma once
#include "gradient_product.h"

namespace vtdge {

constexpr int BLOCK = 128;
constexpr int LEAST_SCALE = 17;                     // e = -110
constexpr uint32_t INFINITE = 0x7f800000u, MOST_ROUNDED_DOWN = 0x7f600000u;      // above the second, e = 120 and 256 2^120 is no fp32 number

// A buffer of blocks: rows of values, filled up with zeros to whole blocks; behind them rows of scales, filled up to whole words.
inline int64_t value_pitch(int64_t n) { return ceil_div(n, BLOCK) * BLOCK; }
inline int64_t scale_pitch(int64_t n) { return ceil_div(ceil_div(n, BLOCK), 4) * 4; }
inline int64_t blocks_bytes(int64_t rows, int64_t n) { return rows * (value_pitch(n) + scale_pitch(n)); }
inline unsigned char *values_of(const void *blocks) { return static_cast<unsigned char *>(const_cast<void *>(blocks)); }
inline unsigned char *scales_of(const void *blocks, int64_t rows, int64_t n) { return values_of(blocks) + rows * value_pitch(n); }

struct QuantizeJob {
    const void *from; int64_t ld; uint32_t rows, per_row; int n;       // nullable: the blocks are there; per_row: blocks
    unsigned char *values, *scales; int64_t value_pitch; int scale_pitch;      // nullable
    bf16_t *expanded; int64_t expanded_pitch;       // nullable: the numbers as bf16, zeros behind the last of a row
};
struct QuantizeArgs {
    QuantizeJob job[2];
    uint32_t first;                                 // workgroups of the first
};
struct DequantizeArgs {
    const unsigned char *values, *scales; uint32_t rows, per_row; int n, scale_pitch; int64_t value_pitch;      // per_row: vectors of eight
    void *to;
};
struct GeluArgs {
    const void *x; int64_t ld; uint32_t rows, per_row; int n;
    void *y; unsigned char *values, *scales; int64_t value_pitch; int scale_pitch;
};
struct NormArgs {
    const void *x; int64_t ld; const void *weight, *bias; float eps; int64_t rows; int n, blocks;
    void *y; unsigned char *values, *scales; int value_pitch, scale_pitch; float *rstd, *part;
};

int check_blocks(const char *what, int64_t rows, int64_t n);
QuantizeJob quantize_job(const void *from, int64_t ld, int64_t rows, int64_t n, void *blocks, bf16_t *expanded, int64_t expanded_pitch);
int launch_quantize(QuantizeArgs &a, int jobs, int dtype, const char *what, hipStream_t st);

// ------------------------------------------------------------------------------------------------ eight numbers of a lane
// `left` of them are there (fewer than one: none), zeros in the place of the others.  Vectors need not lie on 16-byte boundaries: one load
// or store takes them from any boundary of their type.
template <typename T> __device__ __forceinline__ void load8(const T *from, int64_t left, float (&f)[8])
{
    using V = typename Loose<T>::vector;
    if (left >= 8) {
#pragma unroll
        for (int e = 0; e < 8; e += Elem<T>::VEC) Elem<T>::unpack(*reinterpret_cast<const V *>(from + e), f + e);
    } else {
#pragma unroll
        for (int e = 0; e < 8; e++) f[e] = e < left ? Elem<T>::load(from + e) : 0.f;
    }
}
template <typename T> __device__ __forceinline__ void store8(T *to, int64_t left, const float (&f)[8])
{
    using V = typename Loose<T>::vector;
    if (left >= 8) {
#pragma unroll
        for (int e = 0; e < 8; e += Elem<T>::VEC) *reinterpret_cast<V *>(to + e) = Elem<T>::pack(f + e);
    } else {
#pragma unroll
        for (int e = 0; e < 8; e++)
            if (e < left) Elem<T>::store(to + e, f[e]);
    }
}

// the same in two steps, for loads that go out early: as they lie in memory, and as fp32
template <typename T> struct Raw8 {
    static constexpr int N = 8 / Elem<T>::VEC;
    u32x4 v[N];
    __device__ __forceinline__ void load(const T *from, int64_t left)
    {
        using V = typename Loose<T>::vector;
        if (left >= 8) {
#pragma unroll
            for (int e = 0; e < N; e++) v[e] = reinterpret_cast<const V *>(from)[e];
            return;
        }
        float f[8];
        load8<T>(from, left, f);
#pragma unroll
        for (int e = 0; e < N; e++) v[e] = Elem<T>::pack(f + e * Elem<T>::VEC);
    }
    __device__ __forceinline__ void unpack(float (&f)[8]) const
    {
#pragma unroll
        for (int e = 0; e < N; e++) Elem<T>::unpack(v[e], f + e * Elem<T>::VEC);
    }
};

// the largest of sixteen lanes, in each of them
template <int CTRL> __device__ __forceinline__ uint32_t lane_max(uint32_t v)
{
    const uint32_t o = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, true);
    return v > o ? v : o;
}
__device__ __forceinline__ uint32_t max16(uint32_t v)
{
    // a neighbour, the other pair, the half row mirrored, the row mirrored
    return lane_max<0x140>(lane_max<0x141>(lane_max<0x4E>(lane_max<0xB1>(v))));
}

struct Rounded {
    u32x2 bytes; int scale;
};
// The block of sixteen lanes with eight numbers each (all of the wave's lanes take part).
__device__ __forceinline__ Rounded round8(const float (&f)[8])
{
    uint32_t top = 0;
#pragma unroll
    for (int e = 0; e < 8; e++) {
        const uint32_t a = __float_as_uint(f[e]) & 0x7fffffffu;
        top = top > a ? top : a;
    }
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; e++) v[e] = f[e];
    const bool odd = __any(top > MOST_ROUNDED_DOWN);      // rare: without infinities and NaN, and nothing above 240 2^120
    if (odd) {
        top = 0;
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const uint32_t a = __float_as_uint(f[e]) & 0x7fffffffu;
            if (a < INFINITE) top = top > a ? top : a;
        }
    }
    top = max16(top);
    // 448 = 1.75 * 2^8
    int scale = (int)(top >> 23) - 8 + ((top & 0x7fffffu) > 0x600000u ? 1 : 0);
    scale = scale > LEAST_SCALE ? scale : LEAST_SCALE;
    const float inv = __uint_as_float((uint32_t)(254 - scale) << 23);
    if (odd) {
#pragma unroll
        for (int e = 0; e < 8; e++)
            v[e] = (__float_as_uint(f[e]) & 0x7fffffffu) >= INFINITE ? __uint_as_float(0x7fc00000u)
                   : scale == 247 ? __builtin_amdgcn_fmed3f(f[e], -0x1.ep127f, 0x1.ep127f) : f[e];
    }
    Rounded r;
    r.scale = scale;
    int lo = 0, hi = 0;
    lo = __builtin_amdgcn_cvt_pk_fp8_f32(v[0] * inv, v[1] * inv, lo, false);
    lo = __builtin_amdgcn_cvt_pk_fp8_f32(v[2] * inv, v[3] * inv, lo, true);
    hi = __builtin_amdgcn_cvt_pk_fp8_f32(v[4] * inv, v[5] * inv, hi, false);
    hi = __builtin_amdgcn_cvt_pk_fp8_f32(v[6] * inv, v[7] * inv, hi, true);
    r.bytes = u32x2{(uint32_t)lo, (uint32_t)hi};
    return r;
}
// scale byte of a block; behind the last of a row also the bytes that fill its word
__device__ __forceinline__ void put_scale(unsigned char *row, int block, int blocks, int pitch, int scale)
{
    row[block] = (unsigned char)scale;
    if (block == blocks - 1)
        for (int i = blocks; i < pitch; i++) row[i] = 127;
}

// 2^(byte - 127); 255 is NaN
__device__ __forceinline__ float scale_value(int byte)
{
    return __uint_as_float(byte == 0 ? 0x00400000u : byte == 255 ? 0x7fc00000u : (uint32_t)byte << 23);
}
__device__ __forceinline__ void stands_for8(const u32x2 &bytes, int scale, float (&f)[8])
{
    const float s = scale_value(scale);
    const f32x2 a = __builtin_amdgcn_cvt_pk_f32_fp8((int)bytes.x, false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)bytes.x, true);
    const f32x2 c = __builtin_amdgcn_cvt_pk_f32_fp8((int)bytes.y, false), d = __builtin_amdgcn_cvt_pk_f32_fp8((int)bytes.y, true);
    f[0] = a.x * s, f[1] = a.y * s, f[2] = b.x * s, f[3] = b.y * s;
    f[4] = c.x * s, f[5] = c.y * s, f[6] = d.x * s, f[7] = d.y * s;
}
__device__ __forceinline__ u32x4 expand8(const u32x2 &bytes, int scale)
{
    float f[8];
    stands_for8(bytes, scale, f);
    return Elem<bf16_t>::pack(f);
}

// ------------------------------------------------------------------------------------------------ GELU
// x Phi(x) = max(x, 0) - a Phi(-a), a = |x|.  fp32: gelu_fn.  bf16: Phi(-a) is 2 to a polynomial of degree 7, minimax on [0, 10] with the errors up to 4
// weighed four times: 7.2e-5 of the value up to 4, a twenty-seventh of half a bf16 step at its smallest, 2.9e-4 up to 10.  Behind that the value is below
// 8e-23 and the polynomial, whose first coefficient is negative, goes on falling, a quarter off at most.  (1/2 and an odd polynomial on a clamped
// argument, as gelu_fn, leaves 5e-5 |x| in place of nothing below -4.)  +inf is held back from a, NaN is not; -inf is NaN, as inf * 0.
// A Linear of 65536 x 1024 x 4096: 386 us, with degree 9 and 1.1e-5 off 397, by gelu_fn 380.
template <typename T> __device__ __forceinline__ float gelu_value(float v);
template <> __device__ __forceinline__ float gelu_value<float>(float v) { return gelu_fn<float>(v); }
template <> __device__ __forceinline__ float gelu_value<bf16_t>(float v)
{
    const float w = __builtin_elementwise_minimum(v, 64.f), a = fabsf(w);
    float q = -8.870287459e-07f;
    q = __builtin_fmaf(q, a, 3.805294677e-05f);
    q = __builtin_fmaf(q, a, -7.008872890e-04f);
    q = __builtin_fmaf(q, a, 7.399650225e-03f);
    q = __builtin_fmaf(q, a, -5.122005295e-02f);
    q = __builtin_fmaf(q, a, -4.616900438e-01f);
    q = __builtin_fmaf(q, a, -1.149819189e+00f);
    q = __builtin_fmaf(q, a, -1.000101819e+00f);
    return __builtin_fmaf(-a, __builtin_amdgcn_exp2f(q), __builtin_elementwise_max(v, 0.f));
}

// the sum of a wave's lanes, in each of them
__device__ __forceinline__ float wave_total(float v) { return wave_sum(v); }
template <int CTRL, int ROWS> __device__ __forceinline__ double dpp_add(double v)
{
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)u, CTRL, ROWS, 0xf, true);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(u >> 32), CTRL, ROWS, 0xf, true);
    return v + __builtin_bit_cast(double, ((uint64_t)hi << 32) | lo);
}
__device__ __forceinline__ double wave_total(double v)
{
    v = dpp_add<0x142, 0xa>(dpp_add<0x118, 0xf>(dpp_add<0x114, 0xf>(dpp_add<0x112, 0xf>(dpp_add<0x111, 0xf>(v)))));
    v = dpp_add<0x143, 0xc>(v);                     // as wave_sum: the total in the last lane
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)u, 63), hi = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(u >> 32), 63);
    return __builtin_bit_cast(double, ((uint64_t)hi << 32) | lo);
}

}  // namespace vtdge
