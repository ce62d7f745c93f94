// One AdamW step over many tensors (gfx950):  p *= 1 - lr wd;  m = b1 m + (1 - b1) g;  v = b2 v + (1 - b2) g^2;
// p -= lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps), moments in fp32 or in 8 bits.
//
// Bound by memory: 28 bytes an element in fp32, 22 with bf16 weights, 16 and 10 with 8-bit moments.  The tensors of a launch are a
// table in its arguments (no copy to the device, nothing to keep between calls), a workgroup takes a chunk of one of them and finds
// it by halving.  A wave takes 256 consecutive elements at a time, four a lane: weights, gradients and moments all come in one load
// a lane, and the 256 are the block that shares a scale, so that its largest magnitude is one reduction over the wave.  Waves take one
// block each: while some wait others compute, with no loop to keep in order (four blocks a wave 10 to 20 percent slower).
// Measured: 103 M bf16 weights with 32-bit moments 367 us, 6.2 TB/s; the 5.7 M and 22 M fp32 weights of a vision transformer in 200
// tensors 32 us with 32-bit moments (5.1 TB/s) and 67 us with 8-bit ones (5.3 TB/s); a large copy reaches 4.9.
//
// Moments in 8 bits: the first as e4m3 over max|m| / 448, the second as e5m2 over max v / 57344.  Adam's slow decay (b2 = 0.999)
// is far below half a step of either (1/16 and 1/8), and would be lost under rounding to the nearest; a value is therefore rounded
// down or up at random, by 16 random bits added below the last bit that stays, a hash of the element's place in its tensor and of t:
// the same on every run, unbiased to 2^-17 of a step.  A second moment above zero does not become zero, where it would let a
// weight jump by m / eps.  What the codes are made from (m, v, their quotients by the scale) is rounded to fp32 at each
// operation as written, products and sums apart.  A block whose largest magnitude is below 2^-100 is stored as zeros.  Magnitudes
// compare as integers, where NaN is above infinity: a block with either gets a scale that shows it.
#include "common.h"

#include <math.h>

namespace vtdge {

constexpr int OPT_BLOCK = 256;                  // elements of a scale, and of a wave
constexpr int OPT_WAVES = 4;
constexpr int OPT_CHUNK = OPT_WAVES * OPT_BLOCK;        // elements of a workgroup: a block for each wave
constexpr int64_t OPT_MOST_CHUNKS = (1 << 24) - 1;      // of a launch: fewer than 2^32 threads

struct OptScalars {                             // of one step, in fp32; also what vtdge_adamw_scalars leaves on the device
    float decay, beta1, rest1, beta2, rest2, size, root, eps;
    uint32_t step;
};

// The tensors of a launch.  Addresses are below 2^48 and lie in words of 32 and halves of 16 bits, two in a word (scalar loads take
// words): 30 and 42 bytes a tensor in place of 40 and 56, so that the 200 of a vision transformer take two launches and three in
// place of three and four.
template <int BITS> struct OptTable {
    static constexpr int BUFFERS = BITS == 8 ? 6 : 4;         // weight, gradient, moments, their scales
    static constexpr int MOST = BITS == 8 ? 96 : 134;         // 4 KB of kernel arguments hold this many, an even number
    uint32_t low[BUFFERS][MOST], high[BUFFERS / 2][MOST];
    uint32_t first[MOST];                       // chunk it starts with
    uint32_t last[MOST / 2];                    // elements of its last chunk, 1 .. OPT_CHUNK
    uint32_t count, chunks;

    void put(int buffer, uint32_t at, const void *p)
    {
        const uint64_t a = (uint64_t)(uintptr_t)p;
        low[buffer][at] = (uint32_t)a;
        half(high[buffer / 2][at], buffer & 1, (uint32_t)(a >> 32));
    }
    static void half(uint32_t &word, uint32_t upper, uint32_t v) { word = upper ? (word & 0xffffu) | v << 16 : (word & 0xffff0000u) | v; }
    template <typename T> __device__ __forceinline__ T *get(int buffer, uint32_t at) const
    {
        const uintptr_t a = (uintptr_t)low[buffer][at] | (uintptr_t)(high[buffer / 2][at] >> (buffer & 1) * 16 & 0xffffu) << 32;
        return (T *)(__attribute__((address_space(1))) T *)a;        // global memory: no flat loads
    }
};
static_assert(sizeof(OptTable<8>) + sizeof(OptScalars) + 8 <= 4096 && sizeof(OptTable<32>) + sizeof(OptScalars) + 8 <= 4096, "arguments");

// ---- four elements of a lane: a vector where the tensor's buffers allow it, else one by one.  STREAM: past the caches, for weights,
// gradients and moments of more than the last one holds.
template <bool STREAM, typename V> __device__ __forceinline__ V get(const V *p)
{
    if constexpr (STREAM) return __builtin_nontemporal_load(p);
    else return *p;
}
template <bool STREAM, typename V> __device__ __forceinline__ void set(V *p, V v)
{
    if constexpr (STREAM) __builtin_nontemporal_store(v, p);
    else *p = v;
}
template <bool STREAM, typename T> __device__ __forceinline__ void load4(const T *p, int live, bool whole, float (&f)[4])
{
    if (!whole) {
#pragma unroll
        for (int e = 0; e < 4; e++) f[e] = e < live ? Elem<T>::load(p + e) : 0.f;
    } else if constexpr (sizeof(T) == 4) {
        const f32x4 r = get<STREAM>(reinterpret_cast<const f32x4 *>(p));
        f[0] = r.x, f[1] = r.y, f[2] = r.z, f[3] = r.w;
    } else {
        const u32x2 r = get<STREAM>(reinterpret_cast<const u32x2 *>(p));
        f[0] = bf16lo(r.x), f[1] = bf16hi(r.x), f[2] = bf16lo(r.y), f[3] = bf16hi(r.y);
    }
}
template <bool STREAM, typename T> __device__ __forceinline__ void store4(T *p, int live, bool whole, const float (&f)[4])
{
    if (!whole) {
#pragma unroll
        for (int e = 0; e < 4; e++)
            if (e < live) Elem<T>::store(p + e, f[e]);
    } else if constexpr (sizeof(T) == 4) {
        set<STREAM>(reinterpret_cast<f32x4 *>(p), f32x4{f[0], f[1], f[2], f[3]});
    } else {
        set<STREAM>(reinterpret_cast<u32x2 *>(p), u32x2{pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3])});
    }
}
__device__ __forceinline__ uint32_t load_codes(const uint8_t *p, int live, bool whole)
{
    if (whole) return *reinterpret_cast<const uint32_t *>(p);
    uint32_t c = 0;
#pragma unroll
    for (int e = 0; e < 4; e++)
        if (e < live) c |= (uint32_t)p[e] << (8 * e);
    return c;
}
__device__ __forceinline__ void store_codes(uint8_t *p, int live, bool whole, uint32_t c)
{
    if (whole) {
        *reinterpret_cast<uint32_t *>(p) = c;
    } else {
#pragma unroll
        for (int e = 0; e < 4; e++)
            if (e < live) p[e] = (uint8_t)(c >> (8 * e));
    }
}

// ---- 8-bit codes.  M bits of mantissa, SMALL the smallest normal number: FIRST is e4m3, else e5m2.
template <bool FIRST> __device__ __forceinline__ void decode4(uint32_t codes, float scale, float (&f)[4])
{
    f32x2 lo, hi;
    if constexpr (FIRST) {
        lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)codes, false);
        hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)codes, true);
    } else {
        lo = __builtin_amdgcn_cvt_pk_f32_bf8((int)codes, false);
        hi = __builtin_amdgcn_cvt_pk_f32_bf8((int)codes, true);
    }
    f[0] = lo.x * scale, f[1] = lo.y * scale, f[2] = hi.x * scale, f[3] = hi.y * scale;
}
// largest of the wave as an integer
__device__ __forceinline__ uint32_t wave_umax(uint32_t v)
{
#define VT_UMAX(ctrl, mask)                                                                                          \
    {                                                                                                                \
        const uint32_t o = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, ctrl, mask, 0xf, true);                  \
        v = v > o ? v : o;                                                                                           \
    }
    VT_UMAX(0x111, 0xf)
    VT_UMAX(0x112, 0xf)
    VT_UMAX(0x114, 0xf)
    VT_UMAX(0x118, 0xf)
    VT_UMAX(0x142, 0xa)
    VT_UMAX(0x143, 0xc)
#undef VT_UMAX
    return (uint32_t)__builtin_amdgcn_readlane((int)v, 63);
}
// the wave's 256 values as codes, and their scale
template <bool FIRST> __device__ __forceinline__ uint32_t encode4(const float (&f)[4], const uint32_t (&noise)[4], float &scale)
{
#pragma clang fp contract(off)
    constexpr float TOP = FIRST ? 448.f : 57344.f, SMALL = FIRST ? 0x1p-6f : 0x1p-14f;
    constexpr int DROP = FIRST ? 20 : 21;
    uint32_t most = 0;
#pragma unroll
    for (int e = 0; e < 4; e++) {
        const uint32_t a = __float_as_uint(f[e]) & 0x7fffffffu;
        most = most > a ? most : a;
    }
    most = wave_umax(most);
    const bool zero = most < 0x0d800000u;       // 2^-100
    scale = zero ? 0.f : __uint_as_float(most) * (1.0f / TOP);
    const float inverse = zero ? 0.f : TOP / __uint_as_float(most);
    float q[4];
#pragma unroll
    for (int e = 0; e < 4; e++) {
        const float x = fminf(fabsf(f[e]) * inverse, TOP);
        const float lift = x < SMALL ? SMALL : 0.f;            // in the octave above SMALL the last bit kept is that of the numbers below
        const uint32_t n = (FIRST ? noise[e] & 0xffffu : noise[e] >> 16) << (DROP - 16);
        const uint32_t kept = (__float_as_uint(x + lift) + n) & ~((1u << DROP) - 1);
        float r = __uint_as_float(kept) - lift;
        if (!FIRST && x > 0.f) r = fmaxf(r, 0x1p-16f);
        q[e] = __builtin_copysignf(r, f[e]);
    }
    uint32_t c = 0;
    if constexpr (FIRST) {
        c = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(q[0], q[1], 0, false);
        c = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(q[2], q[3], (int)c, true);
    } else {
        c = (uint32_t)__builtin_amdgcn_cvt_pk_bf8_f32(q[0], q[1], 0, false);
        c = (uint32_t)__builtin_amdgcn_cvt_pk_bf8_f32(q[2], q[3], (int)c, true);
    }
    return c;
}
// 32 random bits of an element: odd multipliers, the first 32 bits behind the point of the roots of 2, 3, 5 and 7, last bit set
__device__ __forceinline__ uint32_t dither(uint32_t place, uint32_t step)
{
    uint32_t h = place * 0x6a09e667u + step * 0xbb67ae85u;
    h = (h ^ (h >> 16)) * 0x3c6ef373u;
    h = (h ^ (h >> 15)) * 0xa54ff53bu;
    return h ^ (h >> 16);
}

// m / (sqrt(v) root + eps), the root and the quotient each off by a step of fp32 at most: a step's size, not what codes are made
// from.  Roots below 2^-48 are taken of 2^32 v, which is a normal number wherever v is not zero (v_sqrt_f32 takes others as zero).
__device__ __forceinline__ float change(float m, float v, float root, float eps)
{
    const bool small = v < 0x1p-96f;
    const float r = __builtin_amdgcn_sqrtf(small ? v * 0x1p32f : v);
    return m * __builtin_amdgcn_rcpf((small ? r * 0x1p-16f : r) * root + eps);
}

// A lane's four elements of a block of 256 with 8-bit moments; `live` of them are the tensor's.
template <typename T, bool STREAM> struct Lane {
    float p[4], g[4], sm, sv;
    uint32_t cm, cv;

    __device__ __forceinline__ Lane(const T *from, const T *grad, const uint8_t *m, const uint8_t *v, float m_scale, float v_scale, int live, bool whole)
        : sm(m_scale), sv(v_scale)
    {
        load4<STREAM>(from, live, whole, p);
        load4<STREAM>(grad, live, whole, g);
        cm = load_codes(m, live, whole), cv = load_codes(v, live, whole);
    }
    __device__ __forceinline__ void step(const OptScalars &s, T *to, uint8_t *m, uint8_t *v, float *ms, float *vs, int64_t place, int live, bool whole)
    {
#pragma clang fp contract(off)
        float fm[4], fv[4];
        decode4<true>(cm, sm, fm);
        decode4<false>(cv, sv, fv);
        uint32_t noise[4];
#pragma unroll
        for (int e = 0; e < 4; e++) {
            fm[e] = fm[e] * s.beta1 + g[e] * s.rest1;
            fv[e] = fv[e] * s.beta2 + g[e] * s.rest2 * g[e];
            if (e >= live) fm[e] = fv[e] = 0.f;                // (0 times a scale that is not finite)
            p[e] = p[e] * s.decay - s.size * change(fm[e], fv[e], s.root, s.eps);
            noise[e] = dither((uint32_t)(place + e), s.step);
        }
        const uint32_t em = encode4<true>(fm, noise, sm), ev = encode4<false>(fv, noise, sv);
        store4<STREAM>(to, live, whole, p);
        store_codes(m, live, whole, em);
        store_codes(v, live, whole, ev);
        if ((threadIdx.x & 63) == 0) *ms = sm, *vs = sv;
    }
};

template <typename T, int BITS, bool STREAM>
__global__ __launch_bounds__(64 * OPT_WAVES) void adamw_kernel(OptTable<BITS> t, OptScalars host, const OptScalars *__restrict__ device)
{
#pragma clang fp contract(off)
    const OptScalars s = device != nullptr ? *device : host;
    // the tensor of this chunk: the last one that starts at or before it
    uint32_t n = 0, end = t.count;
    while (end - n > 1) {
        const uint32_t mid = (n + end) >> 1;
        if (t.first[mid] <= blockIdx.x) n = mid;
        else end = mid;
    }
    const uint32_t chunk = blockIdx.x - t.first[n];
    const bool is_last = blockIdx.x + 1 == (n + 1 < t.count ? t.first[n + 1] : t.chunks);
    const int live = is_last ? (int)(t.last[n >> 1] >> (n & 1) * 16 & 0xffffu) : OPT_CHUNK;
    const int64_t base = (int64_t)chunk * OPT_CHUNK;
    T *const p = t.template get<T>(0, n);
    const T *const g = t.template get<const T>(1, n);
    const uint64_t places = (uint64_t)(uintptr_t)p | (uint64_t)(uintptr_t)g;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int block = __builtin_amdgcn_readfirstlane(wave), left = live - block * OPT_BLOCK, at = lane * 4;
    if (left <= 0) return;
    const int64_t i = base + block * OPT_BLOCK + at;
    if constexpr (BITS == 32) {
        float *const m = t.template get<float>(2, n) + i, *const v = t.template get<float>(3, n) + i;
        const bool whole = (places % (4 * sizeof(T))) == 0 && (((uintptr_t)m | (uintptr_t)v) & 15) == 0 && at + 4 <= left;
        float fp[4], fg[4], fm[4], fv[4];
        load4<STREAM>(p + i, left - at, whole, fp);
        load4<STREAM>(g + i, left - at, whole, fg);
        load4<STREAM>(m, left - at, whole, fm);
        load4<STREAM>(v, left - at, whole, fv);
#pragma unroll
        for (int e = 0; e < 4; e++) {
            fm[e] = fm[e] * s.beta1 + fg[e] * s.rest1;
            fv[e] = fv[e] * s.beta2 + fg[e] * s.rest2 * fg[e];
            fp[e] = fp[e] * s.decay - s.size * change(fm[e], fv[e], s.root, s.eps);
        }
        store4<STREAM>(p + i, left - at, whole, fp);
        store4<STREAM>(m, left - at, whole, fm);
        store4<STREAM>(v, left - at, whole, fv);
    } else {
        uint8_t *const m = t.template get<uint8_t>(2, n), *const v = t.template get<uint8_t>(3, n);
        const int64_t k = (int64_t)chunk * OPT_WAVES + block;
        float *const ms = t.template get<float>(4, n) + k, *const vs = t.template get<float>(5, n) + k;
        const bool vec = (places % (4 * sizeof(T))) == 0 && (((uintptr_t)m | (uintptr_t)v) & 3) == 0;
        if (vec && left >= OPT_BLOCK) Lane<T, STREAM>(p + i, g + i, m + i, v + i, *ms, *vs, 4, true).step(s, p + i, m + i, v + i, ms, vs, i, 4, true);
        else {                                                // lanes behind the tensor's end hold zeros
            const bool whole = vec && at + 4 <= left;
            Lane<T, STREAM>(p + i, g + i, m + i, v + i, *ms, *vs, left - at, whole).step(s, p + i, m + i, v + i, ms, vs, i, left - at, whole);
        }
    }
}

static OptScalars scalars_of(double lr, double beta1, double beta2, double eps, double decay, int64_t step)
{
    OptScalars s;
    s.decay = (float)(1.0 - lr * decay);
    s.beta1 = (float)beta1, s.rest1 = (float)(1.0 - beta1);
    s.beta2 = (float)beta2, s.rest2 = (float)(1.0 - beta2);
    s.size = (float)(lr / (1.0 - pow(beta1, (double)step)));
    s.root = (float)(1.0 / sqrt(1.0 - pow(beta2, (double)step)));
    s.eps = (float)eps;
    s.step = (uint32_t)step;
    return s;
}

__global__ void adamw_scalars_kernel(int64_t *step, int64_t skipped, int advance, const float *lr_dev, double lr, double beta1,
                                     double beta2, double eps, double decay, OptScalars *out)
{
    const int64_t t = *step + 1 - skipped;
    if (advance) *step += 1;
    if (lr_dev != nullptr) lr = (double)*lr_dev;
    OptScalars s;
    s.decay = (float)(1.0 - lr * decay);
    s.beta1 = (float)beta1, s.rest1 = (float)(1.0 - beta1);
    s.beta2 = (float)beta2, s.rest2 = (float)(1.0 - beta2);
    s.size = (float)(lr / (1.0 - pow(beta1, (double)t)));
    s.root = (float)(1.0 / sqrt(1.0 - pow(beta2, (double)t)));
    s.eps = (float)eps;
    s.step = (uint32_t)t;
    *out = s;
}

template <typename T, int BITS>
static int go_adamw(const vtdge_adamw_tensor *tensors, int count, const OptScalars &s, const OptScalars *device, hipStream_t st)
{
    // bytes of the call against the last cache's 256 MB: 22 M fp32 weights with 8-bit moments (355 MB) 75 us through the caches, 67 past
    // them, 103 M bf16 weights (2.3 GB) 401 and 365; 5.7 M fp32 weights (160 MB) 31.8 and 32.9
    double bytes = 0;
    for (int k = 0; k < count; k++) bytes += (3.0 * sizeof(T) + (BITS == 8 ? 4 : 16)) * tensors[k].n;
    auto kern = bytes > (256 << 20) ? adamw_kernel<T, BITS, true> : adamw_kernel<T, BITS, false>;
    OptTable<BITS> t{};
    int i = 0;
    while (i < count) {
        uint32_t k = 0;
        int64_t chunks = 0;
        for (; i < count && k < (uint32_t)OptTable<BITS>::MOST; i++) {
            const vtdge_adamw_tensor &x = tensors[i];
            if (x.n == 0) continue;
            const int64_t c = ceil_div(x.n, OPT_CHUNK);
            if (chunks + c > OPT_MOST_CHUNKS) break;
            t.put(0, k, x.param), t.put(1, k, x.grad), t.put(2, k, x.exp_avg), t.put(3, k, x.exp_avg_sq);
            if constexpr (BITS == 8) t.put(4, k, x.exp_avg_scale), t.put(5, k, x.exp_avg_sq_scale);
            t.first[k] = (uint32_t)chunks;
            t.half(t.last[k >> 1], k & 1, (uint32_t)(x.n - (c - 1) * OPT_CHUNK));
            chunks += c;
            k++;
        }
        if (k == 0) break;
        t.count = k;
        t.chunks = (uint32_t)chunks;
        note_kernel(reinterpret_cast<const void *>(kern));
        kern<<<dim3((unsigned)chunks), dim3(64 * OPT_WAVES), 0, st>>>(t, s, device);
        const int rc = check_launch("adamw");
        if (rc != VTDGE_OK) return rc;
    }
    return VTDGE_OK;
}

static bool bad_rates(double lr, double beta1, double beta2, double eps, double decay)
{
    return !(lr >= 0) || !(beta1 >= 0 && beta1 < 1) || !(beta2 >= 0 && beta2 < 1) || !(eps >= 0) || !(decay >= 0);
}

}  // namespace vtdge

using namespace vtdge;

extern "C" int vtdge_adamw_scalars(int64_t *step, int64_t skipped, int advance, const float *lr_dev, double lr, double beta1,
                                   double beta2, double eps, double weight_decay, void *scalars, void *stream)
{
    VT_REQUIRE(step && scalars, VTDGE_ERR_ARG, "adamw_scalars: NULL operand");
    VT_REQUIRE(skipped >= 0, VTDGE_ERR_ARG, "adamw_scalars: skipped is %lld", (long long)skipped);
    VT_REQUIRE(!bad_rates(lr, beta1, beta2, eps, weight_decay), VTDGE_ERR_ARG, "adamw_scalars: lr, betas, eps or weight_decay out of range");
    note_kernel(reinterpret_cast<const void *>(adamw_scalars_kernel));
    adamw_scalars_kernel<<<1, 1, 0, (hipStream_t)stream>>>(step, skipped, advance, lr_dev, lr, beta1, beta2, eps, weight_decay, (OptScalars *)scalars);
    return check_launch("adamw_scalars");
}

extern "C" int vtdge_adamw(const vtdge_adamw_tensor *tensors_host, int count, double lr, double beta1, double beta2, double eps,
                           double weight_decay, int64_t step, const void *scalars, int dtype, int state_bits, void *stream)
{
    VT_REQUIRE(count >= 0 && (tensors_host || count == 0), VTDGE_ERR_ARG, "adamw: bad table of %d tensors", count);
    VT_REQUIRE(dtype == VTDGE_F32 || dtype == VTDGE_BF16, VTDGE_ERR_ARG, "adamw: dtype %d", dtype);
    VT_REQUIRE(state_bits == 32 || state_bits == 8, VTDGE_ERR_UNSUPPORTED, "adamw: moments of %d bits", state_bits);
    VT_REQUIRE(scalars != nullptr || (step >= 1 && !bad_rates(lr, beta1, beta2, eps, weight_decay)), VTDGE_ERR_ARG,
               "adamw: step, lr, betas, eps or weight_decay out of range");
    const int64_t most = OPT_MOST_CHUNKS * OPT_CHUNK;
    for (int i = 0; i < count; i++) {
        const vtdge_adamw_tensor &x = tensors_host[i];
        VT_REQUIRE(x.n >= 0 && x.n <= most, VTDGE_ERR_ARG, "adamw: tensor %d has %lld elements", i, (long long)x.n);
        VT_REQUIRE(x.n == 0 || (x.param && x.grad && x.exp_avg && x.exp_avg_sq && (state_bits == 32 || (x.exp_avg_scale && x.exp_avg_sq_scale))),
                   VTDGE_ERR_ARG, "adamw: NULL operand in tensor %d", i);
        const uint64_t all = (uint64_t)(uintptr_t)x.param | (uint64_t)(uintptr_t)x.grad | (uint64_t)(uintptr_t)x.exp_avg | (uint64_t)(uintptr_t)x.exp_avg_sq
                             | (state_bits == 8 ? (uint64_t)(uintptr_t)x.exp_avg_scale | (uint64_t)(uintptr_t)x.exp_avg_sq_scale : 0);
        VT_REQUIRE(all >> 48 == 0, VTDGE_ERR_UNSUPPORTED, "adamw: tensor %d lies at or behind 2^48", i);
    }
    const OptScalars s = scalars != nullptr ? OptScalars{} : scalars_of(lr, beta1, beta2, eps, weight_decay, step);
    const OptScalars *device = (const OptScalars *)scalars;
    const hipStream_t st = (hipStream_t)stream;
    if (dtype == VTDGE_F32)
        return state_bits == 32 ? go_adamw<float, 32>(tensors_host, count, s, device, st) : go_adamw<float, 8>(tensors_host, count, s, device, st);
    return state_bits == 32 ? go_adamw<bf16_t, 32>(tensors_host, count, s, device, st) : go_adamw<bf16_t, 8>(tensors_host, count, s, device, st);
}
