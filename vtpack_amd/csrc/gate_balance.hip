// Balance of router gates (gfx950):  loss = E sum_e f_e P_e with f_e the fraction of the choices that fell on expert e and P_e its
// mean probability over the tokens, the counts behind f_e, and the gradient of the logits, E / T p_j (f_j - sum_e f_e p_e).
//
// Bound by reading the logits (and writing their gradient) once the tokens are many, by its launches when they are few.
// Sixteen lanes hold a token's logits, up to 32 each, so that every sum and maximum over the experts is four lane exchanges inside a
// row of the register file; a wave works on four tokens at a time.  The choice is made among integer keys, the logit's bits in an
// order where greater is greater (NaN above all) over the expert's complement, so that one maximum finds the largest logit and
// among equals the lowest expert: one 32-bit key where the logits have 16 bits, two where they have 32.
// A workgroup adds probabilities up in registers over its tokens and choices in LDS, and leaves a column of partial sums; one more
// workgroup joins them in their order.  Few tokens are one workgroup's, which joins its own.  Counts are whole numbers and the
// order of the sums is that of the launch: the same bits on every call.  The gradient works the probabilities out again.
#include "common.h"

namespace vtdge {

constexpr int BAL_THREADS = 256, BAL_GROUPS = BAL_THREADS / 16;      // tokens of a workgroup at a time
constexpr int BAL_WORKGROUPS = 512;                                  // columns of partial sums at most
constexpr int BAL_JOIN = 1024;

// ---- lane exchanges inside 16 lanes
template <int O> __device__ __forceinline__ int other16(int v)
{
    static_assert(O == 1 || O == 2 || O == 4 || O == 8, "inside a row of 16 lanes");
    if constexpr (O == 1) return __builtin_amdgcn_update_dpp(0, v, 0xB1, 0xf, 0xf, true);
    else if constexpr (O == 2) return __builtin_amdgcn_update_dpp(0, v, 0x4E, 0xf, 0xf, true);
    else if constexpr (O == 4) return __builtin_amdgcn_update_dpp(0, __builtin_amdgcn_update_dpp(0, v, 0x1B, 0xf, 0xf, true), 0x141, 0xf, 0xf, true);
    else return __builtin_amdgcn_update_dpp(0, v, 0x128, 0xf, 0xf, true);
}
__device__ __forceinline__ uint32_t umax16(uint32_t v)
{
    auto m = [](uint32_t a, int b) { return a > (uint32_t)b ? a : (uint32_t)b; };
    v = m(v, other16<1>((int)v));
    v = m(v, other16<2>((int)v));
    v = m(v, other16<4>((int)v));
    return m(v, other16<8>((int)v));
}
__device__ __forceinline__ float fmax16(float v)
{
    v = fmaxf(v, __int_as_float(other16<1>(__float_as_int(v))));
    v = fmaxf(v, __int_as_float(other16<2>(__float_as_int(v))));
    v = fmaxf(v, __int_as_float(other16<4>(__float_as_int(v))));
    return fmaxf(v, __int_as_float(other16<8>(__float_as_int(v))));
}
__device__ __forceinline__ float sum16(float v)
{
    v += __int_as_float(other16<1>(__float_as_int(v)));
    v += __int_as_float(other16<2>(__float_as_int(v)));
    v += __int_as_float(other16<4>(__float_as_int(v)));
    return v + __int_as_float(other16<8>(__float_as_int(v)));
}

// a float's bits in the order of its value, NaN (of either sign) above infinity, the two zeros equal; never 0 and never ~0
__device__ __forceinline__ uint32_t ordered(float f)
{
    const uint32_t u = __float_as_uint(f == 0.f ? 0.f : f);
    if (f != f) return 0xfffffffeu;
    return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}

// Value i of lane l is that of expert i * 16 + l: neighbouring lanes read neighbouring logits.
template <typename T, int N> struct Token {
    float p[N];                                  // logits, then probabilities; 0 behind the last expert

    __device__ __forceinline__ void load(const T *row, int E, int l)
    {
#pragma unroll
        for (int i = 0; i < N; i++) p[i] = i * 16 + l < E ? Elem<T>::load(row + i * 16 + l) : -INFINITY;
    }
    // the K largest, counted in `counts` (LDS) when `live`; K >= 1
    __device__ __forceinline__ void choose(int E, int l, int K, bool live, uint32_t *counts) const
    {
        uint32_t key[N];
#pragma unroll
        for (int i = 0; i < N; i++) key[i] = i * 16 + l < E ? ordered(p[i]) : 0u;
        if constexpr (sizeof(T) == 2) {          // the low half of a 16-bit logit's bits is its own sign's: the expert goes there
#pragma unroll
            for (int i = 0; i < N; i++) key[i] = i * 16 + l < E ? (key[i] & 0xffff0000u) | (0xffffu - (i * 16 + l)) : 0u;
            uint32_t below = ~0u;
            for (int k = 0; k < K; k++) {
                uint32_t best = 0;
#pragma unroll
                for (int i = 0; i < N; i++) {
                    const uint32_t c = key[i] < below ? key[i] : 0u;
                    best = best > c ? best : c;
                }
                below = umax16(best);
                if (l == 0 && live) atomicAdd(counts + (0xffffu - (below & 0xffffu)), 1u);
            }
        } else {
            for (int k = 0; k < K; k++) {
                uint32_t best = 0;
#pragma unroll
                for (int i = 0; i < N; i++) best = best > key[i] ? best : key[i];
                best = umax16(best);
                uint32_t first = 0;                            // the complement of the lowest expert with it
#pragma unroll
                for (int i = 0; i < N; i++)
                    if (key[i] == best) first = first > 0xffffu - (i * 16 + l) ? first : 0xffffu - (i * 16 + l);
                first = umax16(first);
                const int e = (int)(0xffffu - first);
#pragma unroll
                for (int i = 0; i < N; i++)
                    if (i * 16 + l == e) key[i] = 0u;
                if (l == 0 && live) atomicAdd(counts + e, 1u);
            }
        }
    }
    // the largest logit; -inf where a token has nothing to choose from (NaN is passed over here and shows in the sum)
    __device__ __forceinline__ float largest() const
    {
        float top = p[0];
#pragma unroll
        for (int i = 1; i < N; i++) top = fmaxf(top, p[i]);
        return fmax16(top);
    }
    // every logit -inf, none NaN
    __device__ __forceinline__ bool nothing(float top) const
    {
        float any = 0.f;
#pragma unroll
        for (int i = 0; i < N; i++) any = p[i] != p[i] ? 1.f : any;
        return fmax16(any) == 0.f && top == -INFINITY;
    }
    __device__ __forceinline__ void softmax(float top)
    {
        float total = 0.f;
#pragma unroll
        for (int i = 0; i < N; i++) {
            p[i] = __builtin_amdgcn_exp2f((p[i] - top) * 1.44269504f);
            total += p[i];
        }
        const float inv = 1.0f / sum16(total);
#pragma unroll
        for (int i = 0; i < N; i++) p[i] *= inv;
    }
};

struct BalArgs {
    const void *gate; int64_t pitch; const int64_t *indices; const uint8_t *mask; int64_t tokens; int E, K;
    float *sums; uint32_t *hits; uint32_t *lives;               // partial sums: [E][columns], [E][columns], [columns]
    float *loss; int64_t *counts; float *share;                 // results; share[e] = f_e, share[E] = E / tokens counted
};

// the columns of partial sums, by expert; `share` may not be read by anybody before
__device__ void join_columns(const float *sums, const uint32_t *hits, const uint32_t *lives, int columns, const BalArgs &a, int threads,
                             double *of_wave)
{
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = threads >> 6;
    uint32_t live = 0;
    for (int c = lane; c < columns; c += 64) live += lives[c];
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) live += __shfl_xor(live, o, WAVE);
    const double tokens = live > 0 ? (double)live : 1.0;
    double part = 0.0;
    for (int e = wave; e < a.E; e += waves) {
        double p = 0.0;
        uint64_t n = 0;
        for (int c = lane; c < columns; c += 64) {
            p += (double)sums[(int64_t)e * columns + c];
            n += hits[(int64_t)e * columns + c];
        }
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) {
            p += __shfl_xor(p, o, WAVE);
            n += __shfl_xor(n, o, WAVE);
        }
        const double f = (double)n / (tokens * a.K);
        part += f * (p / tokens);
        if (lane == 0) {
            a.counts[e] = (int64_t)n;
            a.share[e] = (float)f;
        }
    }
    if (lane == 0) of_wave[wave] = part;
    __syncthreads();
    if (threadIdx.x == 0) {
        double sum = 0.0;
        for (int w = 0; w < waves; w++) sum += of_wave[w];
        *a.loss = (float)(sum * a.E);
        a.share[a.E] = (float)(a.E / tokens);
    }
}

// ONE: the only workgroup, which joins its own sums
template <typename T, int N, bool ONE>
__global__ __launch_bounds__(BAL_THREADS) void gate_balance_kernel(BalArgs a)
{
    __shared__ uint32_t counts[16 * N];
    __shared__ float sums[16 * N];
    __shared__ uint32_t lives[4];
    __shared__ double of_wave[BAL_THREADS / 64];
    const int l = threadIdx.x & 15, group = threadIdx.x >> 4, wave = threadIdx.x >> 6;
    for (int e = threadIdx.x; e < 16 * N; e += BAL_THREADS) counts[e] = 0u;
    __syncthreads();
    float acc[N];
#pragma unroll
    for (int i = 0; i < N; i++) acc[i] = 0.f;
    uint32_t live = 0;
    const int64_t step = (int64_t)gridDim.x * BAL_GROUPS;
    // all lanes of a wave take the same number of turns
    for (int64_t t0 = (int64_t)blockIdx.x * BAL_GROUPS; t0 < a.tokens; t0 += step) {
        const int64_t t = t0 + group;
        Token<T, N> x;
        x.load(static_cast<const T *>(a.gate) + (t < a.tokens ? t : a.tokens - 1) * a.pitch, a.E, l);
        const float top = x.largest();
        const bool in = t < a.tokens && (a.mask == nullptr || a.mask[t] != 0) && !x.nothing(top);
        if (a.indices == nullptr) {
            x.choose(a.E, l, a.K, in, counts);
        } else if (in) {
            for (int k = l; k < a.K; k += 16) {
                const int64_t e = a.indices[t * a.K + k];
                if (e >= 0 && e < a.E) atomicAdd(counts + e, 1u);
            }
        }
        x.softmax(top);
        live += in && l == 0 ? 1u : 0u;
#pragma unroll
        for (int i = 0; i < N; i++) acc[i] += in ? x.p[i] : 0.f;
    }
    // the four groups of a wave, then the waves one after the other
#pragma unroll
    for (int i = 0; i < N; i++) {
        acc[i] += __shfl_xor(acc[i], 16, WAVE);
        acc[i] += __shfl_xor(acc[i], 32, WAVE);
    }
#pragma unroll
    for (int o = 16; o <= 32; o <<= 1) live += __shfl_xor(live, o, WAVE);
    for (int w = 0; w < BAL_THREADS / 64; w++) {
        if (wave == w && (threadIdx.x & 63) < 16) {
#pragma unroll
            for (int i = 0; i < N; i++) sums[i * 16 + l] = (w == 0 ? 0.f : sums[i * 16 + l]) + acc[i];
            if (l == 0) lives[w] = live;
        }
        __syncthreads();
    }
    if constexpr (ONE) {
        if (threadIdx.x == 0) lives[0] += lives[1] + lives[2] + lives[3];
        __syncthreads();
        join_columns(sums, counts, lives, 1, a, BAL_THREADS, of_wave);
    } else {
        for (int e = threadIdx.x; e < a.E; e += BAL_THREADS) {
            a.sums[(int64_t)e * gridDim.x + blockIdx.x] = sums[e];
            a.hits[(int64_t)e * gridDim.x + blockIdx.x] = counts[e];
        }
        if (threadIdx.x == 0) a.lives[blockIdx.x] = lives[0] + lives[1] + lives[2] + lives[3];
    }
}

__global__ __launch_bounds__(BAL_JOIN) void gate_balance_join_kernel(BalArgs a, int columns)
{
    __shared__ double of_wave[BAL_JOIN / 64];
    join_columns(a.sums, a.hits, a.lives, columns, a, BAL_JOIN, of_wave);
}

template <typename T, int N>
__global__ __launch_bounds__(BAL_THREADS) void gate_balance_backward_kernel(const T *__restrict__ gate, int64_t pitch,
                                                                            const uint8_t *__restrict__ mask, const float *__restrict__ share,
                                                                            const float *__restrict__ grad_loss, T *__restrict__ grad, int64_t tokens, int E)
{
    const int l = threadIdx.x & 15, group = threadIdx.x >> 4;
    const float scale = *grad_loss * share[E];
    float f[N];
#pragma unroll
    for (int i = 0; i < N; i++) f[i] = i * 16 + l < E ? share[i * 16 + l] : 0.f;
    const int64_t step = (int64_t)gridDim.x * BAL_GROUPS;
    for (int64_t t0 = (int64_t)blockIdx.x * BAL_GROUPS; t0 < tokens; t0 += step) {
        const int64_t t = t0 + group;
        Token<T, N> x;
        x.load(gate + (t < tokens ? t : tokens - 1) * pitch, E, l);
        const float top = x.largest();
        const bool in = t < tokens && (mask == nullptr || mask[t] != 0) && !x.nothing(top);
        x.softmax(top);
        float dot = 0.f;
#pragma unroll
        for (int i = 0; i < N; i++) dot = __builtin_fmaf(x.p[i], f[i], dot);
        dot = sum16(dot);
        if (t < tokens) {
#pragma unroll
            for (int i = 0; i < N; i++)
                if (i * 16 + l < E) Elem<T>::store(grad + t * E + i * 16 + l, in ? scale * (x.p[i] * (f[i] - dot)) : 0.f);
        }
    }
}

static int64_t balance_workgroups(int64_t tokens)
{
    const int64_t wanted = ceil_div(tokens, BAL_GROUPS);
    return wanted < BAL_WORKGROUPS ? wanted : BAL_WORKGROUPS;
}

template <typename T, int N> static int go_balance(BalArgs a, float *workspace, hipStream_t st)
{
    if (a.tokens <= 16 * BAL_GROUPS) {
        auto kern = gate_balance_kernel<T, N, true>;
        note_kernel(reinterpret_cast<const void *>(kern));
        kern<<<1, BAL_THREADS, 0, st>>>(a);
        return check_launch("gate_balance");
    }
    const int columns = (int)balance_workgroups(a.tokens);
    a.sums = workspace;
    a.hits = reinterpret_cast<uint32_t *>(workspace + (int64_t)a.E * columns);
    a.lives = a.hits + (int64_t)a.E * columns;
    auto kern = gate_balance_kernel<T, N, false>;
    note_kernel(reinterpret_cast<const void *>(kern));
    kern<<<columns, BAL_THREADS, 0, st>>>(a);
    const int rc = check_launch("gate_balance");
    if (rc != VTDGE_OK) return rc;
    note_kernel(reinterpret_cast<const void *>(gate_balance_join_kernel));
    gate_balance_join_kernel<<<1, BAL_JOIN, 0, st>>>(a, columns);
    return check_launch("gate_balance");
}

template <typename T, int N>
static int go_balance_backward(const void *gate, int64_t pitch, const uint8_t *mask, const float *share, const float *grad_loss, void *grad,
                               int64_t tokens, int E, hipStream_t st)
{
    const int64_t wanted = ceil_div(tokens, BAL_GROUPS), most = 8 * (int64_t)compute_units();
    auto kern = gate_balance_backward_kernel<T, N>;
    note_kernel(reinterpret_cast<const void *>(kern));
    kern<<<(unsigned)(wanted < most ? wanted : most), BAL_THREADS, 0, st>>>((const T *)gate, pitch, mask, share, grad_loss, (T *)grad, tokens, E);
    return check_launch("gate_balance_backward");
}

// values a lane holds, by the number of experts
#define VT_BY_EXPERTS(E, CALL)          \
    ((E) <= 16    ? CALL(1)             \
     : (E) <= 32  ? CALL(2)             \
     : (E) <= 64  ? CALL(4)             \
     : (E) <= 128 ? CALL(8)             \
     : (E) <= 192 ? CALL(12)            \
     : (E) <= 256 ? CALL(16)            \
                  : CALL(32))

}  // namespace vtdge

using namespace vtdge;

extern "C" int64_t vtdge_gate_balance_workspace(int64_t tokens, int E)
{
    if (tokens <= 16 * BAL_GROUPS || E < 1 || E > VTDGE_MAX_EXPERTS) return 0;
    return balance_workgroups(tokens) * (2 * (int64_t)E + 1) * 4;
}

extern "C" int vtdge_gate_balance(const void *gate, int64_t pitch, const int64_t *indices, const uint8_t *mask, int64_t tokens, int E,
                                  int K, void *workspace, int64_t workspace_bytes, float *loss, int64_t *counts, float *share, int dtype,
                                  void *stream)
{
    VT_REQUIRE(loss && counts && share, VTDGE_ERR_ARG, "gate_balance: NULL operand");
    VT_REQUIRE(tokens > 0 && gate, VTDGE_ERR_ARG, "gate_balance: %lld tokens", (long long)tokens);
    VT_REQUIRE(E >= 1 && pitch >= E, VTDGE_ERR_ARG, "gate_balance: %d experts in rows of %lld", E, (long long)pitch);
    VT_REQUIRE(E <= VTDGE_MAX_EXPERTS, VTDGE_ERR_UNSUPPORTED, "gate_balance: %d experts, at most %d", E, VTDGE_MAX_EXPERTS);
    VT_REQUIRE(K >= 1 && K <= VTDGE_MAX_EXPERTS && (indices || K <= E), VTDGE_ERR_ARG, "gate_balance: %d choices of %d experts", K, E);
    VT_REQUIRE(tokens < (int64_t)1 << 31, VTDGE_ERR_UNSUPPORTED, "gate_balance: %lld tokens", (long long)tokens);
    VT_REQUIRE(dtype == VTDGE_F32 || dtype == VTDGE_BF16, VTDGE_ERR_ARG, "gate_balance: dtype %d", dtype);
    const int64_t need = vtdge_gate_balance_workspace(tokens, E);
    VT_REQUIRE(need == 0 || (workspace && workspace_bytes >= need), VTDGE_ERR_ARG, "gate_balance: workspace of %lld bytes, %lld needed",
               (long long)workspace_bytes, (long long)need);
    const BalArgs a{gate, pitch, indices, mask, tokens, E, K, nullptr, nullptr, nullptr, loss, counts, share};
    const hipStream_t st = (hipStream_t)stream;
#define VT_F32(N) go_balance<float, N>(a, (float *)workspace, st)
#define VT_BF16(N) go_balance<bf16_t, N>(a, (float *)workspace, st)
    return dtype == VTDGE_F32 ? VT_BY_EXPERTS(E, VT_F32) : VT_BY_EXPERTS(E, VT_BF16);
#undef VT_F32
#undef VT_BF16
}

extern "C" int vtdge_gate_balance_backward(const void *gate, int64_t pitch, const uint8_t *mask, const float *share, const float *grad_loss,
                                           void *grad, int64_t tokens, int E, int dtype, void *stream)
{
    VT_REQUIRE(gate && share && grad_loss && grad, VTDGE_ERR_ARG, "gate_balance_backward: NULL operand");
    VT_REQUIRE(tokens > 0 && E >= 1 && pitch >= E, VTDGE_ERR_ARG, "gate_balance_backward: bad sizes");
    VT_REQUIRE(E <= VTDGE_MAX_EXPERTS, VTDGE_ERR_UNSUPPORTED, "gate_balance_backward: %d experts, at most %d", E, VTDGE_MAX_EXPERTS);
    VT_REQUIRE(dtype == VTDGE_F32 || dtype == VTDGE_BF16, VTDGE_ERR_ARG, "gate_balance_backward: dtype %d", dtype);
    const hipStream_t st = (hipStream_t)stream;
#define VT_F32(N) go_balance_backward<float, N>(gate, pitch, mask, share, grad_loss, grad, tokens, E, st)
#define VT_BF16(N) go_balance_backward<bf16_t, N>(gate, pitch, mask, share, grad_loss, grad, tokens, E, st)
    return dtype == VTDGE_F32 ? VT_BY_EXPERTS(E, VT_F32) : VT_BY_EXPERTS(E, VT_BF16);
#undef VT_F32
#undef VT_BF16
}
