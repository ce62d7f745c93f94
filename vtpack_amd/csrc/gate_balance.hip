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
// Measured: 128 tokens of 3 in fp32 5.0 + 3.0 us (forward, gradient); 65536 of 3 in bf16 7.6 + 3 + 5.4; 131071 of 160, the 6 largest, masked, in
// bf16 28 + 5 + 17: there the choice bounds the forward (six times the maximum of ten logits a lane and an exchange), the
// gradient moves its 84 MB at 4.8 TB/s.
#include "common.h"

namespace vtdge {

// threads of a workgroup, 16 a token: as many waves as a compute unit may hold with the registers of N logits a lane
__host__ __device__ constexpr int balance_threads(int n) { return n <= 12 ? 1024 : 512; }
constexpr int BAL_BACKWARD = 256;
constexpr int BAL_WORKGROUPS = 256;                                  // columns of partial sums: one vector a lane of the wave that joins them
constexpr int BAL_JOIN = 1024;

// ---- lane exchanges inside 16 lanes
// (rotations: after 8, 4, 2 and 1 lanes every lane has met all others, in pairs of the same two sums, so that all end with the same bits)
template <int O> __device__ __forceinline__ int other16(int v)
{
    static_assert(O == 1 || O == 2 || O == 4 || O == 8, "inside a row of 16 lanes");
    return __builtin_amdgcn_update_dpp(0, v, 0x120 + O, 0xf, 0xf, true);
}
__device__ __forceinline__ uint32_t umax16(uint32_t v)
{
    auto m = [](uint32_t a, int b) { return a > (uint32_t)b ? a : (uint32_t)b; };
    v = m(v, other16<8>((int)v));
    v = m(v, other16<4>((int)v));
    v = m(v, other16<2>((int)v));
    return m(v, other16<1>((int)v));
}
__device__ __forceinline__ float fmax16(float v)
{
    v = fmaxf(v, __int_as_float(other16<8>(__float_as_int(v))));
    v = fmaxf(v, __int_as_float(other16<4>(__float_as_int(v))));
    v = fmaxf(v, __int_as_float(other16<2>(__float_as_int(v))));
    return fmaxf(v, __int_as_float(other16<1>(__float_as_int(v))));
}
__device__ __forceinline__ float sum16(float v)
{
    v += __int_as_float(other16<8>(__float_as_int(v)));
    v += __int_as_float(other16<4>(__float_as_int(v)));
    v += __int_as_float(other16<2>(__float_as_int(v)));
    return v + __int_as_float(other16<1>(__float_as_int(v)));
}

// a float's bits in the order of its value, all NaN alike above infinity, the two zeros equal; never 0
__device__ __forceinline__ uint32_t ordered(float f)
{
    const uint32_t u = __float_as_uint(f + 0.f);
    return f != f ? 0xffffffffu : u ^ ((uint32_t)((int32_t)u >> 31) | 0x80000000u);
}

// Values 2 j and 2 j + 1 of lane l are those of experts 32 j + 2 l and the next: one load for two where the rows allow it (PAIRS),
// neighbouring lanes side by side.  FULL: PAIRS, and 16 N experts, so that none has to be left out.
enum { ONE_BY_ONE, PAIRS, FULL };
template <typename T, int N> struct Token {
    float p[N];                                  // logits, then probabilities; -inf, then 0 behind the last expert
    static __device__ __forceinline__ int expert(int i, int l) { return (i >> 1) * 32 + 2 * l + (i & 1); }

    template <int WAY> __device__ __forceinline__ void load(const T *row, int E, int l)
    {
#pragma unroll
        for (int i = 0; i < N; i += 2) {
            const int e = expert(i, l);
            if constexpr (WAY == ONE_BY_ONE) {
                const float a = Elem<T>::load(row + min(e, E - 1)), b = Elem<T>::load(row + min(e + 1, E - 1));
                p[i] = e < E ? a : -INFINITY;
                p[i + 1] = e + 1 < E ? b : -INFINITY;
            } else {
                const T *const at = row + (WAY == FULL ? e : min(e, E - 2));
                if constexpr (sizeof(T) == 2) {
                    const uint32_t w = *reinterpret_cast<const uint32_t *>(at);
                    p[i] = bf16lo(w), p[i + 1] = bf16hi(w);
                } else {
                    const f32x2 w = *reinterpret_cast<const f32x2 *>(at);
                    p[i] = w.x, p[i + 1] = w.y;
                }
                if (WAY == PAIRS && e >= E) p[i] = p[i + 1] = -INFINITY;
            }
        }
    }
    // the K largest, counted in `counts` (LDS) when `live`; K >= 1
    template <int WAY> __device__ __forceinline__ void choose(int E, int l, int K, bool live, uint32_t *counts) const
    {
        uint32_t key[N];
        if constexpr (sizeof(T) == 2) {          // a 16-bit logit leaves half of the key to the expert
#pragma unroll
            for (int i = 0; i < N; i++) key[i] = WAY == FULL || expert(i, l) < E ? (ordered(p[i]) & 0xffff0000u) | (0xffffu - expert(i, l)) : 0u;
            // what is chosen already is at or above `chosen`: of differences modulo 2^32, those of smaller keys are the large ones
            uint32_t chosen = 0;
            for (int k = 0; k < K; k++) {
                uint32_t best = 0;
#pragma unroll
                for (int i = 0; i < N; i++) {
                    const uint32_t c = key[i] - chosen;
                    best = best > c ? best : c;
                }
                chosen += umax16(best);
                if (l == 0 && live) atomicAdd(counts + (0xffffu - (chosen & 0xffffu)), 1u);
            }
        } else {
#pragma unroll
            for (int i = 0; i < N; i++) key[i] = WAY == FULL || expert(i, l) < E ? ordered(p[i]) : 0u;
            for (int k = 0; k < K; k++) {
                uint32_t best = 0;
#pragma unroll
                for (int i = 0; i < N; i++) best = best > key[i] ? best : key[i];
                best = umax16(best);
                uint32_t first = 0;                            // the complement of the lowest expert with it
#pragma unroll
                for (int i = N - 1; i >= 0; i--) first = key[i] == best ? 0xffffu - expert(i, l) : first;
                first = umax16(first);
                const int e = (int)(0xffffu - first);
#pragma unroll
                for (int i = 0; i < N; i++) key[i] = expert(i, l) == e ? 0u : key[i];
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
        if (__ballot(top == -INFINITY) == 0) return false;
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
    float *sums; uint32_t *hits; uint32_t *lives;               // partial sums: [E][columns], [E][columns], [columns], 256 columns
    float *loss; int64_t *counts; float *share;                 // results; share[e] = f_e, share[E] = E / tokens counted
};

__device__ __forceinline__ double sum16(double v)
{
    auto add = [](double v, auto other) {
        const uint64_t u = (uint64_t)__double_as_longlong(v);
        return v + __longlong_as_double((long long)(((uint64_t)(uint32_t)other((int)(u >> 32)) << 32) | (uint32_t)other((int)(uint32_t)u)));
    };
    v = add(v, [](int x) { return other16<8>(x); });
    v = add(v, [](int x) { return other16<4>(x); });
    v = add(v, [](int x) { return other16<2>(x); });
    return add(v, [](int x) { return other16<1>(x); });
}

// The columns of partial sums, by expert.  VECS: 256 columns, sixteen lanes an expert; else a single one, in LDS.
template <bool VECS>
__device__ void join_columns(const float *sums, const uint32_t *hits, const uint32_t *lives, const BalArgs &a, int threads, double *of_wave)
{
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = threads >> 6, l = lane & 15;
    uint32_t live = 0;
    if constexpr (VECS) {
        const u32x4 v = reinterpret_cast<const u32x4 *>(lives)[lane];
        live = v.x + v.y + v.z + v.w;
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) live += __shfl_xor(live, o, WAVE);
    } else {
        live = *lives;
    }
    const double tokens = live > 0 ? (double)live : 1.0;
    double part = 0.0;
    for (int e0 = wave * 4; e0 < a.E; e0 += waves * 4) {
        const int e = e0 + (lane >> 4), at = e < a.E ? e : a.E - 1;
        double p, n;                                    // (counts are below 2^41: whole in a double)
        if constexpr (VECS) {
            f32x4 f[4];
            u32x4 h[4];
#pragma unroll
            for (int k = 0; k < 4; k++) {
                f[k] = reinterpret_cast<const f32x4 *>(sums)[at * 64 + k * 16 + l];
                h[k] = reinterpret_cast<const u32x4 *>(hits)[at * 64 + k * 16 + l];
            }
            p = n = 0.0;
#pragma unroll
            for (int k = 0; k < 4; k++) {
                p += ((double)f[k].x + f[k].y) + ((double)f[k].z + f[k].w);
                n += ((double)h[k].x + h[k].y) + ((double)h[k].z + h[k].w);
            }
            p = sum16(p);
            n = sum16(n);
        } else {
            p = sums[at], n = hits[at];
        }
        const double f = n / (tokens * a.K);
        if (l == 0 && e < a.E) {
            part += f * (p / tokens);
            a.counts[e] = (int64_t)n;
            a.share[e] = (float)f;
        }
    }
#pragma unroll
    for (int o = 32; o >= 16; o >>= 1) part += __shfl_xor(part, o, WAVE);
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
template <typename T, int N, int WAY, bool ONE>
__global__ __launch_bounds__(balance_threads(N)) void gate_balance_kernel(BalArgs a)
{
    constexpr int BAL_THREADS = balance_threads(N), BAL_GROUPS = BAL_THREADS / 16;
    __shared__ uint32_t counts[16 * N];
    __shared__ float sums[16 * N];
    __shared__ uint32_t lives[BAL_THREADS / 64];
    __shared__ double of_wave[BAL_THREADS / 64];
    const int l = threadIdx.x & 15, group = threadIdx.x >> 4, wave = threadIdx.x >> 6;
    for (int e = threadIdx.x; e < 16 * N; e += BAL_THREADS) counts[e] = 0u;
    __syncthreads();
    float acc[N];
#pragma unroll
    for (int i = 0; i < N; i++) acc[i] = 0.f;
    uint32_t live = 0;
    const int64_t step = (int64_t)gridDim.x * BAL_GROUPS;
    const T *const gate = static_cast<const T *>(a.gate);
    // (the last token stands in for those behind it; its lanes read and are not counted)
    auto row_of = [&](int64_t t) { return gate + (t < a.tokens ? t : a.tokens - 1) * a.pitch; };
    Token<T, N> next;
    next.template load<WAY>(row_of((int64_t)blockIdx.x * BAL_GROUPS + group), a.E, l);
    // all lanes of a wave take the same number of turns
    for (int64_t t0 = (int64_t)blockIdx.x * BAL_GROUPS; t0 < a.tokens; t0 += step) {
        const int64_t t = t0 + group;
        Token<T, N> x = next;
        if (N <= 16) next.template load<WAY>(row_of(t + step), a.E, l);      // a token ahead, where the registers allow it
        const float top = x.largest();
        const bool in = t < a.tokens && (a.mask == nullptr || a.mask[t] != 0) && !x.nothing(top);
        if (a.indices == nullptr) {
            x.template choose<WAY>(a.E, l, a.K, in, counts);
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
        if (N > 16) next.template load<WAY>(row_of(t + step), a.E, l);
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
            for (int i = 0; i < N; i++) {
                float &s = sums[Token<T, N>::expert(i, l)];
                s = (w == 0 ? 0.f : s) + acc[i];
            }
            if (l == 0) lives[w] = live;
        }
        __syncthreads();
    }
    if (threadIdx.x == 0)
        for (int w = 1; w < BAL_THREADS / 64; w++) lives[0] += lives[w];
    if constexpr (ONE) {
        __syncthreads();
        join_columns<false>(sums, counts, lives, a, BAL_THREADS, of_wave);
    } else {
        // (the columns of workgroups that there are not are the first one's to clear)
        for (int e = threadIdx.x; e < a.E; e += BAL_THREADS) {
            a.sums[(int64_t)e * BAL_WORKGROUPS + blockIdx.x] = sums[e];
            a.hits[(int64_t)e * BAL_WORKGROUPS + blockIdx.x] = counts[e];
        }
        if (threadIdx.x == 0) a.lives[blockIdx.x] = lives[0];
        if (blockIdx.x == 0) {
            const int none = BAL_WORKGROUPS - gridDim.x;
            for (int i = threadIdx.x; i < (a.E + 1) * none; i += BAL_THREADS) {
                const int e = i / none, c = gridDim.x + i % none;
                if (e < a.E) a.sums[(int64_t)e * BAL_WORKGROUPS + c] = 0.f, a.hits[(int64_t)e * BAL_WORKGROUPS + c] = 0u;
                else a.lives[c] = 0u;
            }
        }
    }
}

__global__ __launch_bounds__(BAL_JOIN) void gate_balance_join_kernel(BalArgs a)
{
    __shared__ double of_wave[BAL_JOIN / 64];
    join_columns<true>(a.sums, a.hits, a.lives, a, BAL_JOIN, of_wave);
}

template <typename T, int N, int WAY>
__global__ __launch_bounds__(BAL_BACKWARD) void gate_balance_backward_kernel(const T *__restrict__ gate, int64_t pitch,
                                                                            const uint8_t *__restrict__ mask, const float *__restrict__ share,
                                                                            const float *__restrict__ grad_loss, T *__restrict__ grad, int64_t tokens, int E)
{
    const int l = threadIdx.x & 15, group = threadIdx.x >> 4;
    const float scale = *grad_loss * share[E];
    float f[N];
#pragma unroll
    for (int i = 0; i < N; i++) f[i] = Token<T, N>::expert(i, l) < E ? share[Token<T, N>::expert(i, l)] : 0.f;
    const int64_t step = (int64_t)gridDim.x * (BAL_BACKWARD / 16);
    for (int64_t t0 = (int64_t)blockIdx.x * (BAL_BACKWARD / 16); t0 < tokens; t0 += step) {
        const int64_t t = t0 + group;
        Token<T, N> x;
        x.template load<WAY>(gate + (t < tokens ? t : tokens - 1) * pitch, E, l);
        const float top = x.largest();
        const bool in = t < tokens && (mask == nullptr || mask[t] != 0) && !x.nothing(top);
        x.softmax(top);
        float dot = 0.f;
#pragma unroll
        for (int i = 0; i < N; i++) dot = __builtin_fmaf(x.p[i], f[i], dot);
        dot = sum16(dot);
        if (t >= tokens) continue;
#pragma unroll
        for (int i = 0; i < N; i += 2) {
            const int e = Token<T, N>::expert(i, l);
            const float a = in ? scale * (x.p[i] * (f[i] - dot)) : 0.f, b = in ? scale * (x.p[i + 1] * (f[i + 1] - dot)) : 0.f;
            T *const to = grad + t * E + e;
            if constexpr (WAY != ONE_BY_ONE) {
                if (e < E) {
                    if constexpr (sizeof(T) == 2) *reinterpret_cast<uint32_t *>(to) = pack_bf16x2(a, b);
                    else *reinterpret_cast<f32x2 *>(to) = f32x2{a, b};
                }
            } else {
                if (e < E) Elem<T>::store(to, a);
                if (e + 1 < E) Elem<T>::store(to + 1, b);
            }
        }
    }
}

template <typename T> static int way_of(const void *gate, int64_t pitch, int E, int N)
{
    if (E % 2 != 0 || pitch % 2 != 0 || ((uintptr_t)gate % (2 * sizeof(T))) != 0) return ONE_BY_ONE;
    return E == 16 * N ? FULL : PAIRS;
}
constexpr int64_t BAL_ONE = 512;                   // tokens a single workgroup takes: as fast as a second launch

template <typename T, int N, int WAY> static int go_balance(BalArgs a, float *workspace, hipStream_t st)
{
    if (a.tokens <= BAL_ONE) {
        auto kern = gate_balance_kernel<T, N, WAY, true>;
        note_kernel(reinterpret_cast<const void *>(kern));
        kern<<<1, balance_threads(N), 0, st>>>(a);
        return check_launch("gate_balance");
    }
    a.sums = workspace;
    a.hits = reinterpret_cast<uint32_t *>(workspace + (int64_t)a.E * BAL_WORKGROUPS);
    a.lives = a.hits + (int64_t)a.E * BAL_WORKGROUPS;
    auto kern = gate_balance_kernel<T, N, WAY, false>;
    note_kernel(reinterpret_cast<const void *>(kern));
    const int64_t wanted = ceil_div(a.tokens, balance_threads(N) / 16);
    kern<<<(unsigned)(wanted < BAL_WORKGROUPS ? wanted : BAL_WORKGROUPS), balance_threads(N), 0, st>>>(a);
    const int rc = check_launch("gate_balance");
    if (rc != VTDGE_OK) return rc;
    note_kernel(reinterpret_cast<const void *>(gate_balance_join_kernel));
    gate_balance_join_kernel<<<1, BAL_JOIN, 0, st>>>(a);
    return check_launch("gate_balance");
}
template <typename T, int N> static int go_balance(const BalArgs &a, float *workspace, hipStream_t st)
{
    const int way = way_of<T>(a.gate, a.pitch, a.E, N);
    return way == FULL ? go_balance<T, N, FULL>(a, workspace, st) : way == PAIRS ? go_balance<T, N, PAIRS>(a, workspace, st) : go_balance<T, N, ONE_BY_ONE>(a, workspace, st);
}

template <typename T, int N>
static int go_balance_backward(const void *gate, int64_t pitch, const uint8_t *mask, const float *share, const float *grad_loss, void *grad,
                               int64_t tokens, int E, hipStream_t st)
{
    const int64_t wanted = ceil_div(tokens, BAL_BACKWARD / 16), most = 8 * (int64_t)compute_units();
    const int way = way_of<T>(grad, E, E, N) == ONE_BY_ONE ? ONE_BY_ONE : way_of<T>(gate, pitch, E, N);
    auto kern = way == FULL ? gate_balance_backward_kernel<T, N, FULL> : way == PAIRS ? gate_balance_backward_kernel<T, N, PAIRS> : gate_balance_backward_kernel<T, N, ONE_BY_ONE>;
    note_kernel(reinterpret_cast<const void *>(kern));
    kern<<<(unsigned)(wanted < most ? wanted : most), BAL_BACKWARD, 0, st>>>((const T *)gate, pitch, mask, share, grad_loss, (T *)grad, tokens, E);
    return check_launch("gate_balance_backward");
}

// values a lane holds, by the number of experts
#define VT_BY_EXPERTS(E, CALL)          \
    ((E) <= 32    ? CALL(2)             \
     : (E) <= 64  ? CALL(4)             \
     : (E) <= 96  ? CALL(6)             \
     : (E) <= 128 ? CALL(8)             \
     : (E) <= 160 ? CALL(10)            \
     : (E) <= 192 ? CALL(12)            \
     : (E) <= 256 ? CALL(16)            \
                  : CALL(32))

}  // namespace vtdge

using namespace vtdge;

extern "C" int64_t vtdge_gate_balance_workspace(int64_t tokens, int E)
{
    if (tokens <= BAL_ONE || E < 1 || E > VTDGE_MAX_EXPERTS) return 0;
    return BAL_WORKGROUPS * (2 * (int64_t)E + 1) * 4;
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
    VT_REQUIRE(need == 0 || (workspace && workspace_bytes >= need && ((uintptr_t)workspace & 15) == 0), VTDGE_ERR_ARG, "gate_balance: workspace of %lld bytes, %lld needed",
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
