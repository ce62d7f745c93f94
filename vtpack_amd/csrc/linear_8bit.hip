// A Linear over blocks of 8-bit numbers, y = act(Q(x) Q(W)^T + b), and its gradients dx = g Q(W), dW = g^T Q(x), db = sum g (gfx950), g the
// gradient of y rounded to bf16 (an error of half a step on each of many terms, as on any bf16 operand).
//
// Many rows: x (and W, where it is not given in blocks) is brought into blocks by a launch of its own, bound by memory (65536 x 1024 in bf16:
// 39 us), and multiplied by tiles (65536 x 1024 x 4096: 310 to 330 us with that launch, 387 with GELU; 8192 x 8192 x 8192: 470 to 480, 2.3
// PFLOP/s, where the library's product of 8-bit tensors reaches 2.8).  A width of 1024 is eight slabs of a 256 x 256 tile, which has its compute unit to itself: its
// first loads, GELU and 128 KB of results run with no product beside them, and the matrix units are busy 42 % of the time, 35 % with GELU, at 1.9
// GHz.  In long sums they and the clock bound it (1.6 - 1.8 GHz of 2.4 under products of random numbers, whatever the order of reads and
// products; another two of them were 3 and 5 % slower).  Short sums: the results' way to memory.
// Gradients: W and x expanded and laid out along the sums by one launch (32768 x 1024 and 4096 x 1024: 20 us), one launch of tiles for both
// products (515 us, 1.07 PFLOP/s; the library's bf16 product of 65536 x 1024 x 4096 runs at 1.05), and one that adds up their parts (14 us).
#include "eight_bit.h"

namespace vtdge {

struct ForwardArgs {
    Operand x, w;                                   // bf16; or blocks, two numbers an element
    const unsigned char *x_scales, *w_scales; int scale_pitch;
    const void *bias; void *y; int64_t rows, out; int stages;
    bool stream_y;                                  // the result past the caches
};

// ------------------------------------------------------------------------------------------------ the product of a tile of blocks
// As multiply_tile, on the 8-bit matrix instructions, which take the scales themselves: a slab of 2 SLAB numbers is one block, so that all of
// an instruction's sum has one scale for each row.  Scale bytes come four blocks at a time, the word of each row, into one of two places of
// their own (65536 x 1024 x 4096: 15 us less than a word with every slab).
template <class S> struct EightBit {
    static constexpr int SCALE_CHUNKS = (S::ROWS + S::COLS) / 64, SCALE_LOADS = (SCALE_CHUNKS + S::WAVES - 1) / S::WAVES;
    static constexpr int WORDS = SCALE_LOADS * S::WAVES * 256, SCALES = S::RING, RING = SCALES + 2 * WORDS, LDS = RING + S::COLS * 4;
    static_assert(LDS <= 160 * 1024 && S::ROWS % 64 == 0 && S::COLS % 64 == 0 && S::PARTS == 1, "LDS");
};
typedef int i32x8 __attribute__((ext_vector_type(8)));

template <class S, class LA, class LB, class F>
__device__ __forceinline__ void multiply_blocks(const LA &a, const LB &b, const ForwardArgs &p, int64_t r0, int64_t c0, unsigned char *smem, f32x16 (&acc)[S::IM][S::JN], F &&meanwhile)
{
    using E = EightBit<S>;
    constexpr int IM = S::IM, JN = S::JN, SLOTS = S::SLOTS, A_BYTES = LA::STAGE;
    constexpr int LOADS = LA::PIECES + LB::PIECES;          // and now and then those of scales: what waits for fewer waits for enough
    constexpr int GROUP = 4;                                // blocks, a slab each, whose scales are a word
    static_assert(LOADS * (SLOTS - 2) < 64, "the counter of outstanding loads");
    const int lane = threadIdx.x & 63, lr = lane & 31, wid = wave_uniform(threadIdx.x >> 6), wm = wid / S::WN, wn = wid % S::WN;
    const uint32_t lds0 = (uint32_t)(uintptr_t)smem;
    // this wave's rows of scales
    const void *scales[E::SCALE_LOADS];
    uint32_t offset[E::SCALE_LOADS];
#pragma unroll
    for (int d = 0; d < E::SCALE_LOADS; d++) {
        const int chunk = min(d * S::WAVES + wid, E::SCALE_CHUNKS - 1);
        const bool of_x = chunk < S::ROWS / 64;
        const int row = (of_x ? chunk : chunk - S::ROWS / 64) * 64 + lane;
        const int64_t first = of_x ? r0 : c0, there = (of_x ? p.rows : p.out) - first;
        scales[d] = uniform_ptr((of_x ? p.x_scales : p.w_scales) + first * p.scale_pitch);
        offset[d] = (uint32_t)(row < there ? row : (int)there - 1) * (uint32_t)p.scale_pitch;
    }
    auto issue = [&](int t, int slot) {
        const uint32_t at = lds0 + slot * S::STAGE;
        if (t % GROUP == 0) {
#pragma unroll
            for (int d = 0; d < E::SCALE_LOADS; d++)
                dma4(scales[d], offset[d] + (uint32_t)(t / GROUP) * 4, wave_uniform(lds0 + E::SCALES + (t / GROUP & 1) * E::WORDS + (d * S::WAVES + wid) * 256));
        }
        a.load(0, t, at);
        b.load(0, t, at + A_BYTES);
    };
    uint32_t words_a[IM], words_b[JN];
    int in = 0, out = 0;
#pragma unroll
    for (int d = 0; d < SLOTS - 1; d++)
        if (d < p.stages) {
            issue(d, in);
            in++;
        }
    meanwhile();
    for (int t = 0; t < p.stages; t++) {
        const int behind = min(p.stages - 1 - t, SLOTS - 2);
        static_for<SLOTS - 1>([&](auto X) {
            constexpr int x = decltype(X)::value;
            if (behind == x) wait_vmcnt<x * LOADS>();
        });
        lds_barrier();
        const unsigned char *sa = smem + out * S::STAGE, *sb = sa + A_BYTES;
        out = out == SLOTS - 1 ? 0 : out + 1;
        constexpr int STEPS = S::SLAB / 32;
        u32x4 fa[2][IM][2], fb[2][JN][2];
        auto fetch = [&](int s) {
#pragma unroll
            for (int h = 0; h < 2; h++) {
#pragma unroll
                for (int i = 0; i < IM; i++) fa[s & 1][i][h] = LA::fragment(sa, wm * IM + i, 2 * s + h);
#pragma unroll
                for (int j = 0; j < JN; j++) fb[s & 1][j][h] = LB::fragment(sb, wn * JN + j, 2 * s + h);
            }
        };
        if (t % GROUP == 0) {
            const unsigned char *ss = smem + E::SCALES + (t / GROUP & 1) * E::WORDS;
#pragma unroll
            for (int i = 0; i < IM; i++) words_a[i] = *reinterpret_cast<const uint32_t *>(ss + ((wm * IM + i) * 32 + lr) * 4);
#pragma unroll
            for (int j = 0; j < JN; j++) words_b[j] = *reinterpret_cast<const uint32_t *>(ss + (S::ROWS + (wn * JN + j) * 32 + lr) * 4);
        }
        fetch(0);
        __builtin_amdgcn_sched_barrier(0);
        if (t + SLOTS - 1 < p.stages) {
            issue(t + SLOTS - 1, in);
            in = in == SLOTS - 1 ? 0 : in + 1;
        }
        const int shift = t % GROUP * 8;
        uint32_t qa[IM], qb[JN];
#pragma unroll
        for (int i = 0; i < IM; i++) qa[i] = words_a[i] >> shift;
#pragma unroll
        for (int j = 0; j < JN; j++) qb[j] = words_b[j] >> shift;
        auto eight = [](const u32x4 (&f)[2]) {
            return i32x8{(int)f[0].x, (int)f[0].y, (int)f[0].z, (int)f[0].w, (int)f[1].x, (int)f[1].y, (int)f[1].z, (int)f[1].w};
        };
#pragma unroll
        for (int s = 0; s < STEPS; s++) {
            __builtin_amdgcn_sched_barrier(0);
            if (s + 1 < STEPS) fetch(s + 1);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int i = 0; i < IM; i++)
#pragma unroll
                for (int j = 0; j < JN; j++)
                    acc[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(eight(fb[s & 1][j]), eight(fa[s & 1][i]), acc[i][j], 0, 0, 0, (int)qb[j], 0, (int)qa[i]);
        }
    }
    lds_barrier();
}

// fp32 results: bf16 operands, whose products are exact and whose sums are fp32 (bf16 sums of 128 normal numbers are 1e-8 off).  bf16
// results: 8-bit operands, at twice the rate.  Those instructions cut the products of eight neighbours, toward zero, 13 bits below the largest sum of
// two exponents among them, before they join an fp32 sum: 1.4e-5 of the results in the 2-norm for normal numbers, 2.4e-5 where some channels are
// larger, a hundredth of bf16's rounding; at worst seven of the eight are lost, 7 2^-13 of the largest, which is more than a result's half step
// where the sum cancels to less than two fifths of it.
template <class S, typename T, bool GELU> __global__ __launch_bounds__(S::THREADS, S::PER_SIMD) void linear_8bit_kernel(ForwardArgs p, int tm, int tn)
{
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    constexpr int IM = S::IM, JN = S::JN;
    constexpr bool EIGHT = sizeof(T) == 2;
    int m, n;
    tile_at(place_of(blockIdx.x, tm * tn), tm, tn, m, n);
    const int64_t r0 = (int64_t)m * S::ROWS, c0 = (int64_t)n * S::COLS;
    float *const bias = reinterpret_cast<float *>(smem + (EIGHT ? EightBit<S>::RING : S::RING));
    // (behind the first direct loads: in front of them its way from memory would be waited for)
    auto read_bias = [&] {
        for (int c = threadIdx.x; c < S::COLS; c += S::THREADS)
            bias[c] = p.bias != nullptr && c0 + c < p.out ? Elem<T>::load(static_cast<const T *>(p.bias) + c0 + c) : 0.f;
    };
    f32x16 acc[IM][JN] = {};
    const Loader<true, S::ROWS, S::SLAB, S::WAVES> a(p.x, r0, p.rows, 0);
    const Loader<true, S::COLS, S::SLAB, S::WAVES> b(p.w, c0, p.out, 0);
    if constexpr (EIGHT) {
        multiply_blocks<S>(a, b, p, r0, c0, smem, acc, read_bias);
    } else {
        float none[IM];
        read_bias();
        multiply_tile<S, false>(a, b, 0, p.stages, smem, acc, false, none);
    }
    const int lg = (threadIdx.x & 63) >> 5, wn = wave_uniform(threadIdx.x >> 6) % S::WN;
    // (bf16 65536 x 1024 x 4096 with GELU: 470 us in pieces of 32 bytes from the registers, 400 so)
    auto finish = [&](int j, int q, f32x4 &v) {
        v += *reinterpret_cast<const f32x4 *>(bias + (wn * JN + j) * 32 + 8 * q + 4 * lg);
        if constexpr (GELU)
#pragma unroll
            for (int e = 0; e < 4; e++) v[e] = gelu_value<T>(v[e]);
    };
    put_tile<S>(smem, acc, finish, static_cast<T *>(p.y), p.rows, p.out, r0, c0, p.stream_y);
}

// ------------------------------------------------------------------------------------------------ few rows
// Up to 16 rows against a weight in blocks, bound by the reading of the weight: one launch, x is brought into blocks by every workgroup for
// itself while the first of its weights are on their way.  A workgroup has 16 outputs, its four waves take four blocks of them in turn; a
// lane loads 32 bytes of a block of one output, four of them the whole line, and multiplies as it came (both operands' numbers are in the
// same order).  us of a call, so / by tiles behind a launch for x, in bf16: 1 row x 4096 x 16384 16.0 (4.2 TB/s) / 15.2, 4 x 4096 x 4096 9.1 / 14.0,
// 1 x 384 x 1536 3.5 / 8.0, 16 x 1024 x 4096 6.6 / 7.8, 8 x 2048 x 8192 8.3 / 9.9, 16 x 1024 x 16384 10.3 / 8.2; in fp32, where tiles read a weight that
// every call expands to bf16 first: 20 / 53, 10.0 / 38, 3.7 / 7.8, 7.0 / 14.6, 9.2 / 31, 14 / 28.  (More numbers of x than FEW_BYTES go by tiles, in fp32 at their cost: 5
// rows x 4096 x 4096 38 us, 64 rows x 4096 x 16384 58, bf16 15 and 16.)
struct FewArgs {
    const void *x; int64_t ldx; int rows, width;
    const unsigned char *w, *w_scales; int64_t value_pitch; int scale_pitch;
    const void *bias; void *y; int64_t out;
};
constexpr int FEW = 16, FEW_BYTES = 16384;          // rows; numbers of x in LDS
template <typename T> static constexpr int few_lds(int rows, int64_t pitch, int scales)
{
    return (int)(rows * pitch * (sizeof(T) == 2 ? 1 : 2)) + (rows * scales + 15) / 16 * 16 + 4 * 64 * 16;
}
template <typename T, bool GELU> __global__ __launch_bounds__(256) void linear_8bit_few_kernel(FewArgs p)
{
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    constexpr bool EIGHT = sizeof(T) == 2;
    constexpr int SIZE = EIGHT ? 1 : 2;             // bytes of a number of x: 8-bit, or expanded
    const int lane = threadIdx.x & 63, wid = wave_uniform(threadIdx.x >> 6), at16 = lane & 15, g = lane >> 4;
    const int blocks = (p.width + BLOCK - 1) / BLOCK, x_pitch = blocks * BLOCK * SIZE;
    unsigned char *const xq = smem, *const xs = smem + p.rows * x_pitch;
    f32x4 *const sums = reinterpret_cast<f32x4 *>(xs + (p.rows * p.scale_pitch + 15) / 16 * 16);
    const int64_t o0 = (int64_t)blockIdx.x * 16, o = o0 + at16 < p.out ? o0 + at16 : p.out - 1;
    const unsigned char *const w = p.w + o * p.value_pitch + g * 16, *const ws = p.w_scales + o * p.scale_pitch;
    struct Unit {
        u32x4 v[4][2];
        uint32_t scales;
    };
    auto load = [&](Unit &u, int unit) {
        if (unit * 4 >= blocks) return;
        u.scales = *reinterpret_cast<const uint32_t *>(ws + unit * 4);
#pragma unroll
        for (int b = 0; b < 4; b++) {
            const int block = min(unit * 4 + b, blocks - 1);          // (behind the last: not used)
#pragma unroll
            for (int h = 0; h < 2; h++) u.v[b][h] = *reinterpret_cast<const u32x4 *>(w + block * BLOCK + h * 64);
        }
    };
    float add[4];                                   // the outputs' own, see below
#pragma unroll
    for (int e = 0; e < 4; e++) add[e] = p.bias != nullptr && o0 + 4 * g + e < p.out ? Elem<T>::load(static_cast<const T *>(p.bias) + o0 + 4 * g + e) : 0.f;
    Unit next[2];                                   // two ahead: 4096 numbers of the four waves
    load(next[0], wid);
    load(next[1], wid + 4);
    for (int first = 0; first < p.rows * blocks; first += 16) {        // the same for all: the lanes of a block take part together
        const int id = first + (threadIdx.x >> 4), row = id / blocks, block = id - row * blocks, c = block * BLOCK + at16 * 8;
        const bool in = id < p.rows * blocks;
        float f[8];
        load8<T>(static_cast<const T *>(p.x) + (int64_t)row * p.ldx + c, in ? p.width - c : 0, f);
        const Rounded q = round8(f);
        if (!in) continue;
        if constexpr (EIGHT) {
            *reinterpret_cast<u32x2 *>(xq + row * x_pitch + c) = q.bytes;
            if (at16 == 0) xs[row * p.scale_pitch + block] = (unsigned char)q.scale;
        } else {
            *reinterpret_cast<u32x4 *>(xq + row * x_pitch + c * 2) = expand8(q.bytes, q.scale);
        }
    }
    lds_barrier();
    const int row = at16 < p.rows ? at16 : p.rows - 1;
    const unsigned char *const xr = xq + row * x_pitch + g * 16 * SIZE, *const xsr = xs + row * p.scale_pitch;
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    auto multiply = [&](const Unit &now, int unit) {
#pragma unroll
        for (int b = 0; b < 4; b++) {
            const int block = unit * 4 + b;
            if (block >= blocks) break;
            if constexpr (EIGHT) {
                const u32x4 x0 = *reinterpret_cast<const u32x4 *>(xr + block * BLOCK), x1 = *reinterpret_cast<const u32x4 *>(xr + block * BLOCK + 64);
                const u32x4 w0 = now.v[b][0], w1 = now.v[b][1];
                acc = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(
                    i32x8{(int)w0.x, (int)w0.y, (int)w0.z, (int)w0.w, (int)w1.x, (int)w1.y, (int)w1.z, (int)w1.w},
                    i32x8{(int)x0.x, (int)x0.y, (int)x0.z, (int)x0.w, (int)x1.x, (int)x1.y, (int)x1.z, (int)x1.w}, acc, 0, 0, 0,
                    (int)(now.scales >> (8 * b)), 0, (int)xsr[block]);
            } else {
#pragma unroll
                for (int q = 0; q < 4; q++) {
                    const u32x4 part = now.v[b][q >> 1];
                    const u32x4 we = expand8(q & 1 ? u32x2{part.z, part.w} : u32x2{part.x, part.y}, (int)(now.scales >> (8 * b) & 255u));
                    const u32x4 xe = *reinterpret_cast<const u32x4 *>(xr + (block * BLOCK + (q >> 1) * 64 + (q & 1) * 8) * 2);
                    acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, we), __builtin_bit_cast(bf16x8, xe), acc, 0, 0, 0);
                }
            }
        }
    };
    for (int unit = wid; unit * 4 < blocks; unit += 8) {
        const Unit now = next[0];
        load(next[0], unit + 8);
        multiply(now, unit);
        const Unit then = next[1];
        load(next[1], unit + 12);
        multiply(then, unit + 4);
    }
    // a lane has outputs 4 g .. 4 g + 3 of row at16
    sums[wid * 64 + lane] = acc;
    lds_barrier();
    if (wid != 0 || at16 >= p.rows) return;
    acc = (sums[lane] + sums[64 + lane]) + (sums[128 + lane] + sums[192 + lane]);
#pragma unroll
    for (int e = 0; e < 4; e++) {
        const int64_t c = o0 + 4 * g + e;
        if (c >= p.out) break;
        float v = acc[e] + add[e];
        if (GELU) v = gelu_value<T>(v);
        Elem<T>::store(static_cast<T *>(p.y) + at16 * p.out + c, v);
    }
}

// Blocks [rows, n] as bf16 [n, pitch], zeros behind the rows: what both gradients multiply lies along their sums then, and is read from LDS
// in 16 bytes a lane (32768 x 1024 x 4096: 605 us of gradients where the LDS reads transpose, 554 so, and 515 since with whole lines and no bank
// conflicts).  Bound by memory: three bytes a number, 113 MB in 20 us there.
struct ExpandJob {
    const unsigned char *values, *scales; uint32_t rows, down; int64_t value_pitch; int scale_pitch, n; bf16_t *to; int64_t pitch;     // down: tiles of 64 rows
};
// Rows of g: bf16, filled up with zeros to whole slabs.
struct PackJob {
    const void *from; int64_t ld; uint32_t rows, per_row; int n; bf16_t *to;      // per_row: vectors of eight; rows 0: g lies as it is read
};
struct PrepareArgs {
    ExpandJob job[2];
    PackJob pack;
    uint32_t first, second;                         // workgroups of the first, of both
};
template <typename T> __global__ __launch_bounds__(256) void prepare_gradients_kernel(PrepareArgs p)
{
    if (blockIdx.x >= p.second) {
        const PackJob &g = p.pack;
        const uint32_t id = (blockIdx.x - p.second) * 256 + threadIdx.x, row = id / g.per_row, c = (id - row * g.per_row) * 8;
        if (row >= g.rows) return;
        float f[8];
        load8<T>(static_cast<const T *>(g.from) + (int64_t)row * g.ld + c, g.n - (int)c, f);
        *reinterpret_cast<u32x4 *>(g.to + ((int64_t)row * g.per_row * 8 + c)) = Elem<bf16_t>::pack(f);
        return;
    }
    // [column][two rows a word]; pieces of four words are XOR-ed by the column's eight, and the columns of the upper half swapped in pairs, so that the
    // sixteen columns that a wave writes at once lie in all 64 banks
    __shared__ __attribute__((aligned(16))) uint32_t tile[BLOCK * 32];
    auto word = [](int column, int piece) { return (column ^ (column >> 6 & 1)) * 32 + (piece ^ (column >> 3 & 7)) * 4; };
    const bool second = blockIdx.x >= p.first;
    const ExpandJob &job = p.job[second ? 1 : 0];
    const uint32_t id = blockIdx.x - (second ? p.first : 0), block = id / job.down, r0 = (id - block * job.down) * 64;
#pragma unroll
    for (int k = 0; k < 2; k++) {
        const int pair = (threadIdx.x >> 4) + 16 * k, c = (threadIdx.x & 15) * 8;
        float f[2][8];
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const uint32_t r = r0 + 2 * pair + h;
            if (r < job.rows) {
                stands_for8(*reinterpret_cast<const u32x2 *>(job.values + (int64_t)r * job.value_pitch + block * BLOCK + c), job.scales[(int64_t)r * job.scale_pitch + block], f[h]);
            } else {
#pragma unroll
                for (int e = 0; e < 8; e++) f[h][e] = 0.f;
            }
        }
#pragma unroll
        for (int e = 0; e < 8; e++) tile[word(c + e, pair >> 2) + (pair & 3)] = pack_bf16x2(f[0][e], f[1][e]);
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 4; k++) {
        const int at = threadIdx.x + 256 * k, column = at >> 3, piece = at & 7;
        if ((int)(block * BLOCK) + column < job.n)
            *reinterpret_cast<u32x4 *>(job.to + (int64_t)(block * BLOCK + column) * job.pitch + r0 + piece * 8) =
                *reinterpret_cast<const u32x4 *>(tile + word(column, piece));
    }
}

// ------------------------------------------------------------------------------------------------ on the host
using ForwardLarge = Shape<2, 4, 4, 2, 64, 2, 1>;
using ForwardSquare = Shape<2, 2, 2, 2, 64, 2, 1>;
using ForwardSmall = Shape<1, 1, 2, 2, 64, 3, 1>;
static_assert(ForwardLarge::SLAB == 64 && ForwardSquare::SLAB == 64 && ForwardSmall::SLAB == 64, "slabs of a block");

constexpr int SLAB = 64;
static int64_t take(int64_t &at, int64_t bytes)
{
    const int64_t here = at;
    at += (bytes + 255) / 256 * 256;
    return here;
}
static int64_t padded(int64_t n) { return ceil_div(n, SLAB) * SLAB; }

static bool few_rows(int64_t rows, int64_t width) { return rows <= FEW && rows * value_pitch(width) <= FEW_BYTES; }

struct ForwardPlan {
    int64_t x_at, w_at, bytes;
};
static ForwardPlan plan_forward(int64_t rows, int64_t out, int64_t width, int how, int dtype)
{
    ForwardPlan p{};
    int64_t at = 0;
    const bool few = few_rows(rows, width), blocks = few || dtype != VTDGE_F32;        // blocks are multiplied, or what they expand to
    p.x_at = take(at, few || (blocks && (how & VTDGE_8BIT_X_KEPT)) ? 0 : blocks ? blocks_bytes(rows, width) : rows * padded(width) * 2);
    p.w_at = take(at, blocks && (how & (VTDGE_8BIT_WEIGHT_KEPT | VTDGE_8BIT_WEIGHT_GIVEN)) ? 0 : blocks ? blocks_bytes(out, width) : out * padded(width) * 2);
    p.bytes = at;
    return p;
}
struct BackwardPlan : GradPlan {
    int64_t g_at, x_at, w_at, dx_at, dw_at, db_at, bytes;
};
// whether the products read the gradient where it lies
static bool gradient_lies(const void *g, int64_t ld, int64_t out, int dtype)
{
    return dtype == VTDGE_BF16 && out % SLAB == 0 && ld % 8 == 0 && ld < (1 << 22) && ((uintptr_t)g & 15) == 0;
}
// (the cuts are the same whichever gradients are wanted, and so are their bits)
static BackwardPlan plan_backward(int64_t rows, int64_t out, int64_t width, int how)
{
    BackwardPlan p{};
    plan_gradients(p, rows, out, (int)width, false, true);
    int64_t at = 0;
    const bool dx = !(how & VTDGE_8BIT_NO_DX), dw = !(how & VTDGE_8BIT_NO_DWEIGHT), db = !(how & VTDGE_8BIT_NO_DBIAS);
    p.g_at = take(at, how & VTDGE_8BIT_GRADIENT_LIES ? 0 : rows * padded(out) * 2);
    p.x_at = take(at, dw ? width * padded(rows) * 2 : 0);
    p.w_at = take(at, dx ? width * padded(out) * 2 : 0);
    // (a sum that is not cut leaves for its place)
    p.dx_at = take(at, dx && p.dx_splits > 1 ? part_of(rows * width) * 4 * p.dx_splits : 0);
    p.dw_at = take(at, dw && p.dw_splits > 1 ? part_of(out * width) * 4 * p.dw_splits : 0);
    p.db_at = take(at, db && p.dw_splits > 1 ? part_of(out) * 4 * p.dw_splits : 0);
    p.bytes = at;
    return p;
}

static int check_linear(const char *what, int64_t rows, int64_t out, int64_t width, int dtype)
{
    VT_REQUIRE(dtype == VTDGE_F32 || dtype == VTDGE_BF16, VTDGE_ERR_ARG, "%s: dtype %d", what, dtype);
    VT_STEP(check_blocks(what, rows, width));
    VT_STEP(check_blocks(what, out, width));
    VT_STEP(check_blocks(what, rows, out));
    VT_REQUIRE(out <= (1 << 20) && ceil_div(rows, 64) * ceil_div(out, 64) < (1 << 23), VTDGE_ERR_UNSUPPORTED, "%s: %lld rows, %lld outputs", what,
               (long long)rows, (long long)out);
    return VTDGE_OK;
}

template <class S, typename T, bool GELU> static int go_forward_as(const ForwardArgs &a, hipStream_t st)
{
    const int64_t tm = ceil_div(a.rows, S::ROWS), tn = ceil_div(a.out, S::COLS);
    auto kern = linear_8bit_kernel<S, T, GELU>;
    constexpr int LDS = sizeof(T) == 2 ? EightBit<S>::LDS : S::LDS;
    VT_RESERVE_LDS(kern, LDS, "linear_8bit");
    note_kernel(reinterpret_cast<const void *>(kern));
    kern<<<(unsigned)(tm * tn), S::THREADS, LDS, st>>>(a, (int)tm, (int)tn);
    return check_launch("linear_8bit");
}
template <class S> static int go_forward(const ForwardArgs &a, int act, int dtype, hipStream_t st)
{
    if (dtype == VTDGE_F32) return act == VTDGE_ACT_GELU ? go_forward_as<S, float, true>(a, st) : go_forward_as<S, float, false>(a, st);
    return act == VTDGE_ACT_GELU ? go_forward_as<S, bf16_t, true>(a, st) : go_forward_as<S, bf16_t, false>(a, st);
}

}  // namespace vtdge

using namespace vtdge;

extern "C" int64_t vtdge_linear_8bit_workspace(int64_t rows, int64_t out, int64_t width, int how, int dtype)
{
    if (check_linear("linear_8bit_workspace", rows, out, width, dtype) != VTDGE_OK) return -1;
    return plan_forward(rows, out, width, how, dtype).bytes;
}

template <typename T> static int go_few(const FewArgs &a, int act, hipStream_t st)
{
    auto kern = act == VTDGE_ACT_GELU ? linear_8bit_few_kernel<T, true> : linear_8bit_few_kernel<T, false>;
    note_kernel(reinterpret_cast<const void *>(kern));
    kern<<<(unsigned)ceil_div(a.out, 16), 256, few_lds<T>(a.rows, value_pitch(a.width), a.scale_pitch), st>>>(a);
    return check_launch("linear_8bit");
}

extern "C" int vtdge_linear_8bit(const void *x, int64_t ldx, const void *weight, int64_t ldw, void *w_blocks, const void *bias, void *y, void *x_blocks,
                                 int64_t rows, int64_t out, int64_t width, int act, void *workspace, int64_t workspace_bytes, int dtype, void *stream)
{
    VT_STEP(check_linear("linear_8bit", rows, out, width, dtype));
    VT_REQUIRE(x && y && (weight || w_blocks), VTDGE_ERR_ARG, "linear_8bit: NULL operand");
    VT_REQUIRE(act == VTDGE_ACT_NONE || act == VTDGE_ACT_GELU, VTDGE_ERR_ARG, "linear_8bit: act %d", act);
    VT_REQUIRE((ldx >= width || rows == 1) && (weight == nullptr || ldw >= width || out == 1), VTDGE_ERR_ARG, "linear_8bit: rows of %lld, %lld and %lld apart",
               (long long)width, (long long)ldx, (long long)ldw);
    VT_REQUIRE(((uintptr_t)w_blocks & 127) == 0 && ((uintptr_t)x_blocks & 127) == 0, VTDGE_ERR_ARG, "linear_8bit: blocks off their boundary");
    const int how = (weight == nullptr ? VTDGE_8BIT_WEIGHT_GIVEN : w_blocks != nullptr ? VTDGE_8BIT_WEIGHT_KEPT : 0) | (x_blocks != nullptr ? VTDGE_8BIT_X_KEPT : 0);
    const ForwardPlan p = plan_forward(rows, out, width, how, dtype);
    VT_REQUIRE((workspace != nullptr || p.bytes == 0) && workspace_bytes >= p.bytes && ((uintptr_t)workspace & 255) == 0, VTDGE_ERR_ARG,
               "linear_8bit: workspace of %lld bytes, %lld needed", (long long)workspace_bytes, (long long)p.bytes);
    unsigned char *const ws = (unsigned char *)workspace;
    const hipStream_t st = (hipStream_t)stream;
    QuantizeArgs q{};
    if (few_rows(rows, width)) {
        void *const wq = w_blocks != nullptr ? w_blocks : ws + p.w_at;
        int jobs = 0;
        if (weight != nullptr) q.job[jobs++] = quantize_job(weight, ldw, out, width, wq, nullptr, 0);
        if (x_blocks != nullptr) q.job[jobs++] = quantize_job(x, ldx, rows, width, x_blocks, nullptr, 0);
        if (jobs > 0) VT_STEP(launch_quantize(q, jobs, dtype, "linear_8bit", st));
        FewArgs f{};
        f.x = x, f.ldx = ldx, f.rows = (int)rows, f.width = (int)width, f.w = values_of(wq), f.w_scales = scales_of(wq, out, width);
        f.value_pitch = value_pitch(width), f.scale_pitch = (int)scale_pitch(width), f.bias = bias, f.y = y, f.out = out;
        return dtype == VTDGE_F32 ? go_few<float>(f, act, st) : go_few<bf16_t>(f, act, st);
    }
    ForwardArgs a{};
    a.bias = bias, a.y = y, a.rows = rows, a.out = out;
    // Past the caches where the result fills the last of them (us so / kept: bf16 131072 x 1024 x 1024 224 / 244, 65536 x 1024 x 4096 300 / 338;
    // below it 16384 x 1024 x 4096 97 / 91)
    a.stream_y = rows * out * (dtype == VTDGE_F32 ? 4 : 2) >= (256ll << 20);
    int64_t slabs;                                  // of 64 elements
    if (dtype == VTDGE_F32) {
        bf16_t *const xb = (bf16_t *)(ws + p.x_at), *const wb = (bf16_t *)(ws + p.w_at);
        q.job[0] = quantize_job(x, ldx, rows, width, x_blocks, xb, padded(width));
        q.job[1] = quantize_job(weight, ldw, out, width, w_blocks, wb, padded(width));
        VT_STEP(launch_quantize(q, 2, dtype, "linear_8bit", st));
        a.x = Operand{xb, padded(width), 0}, a.w = Operand{wb, padded(width), 0};
        slabs = padded(width) / SLAB;
    } else {
        void *const xq = x_blocks != nullptr ? x_blocks : ws + p.x_at, *const wq = w_blocks != nullptr ? w_blocks : ws + p.w_at;
        q.job[0] = quantize_job(x, ldx, rows, width, xq, nullptr, 0);
        if (weight != nullptr) q.job[1] = quantize_job(weight, ldw, out, width, wq, nullptr, 0);
        VT_STEP(launch_quantize(q, weight != nullptr ? 2 : 1, dtype, "linear_8bit", st));
        a.x = Operand{(const bf16_t *)xq, value_pitch(width) / 2, 0}, a.w = Operand{(const bf16_t *)wq, value_pitch(width) / 2, 0};
        a.x_scales = scales_of(xq, rows, width), a.w_scales = scales_of(wq, out, width), a.scale_pitch = (int)scale_pitch(width);
        slabs = value_pitch(width) / BLOCK;
    }
    // Many tiles by 256 x 256, two of 128 x 128 beside each other on a compute unit for fewer, and for short sums without an activation (whose
    // results leave while the other multiplies), 64 x 64 where those would leave compute units without work.  us of a call in bf16 (64 x 64,
    // 128 x 128, 256 x 256): 4112 x 384 x 384 8.6, 9.1, 13.1; 4112 x 384 x 1536 13.9, 11.7, 14.9; 8192 x 1024 x 1024 26.4, 21.4, 27.0;
    // 65536 x 384 x 384 41, 34, 36; 32768 x 384 x 1536 with GELU 65, 51, 46; 16384 x 1024 x 1024 42.7, 34.0, 33.3; 8192 x 4096 x 4096 226, 154, 139;
    // in fp32 4112 x 384 x 384 10.5, 12.5, 19.5; 8192 x 1024 x 1024 38, 31, 40; 65536 x 384 x 384 60, 56, 61; 8192 x 4096 x 4096 420, 280, 263
    const int64_t cu = compute_units();
    a.stages = (int)slabs;
    if (ceil_div(rows, 128) * ceil_div(out, 128) * 4 < 5 * cu) return go_forward<ForwardSmall>(a, act, dtype, st);
    if (ceil_div(rows, 256) * ceil_div(out, 256) < cu || (act == VTDGE_ACT_NONE && width <= 640)) return go_forward<ForwardSquare>(a, act, dtype, st);
    return go_forward<ForwardLarge>(a, act, dtype, st);
}

extern "C" int64_t vtdge_linear_8bit_backward_workspace(int64_t rows, int64_t out, int64_t width, int how, int dtype)
{
    if (check_linear("linear_8bit_backward_workspace", rows, out, width, dtype) != VTDGE_OK) return -1;
    if (dtype != VTDGE_BF16 || out % SLAB != 0) how &= ~VTDGE_8BIT_GRADIENT_LIES;
    return plan_backward(rows, out, width, how).bytes;
}

extern "C" int vtdge_linear_8bit_backward(const void *grad, int64_t ldg, const void *x_blocks, const void *w_blocks, int64_t rows, int64_t out,
                                          int64_t width, void *workspace, int64_t workspace_bytes, void *dx, void *dweight, void *dbias, int dtype,
                                          void *stream)
{
    VT_STEP(check_linear("linear_8bit_backward", rows, out, width, dtype));
    if (dx == nullptr && dweight == nullptr && dbias == nullptr) return VTDGE_OK;
    VT_REQUIRE(grad && (dx == nullptr || w_blocks) && (dweight == nullptr || x_blocks), VTDGE_ERR_ARG, "linear_8bit_backward: NULL operand");
    VT_REQUIRE(rows <= VTDGE_MAX_ROWS_8BIT, VTDGE_ERR_UNSUPPORTED, "linear_8bit_backward: %lld rows, %d at most", (long long)rows, VTDGE_MAX_ROWS_8BIT);
    VT_REQUIRE(ldg >= out || rows == 1, VTDGE_ERR_ARG, "linear_8bit_backward: rows of %lld, %lld apart", (long long)out, (long long)ldg);
    VT_REQUIRE(((uintptr_t)w_blocks & 127) == 0 && ((uintptr_t)x_blocks & 127) == 0, VTDGE_ERR_ARG, "linear_8bit_backward: blocks off their boundary");
    const bool lies = gradient_lies(grad, rows > 1 ? ldg : 0, out, dtype);
    const BackwardPlan p = plan_backward(rows, out, width, (lies ? VTDGE_8BIT_GRADIENT_LIES : 0) | (dx == nullptr ? VTDGE_8BIT_NO_DX : 0) |
                                                               (dweight == nullptr ? VTDGE_8BIT_NO_DWEIGHT : 0) | (dbias == nullptr ? VTDGE_8BIT_NO_DBIAS : 0));
    VT_REQUIRE((workspace != nullptr || p.bytes == 0) && workspace_bytes >= p.bytes && ((uintptr_t)workspace & 255) == 0, VTDGE_ERR_ARG, "linear_8bit_backward: workspace of %lld bytes, %lld needed",
               (long long)workspace_bytes, (long long)p.bytes);
    unsigned char *const ws = (unsigned char *)workspace;
    const hipStream_t st = (hipStream_t)stream;
    bf16_t *const xb = (bf16_t *)(ws + p.x_at), *const wb = (bf16_t *)(ws + p.w_at);
    Operand g_op{(const bf16_t *)grad, rows > 1 ? ldg : out, 0};
    PrepareArgs d{};
    int jobs = 0;
    int64_t tiles = 0;
    auto expand = [&](const void *blocks, int64_t r, bf16_t *to) {
        ExpandJob &j = d.job[jobs++];
        j.values = values_of(blocks), j.scales = scales_of(blocks, r, width), j.rows = (uint32_t)r, j.down = (uint32_t)ceil_div(r, 64);
        j.value_pitch = value_pitch(width), j.scale_pitch = (int)scale_pitch(width), j.n = (int)width, j.to = to, j.pitch = padded(r);
        tiles += j.down * ceil_div(width, BLOCK);
        if (jobs == 1) d.first = (uint32_t)tiles;
    };
    if (dx != nullptr) expand(w_blocks, out, wb);
    if (dweight != nullptr) expand(x_blocks, rows, xb);
    d.second = (uint32_t)tiles;
    if (!lies) {
        bf16_t *const to = (bf16_t *)(ws + p.g_at);
        d.pack = PackJob{grad, ldg, (uint32_t)rows, (uint32_t)(padded(out) / 8), (int)out, to};
        tiles += ceil_div(rows * d.pack.per_row, 256);
        g_op = Operand{to, padded(out), 0};
    }
    VT_REQUIRE(tiles < (1 << 24), VTDGE_ERR_UNSUPPORTED, "linear_8bit_backward: %lld rows of %lld and %lld", (long long)rows, (long long)width, (long long)out);
    if (tiles > 0) {
        auto kern = dtype == VTDGE_F32 ? prepare_gradients_kernel<float> : prepare_gradients_kernel<bf16_t>;
        note_kernel(reinterpret_cast<const void *>(kern));
        kern<<<(unsigned)tiles, 256, 0, st>>>(d);
        VT_STEP(check_launch("linear_8bit_backward"));
    }
    GradPair g{};
    g.f32 = dtype == VTDGE_F32, g.ends = true;
    if (dx != nullptr) {
        g.dx.a = g_op, g.dx.b = Operand{wb, padded(out), 0};
        g.dx.rows = rows, g.dx.cols = width, g.dx.sum_b = out;
        g.dx.stages = (int)ceil_div(out, p.slab_g), g.dx.splits = p.dx_splits;
        g.dx.part = p.dx_splits == 1 ? nullptr : (float *)(ws + p.dx_at), g.dx.part_stride = part_of(rows * width), g.dx.out = dx;
    }
    if (dweight != nullptr || dbias != nullptr) {
        // (without dW the second operand is not multiplied to any end: the gradient's memory stands in its place, a row of it of any length
        // within)
        g.dw.a = g_op, g.dw.b = dweight != nullptr ? Operand{xb, padded(rows), 0} : g_op;
        g.dw.rows = out, g.dw.cols = dweight != nullptr ? width : 1, g.dw.sum_a = rows, g.dw.span_a = padded(out), g.dw.sum_b = rows;
        g.dw.stages = (int)ceil_div(rows, p.slab_g), g.dw.splits = p.dw_splits;
        const bool cut = p.dw_splits > 1;
        g.dw.part = cut && dweight != nullptr ? (float *)(ws + p.dw_at) : nullptr, g.dw.part_stride = part_of(out * width), g.dw.out = dweight;
        g.dw.sums_part = cut && dbias != nullptr ? (float *)(ws + p.db_at) : nullptr, g.dw.sums_stride = part_of(out), g.dw.sums = dbias;
    }
    VT_STEP(launch_gradients(p, g, "linear_8bit_backward", st));
    const SumJob sums[3] = {{g.dx.part, dx, rows * width, g.dx.part_stride, p.dx_splits},
                            {g.dw.part, dweight, out * width, g.dw.part_stride, p.dw_splits},
                            {g.dw.sums_part, dbias, out, g.dw.sums_stride, p.dw_splits}};
    return sum_parts(sums, 3, nullptr, nullptr, g.f32, "linear_8bit_backward", st);
}
