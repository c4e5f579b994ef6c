// hpf_softmax.hip -- softmax cross entropy of rows against a whole catalogue, with its gradients, without keeping the logits.
//
//   z[n, v] = scale <x[n], w[v]> + bias[v];   lse[n] = log sum_v exp z[n, v];   loss[n] = lse[n] - z[n, t[n]]
//   G[n, v] = weight[n] (exp(z[n, v] - lse[n]) - [v = t[n]])
//   dx = scale G w;   dw = scale G^T x;   dbias[v] = sum_n G[n, v]
//
// Every product is a matrix instruction (32 x 32 x 16); a row's statistics are kept in base 2 (z log2(e)).
//
// PASSES.  A wavefront keeps 32 (or 64) rows of one matrix in registers -- the STATIONARY rows -- and the other matrix streams
// by in tiles of 32 rows through shared memory, four or eight wavefronts reading each.  A tile's logits come out with the
// stationary row in the lane and the streamed row in the register, so that what belongs to a stationary row is a lane's own.
//   rows pass:   x stationary, w streamed: running maximum and sum of a softmax, and the sum of exp(z - max) w over the tiles
//                -- dx before its normalisation -- in the same pass, rescaled when a maximum grows
//   items pass:  w stationary, x streamed: G from the finished lse, and its product with x
// so the logits are computed twice and nothing of their size is written.  An output register's row (8 (i / 4) + 4 (lane / 32) +
// i % 4) is not an operand's (8 (lane / 32) + j), but a contraction may take its terms in any order: the second product's
// other operand is laid out in the order in which the first product's output lies in the registers, and the probabilities
// never leave the lane that made them.
//
// 32-BIT MATRICES are split into three bfloat16 parts (8 + 8 + 8 bits of mantissa) and multiplied in six products, all those
// of at least 2^-16 of the whole: what is left out is below 2^-24 of |a| |b|, the size of one 32-bit rounding.  bfloat16 and
// half matrices take one product; their probabilities are rounded to the same type (half: times 2^14, so that 2^-28 of a row's
// largest is still a normal number), everything else stays in 32 bits.
//
// THE TARGET's logit is kept out of the sums and joined at the end: 1 - p(target) is then the sum of the others' shares and not a
// difference of near equals, and the loss of a row that is sure of its target log1p(others / target).
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "hpf_hip.h"

namespace {

constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.693147180559945309417f;
constexpr float kNothing = -0x1p126f;     // a running maximum before anything: logits (base 2) at or below it are masked
constexpr int kNoTarget = 0x3FFFFFFF;     // block 2^25 of 32 items: beyond every catalogue
constexpr int kNegative = 0x40000000;     // flag beside a row's target: its weight is negative
constexpr int kPadTiles = 8;              // packed matrices end on a multiple of so many tiles: staging reads whole groups

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

struct Bf {
    typedef __bf16 e;
    typedef __bf16 v8 __attribute__((ext_vector_type(8)));
    static __device__ __forceinline__ f32x16 mfma(v8 a, v8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
};
struct Hf {
    typedef _Float16 e;
    typedef _Float16 v8 __attribute__((ext_vector_type(8)));
    static __device__ __forceinline__ f32x16 mfma(v8 a, v8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
};

// what a user's matrix is, what it is multiplied in, in how many parts, and the power of two its probabilities are held times
struct F32 { typedef float t; typedef Bf m; static constexpr int S = 3, shift = 0; };
struct B16 { typedef __bf16 t; typedef Bf m; static constexpr int S = 1, shift = 0; };
struct H16 { typedef _Float16 t; typedef Hf m; static constexpr int S = 1, shift = 14; };

template <class Y> struct Parts { typename Y::m::v8 p[Y::S]; };   // 8 values of an operand

template <class Y> __device__ __forceinline__ void split(float x, Parts<Y> &to, int j)
{
    typedef typename Y::m::e e;
    to.p[0][j] = (e)x;
    if constexpr (Y::S == 3) {
        const float r = x - (float)to.p[0][j];
        to.p[1][j] = (e)r;
        to.p[2][j] = (e)(r - (float)to.p[1][j]);
    }
}

// c += a b, smallest products first
template <class Y> __device__ __forceinline__ f32x16 product(const Parts<Y> &a, const Parts<Y> &b, f32x16 c)
{
    if constexpr (Y::S == 3) {
        c = Y::m::mfma(a.p[2], b.p[0], c);
        c = Y::m::mfma(a.p[0], b.p[2], c);
        c = Y::m::mfma(a.p[1], b.p[1], c);
        c = Y::m::mfma(a.p[1], b.p[0], c);
        c = Y::m::mfma(a.p[0], b.p[1], c);
    }
    return Y::m::mfma(a.p[0], b.p[0], c);
}

// the larger of two, NaN if either is
__device__ __forceinline__ float larger(float a, float b) { return a != a || a >= b ? a : b; }

__device__ __forceinline__ float other_half(float x) { return __shfl_xor(x, 32); }

// A UNIT is one operand of a matrix instruction as it lies in memory: 64 lanes x 8 values, 1 KB.
constexpr int kUnit = 1024;

// ---------------------------------------------------------------------------------------------------------------------
// packing: rows [R][K] (row stride ld) -> units.  `by_row`: tile of 32 rows after tile, in it K / 16 units (lane: row lane % 32,
// columns 16 cb + 8 (lane / 32) + j).  `by_col`: tile after tile, in it (K / 32) x 2 units (lane: column 32 ko + lane % 32, rows
// 16 t + 8 (j / 4) + 4 (lane / 32) + j % 4: the order of a product's output registers).  Columns and rows beyond the matrix
// are zero, and so are rows whose target is no item (padding: whatever they hold must not reach a sum).  Bound by memory:
// one workgroup takes 32 rows x 128 columns through shared memory, read once for both forms.
// ---------------------------------------------------------------------------------------------------------------------
template <class Y>
__global__ __launch_bounds__(256) void pack_kernel(const typename Y::t *src, int64_t ld, int64_t R, int K, int CB, int KO, char *by_row,
                                                   char *by_col, const int64_t *target, int64_t items, float sign)
{
    __shared__ float tile[32][129];
    const int64_t rb = blockIdx.x;
    const int c0 = blockIdx.y * 128;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const int at = i * 256 + threadIdx.x, r = at >> 7, c = c0 + (at & 127);
        const int64_t row = rb * 32 + r;
        float x = 0.0f;
        if (row < R && c < K && !(target && (uint64_t)target[row] >= (uint64_t)items))
            x = (float)src[row * ld + c];
        tile[r][at & 127] = x;
    }
    __syncthreads();
    const int lane = threadIdx.x & 63, low = lane & 31, h = lane >> 5;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int u = i * 4 + (threadIdx.x >> 6), cb = blockIdx.y * 8 + u;
        if (by_row && cb < CB) {
            Parts<Y> q;
#pragma unroll
            for (int j = 0; j < 8; ++j)
                split<Y>(sign * tile[low][16 * u + 8 * h + j], q, j);
            for (int s = 0; s < Y::S; ++s)
                *(typename Y::m::v8 *)(by_row + (((rb * CB + cb) * Y::S + s) * 64 + lane) * 16) = q.p[s];
        }
        const int ko = blockIdx.y * 4 + (u >> 1), t = u & 1;
        if (by_col && ko < KO) {
            Parts<Y> q;
#pragma unroll
            for (int j = 0; j < 8; ++j)
                split<Y>(tile[16 * t + 8 * (j >> 2) + 4 * h + (j & 3)][32 * (u >> 1) + low], q, j);
            for (int s = 0; s < Y::S; ++s)
                *(typename Y::m::v8 *)(by_col + ((((rb * KO + ko) * 2 + t) * Y::S + s) * 64 + lane) * 16) = q.p[s];
        }
    }
}

// bias in base 2, -inf beyond the catalogue (and nothing but that where there is no bias)
__global__ void bias_kernel(const float *bias, int64_t V, int64_t padded, float *out)
{
    const int64_t v = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (v < padded)
        out[v] = v >= V ? -INFINITY : bias ? bias[v] * kLog2e : 0.0f;
}

// the smallest power of two that is no less than any |weight| (1 if there is none): G is held as a share of it
__global__ __launch_bounds__(1024) void weight_kernel(const float *weight, int64_t N, float *out)
{
    __shared__ float top[16];
    float m = 0.0f;
    if (weight)
        for (int64_t n = threadIdx.x; n < N; n += 1024)
            m = fmaxf(m, fabsf(weight[n]));
    for (int d = 32; d; d >>= 1)
        m = fmaxf(m, __shfl_xor(m, d));
    if ((threadIdx.x & 63) == 0)
        top[threadIdx.x >> 6] = m;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int i = 1; i < 16; ++i)
            m = fmaxf(m, top[i]);
        int e = 0;
        if (m > 0.0f && m < INFINITY)
            frexpf(m, &e);                       // m in [2^(e-1), 2^e)
        out[0] = ldexpf(1.0f, e > 100 ? 100 : e < -100 ? -100 : e);
    }
}

// ---------------------------------------------------------------------------------------------------------------------
// the passes
// ---------------------------------------------------------------------------------------------------------------------
enum { kNll, kRows, kItems };

struct PassArgs {
    const char *still;        // stationary matrix, by_row
    const char *by_row;       // streamed matrix
    const char *by_col;
    const float *reg_bias;    // per streamed row: rows passes: its bias (base 2); items pass: log2 |weight| - lse
    const float *lane_bias;   // items pass: the stationary item's bias
    const int32_t *meta;      // items pass: per streamed row its target and flag; rows passes: per stationary row
    const float *target_g;    // items pass: per streamed row, G at its target
    float *stats;             // rows passes: [split][3][still rows]: maximum, sum without the target, target's logit
    float *part;              // [split][still rows][32 KO]
    float *part_sum;          // items pass: [split][still rows], sums of G
    int64_t still_tiles, still_rows, stream_tiles;   // tiles of 32; still_rows = 32 still_tiles
    float c;                  // |scale| log2(e)
    int splits, bias;
};

// every wavefront's staged units are in shared memory (a barrier alone does not wait for them)
__device__ __forceinline__ void staged_barrier()
{
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
}

template <class Y, int KO, int MODE> struct Shape {
    static constexpr int S = Y::S, CB = 2 * KO;
    static constexpr int row_units = CB * S, col_units = MODE == kNll ? 0 : 2 * KO * S, units = row_units + col_units;   // per tile
    static constexpr int NW = S == 3 && KO == 4 ? 8 : 4;                      // wavefronts
    static constexpr int QB = (S == 1 && KO <= 4) || KO == 1 ? 2 : 1;         // stationary tiles of a wavefront
    static constexpr int RT = units <= 4 ? 4 : units <= 12 ? 2 : 1;           // streamed tiles a stage
    static constexpr int bufs = 2 * RT * units > 150 ? 1 : 2;
    static constexpr int waves = S == 3 && KO == 8 ? 1 : 2;                   // per SIMD: 512 or 256 registers
};

__device__ __forceinline__ void stage_unit(const char *from, char *to)
{
    __builtin_amdgcn_global_load_lds((__attribute__((address_space(1))) const void *)(from + (threadIdx.x & 63) * 16),
                                     (__attribute__((address_space(3))) void *)(uintptr_t)to, 16, 0, 0);
}

// One block of logits (base 2; lane: stationary row, register: item) into a running softmax: the target's own is taken out to `at`, the
// rest become probabilities relative to the new maximum (times 2^shift); `rescale(f)` is called where the maximum grew.
template <class Y, class F>
__device__ __forceinline__ void online(f32x16 &x, int tile, int h, int target, float &top, float &sum, float &at, const F &rescale)
{
    if (__any((target >> 5) == tile))
#pragma unroll
        for (int i = 0; i < 16; ++i)
            if (target == tile * 32 + 8 * (i >> 2) + 4 * h + (i & 3)) {
                at = x[i];
                x[i] = -INFINITY;
            }
    float m = x[0];
#pragma unroll
    for (int i = 1; i < 16; ++i)
        m = fmaxf(m, x[i]);
    m = fmaxf(m, other_half(m));
    if (__any(m > top)) {
        const float grown = fmaxf(m, top), f = __builtin_amdgcn_exp2f(top - grown);
        sum *= f;
        top = grown;
        rescale(f);
    }
    const float down = (float)Y::shift - top;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        x[i] = __builtin_amdgcn_exp2f(x[i] + down);
        sum += x[i];
    }
}

__device__ __forceinline__ void store_stats(float *to, int64_t rows, int h, float top, float sum, float at)
{
    const float both = sum + other_half(sum), hit = larger(at, other_half(at));
    if (h == 0) {
        to[0] = top;
        to[rows] = both;
        to[2 * rows] = hit;
    }
}

template <class Y, int KO, int MODE>
__global__ __launch_bounds__((Shape<Y, KO, MODE>::NW * 64), (Shape<Y, KO, MODE>::waves)) void pass_kernel(PassArgs A)
{
    typedef Shape<Y, KO, MODE> Z;
    constexpr int S = Z::S, CB = Z::CB, QB = Z::QB, RT = Z::RT, NW = Z::NW;
    __shared__ __attribute__((aligned(1024))) char lds[Z::bufs][RT * Z::units * kUnit];

    const int lane = threadIdx.x & 63, low = lane & 31, h = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int sp = blockIdx.x % A.splits;                                  // equal splits stream the same tiles: ids a multiple of 8 apart
    const int64_t q0 = ((int64_t)(blockIdx.x / A.splits) * NW + wave) * QB;   // meet on one die and its cache
    const int64_t groups = (A.stream_tiles + RT - 1) / RT;
    const int64_t g0 = groups * sp / A.splits, g1 = groups * (sp + 1) / A.splits;

    Parts<Y> still[QB][CB];
    int target[QB];
    float lane_bias[QB];
#pragma unroll
    for (int q = 0; q < QB; ++q) {
        const bool in = q0 + q < A.still_tiles;
#pragma unroll
        for (int cb = 0; cb < CB; ++cb)
            for (int s = 0; s < S; ++s) {
                typename Y::m::v8 z = {};
                still[q][cb].p[s] = in ? *(const typename Y::m::v8 *)(A.still + (((q0 + q) * CB + cb) * S + s) * kUnit + lane * 16) : z;
            }
        target[q] = MODE != kItems && in ? A.meta[(q0 + q) * 32 + low] : kNoTarget;
        lane_bias[q] = MODE == kItems && in && A.bias ? A.lane_bias[(q0 + q) * 32 + low] : 0.0f;
    }

    f32x16 acc[QB][MODE == kNll ? 1 : KO];
    float top[QB], sum[QB], at[QB];
#pragma unroll
    for (int q = 0; q < QB; ++q) {
        top[q] = kNothing;
        sum[q] = 0.0f;
        at[q] = -INFINITY;
        if constexpr (MODE != kNll)
            for (int ko = 0; ko < KO; ++ko)
                acc[q][ko] = (f32x16)(0.0f);
    }

    auto stage = [&](int64_t g, int buf) {
        const char *from = A.by_row + g * RT * Z::row_units * kUnit;
#pragma unroll
        for (int u = 0; u < RT * Z::row_units; u += NW)
            if (u + wave < RT * Z::row_units)
                stage_unit(from + (u + wave) * kUnit, &lds[buf][(u + wave) * kUnit]);
        if constexpr (MODE != kNll) {
            from = A.by_col + g * RT * Z::col_units * kUnit;
#pragma unroll
            for (int u = 0; u < RT * Z::col_units; u += NW)
                if (u + wave < RT * Z::col_units)
                    stage_unit(from + (u + wave) * kUnit, &lds[buf][(RT * Z::row_units + u + wave) * kUnit]);
        }
    };
    auto fetch = [&](const char *unit) {
        Parts<Y> x;
        for (int s = 0; s < S; ++s)
            x.p[s] = *(const typename Y::m::v8 *)(unit + s * kUnit + lane * 16);
        return x;
    };

    if (Z::bufs == 2 && g0 < g1)
        stage(g0, 0);
    for (int64_t g = g0; g < g1; ++g) {
        int buf = 0;
        if constexpr (Z::bufs == 2) {
            buf = (int)(g - g0) & 1;
            staged_barrier();                     // this group has arrived, and the other buffer has been read
            if (g + 1 < g1)
                stage(g + 1, buf ^ 1);
        } else {
            __syncthreads();
            stage(g, 0);
            staged_barrier();
        }
#pragma unroll 1
        for (int rt = 0; rt < RT; ++rt) {
            const int64_t tile = g * RT + rt;
            if (tile >= A.stream_tiles)
                break;
            const char *rows = &lds[buf][rt * Z::row_units * kUnit], *cols = &lds[buf][(RT * Z::row_units + rt * Z::col_units) * kUnit];
            const bool biased = MODE == kItems || A.bias || tile == A.stream_tiles - 1;
            f32x4 rb[4];
            if (biased)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    rb[i] = *(const f32x4 *)(A.reg_bias + tile * 32 + 8 * i + 4 * h);
            int meta = 0;
            if constexpr (MODE == kItems)
                meta = A.meta[tile * 32 + low];

            f32x16 z[QB];
#pragma unroll
            for (int q = 0; q < QB; ++q)
                z[q] = (f32x16)(0.0f);
#pragma unroll
            for (int cb = 0; cb < CB; ++cb) {
                const Parts<Y> a = fetch(rows + cb * S * kUnit);
#pragma unroll
                for (int q = 0; q < QB; ++q)
                    z[q] = product<Y>(a, still[q][cb], z[q]);
            }

            Parts<Y> p[QB][2];
#pragma unroll
            for (int q = 0; q < QB; ++q) {
                f32x16 &x = z[q];
                if constexpr (MODE == kItems) {
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        x[i] = __builtin_amdgcn_exp2f(fmaf(x[i], A.c, rb[i >> 2][i & 3] + lane_bias[q]));
                    if (__any(meta & kNegative))
#pragma unroll
                        for (int i = 0; i < 16; ++i)
                            if (__shfl(meta, 8 * (i >> 2) + 4 * h + (i & 3)) & kNegative)
                                x[i] = -x[i];
                    if (__any(((meta & ~kNegative) >> 5) == (int)(q0 + q)))
#pragma unroll
                        for (int i = 0; i < 16; ++i) {
                            const int r = 8 * (i >> 2) + 4 * h + (i & 3);
                            if ((__shfl(meta, r) & ~kNegative) == (int)(q0 + q) * 32 + low)
                                x[i] = A.target_g[tile * 32 + r];
                        }
                    if (A.bias)
#pragma unroll
                        for (int i = 0; i < 16; ++i)
                            sum[q] += x[i];
                } else {
                    if (biased) {
#pragma unroll
                        for (int i = 0; i < 16; ++i)
                            x[i] = fmaf(x[i], A.c, rb[i >> 2][i & 3]);
                    } else {
#pragma unroll
                        for (int i = 0; i < 16; ++i)
                            x[i] = x[i] * A.c;
                    }
                    online<Y>(x, (int)tile, h, target[q], top[q], sum[q], at[q], [&](float f) {
                        if constexpr (MODE == kRows)
#pragma unroll
                            for (int ko = 0; ko < KO; ++ko)
                                acc[q][ko] *= f;
                    });
                }
                if constexpr (MODE != kNll)
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        split<Y>(x[i], p[q][i >> 3], i & 7);
            }

            if constexpr (MODE != kNll)
#pragma unroll
                for (int ko = 0; ko < KO; ++ko)
#pragma unroll
                    for (int t = 0; t < 2; ++t) {
                        const Parts<Y> a = fetch(cols + (ko * 2 + t) * S * kUnit);
#pragma unroll
                        for (int q = 0; q < QB; ++q)
                            acc[q][ko] = product<Y>(a, p[q][t], acc[q][ko]);
                    }
        }
    }

#pragma unroll
    for (int q = 0; q < QB; ++q) {
        if (q0 + q >= A.still_tiles)
            break;
        const int64_t row = (q0 + q) * 32 + low;
        if constexpr (MODE == kItems) {
            const float both = sum[q] + other_half(sum[q]);
            if (A.bias && h == 0)
                A.part_sum[sp * A.still_rows + row] = both;
        } else {
            store_stats(A.stats + (int64_t)sp * 3 * A.still_rows + row, A.still_rows, h, top[q], sum[q], at[q]);
        }
        if constexpr (MODE != kNll) {
            float *to = A.part + (sp * A.still_rows + row) * (32 * KO) + 4 * h;
#pragma unroll
            for (int ko = 0; ko < KO; ++ko)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const f32x4 o = {acc[q][ko][4 * i], acc[q][ko][4 * i + 1], acc[q][ko][4 * i + 2], acc[q][ko][4 * i + 3]};
                    *(f32x4 *)(to + 32 * ko + 8 * i) = o;
                }
        }
    }
}

// ---------------------------------------------------------------------------------------------------------------------
// Rows too wide for a wavefront's registers (k > 256): plain tiled products of packed matrices, the catalogue in chunks.  The
// statistics come from a first run over all logits; then, chunk by chunk, G is written in both operand layouts (16-bit parts,
// a chunk at a time: at most kChunkBytes) and multiplied with the items (dx, summed over the chunks) and with x (dw).
// Bound by the matrix instructions: 8 N V K operations, 128 x 128 outputs a workgroup, 64 x 64 a wavefront.
// ---------------------------------------------------------------------------------------------------------------------
constexpr int64_t kChunkBytes = 192ll << 20;

template <class Y, int KC_> struct Wide {
    static constexpr int S = Y::S, KC = KC_;                // units of the contraction a stage
    static constexpr int stage = 8 * KC * S * kUnit;        // 4 tiles of each matrix
};
template <class Y> struct Logits : Wide<Y, Y::S == 1 ? 4 : 2> {};

// For each group: the 128 x 128 product of 4 + 4 tiles over `steps` stages, handed to `done(group, acc)`.  a(group, step, tile) and
// b(group, step, tile) are a tile's KC S consecutive units.
template <class Y, class Z, class A, class B, class D>
__device__ __forceinline__ void wide_core(char *lds, int64_t groups, int steps, const A &a, const B &b, const D &done)
{
    constexpr int S = Z::S, KC = Z::KC, per = KC * S;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wa = wave >> 1, wb = wave & 1;
    auto stage = [&](int64_t g, int step, int buf) {
        const char *pa = a(g, step, wave), *pb = b(g, step, wave);       // wavefront w brings tile w of each matrix
#pragma unroll
        for (int u = 0; u < per; ++u) {
            stage_unit(pa + u * kUnit, lds + buf * Z::stage + (wave * per + u) * kUnit);
            stage_unit(pb + u * kUnit, lds + buf * Z::stage + ((4 + wave) * per + u) * kUnit);
        }
    };
    f32x16 acc[2][2];
    int buf = 0;
    if (groups > 0 && steps > 0)
        stage(0, 0, 0);
    for (int64_t g = 0; g < groups; ++g) {
#pragma unroll
        for (int i = 0; i < 2; ++i)
            for (int j = 0; j < 2; ++j)
                acc[i][j] = (f32x16)(0.0f);
        for (int step = 0; step < steps; ++step, buf ^= 1) {
            staged_barrier();                      // this stage has arrived, the other has been read
            if (step + 1 < steps)
                stage(g, step + 1, buf ^ 1);
            else if (g + 1 < groups)   // (groups of one length: steps > 0 here)
                stage(g + 1, 0, buf ^ 1);
            const char *at = lds + buf * Z::stage + lane * 16;
#pragma unroll
            for (int c = 0; c < KC; ++c) {
                Parts<Y> x[2], y[2];
#pragma unroll
                for (int i = 0; i < 2; ++i)
                    for (int s = 0; s < S; ++s) {
                        x[i].p[s] = *(const typename Y::m::v8 *)(at + ((2 * wa + i) * per + c * S + s) * kUnit);
                        y[i].p[s] = *(const typename Y::m::v8 *)(at + ((4 + 2 * wb + i) * per + c * S + s) * kUnit);
                    }
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int j = 0; j < 2; ++j)
                        acc[i][j] = product<Y>(x[i], y[j], acc[i][j]);
            }
        }
        done(g, acc);
    }
}

struct WideArgs {
    const char *w, *x;              // by_row units
    const float *bias, *reg_bias, *target_g;
    const int32_t *meta;
    float *stats, *part_sum;
    char *g_rows, *g_items;         // G of a chunk: rows n / contraction v, and rows v / contraction n
    int64_t n_tiles, v_tiles, rows, v0, v_count;   // tiles; v0, v_count: the chunk
    float c;
    int CB, splits, has_bias;
};

// logits in base 2 of one 32 x 32 block: lane: row n, register: item
__device__ __forceinline__ void wide_bias(f32x16 &x, const WideArgs &A, int64_t tile, int h)
{
    if (A.has_bias || tile == A.v_tiles - 1) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const f32x4 b = *(const f32x4 *)(A.bias + tile * 32 + 8 * i + 4 * h);
#pragma unroll
            for (int j = 0; j < 4; ++j)
                x[4 * i + j] = fmaf(x[4 * i + j], A.c, b[j]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 16; ++i)
            x[i] *= A.c;
    }
}

template <class Y> __global__ __launch_bounds__(256, 2) void wide_stats_kernel(WideArgs A)
{
    typedef Logits<Y> Z;
    __shared__ __attribute__((aligned(1024))) char lds[2 * Z::stage];
    const int lane = threadIdx.x & 63, low = lane & 31, h = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wa = wave >> 1, wb = wave & 1;
    const int sp = blockIdx.x % A.splits;
    const int64_t n0 = (int64_t)(blockIdx.x / A.splits) * 4;
    const int64_t all = (A.v_tiles + 3) / 4, g0 = all * sp / A.splits, g1 = all * (sp + 1) / A.splits;
    int target[2];
    float top[2], sum[2], at[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const int64_t tile = n0 + 2 * wb + j;
        target[j] = tile < A.n_tiles ? A.meta[tile * 32 + low] : kNoTarget;
        top[j] = kNothing;
        sum[j] = 0.0f;
        at[j] = -INFINITY;
    }
    wide_core<Y, Z>(
        lds, g1 - g0, A.CB / Z::KC,
        [&](int64_t g, int step, int tile) { return A.w + (((g0 + g) * 4 + tile) * A.CB + step * Z::KC) * Z::S * kUnit; },
        [&](int64_t, int step, int tile) { return A.x + ((n0 + tile) * A.CB + step * Z::KC) * Z::S * kUnit; },
        [&](int64_t g, f32x16 (&acc)[2][2]) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int64_t tile = (g0 + g) * 4 + 2 * wa + i;
                if (tile >= A.v_tiles)
                    break;
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    f32x16 &x = acc[i][j];
                    wide_bias(x, A, tile, h);
                    online<Y>(x, (int)tile, h, target[j], top[j], sum[j], at[j], [](float) {});
                }
            }
        });
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const int64_t tile = n0 + 2 * wb + j;
        if (tile < A.n_tiles)
            store_stats(A.stats + (int64_t)(2 * sp + wa) * 3 * A.rows + tile * 32 + low, A.rows, h, top[j], sum[j], at[j]);
    }
}

// G of 4 tiles of rows against 4 tiles of items of the chunk, in both layouts, and the sums over its rows
template <class Y> __global__ __launch_bounds__(256, 2) void wide_g_kernel(WideArgs A)
{
    typedef Logits<Y> Z;
    typedef typename Y::m::e e;
    constexpr int S = Y::S;
    __shared__ __attribute__((aligned(1024))) char lds[2 * Z::stage];
    __shared__ __attribute__((aligned(16))) e turn_all[4][32][36];      // a block a wavefront, to exchange its lanes and registers
    const int lane = threadIdx.x & 63, low = lane & 31, h = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wa = wave >> 1, wb = wave & 1;
    e(*turn)[36] = turn_all[wave];
    const int64_t ngroups = (A.n_tiles + 3) / 4, n0 = blockIdx.x % ngroups * 4, vg = blockIdx.x / ngroups * 4;   // vg: within the chunk
    int meta[2];
    float down[2], tg[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const int64_t tile = n0 + 2 * wb + j;
        const bool in = tile < A.n_tiles;
        meta[j] = in ? A.meta[tile * 32 + low] : kNoTarget;
        down[j] = in ? A.reg_bias[tile * 32 + low] : -INFINITY;
        tg[j] = in ? A.target_g[tile * 32 + low] : 0.0f;
    }
    wide_core<Y, Z>(
        lds, 1, A.CB / Z::KC,
        [&](int64_t, int step, int tile) { return A.w + ((A.v0 + vg + tile) * A.CB + step * Z::KC) * Z::S * kUnit; },
        [&](int64_t, int step, int tile) { return A.x + ((n0 + tile) * A.CB + step * Z::KC) * Z::S * kUnit; },
        [&](int64_t, f32x16 (&acc)[2][2]) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int64_t vt = vg + 2 * wa + i, tile = A.v0 + vt;
                if (vt >= A.v_count)
                    break;
                f32x16 total = (f32x16)(0.0f);
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const int64_t nt = n0 + 2 * wb + j;
                    if (nt >= A.n_tiles)
                        break;
                    f32x16 &x = acc[i][j];
                    wide_bias(x, A, tile, h);
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        x[r] = __builtin_amdgcn_exp2f(x[r] + down[j]);
                        if (meta[j] & kNegative)
                            x[r] = -x[r];
                    }
                    if (__any(((meta[j] & ~kNegative) >> 5) == (int)tile))
#pragma unroll
                        for (int r = 0; r < 16; ++r)
                            if ((meta[j] & ~kNegative) == (int)tile * 32 + 8 * (r >> 2) + 4 * h + (r & 3))
                                x[r] = tg[j];
                    total += x;
                    Parts<Y> p[2];
#pragma unroll
                    for (int r = 0; r < 16; ++r)
                        split<Y>(x[r], p[r >> 3], r & 7);
                    for (int s = 0; s < S; ++s) {
#pragma unroll
                        for (int t = 0; t < 2; ++t)
                            *(typename Y::m::v8 *)(A.g_rows + (((nt * A.v_count + vt) * 2 + t) * S + s) * kUnit + lane * 16) = p[t].p[s];
#pragma unroll
                        for (int r = 0; r < 16; ++r)
                            turn[low][8 * (r >> 2) + 4 * h + (r & 3)] = p[r >> 3].p[s][r & 7];
                        // (one wavefront's own block: its accesses to shared memory are served in order)
                        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
                        for (int t = 0; t < 2; ++t) {
                            typename Y::m::v8 q;
#pragma unroll
                            for (int r = 0; r < 8; ++r)
                                q[r] = turn[16 * t + 8 * (r >> 2) + 4 * h + (r & 3)][low];
                            *(typename Y::m::v8 *)(A.g_items + (((vt * A.n_tiles + nt) * 2 + t) * S + s) * kUnit + lane * 16) = q;
                        }
                        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                    }
                }
                if (A.has_bias) {   // over the lanes of each half: [64 rows][chunk's items]
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        float v = total[r];
                        for (int d = 16; d; d >>= 1)
                            v += __shfl_xor(v, d);
                        if (low == 0)
                            A.part_sum[((n0 / 2 + wb) * A.v_count + vt) * 32 + 8 * (r >> 2) + 4 * h + (r & 3)] = v;
                    }
                }
            }
        });
}

// c[m][k] = sum over the contraction's tiles of a (by_row units, U of them a tile) times b (by_col units)
struct ProductArgs {
    const char *a, *b;
    int64_t a_tiles, a_units, tiles;      // output tiles, units of one, contraction tiles (32 each)
    int KO, splits;
    float *part;                          // [split][32 a_tiles][32 KO] sums; `more`: added to what is there
    int more;
};

template <class Y> __global__ __launch_bounds__(256, 2) void wide_product_kernel(ProductArgs A)
{
    typedef Wide<Y, 2> Z;
    __shared__ __attribute__((aligned(1024))) char lds[2 * Z::stage];
    const int lane = threadIdx.x & 63, low = lane & 31, h = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wa = wave >> 1, wb = wave & 1;
    const int kgroups = (A.KO + 3) / 4;
    int64_t id = blockIdx.x;
    const int kg = (int)(id % kgroups) * 4;
    id /= kgroups;
    const int sp = (int)(id % A.splits);
    const int64_t m0 = id / A.splits * 4;
    const int64_t s0 = A.tiles * sp / A.splits, s1 = A.tiles * (sp + 1) / A.splits;   // a contraction tile a stage
    wide_core<Y, Z>(
        lds, 1, (int)(s1 - s0),
        [&](int64_t, int step, int tile) { return A.a + ((m0 + tile) * A.a_units + (s0 + step) * Z::KC) * Z::S * kUnit; },
        [&](int64_t, int step, int tile) { return A.b + ((s0 + step) * A.KO + (kg + tile < A.KO ? kg + tile : A.KO - 1)) * Z::KC * Z::S * kUnit; },
        [&](int64_t, f32x16 (&acc)[2][2]) {
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const int64_t mt = m0 + 2 * wa + i;
                    const int ko = kg + 2 * wb + j;
                    if (mt >= A.a_tiles || ko >= A.KO)
                        continue;
                    float *to = A.part + ((sp * A.a_tiles + mt) * 32) * (int64_t)(32 * A.KO) + 32 * ko + low;
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        float *o = to + (8 * (r >> 2) + 4 * h + (r & 3)) * (int64_t)(32 * A.KO);
                        *o = A.more ? *o + acc[i][j][r] : acc[i][j][r];
                    }
                }
        });
}

// meta of the rows before their passes: targets as 32-bit numbers
__global__ void targets_kernel(const int64_t *target, int64_t N, int64_t V, int64_t padded, int32_t *meta)
{
    const int64_t n = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (n < padded) {
        const int64_t t = n < N ? target[n] : -1;
        meta[n] = t >= 0 && t < V ? (int32_t)t : kNoTarget;
    }
}

// ---------------------------------------------------------------------------------------------------------------------
// Joins a row's splits: loss and lse, what the items pass needs of the row, and dx (a wavefront a row).
// ---------------------------------------------------------------------------------------------------------------------
struct FinishArgs {
    const float *stats, *part;
    const int64_t *target;
    const float *weight, *wpow;
    const void *w;                 // items, for the target's own row
    float *loss, *lse, *reg_bias, *target_g;
    int32_t *meta;
    void *dx;
    int64_t N, V, rows, ldw, lddx;
    int K, KP, splits;
    float scale;
};

template <class Y, bool GRAD> __global__ __launch_bounds__(256) void finish_rows_kernel(FinishArgs A)
{
    const int lane = threadIdx.x & 63;
    const int64_t n = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (n >= A.rows)
        return;
    if (n >= A.N) {                // rows that only fill the last tile: no share of any sum
        if (GRAD && lane == 0) {
            A.reg_bias[n] = -INFINITY;
            A.target_g[n] = 0.0f;
            A.meta[n] = kNoTarget;
        }
        return;
    }
    float top = kNothing, others = 0.0f, at = -INFINITY;
    for (int s = 0; s < A.splits; ++s) {
        top = fmaxf(top, A.stats[(3 * s + 0) * A.rows + n]);
        at = larger(at, A.stats[(3 * s + 2) * A.rows + n]);
    }
    for (int s = 0; s < A.splits; ++s)
        others += A.stats[(3 * s + 1) * A.rows + n] * __builtin_amdgcn_exp2f(A.stats[3 * s * A.rows + n] - top);
    others *= __builtin_amdgcn_exp2f(-(float)Y::shift);
    // `top` is that of the others; the target's own logit may be far above it
    const float peak = fmaxf(top, at);
    const float rest = others * __builtin_amdgcn_exp2f(top - peak), own = __builtin_amdgcn_exp2f(at - peak), all = rest + own;
    const float lse2 = all > 0.0f || all != all ? peak + log2f(all) : -INFINITY;
    const int64_t t = A.target[n];
    float loss = 0.0f;
    bool alive = t >= 0;
    if (t >= A.V) {                // no such item: said in the loss, and kept out of the gradients
        loss = __builtin_nanf("");
        alive = false;
    } else if (t >= 0) {
        if (!(at > kNothing) && at == at && all == all) {   // a masked target
            loss = INFINITY;
            alive = false;
        } else if (own > 0.0f && rest < 0x1p20f * own) {
            loss = log1pf(rest / own);
        } else {
            loss = (lse2 - at) * kLn2;
        }
    }
    if (lane == 0) {
        A.loss[n] = loss;
        if (A.lse)
            A.lse[n] = lse2 * kLn2;
    }
    if constexpr (GRAD) {
        const float weight = alive ? (A.weight ? A.weight[n] : 1.0f) : 0.0f, wpow = *A.wpow;
        const float gt = -(weight / wpow) * (rest / all);          // G at the target, as a share of wpow
        if (lane == 0) {
            A.reg_bias[n] = alive ? (log2f(fabsf(weight) / wpow) - lse2) + (float)Y::shift : -INFINITY;
            A.target_g[n] = alive ? gt * __builtin_amdgcn_exp2f((float)Y::shift) : 0.0f;
            A.meta[n] = alive ? (int32_t)t | (weight < 0.0f ? kNegative : 0) : kNoTarget;
        }
        if (!A.dx)
            return;
        typedef typename Y::t T;
        T *dx = (T *)A.dx + n * A.lddx;
        const T *w = (const T *)A.w + (alive ? t : 0) * A.ldw;
        const float share = weight / all * __builtin_amdgcn_exp2f(top - peak - (float)Y::shift);
        for (int k = lane; k < A.K; k += 64) {
            float sum = 0.0f;
            if (alive) {
                for (int s = 0; s < A.splits; ++s)
                    sum += A.part[(s * A.rows + n) * A.KP + k] * __builtin_amdgcn_exp2f(A.stats[3 * s * A.rows + n] - top);
                sum = A.scale * (sum * share + gt * wpow * (float)w[k]);
            }
            dx[k] = (T)sum;
        }
    }
}

// joins the splits of a product with G: out = scale wpow sum, dbias = wpow sum (a wavefront a row)
template <class Y>
__global__ __launch_bounds__(256) void finish_items_kernel(const float *part, const float *part_sum, const float *wpow, int64_t V, int64_t rows,
                                                           int K, int KP, int splits, int sum_splits, float scale, typename Y::t *dw, int64_t lddw, float *dbias)
{
    const int lane = threadIdx.x & 63;
    const int64_t v = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (v >= V)
        return;
    const float f = *wpow * __builtin_amdgcn_exp2f(-(float)Y::shift);
    for (int k = lane; k < K; k += 64) {
        float sum = 0.0f;
        for (int s = 0; s < splits; ++s)
            sum += part[(s * rows + v) * KP + k];
        dw[v * lddw + k] = (typename Y::t)(scale * (f * sum));
    }
    if (dbias && lane == 0) {
        float sum = 0.0f;
        for (int s = 0; s < sum_splits; ++s)
            sum += part_sum[s * rows + v];
        dbias[v] = f * sum;
    }
}

template <class T> __global__ void zero_rows_kernel(T *p, int64_t rows, int K, int64_t ld)
{
    for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < rows * K; i += (int64_t)gridDim.x * blockDim.x)
        p[i / K * ld + i % K] = (T)0.0f;
}

// ---------------------------------------------------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------------------------------------------------
int64_t up(int64_t a, int64_t b) { return (a + b - 1) / b * b; }

struct Plan {
    bool wide;
    int KO, KP, row_splits, item_splits, stats_splits, sum_splits;
    int64_t chunk;                                  // wide: tiles of items at a time
    int64_t n_tiles, v_tiles;                       // of 32, without padding
    int64_t x_row, x_col, w_row, w_col, bias, reg, tg, meta, wpow, stats, part, part_sum, dx_part, g_rows, g_items, bytes;   // offsets
};

int64_t tiles_padded(int64_t tiles) { return up(tiles, kPadTiles); }

// how many pieces the streamed side is cut into: enough workgroups for four on each compute unit, each with 8 tiles at least, in eights
// (one a die) once there are that many
int64_t pick_splits(int64_t workgroups, int64_t stream_tiles, int cus)
{
    int64_t s = (4 * cus + workgroups - 1) / workgroups;
    if (s > stream_tiles / 8)
        s = stream_tiles / 8;
    if (s > 8)
        s = s / 8 * 8;
    return s < 1 ? 1 : s;
}

// wide: pieces of a chunk's contraction for dx
int dx_splits(const Plan &P, int cus) { return (int)pick_splits(2 * ((P.n_tiles + 3) / 4) * ((P.KO + 3) / 4), P.chunk, cus); }

template <class Y, int KO, int MODE> int64_t workgroups(int64_t tiles)
{
    typedef Shape<Y, KO, MODE> Z;
    return (tiles + Z::NW * Z::QB - 1) / (Z::NW * Z::QB);
}

template <class Y> void make_plan(Plan &P, int64_t n, int64_t v, int64_t k, bool grad, int cus)
{
    const int need = (int)((k + 31) / 32);
    P.wide = need > 8;
    P.KO = need <= 1 ? 1 : need <= 2 ? 2 : need <= 4 ? 4 : need <= 8 ? 8 : (need + 1) / 2 * 2;
    P.KP = 32 * P.KO;
    P.n_tiles = (n + 31) / 32;
    P.v_tiles = (v + 31) / 32;
    int64_t gr = 1, gi = 1;
    if (!P.wide) switch (P.KO) {
    case 1: gr = grad ? workgroups<Y, 1, kRows>(P.n_tiles) : workgroups<Y, 1, kNll>(P.n_tiles); gi = workgroups<Y, 1, kItems>(P.v_tiles); break;
    case 2: gr = grad ? workgroups<Y, 2, kRows>(P.n_tiles) : workgroups<Y, 2, kNll>(P.n_tiles); gi = workgroups<Y, 2, kItems>(P.v_tiles); break;
    case 4: gr = grad ? workgroups<Y, 4, kRows>(P.n_tiles) : workgroups<Y, 4, kNll>(P.n_tiles); gi = workgroups<Y, 4, kItems>(P.v_tiles); break;
    default: gr = grad ? workgroups<Y, 8, kRows>(P.n_tiles) : workgroups<Y, 8, kNll>(P.n_tiles); gi = workgroups<Y, 8, kItems>(P.v_tiles);
    }
    P.row_splits = (int)pick_splits(gr, P.v_tiles, cus);
    P.item_splits = (int)pick_splits(gi, P.n_tiles, cus);
    P.stats_splits = P.row_splits;
    if (P.wide) {
        const int64_t ng = (P.n_tiles + 3) / 4;
        P.row_splits = (int)pick_splits(2 * ng, P.v_tiles, cus);
        P.stats_splits = 2 * P.row_splits;
        const int64_t tile_bytes = up(P.n_tiles, 4) * 32 * 32 * 2 * Y::S * 2;
        P.chunk = kChunkBytes / tile_bytes / 4 * 4;
        P.chunk = P.chunk < 4 ? 4 : P.chunk > up(P.v_tiles, 4) ? up(P.v_tiles, 4) : P.chunk;
        const int64_t kg = (P.KO + 3) / 4;
        P.item_splits = (int)pick_splits(2 * kg * (P.chunk / 4), P.n_tiles, cus);   // dw: contraction over the rows
        P.sum_splits = (int)(2 * ng);
    }
    const int64_t nt = tiles_padded(P.n_tiles), vt = tiles_padded(P.v_tiles), unit = (int64_t)2 * P.KO * Y::S * kUnit;
    const int64_t nr = P.n_tiles * 32, vr = P.v_tiles * 32;
    int64_t at = 0;
    auto take = [&](int64_t bytes) {
        const int64_t here = at;
        at += up(bytes, 1024);
        return here;
    };
    P.x_row = take(nt * unit);
    P.w_row = take(vt * unit);
    P.bias = take(vt * 32 * 4);
    P.meta = take(nt * 32 * 4);
    P.stats = take((int64_t)P.stats_splits * 3 * nr * 4);
    if (grad) {
        P.x_col = take(nt * unit);
        P.w_col = take(vt * unit);
        P.reg = take(nt * 32 * 4);
        P.tg = take(nt * 32 * 4);
        P.wpow = take(4);
        if (P.wide) {
            P.part = take(P.item_splits * P.chunk * 32 * P.KP * 4);
            P.part_sum = take(P.sum_splits * P.chunk * 32 * 4);
            P.dx_part = take(dx_splits(P, cus) * nr * P.KP * 4);
            P.g_rows = take(up(P.n_tiles, 4) * P.chunk * 2 * Y::S * kUnit);
            P.g_items = take(up(P.n_tiles, 4) * P.chunk * 2 * Y::S * kUnit);
            P.bytes = at;
            return;
        }
        const int64_t rows_part = P.row_splits * nr * P.KP * 4, items_part = P.item_splits * vr * P.KP * 4;
        P.part = take(rows_part > items_part ? rows_part : items_part);   // (the rows' is read before the items' is written)
        P.part_sum = take(P.item_splits * vr * 4);
    }
    P.bytes = at;
}

template <class Y, int MODE> void launch_pass(int KO, const PassArgs &A, hipStream_t st)
{
    switch (KO) {
    case 1: pass_kernel<Y, 1, MODE><<<(unsigned)(workgroups<Y, 1, MODE>(A.still_tiles) * A.splits), Shape<Y, 1, MODE>::NW * 64, 0, st>>>(A); break;
    case 2: pass_kernel<Y, 2, MODE><<<(unsigned)(workgroups<Y, 2, MODE>(A.still_tiles) * A.splits), Shape<Y, 2, MODE>::NW * 64, 0, st>>>(A); break;
    case 4: pass_kernel<Y, 4, MODE><<<(unsigned)(workgroups<Y, 4, MODE>(A.still_tiles) * A.splits), Shape<Y, 4, MODE>::NW * 64, 0, st>>>(A); break;
    default: pass_kernel<Y, 8, MODE><<<(unsigned)(workgroups<Y, 8, MODE>(A.still_tiles) * A.splits), Shape<Y, 8, MODE>::NW * 64, 0, st>>>(A);
    }
}

struct Call {
    const void *x, *w;
    const int64_t *target;
    const float *weight, *bias;
    float *loss, *lse, *dbias;
    void *dx, *dw;
    int64_t n, v, k, ldx, ldw, lddx, lddw;
    float scale;
    bool grad;
    int cus;
    char *ws;
    int64_t ws_bytes;
    hipStream_t st;
};

template <class Y> int run(const Call &C)
{
    typedef typename Y::t T;
    Plan P = {};
    make_plan<Y>(P, C.n, C.v, C.k, C.grad, C.cus);
    if (C.ws_bytes < P.bytes)
        return HPF_EINVAL;
    const int K = (int)C.k, CB = 2 * P.KO;
    const dim3 groups_w((unsigned)P.v_tiles, (unsigned)((P.KP + 127) / 128)), groups_x((unsigned)P.n_tiles, (unsigned)((P.KP + 127) / 128));
    const float sign = C.scale < 0.0f ? -1.0f : 1.0f;     // goes into the packed x, so that logits rise with the product
    char *const ws = C.ws;
    pack_kernel<Y><<<groups_w, 256, 0, C.st>>>((const T *)C.w, C.ldw, C.v, K, CB, P.KO, ws + P.w_row, C.grad ? ws + P.w_col : nullptr, nullptr, 0, 1.0f);
    pack_kernel<Y><<<groups_x, 256, 0, C.st>>>((const T *)C.x, C.ldx, C.n, K, CB, P.KO, ws + P.x_row, C.grad ? ws + P.x_col : nullptr,
                                              C.grad ? C.target : nullptr, C.v, sign);
    const int64_t vp = tiles_padded(P.v_tiles) * 32, np = tiles_padded(P.n_tiles) * 32;
    bias_kernel<<<(unsigned)((vp + 255) / 256), 256, 0, C.st>>>(C.bias, C.v, vp, (float *)(ws + P.bias));
    targets_kernel<<<(unsigned)((np + 255) / 256), 256, 0, C.st>>>(C.target, C.n, C.v, np, (int32_t *)(ws + P.meta));
    if (C.grad)
        weight_kernel<<<1, 1024, 0, C.st>>>(C.weight, C.n, (float *)(ws + P.wpow));

    PassArgs A = {};
    A.still = ws + P.x_row;
    A.by_row = ws + P.w_row;
    A.by_col = ws + P.w_col;
    A.reg_bias = (const float *)(ws + P.bias);
    A.meta = (const int32_t *)(ws + P.meta);
    A.stats = (float *)(ws + P.stats);
    A.part = (float *)(ws + P.part);
    A.still_tiles = P.n_tiles;
    A.still_rows = P.n_tiles * 32;
    A.stream_tiles = P.v_tiles;
    A.c = fabsf(C.scale) * kLog2e;
    A.splits = P.row_splits;
    A.bias = C.bias != nullptr;
    WideArgs W = {};
    if (P.wide) {
        W.w = A.by_row;
        W.x = A.still;
        W.bias = A.reg_bias;
        W.meta = A.meta;
        W.stats = A.stats;
        W.n_tiles = P.n_tiles;
        W.v_tiles = P.v_tiles;
        W.rows = A.still_rows;
        W.c = A.c;
        W.CB = CB;
        W.splits = P.row_splits;
        W.has_bias = A.bias;
        wide_stats_kernel<Y><<<(unsigned)((P.n_tiles + 3) / 4 * P.row_splits), 256, 0, C.st>>>(W);
    } else if (C.grad)
        launch_pass<Y, kRows>(P.KO, A, C.st);
    else
        launch_pass<Y, kNll>(P.KO, A, C.st);

    FinishArgs F = {};
    F.stats = A.stats;
    F.part = A.part;
    F.target = C.target;
    F.weight = C.weight;
    F.wpow = (const float *)(ws + P.wpow);
    F.w = C.w;
    F.loss = C.loss;
    F.lse = C.lse;
    F.reg_bias = (float *)(ws + P.reg);
    F.target_g = (float *)(ws + P.tg);
    F.meta = (int32_t *)(ws + P.meta);
    F.dx = P.wide ? nullptr : C.dx;
    F.N = C.n;
    F.V = C.v;
    F.rows = A.still_rows;
    F.ldw = C.ldw;
    F.lddx = C.lddx;
    F.K = K;
    F.KP = P.KP;
    F.splits = P.stats_splits;
    F.scale = C.scale;
    const unsigned row_blocks = (unsigned)((F.rows + 3) / 4);
    if (!C.grad) {
        finish_rows_kernel<Y, false><<<row_blocks, 256, 0, C.st>>>(F);
        return (int)hipGetLastError();
    }
    finish_rows_kernel<Y, true><<<row_blocks, 256, 0, C.st>>>(F);

    if (P.wide) {
        W.reg_bias = F.reg_bias;
        W.target_g = F.target_g;
        W.part_sum = (float *)(ws + P.part_sum);
        W.g_rows = ws + P.g_rows;
        W.g_items = ws + P.g_items;
        const int kg = (P.KO + 3) / 4, zs = dx_splits(P, C.cus);
        float *const dx_part = (float *)(ws + P.dx_part), *const dw_part = (float *)(ws + P.part);
        for (int64_t v0 = 0; v0 < P.v_tiles; v0 += P.chunk) {
            W.v0 = v0;
            W.v_count = P.v_tiles - v0 < P.chunk ? P.v_tiles - v0 : P.chunk;
            wide_g_kernel<Y><<<(unsigned)((P.n_tiles + 3) / 4 * ((W.v_count + 3) / 4)), 256, 0, C.st>>>(W);
            ProductArgs D = {W.g_rows, ws + P.w_col + v0 * 2 * P.KO * Y::S * kUnit, P.n_tiles, W.v_count * 2, W.v_count, P.KO, zs, dx_part, v0 > 0};
            wide_product_kernel<Y><<<(unsigned)((P.n_tiles + 3) / 4 * kg * zs), 256, 0, C.st>>>(D);
            D = {W.g_items, ws + P.x_col, W.v_count, P.n_tiles * 2, P.n_tiles, P.KO, P.item_splits, dw_part, 0};
            wide_product_kernel<Y><<<(unsigned)((W.v_count + 3) / 4 * kg * P.item_splits), 256, 0, C.st>>>(D);
            const int64_t first = v0 * 32, count = C.v - first < W.v_count * 32 ? C.v - first : W.v_count * 32;
            finish_items_kernel<Y><<<(unsigned)((count + 3) / 4), 256, 0, C.st>>>(dw_part, W.part_sum, F.wpow, count, W.v_count * 32, K, P.KP,
                                                                                 P.item_splits, P.sum_splits, C.scale, (T *)C.dw + first * C.lddw,
                                                                                 C.lddw, C.bias ? C.dbias + first : nullptr);
        }
        finish_items_kernel<Y><<<(unsigned)((C.n + 3) / 4), 256, 0, C.st>>>(dx_part, nullptr, F.wpow, C.n, F.rows, K, P.KP, zs, 0, C.scale,
                                                                            (T *)C.dx, C.lddx, nullptr);
        return (int)hipGetLastError();
    }
    A.still = ws + P.w_row;
    A.by_row = ws + P.x_row;
    A.by_col = ws + P.x_col;
    A.reg_bias = F.reg_bias;
    A.lane_bias = (const float *)(ws + P.bias);
    A.target_g = F.target_g;
    A.part_sum = (float *)(ws + P.part_sum);
    A.still_tiles = P.v_tiles;
    A.still_rows = P.v_tiles * 32;
    A.stream_tiles = P.n_tiles;
    A.splits = P.item_splits;
    launch_pass<Y, kItems>(P.KO, A, C.st);
    finish_items_kernel<Y><<<(unsigned)((C.v + 3) / 4), 256, 0, C.st>>>(A.part, A.part_sum, F.wpow, C.v, A.still_rows, K, P.KP, P.item_splits,
                                                                        P.item_splits, C.scale, (T *)C.dw, C.lddw, C.bias ? C.dbias : nullptr);
    return (int)hipGetLastError();
}

int run_type(int type, const Call &C) { return type == HPF_F32 ? run<F32>(C) : type == HPF_BF16 ? run<B16>(C) : run<H16>(C); }

bool sizes_ok(int64_t n, int64_t v, int64_t k) { return n >= 0 && v > 0 && k > 0 && n < kNoTarget - 31 && v < kNoTarget - 31 && k < (1 << 20); }

}  // namespace

extern "C" int64_t hpf_hip_softmax_workspace(int64_t n, int64_t v, int64_t k, int type, int grad, int cu_count)
{
    if (!sizes_ok(n, v, k) || cu_count <= 0)
        return HPF_EINVAL;
    if (type < HPF_F32 || type > HPF_F16)
        return HPF_EUNSUPPORTED;
    if (n == 0)
        return 0;
    Plan P = {};
    if (type == HPF_F32)
        make_plan<F32>(P, n, v, k, grad != 0, cu_count);
    else if (type == HPF_BF16)
        make_plan<B16>(P, n, v, k, grad != 0, cu_count);
    else
        make_plan<H16>(P, n, v, k, grad != 0, cu_count);
    return P.bytes;
}

extern "C" int hpf_hip_softmax_nll(const void *x, int64_t ldx, const void *items, int64_t ld_items, const int64_t *target, const float *bias,
                                   float scale, int64_t n, int64_t v, int64_t k, int type, float *loss, float *lse, void *workspace,
                                   int64_t workspace_bytes, int cu_count, void *stream)
{
    if (!sizes_ok(n, v, k) || cu_count <= 0 || ldx < k || ld_items < k)
        return HPF_EINVAL;
    if (type < HPF_F32 || type > HPF_F16)
        return HPF_EUNSUPPORTED;
    if (n == 0)
        return 0;
    if (!x || !items || !target || !loss || !workspace || ((uintptr_t)workspace & 255))
        return HPF_EINVAL;
    Call C = {};
    C.x = x;
    C.w = items;
    C.target = target;
    C.bias = bias;
    C.loss = loss;
    C.lse = lse;
    C.n = n;
    C.v = v;
    C.k = k;
    C.ldx = ldx;
    C.ldw = ld_items;
    C.scale = scale;
    C.cus = cu_count;
    C.ws = (char *)workspace;
    C.ws_bytes = workspace_bytes;
    C.st = (hipStream_t)stream;
    return run_type(type, C);
}

extern "C" int hpf_hip_softmax_nll_grad(const void *x, int64_t ldx, const void *items, int64_t ld_items, const int64_t *target,
                                        const float *weight, const float *bias, float scale, int64_t n, int64_t v, int64_t k, int type,
                                        float *loss, void *dx, int64_t ld_dx, void *ditems, int64_t ld_ditems, float *dbias, void *workspace,
                                        int64_t workspace_bytes, int cu_count, void *stream)
{
    if (!sizes_ok(n, v, k) || cu_count <= 0 || ldx < k || ld_items < k || ld_dx < k || ld_ditems < k)
        return HPF_EINVAL;
    if (type < HPF_F32 || type > HPF_F16)
        return HPF_EUNSUPPORTED;
    if (!ditems || (bias != nullptr) != (dbias != nullptr))
        return HPF_EINVAL;
    const hipStream_t st = (hipStream_t)stream;
    if (n == 0) {              // no rows: the items' gradients are zero
        if (type == HPF_F32)
            zero_rows_kernel<<<1024, 256, 0, st>>>((float *)ditems, v, (int)k, ld_ditems);
        else
            zero_rows_kernel<<<1024, 256, 0, st>>>((_Float16 *)ditems, v, (int)k, ld_ditems);
        if (dbias)
            zero_rows_kernel<<<64, 256, 0, st>>>(dbias, v, 1, 1);
        return (int)hipGetLastError();
    }
    if (!x || !items || !target || !loss || !dx || !workspace || ((uintptr_t)workspace & 255))
        return HPF_EINVAL;
    Call C = {};
    C.x = x;
    C.w = items;
    C.target = target;
    C.weight = weight;
    C.bias = bias;
    C.loss = loss;
    C.dx = dx;
    C.dw = ditems;
    C.dbias = dbias;
    C.n = n;
    C.v = v;
    C.k = k;
    C.ldx = ldx;
    C.ldw = ld_items;
    C.lddx = ld_dx;
    C.lddw = ld_ditems;
    C.scale = scale;
    C.grad = true;
    C.cus = cu_count;
    C.ws = (char *)workspace;
    C.ws_bytes = workspace_bytes;
    C.st = st;
    return run_type(type, C);
}
