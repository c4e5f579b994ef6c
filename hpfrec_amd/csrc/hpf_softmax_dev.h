// hpf_softmax_dev.h -- softmax cross entropy of rows against a whole catalogue, with its gradients, without keeping the logits.
//
//   z[n, v] = scale <x[n], w[v]> + bias[v];   lse[n] = log sum_v exp z[n, v];   loss[n] = lse[n] - z[n, t[n]]
//   G[n, v] = weight[n] (exp(z[n, v] - lse[n]) - [v = t[n]])
//   dx = scale G w;   dw = scale G^T x;   dbias[v] = sum_n G[n, v]
//
// Every product is a matrix instruction (32 x 32 x 16); a row's statistics are kept in base 2 (z log2(e)).
//
// THREE FORMS, chosen by sizes and types alone (times: 4,096 rows with gradients, 50k items, or what is said):
//   few rows     loss alone, up to 64 rows: items read once, unpacked; rows that shared memory holds beside tiles of items (256 values, 128
//                in 32 bits) whole, wider ones in parts.  64 rows, 100k items: of 100 in bf16 24.8 us against 39.9 by the passes, in 32 bits 44.8 : 55.2, of
//                256 in bf16 49.3 : 64.1; one row, 27k items of 50 in 32 bits 21.0 : 27.8, 380k of
//                1000 395 : 1,911 by wide products; 64 rows, 100k items of 1000 in bf16 110 : 290
//   passes       rows of up to 256 values, which a wavefront's registers hold: of 60 in bf16 212 us against 762 by wide products,
//                of 256 475 : 1,013; of 50 in 32 bits 395 : 1,970, of 200 1,350 : 2,840; 100 rows, 1k items: 42 : 115
//   wide         wider ones
//
// PASSES.  A wavefront keeps 32 rows of one matrix in registers -- the STATIONARY rows -- and the other matrix streams by in tiles of
// 32 rows through shared memory, four or eight wavefronts reading each.  A tile's logits come out with the stationary row in the
// lane and the streamed row in the register, so that what belongs to a stationary row is a lane's own.
//   rows pass:   x stationary, w streamed: running maximum and sum of a softmax, and the sum of exp(z - max) w over the tiles
//                -- dx before its normalisation -- in the same pass, rescaled when a maximum grows
//   items pass:  w stationary, x streamed: G from the finished lse, and its product with x, held relative to the item's largest
// so the logits are computed twice and nothing of their size is written: 8 N V K operations with gradients, 2 N V K without.  An
// output register's row (8 (i / 4) + 4 (lane / 32) + i % 4) is not an operand's (8 (lane / 32) + j), but a contraction may take its
// terms in any order: the second product's other operand is laid out in the order in which the first product's output lies in
// the registers, and the probabilities never leave the lane that made them.
//
// 32-BIT MATRICES are split into two half-precision parts (11 + 11 bits of mantissa and the second's sign: a value is held to
// 2^-23) and multiplied in three products; the fourth, low times low, is below 2^-22 of |a| |b| and of either sign.  For
// half's range they are scaled by powers of two: 32 rows share one where rows are multiplied with rows (the largest becomes
// 2^14 .. 2^15; rows of x without gradients have one each), all rows of a column one where the sum is over rows; what is below
// 2^-17 of the largest is held to 2^-40 of it.  Probabilities are held times 2^14 relative to a running maximum of their row (or
// item).  bfloat16 and half matrices take one product; their probabilities are rounded to the same type -- up to 2^-8 or 2^-11
// of a term, of either sign, which is what the matrices' own rounding did to theirs -- and everything else stays in 32 bits.
//
// A running maximum is rounded up to a whole number: rescaling by a power of two changes no digit.
//
// THE TARGET's logit is kept out of the sums and joined at the end: 1 - p(target) is then the sum of the others' shares and not a
// difference of near equals, and the loss of a row that is sure of its target log1p(others / target).
#ifndef HPF_SOFTMAX_DEV_H
#define HPF_SOFTMAX_DEV_H
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "hpf_hip.h"

namespace hpf_softmax {

constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.693147180559945309417f;
constexpr float kNothing = -0x1p126f;     // a running maximum before anything: logits (base 2) at or below it are masked
constexpr int kNoTarget = 0x3FFFFFFF;     // in tile 2^25 - 1 of 32 items: the one behind the largest catalogue's last
constexpr int kNegative = 0x40000000;     // flags beside a row's target: its weight is negative
constexpr int kAway = -0x7FFFFFFF - 1;    //   its lse is over kAwayFrom in size: see FinishArgs::away
constexpr int kTarget = 0x3FFFFFFF;       //   the target itself
constexpr float kAwayFrom = 128.0f;
constexpr int kPadTiles = 8;              // packed matrices end on a multiple of so many tiles: staging reads whole groups

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef int i32x4 __attribute__((ext_vector_type(4)));

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

// What a user's matrix is, what it is multiplied in, in how many parts, and the power of two its probabilities are held times;
// ranged: G is held relative to a running maximum (half's range); scaled: the parts are.
struct F32 { typedef float t; typedef Hf m; static constexpr int S = 2, shift = 14; static constexpr bool ranged = true, scaled = true; };
struct B16 { typedef __bf16 t; typedef Bf m; static constexpr int S = 1, shift = 0; static constexpr bool ranged = false, scaled = false; };
struct H16 { typedef _Float16 t; typedef Hf m; static constexpr int S = 1, shift = 14; static constexpr bool ranged = true, scaled = false; };
// 32-bit rows over 256 wide: three bfloat16 parts, whose range needs neither scales nor maxima, in six products
struct W32 { typedef float t; typedef Bf m; static constexpr int S = 3, shift = 0; static constexpr bool ranged = false, scaled = false; };

template <class Y> struct Parts { typename Y::m::v8 p[Y::S]; };   // 8 values of an operand

template <class Y> __device__ __forceinline__ void split(float x, Parts<Y> &to, int j)
{
    typedef typename Y::m::e e;
    // (three bfloat16 parts: a value above bfloat16's largest would round to infinity and leave minus infinity)
    to.p[0][j] = (e)(Y::S == 3 ? __builtin_amdgcn_fmed3f(x, -0x1.FEp127f, 0x1.FEp127f) : x);
    if constexpr (Y::S > 1) {
        const float r = x - (float)to.p[0][j];
        to.p[1][j] = (e)r;
        if constexpr (Y::S > 2)
            to.p[2][j] = (e)(r - (float)to.p[1][j]);
    }
}

// two neighbouring values (j even), rounded together; what is left of each by one multiply-add that reads the half in place
template <class Y> __device__ __forceinline__ void split2(float x0, float x1, Parts<Y> &to, int j)
{
    if constexpr (Y::S == 3) {
        split<Y>(x0, to, j);
        split<Y>(x1, to, j + 1);
    } else {
        typedef float f2 __attribute__((ext_vector_type(2)));
        typedef typename Y::m::e e2 __attribute__((ext_vector_type(2)));
        const e2 hi = __builtin_convertvector((f2){x0, x1}, e2);
        to.p[0][j] = hi[0];
        to.p[0][j + 1] = hi[1];
        if constexpr (Y::S == 2) {
            const e2 lo = __builtin_convertvector(((f2){fmaf((float)hi[0], -1.0f, x0), fmaf((float)hi[1], -1.0f, x1)}), e2);
            to.p[1][j] = lo[0];
            to.p[1][j + 1] = lo[1];
        }
    }
}

// c += a b, smallest products first
template <class Y> __device__ __forceinline__ f32x16 product(const Parts<Y> &a, const Parts<Y> &b, f32x16 c)
{
    if constexpr (Y::S == 3) {
        c = Y::m::mfma(a.p[2], b.p[0], c);
        c = Y::m::mfma(a.p[0], b.p[2], c);
        c = Y::m::mfma(a.p[1], b.p[1], c);
    }
    if constexpr (Y::S > 1) {
        c = Y::m::mfma(a.p[1], b.p[0], c);
        c = Y::m::mfma(a.p[0], b.p[1], c);
    }
    return Y::m::mfma(a.p[0], b.p[0], c);
}

// the larger of two, NaN if either is
__device__ __forceinline__ float larger(float a, float b) { return a != a || a >= b ? a : b; }

// a lane's value in the lower half of the wavefront, and in the upper one: both, in every lane
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ float halves_max(float x)
{
    const u32x2 r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float other_half(float x) { return __shfl_xor(x, 32); }

// Workgroups of launches that may pass 2^32 threads are numbered over two dimensions: see blocks_of().
constexpr int kGridX = 1 << 16;
__device__ __forceinline__ int64_t block_number() { return (int64_t)blockIdx.y * kGridX + blockIdx.x; }
inline dim3 blocks_of(int64_t n) { return dim3((unsigned)(n < kGridX ? n : kGridX), (unsigned)((n + kGridX - 1) / kGridX)); }

// a word that earlier launches wrote, the same for all lanes
__device__ __forceinline__ int uniform_word(const int32_t *p) { return *(const __attribute__((address_space(4))) int32_t *)(uintptr_t)p; }

// A UNIT is one operand of a matrix instruction as it lies in memory: 64 lanes x 8 values, 1 KB.
constexpr int kUnit = 1024;

// the exponent that brings a largest magnitude into [2^14, 2^15) when it is taken away; 0 for nothing but zeros
__device__ __forceinline__ int half_exponent(float top) { return top > 0.0f ? (int)(__float_as_uint(top) >> 23) - 127 - 14 : 0; }
// of four columns (k a multiple of 4) from their largest magnitudes, which earlier launches wrote
__device__ __forceinline__ f32x4 column_exponents(const uint32_t *top, int k)
{
    const f32x4 t = *(const __attribute__((address_space(4))) f32x4 *)(uintptr_t)(top + k);
    return (f32x4){(float)half_exponent(t[0]), (float)half_exponent(t[1]), (float)half_exponent(t[2]), (float)half_exponent(t[3])};
}
__device__ __forceinline__ float finite_size(float x) { return fabsf(x) < INFINITY ? fabsf(x) : 0.0f; }

// a bias that takes its item out: what remains of it in base 2 is no number above kNothing
__device__ __forceinline__ bool masks(float bias) { return bias * kLog2e <= kNothing; }

__device__ __forceinline__ float wave_max(float m)
{
    for (int d = 32; d; d >>= 1)
        m = fmaxf(m, __shfl_xor(m, d));
    return m;
}

// ---------------------------------------------------------------------------------------------------------------------
// Preparation.
// ---------------------------------------------------------------------------------------------------------------------
struct PrepArgs {
    const int64_t *target;
    const float *bias;
    int64_t N, V, np, vp;          // np, vp: padded
    float *bias2;                  // bias in base 2, -inf beyond the catalogue and where it masks
    int32_t *meta;                 // targets as 32-bit numbers, kNoTarget where there is none or a masked one
    uint32_t *zero;                // what later launches take maxima into
    int zeros;
};

// An item and a row a thread; a launch's latency (2 us at 1,000 items, 5 at 380k).
static __global__ __launch_bounds__(256) void prepare_kernel(PrepArgs A)
{
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i < A.zeros)
        A.zero[i] = 0;
    if (i < A.vp)
        A.bias2[i] = i >= A.V || (A.bias && masks(A.bias[i])) ? -INFINITY : A.bias ? A.bias[i] * kLog2e : 0.0f;
    if (i < A.np) {
        const int64_t t = i < A.N ? A.target[i] : -1;
        A.meta[i] = t >= 0 && t < A.V && !(A.bias && masks(A.bias[t])) ? (int32_t)t : kNoTarget;
    }
}

struct Matrix {
    const void *p;
    int64_t ld, rows;
    float sign;                    // goes into by_row
    const float *bias2;            // items with a bias: theirs
    const int32_t *meta;           // x with its gradients: its targets
    const float *weight;           //   its weights (NULL: ones), and the largest magnitude among them (bits)
    uint32_t *weight_top;
    char *by_row, *by_col;
    int32_t *exps;                 // scaled: of the tiles, or with `each` of the rows
    int each;
    uint32_t *col_top;             // scaled: of the columns (as magnitudes' bits)
};

// Rows that take no part count as zeros, since whatever they hold must reach no sum and no scale: masked items, and in the gradients
// rows without a target or with a masked one.
__device__ __forceinline__ bool takes_part(const Matrix &M, int64_t row)
{
    return row < M.rows && !(M.bias2 && M.bias2[row] <= kNothing) && !(M.meta && M.meta[row] == kNoTarget);
}
__device__ __forceinline__ uint32_t tile_rows(const Matrix &M, int64_t tile)      // a bit a row
{
    return (uint32_t)__ballot(takes_part(M, tile * 32 + (threadIdx.x & 31)));
}

// by one wavefront for a tile of x
__device__ __forceinline__ void largest_weight(const Matrix &M, int64_t tile, uint32_t rows)
{
    const int low = threadIdx.x & 31;
    const float top = wave_max(rows >> low & 1 ? M.weight ? fabsf(M.weight[tile * 32 + low]) : 1.0f : 0.0f);
    if ((threadIdx.x & 63) == 0 && __float_as_uint(top) > __hip_atomic_load(M.weight_top, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT))
        atomicMax(M.weight_top, __float_as_uint(top));
}

// G is held as a share of the power of two above every |weight| (2^-100 .. 2^127, so that no share is above two; 1 where there is none or
// no finite weight)
__device__ __forceinline__ int weight_exponent(const uint32_t *top)
{
    const uint32_t bits = *top;
    const int e = (int)(bits >> 23) - 126;
    return bits == 0 || bits >= 0x7F800000u ? 0 : e > 127 ? 127 : e < -100 ? -100 : e;
}

// Largest magnitudes of the columns of both matrices; a wavefront reads whole rows, 8 at a time.  One workgroup of 16 wavefronts a
// compute unit: each ends in an atomic maximum a column (in no order that matters), and those of one column are served one after the
// other.  Bound by memory: 388k rows of 100 in 54 us, 2.9 TB/s; 31k of 50 in 7.7, which is latency.
static __global__ __launch_bounds__(1024) void columns_kernel(Matrix W, Matrix X, int K, int w_blocks)
{
    __shared__ float top[16][256];
    const bool second = (int)blockIdx.x >= w_blocks;
    const Matrix &M = second ? X : W;
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int64_t first = (second ? blockIdx.x - w_blocks : blockIdx.x) * 16 + wave, step = (second ? gridDim.x - w_blocks : w_blocks) * 16;
    float m[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int64_t r = first; r < M.rows; r += 8 * step) {
        float x[8][4];
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (64 * j < K)
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const int64_t row = r + i * step < M.rows ? r + i * step : r;
                    x[i][j] = ((const float *)M.p)[row * M.ld + (lane + 64 * j < K ? lane + 64 * j : K - 1)];
                }
        const uint64_t rows = __ballot(takes_part(M, r + (lane & 7) * step));
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (rows >> i & 1)
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (64 * j < K)
                        m[j] = fmaxf(m[j], finite_size(x[i][j]));
    }
    for (int j = 0; j < 4; ++j)
        top[wave][lane + 64 * j] = m[j];
    __syncthreads();
    const int c = threadIdx.x;
    if (c < K) {
        float all = top[0][c];
        for (int i = 1; i < 16; ++i)
            all = fmaxf(all, top[i][c]);
        if (__float_as_uint(all) > __hip_atomic_load(&M.col_top[c], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT))
            atomicMax(&M.col_top[c], __float_as_uint(all));
    }
}

// packing: rows -> units, one workgroup 32 rows.  `by_row`: tile of 32 rows after tile, in it K / 16 units (lane: row lane % 32,
// columns 16 cb + 8 (lane / 32) + j).  `by_col`: tile after tile, in it (K / 32) x 2 units (lane: column 32 ko + lane % 32, rows
// 16 t + 8 (j / 4) + 4 (lane / 32) + j % 4: the order of a product's output registers).  Columns and rows beyond the matrix
// are zero.  Bound by memory, read once for both forms: 388k rows of 100 in 32 bits, 155 MB in and 400 MB out, in 126 us, 4.4 TB/s;
// 108k of 200 in bf16 36 us.
template <class Y, int KO> __global__ __launch_bounds__(256) void pack_kernel(Matrix W, Matrix X, int K, int CB, int64_t w_tiles)
{
    constexpr int KP = 32 * KO;
    __shared__ float tile[32][KP + 1];
    __shared__ float tops[32];
    const int64_t id = block_number();
    const bool second = id >= w_tiles;
    const Matrix &M = second ? X : W;
    const int64_t rb = second ? id - w_tiles : id;
    if (rb * 32 >= M.rows)
        return;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, low = lane & 31, h = lane >> 5;
    const uint32_t rows = tile_rows(M, rb);
    if (M.weight_top && wave == 0)
        largest_weight(M, rb, rows);
    float top = 0.0f;
#pragma unroll 4
    for (int i = 0; i < 8; ++i) {
        const int r = wave * 8 + i;
        const int64_t row = rb * 32 + r < M.rows ? rb * 32 + r : rb * 32;
#pragma unroll
        for (int j = 0; j < (KP + 63) / 64; ++j) {
            const int c = lane + 64 * j;
            float x = (float)((const typename Y::t *)M.p)[row * M.ld + (c < K ? c : K - 1)];
            x = (rows >> r & 1) && c < K ? x : 0.0f;
            if (c < KP)
                tile[r][c] = x;
            top = fmaxf(top, finite_size(x));
        }
        if (Y::scaled && M.each) {
            top = wave_max(top);
            if (lane == 0)
                tops[r] = top;
            top = 0.0f;
        }
    }
    if (Y::scaled && !M.each) {
        top = wave_max(top);
        if (lane == 0)
            tops[wave] = top;
    }
    __syncthreads();
    int e = 0;
    if constexpr (Y::scaled) {
        e = half_exponent(M.each ? tops[low] : fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3])));
        if (M.each && threadIdx.x < 32)
            M.exps[rb * 32 + low] = e;
        else if (!M.each && threadIdx.x == 0)
            M.exps[rb] = e;
    }
    for (int cb = wave; cb < CB; cb += 4) {
        Parts<Y> q;
#pragma unroll
        for (int j = 0; j < 8; ++j)
            split<Y>(ldexpf(M.sign * tile[low][16 * cb + 8 * h + j], -e), q, j);
        for (int s = 0; s < Y::S; ++s)
            *(typename Y::m::v8 *)(M.by_row + (((rb * CB + cb) * Y::S + s) * 64 + lane) * 16) = q.p[s];
    }
    if (!M.by_col)
        return;
    for (int u = wave; u < 2 * KO; u += 4) {
        const int ko = u >> 1, t = u & 1, c = 32 * ko + low;
        const int ce = Y::scaled && c < K ? half_exponent(__uint_as_float(M.col_top[c])) : 0;
        Parts<Y> q;
#pragma unroll
        for (int j = 0; j < 8; ++j)
            split<Y>(ldexpf(tile[16 * t + 8 * (j >> 2) + 4 * h + (j & 3)][c], -ce), q, j);
        for (int s = 0; s < Y::S; ++s)
            *(typename Y::m::v8 *)(M.by_col + ((((rb * KO + ko) * 2 + t) * Y::S + s) * 64 + lane) * 16) = q.p[s];
    }
}

// The same for rows of any width, without scales: 32 rows x 128 columns a workgroup.
// Bound by memory, short of it where rows do not begin on 16 bytes: 50,001 rows of 1000 in half precision in 105 us, 2.9 TB/s.
template <class Y> __global__ __launch_bounds__(256) void pack_wide_kernel(Matrix M, int K, int CB, int KO)
{
    __shared__ float tile[32][129];
    const int64_t rb = blockIdx.x;
    const int c0 = blockIdx.y * 128;
    const uint32_t rows = tile_rows(M, rb);
    if (M.weight_top && blockIdx.y == 0 && threadIdx.x < 64)
        largest_weight(M, rb, rows);
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const int at = i * 256 + threadIdx.x, r = at >> 7, c = c0 + (at & 127);
        const int64_t row = rb * 32 + r < M.rows ? rb * 32 + r : rb * 32;
        const float x = (float)((const typename Y::t *)M.p)[row * M.ld + (c < K ? c : K - 1)];
        tile[r][at & 127] = (rows >> r & 1) && c < K ? x : 0.0f;
    }
    __syncthreads();
    const int lane = threadIdx.x & 63, low = lane & 31, h = lane >> 5;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int u = i * 4 + (threadIdx.x >> 6), cb = blockIdx.y * 8 + u;
        if (cb < CB) {
            Parts<Y> q;
#pragma unroll
            for (int j = 0; j < 8; ++j)
                split<Y>(M.sign * tile[low][16 * u + 8 * h + j], q, j);
            for (int s = 0; s < Y::S; ++s)
                *(typename Y::m::v8 *)(M.by_row + (((rb * CB + cb) * Y::S + s) * 64 + lane) * 16) = q.p[s];
        }
        const int ko = blockIdx.y * 4 + (u >> 1), t = u & 1;
        if (M.by_col && ko < KO) {
            Parts<Y> q;
#pragma unroll
            for (int j = 0; j < 8; ++j)
                split<Y>(tile[16 * t + 8 * (j >> 2) + 4 * h + (j & 3)][32 * (u >> 1) + low], q, j);
            for (int s = 0; s < Y::S; ++s)
                *(typename Y::m::v8 *)(M.by_col + ((((rb * KO + ko) * 2 + t) * Y::S + s) * 64 + lane) * 16) = q.p[s];
        }
    }
}

// ---------------------------------------------------------------------------------------------------------------------
// the passes
// ---------------------------------------------------------------------------------------------------------------------
enum { kNll, kRows, kItems };

struct PassArgs {
    const char *still;              // stationary matrix, by_row
    const char *by_row, *by_col;    // streamed matrix
    const int32_t *still_exp, *stream_exp;   // scaled: their tiles' (stationary rows without gradients: each row's)
    const float *reg_bias;          // per streamed row: rows passes: its bias (base 2); items pass: log2(|weight|), less weight_exponent, less lse (less `away`)
    const float *lane_bias;         // items pass: the stationary item's bias
    const int32_t *meta;            // items pass: per streamed row its target and flag; rows passes: per stationary row
    const float *target_log;        // items pass: per streamed row, log2 of |G| at its target
    const float *away;              //   and of rows whose meta has kAway: what is added ahead of reg_bias
    float *stats;                   // [split][3][still rows]: what sums are relative to (base 2), sum (rows: without the target), rows: target's logit
    float *part;                    // [split][still rows][32 KO]
    int64_t still_tiles, still_rows, stream_tiles;   // tiles of 32; still_rows = 32 still_tiles
    float c;                        // |scale| log2(e)
    int splits, bias, base, more;   // pieces of the streamed groups: `more` of base + 1, the rest of base
    // items pass in one piece: the results themselves
    void *out;
    float *dbias;
    const uint32_t *col_top;
    const uint32_t *weight_top;
    int64_t ld_out, count;
    int K, quads;                   // quads: rows of `out` allow four values at once
    float scale;
};

constexpr int kGridY = 32768;

// every wavefront's staged units are in shared memory (a barrier alone does not wait for them)
__device__ __forceinline__ void staged_barrier()
{
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
}

// KO: K / 32 rounded up; ODD: the last 16 of these columns are beyond K, and the products with rows leave them out.
// (Times: 4,096 rows x 50k items with gradients, or 8,192 x 100k without.)
//   waves  a SIMD holds as many as registers allow (512, 256 or 168 each) beside the stationary rows and the sums: without gradients,
//          of 50 in 32 bits, three 392 us, two 430; with them three 402, two 422; of 128 in bf16 three 331, two 313; of 256 in bf16
//          two 523, one 737
//   NW     where two share a SIMD a workgroup has all eight of a compute unit, which read each tile once: of 100 in 32 bits 586 us,
//          four 632; of 160 in bf16 339 : 351; where three do, it is three workgroups that overlap their barriers
//   RT     short stages cost a barrier each, long ones room: of 30 in bf16 four tiles 179 us, one 184; of 50 in 32 bits one tile 402
//          us, two 449
template <class Y, int KO, int ODD, int MODE> struct Shape {
    static constexpr int S = Y::S, CB = 2 * KO - ODD;
    static constexpr int row_units = CB * S, col_units = MODE == kNll ? 0 : 2 * KO * S, units = row_units + col_units;   // per tile
    static constexpr int waves = S == 2 && KO > 4 && MODE != kNll ? 1 : (S + (MODE == kNll ? 0 : 2)) * KO <= 9 ? 3 : 2;   // a SIMD
    static constexpr int NW = waves == 2 ? 8 : 4;                             // wavefronts of a workgroup
    static constexpr int RT = units <= 4 ? 4 : units <= 12 ? 2 : 1;           // streamed tiles a stage
    static constexpr int side = RT * 64 * 4 * (MODE == kItems ? 3 : 1);       // reg_bias (and meta, target_log) of a stage: 64 values a tile, 32 of them its own
    static constexpr int stage = RT * units * kUnit + side;
};

__device__ __forceinline__ void stage_unit(const char *from, char *to)
{
    __builtin_amdgcn_global_load_lds((__attribute__((address_space(1))) const void *)(from + (threadIdx.x & 63) * 16),
                                     (__attribute__((address_space(3))) void *)(uintptr_t)to, 16, 0, 0);
}
__device__ __forceinline__ void stage_words(const void *from, char *to)   // 64 of 32 bits
{
    __builtin_amdgcn_global_load_lds((__attribute__((address_space(1))) const void *)((const char *)from + (threadIdx.x & 63) * 4),
                                     (__attribute__((address_space(3))) void *)(uintptr_t)to, 4, 0, 0);
}

// a sum with its own rounding error carried along
struct Sum {
    float s, c;
    __device__ __forceinline__ void add(float x)
    {
        const float y = x - c, t = s + y;
        c = (t - s) - y;
        s = t;
    }
};

template <int READS, int PRODUCTS, int STEPS> __device__ __forceinline__ void order_pairs()
{
    if constexpr (STEPS > 0) {
        __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
        if constexpr (STEPS > 2)
            __builtin_amdgcn_sched_group_barrier(0x100, (STEPS > 3 ? 2 : 1) * READS, 0);
        if constexpr ((STEPS > 1 ? 2 : 1) * PRODUCTS > 1)
            __builtin_amdgcn_sched_group_barrier(0x8, (STEPS > 1 ? 2 : 1) * PRODUCTS - 1, 0);
        order_pairs<READS, PRODUCTS, STEPS - 2>();
    }
}

// Order for the scheduler, in a block of STEPS x (READS reads of shared memory, then PRODUCTS matrix instructions that use them): two
// steps' reads behind the first product of the two steps before.  (Left alone it puts each read right ahead of its product, and a
// wavefront waits for shared memory half of its time.)
template <int READS, int PRODUCTS, int STEPS> __device__ __forceinline__ void order_reads()
{
    if constexpr (STEPS > 0)
        __builtin_amdgcn_sched_group_barrier(0x100, (STEPS > 1 ? 2 : 1) * READS, 0);
    order_pairs<READS, PRODUCTS, STEPS>();
}

__device__ __forceinline__ float sum16(const f32x16 &x)
{
    return (((x[0] + x[1]) + (x[2] + x[3])) + ((x[4] + x[5]) + (x[6] + x[7]))) + (((x[8] + x[9]) + (x[10] + x[11])) + ((x[12] + x[13]) + (x[14] + x[15])));
}

// What a stationary row's exponentials are held relative to: they are 2^(z + down), and at most 2^shift.  `down` is a whole number, so that
// rescaling changes no digit.  far: the same for all lanes, some of which hold logits so large that floats lie a whole number or more
// apart and the shift would be lost in them: their largest is held as one, and every logit is rounded as the largest was (later blocks
// come with c = 1).
constexpr float kFar = 0x1p23f;
struct Held {
    float down;
    bool far;
    __device__ __forceinline__ void begin()
    {
        down = -kNothing;
        far = false;
    }
};

// One block (lane: stationary row, register: streamed row) whose logarithms in base 2 are c x becomes its exponentials relative to a
// running maximum; `rescale(f)` is called where the maximum grew.  c > 0.
template <class Y, class F> __device__ __forceinline__ void exponentials(f32x16 &x, float c, Held &held, Sum &sum, const F &rescale)
{
    float m = x[0];
#pragma unroll
    for (int i = 1; i < 16; ++i)
        m = fmaxf(m, x[i]);
    m = halves_max(m) * c;
    if (__any(m + held.down > (float)Y::shift)) {
        const float top = ceilf(m), down = m + held.down > (float)Y::shift ? fabsf(top) < kFar ? (float)Y::shift - top : -top : held.down;
        const float f = __builtin_amdgcn_exp2f(down - held.down);
        sum.s *= f;
        sum.c *= f;
        held.down = down;
        held.far = __any(fabsf(down) >= kFar && down < -kNothing);
        rescale(f);
        if (held.far) {
#pragma unroll
            for (int i = 0; i < 16; ++i)
                x[i] *= c;
            c = 1.0f;
        }
    }
    const float down = held.down < -kNothing ? held.down : -INFINITY;     // (nothing yet: all of it is masked)
#pragma unroll
    for (int i = 0; i < 16; ++i)
        x[i] = __builtin_amdgcn_exp2f(fmaf(x[i], c, down));
}

// the register of a block that holds streamed row r (0 .. 31), for the lanes of half h: i with row_of(i, h) = r
__device__ __forceinline__ constexpr int row_of(int i, int h) { return 8 * (i >> 2) + 4 * h + (i & 3); }

// takes the target's logit out of its block
__device__ __forceinline__ void take_target(f32x16 &x, float c, int tile, int h, int target, float &at)
{
    if (__any((target >> 5) == tile))
#pragma unroll
        for (int i = 0; i < 16; ++i)
            if (target == tile * 32 + row_of(i, h)) {
                at = x[i] * c;
                x[i] = -INFINITY;
            }
}

// The logarithm of a share as it comes out of the roundings of its logit and its row's lse: no share is above two (weight_exponent).
// (NaN stays.)
__device__ __forceinline__ float share_log(float x) { return __builtin_elementwise_minimum(x, 1.0f); }

__device__ __forceinline__ void store_stats(float *to, int64_t rows, int h, const Held &held, const Sum &sum, float at)
{
    const float both = sum.s + other_half(sum.s), hit = larger(at, other_half(at));
    if (h == 0) {
        to[0] = -held.down;
        to[rows] = both;
        to[2 * rows] = hit;
    }
}

// x 2^e for whole numbers held as floats (very low ones: a maximum of nothing)
__device__ __forceinline__ float times_power(float x, float e) { return ldexpf(x, (int)fmaxf(e, -1000.0f)); }

// Bound by the matrix instructions where rows are wide and by the exponentials where they are narrow: a logit costs a wavefront's lane
// about ten vector instructions and an exponential, and the two kinds of instruction were seen to take turns rather than to overlap
// (raised priorities changed nothing, logits made a tile ahead beside the exponentials cost 1 to 8 per cent).  Least and mean of six calls,
// 8,192 x 380k of 100 in 32 bits: rows 3.45 and 3.59 ms, items 3.58 and 3.75 ms, 1.04 and 1.00 PFLOP/s of half-precision products in the mean,
// while one of 8192 x 8192 x 8192 of the library runs at 1.16; loss alone, of 50: 1.28 and 1.43 ms.  8,192 x 100k of 200 in bf16: 0.72 and
// 0.76, 0.80 and 0.84 ms, 0.86 and 0.78 PFLOP/s.  Rows away from zero (kAway) cost the items 2 to 8 per cent of the call.
template <class Y, int KO, int ODD, int MODE>
__global__ __launch_bounds__((Shape<Y, KO, ODD, MODE>::NW * 64), (Shape<Y, KO, ODD, MODE>::waves)) void pass_kernel(PassArgs A)
{
    typedef Shape<Y, KO, ODD, MODE> Z;
    constexpr int S = Z::S, CB = Z::CB, RT = Z::RT, NW = Z::NW;
    __shared__ __attribute__((aligned(1024))) char lds[2][Z::stage];

    const int lane = threadIdx.x & 63, low = lane & 31, h = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int sp = blockIdx.x;      // equal splits stream the same tiles: where there are eight, they meet on one die and its cache
    const int64_t mine = ((int64_t)blockIdx.z * kGridY + blockIdx.y) * NW + wave;     // the stationary tile
    if (mine - wave >= A.still_tiles)
        return;
    const bool in = mine < A.still_tiles;
    const int g0 = A.base * sp + (sp < A.more ? sp : A.more), g1 = g0 + A.base + (sp < A.more);      // (at most 2^25 tiles)

    Parts<Y> still[CB];
#pragma unroll
    for (int cb = 0; cb < CB; ++cb)
        for (int s = 0; s < S; ++s) {
            typename Y::m::v8 z = {};
            still[cb].p[s] = in ? *(const typename Y::m::v8 *)(A.still + ((mine * CB + cb) * S + s) * kUnit + lane * 16) : z;
        }
    const int target = MODE != kItems && in ? A.meta[mine * 32 + low] : kNoTarget;
    const float lane_bias = MODE == kItems && in && A.bias ? A.lane_bias[mine * 32 + low] : 0.0f;
    const int still_exp = Y::scaled && in ? MODE == kNll ? A.still_exp[mine * 32 + low] : uniform_word(A.still_exp + mine) : 0;

    f32x16 acc[MODE == kNll ? 1 : KO];
    if constexpr (MODE != kNll)
        for (int ko = 0; ko < KO; ++ko)
            acc[ko] = (f32x16)(0.0f);
    float at = -INFINITY;
    Held held = {0.0f, false};
    if (MODE != kItems || Y::ranged)
        held.begin();
    Sum sum = {0.0f, 0.0f};

    auto stage = [&](int g, int buf) {
        const char *from = A.by_row + (int64_t)g * RT * Z::row_units * kUnit;
#pragma unroll
        for (int u = 0; u < RT * Z::row_units; u += NW)
            if (u + wave < RT * Z::row_units)
                stage_unit(from + (u + wave) * kUnit, &lds[buf][(u + wave) * kUnit]);
        if constexpr (MODE != kNll) {
            from = A.by_col + (int64_t)g * RT * Z::col_units * kUnit;
#pragma unroll
            for (int u = 0; u < RT * Z::col_units; u += NW)
                if (u + wave < RT * Z::col_units)
                    stage_unit(from + (u + wave) * kUnit, &lds[buf][(RT * Z::row_units + u + wave) * kUnit]);
        }
        if (wave < RT) {
            stage_words(A.reg_bias + ((int64_t)g * RT + wave) * 32, &lds[buf][RT * Z::units * kUnit + wave * 256]);
            if constexpr (MODE == kItems) {
                stage_words(A.meta + ((int64_t)g * RT + wave) * 32, &lds[buf][RT * Z::units * kUnit + (RT + wave) * 256]);
                stage_words(A.target_log + ((int64_t)g * RT + wave) * 32, &lds[buf][RT * Z::units * kUnit + (2 * RT + wave) * 256]);
            }
        }
    };
    auto fetch = [&](const char *unit) {
        Parts<Y> x;
        for (int s = 0; s < S; ++s)
            x.p[s] = *(const typename Y::m::v8 *)(unit + s * kUnit + lane * 16);
        return x;
    };

    if (g0 < g1)
        stage(g0, 0);
    for (int g = g0; g < g1; ++g) {
        const int buf = (g - g0) & 1;
        staged_barrier();                         // this group has arrived, and the other buffer has been read
        if (g + 1 < g1)
            stage(g + 1, buf ^ 1);
#pragma unroll 1
        for (int rt = 0; rt < RT; ++rt) {
            const int tile = (int)g * RT + rt;
            if (tile >= (int)A.stream_tiles)
                break;
            const char *rows = &lds[buf][rt * Z::row_units * kUnit], *cols = &lds[buf][(RT * Z::row_units + rt * Z::col_units) * kUnit];
            const char *side = &lds[buf][RT * Z::units * kUnit + rt * 256];
            const bool biased = MODE == kItems || A.bias || tile == (int)A.stream_tiles - 1;
            const int stream_exp = Y::scaled ? uniform_word(A.stream_exp + tile) : 0;

            f32x16 x = (f32x16)(0.0f);
#pragma unroll
            for (int cb = 0; cb < CB; ++cb)
                x = product<Y>(fetch(rows + cb * S * kUnit), still[cb], x);
            order_reads<S, 2 * S - 1, CB>();

            float c = Y::scaled ? ldexpf(A.c, stream_exp + still_exp) : A.c;
            const int meta = MODE == kItems ? ((const int32_t *)(side + RT * 256))[low] : 0;
            if (MODE == kItems && __any(meta < 0)) {       // (logits first, then down to their row's, then shares: small numbers beside small ones)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const f32x4 b = *(const f32x4 *)(side + (8 * i + 4 * h) * 4), away = *(const f32x4 *)(A.away + (int64_t)tile * 32 + 8 * i + 4 * h);
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        x[4 * i + j] = share_log((fmaf(x[4 * i + j], c, lane_bias) + away[j]) + b[j]);
                }
                c = 1.0f;
            } else if (biased || held.far || __any(c == 0.0f)) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const f32x4 b = *(const f32x4 *)(side + (8 * i + 4 * h) * 4);
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        x[4 * i + j] = fmaf(x[4 * i + j], c, b[j]);
                }
                // (the bias goes to the item's logits by themselves: a target's share and a large bias would lose each other's digits)
                if (MODE == kItems && A.bias)
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        x[i] += lane_bias;
                c = 1.0f;
            }
            const auto rescale = [&](float f) {
                if constexpr (MODE != kNll)
#pragma unroll
                    for (int ko = 0; ko < KO; ++ko)
                        acc[ko] *= f;
            };
            if constexpr (MODE == kItems) {
                unsigned flip = 0;             // registers of negative G: negative weights, and targets of positive ones
                const bool hit = __any(((meta & kTarget) >> 5) == (int)mine), negative = __any(meta & kNegative);
                if (hit || negative) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const i32x4 of = *(const i32x4 *)(side + RT * 256 + (8 * i + 4 * h) * 4);
                        const f32x4 log = *(const f32x4 *)(side + 2 * RT * 256 + (8 * i + 4 * h) * 4);
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const bool own = (of[j] & kTarget) == (int)mine * 32 + low;
                            x[4 * i + j] = own ? log[j] : x[4 * i + j];
                            flip |= (unsigned)(own != ((of[j] & kNegative) != 0)) << (4 * i + j);
                        }
                    }
                }
                if constexpr (Y::ranged) {
                    exponentials<Y>(x, c, held, sum, rescale);
                } else {
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        x[i] = __builtin_amdgcn_exp2f(x[i]);
                }
                if (hit || negative)
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        x[i] = flip >> i & 1 ? -x[i] : x[i];
                if (A.bias)
                    sum.add(sum16(x));
            } else {
                take_target(x, c, tile, h, target, at);
                exponentials<Y>(x, c, held, sum, rescale);
                sum.add(sum16(x));
            }

            if constexpr (MODE != kNll) {
                Parts<Y> p[2];
#pragma unroll
                for (int i = 0; i < 16; i += 2)
                    split2<Y>(x[i], x[i + 1], p[i >> 3], i & 7);
#pragma unroll
                for (int u = 0; u < 2 * KO; ++u)
                    acc[u >> 1] = product<Y>(fetch(cols + u * S * kUnit), p[u & 1], acc[u >> 1]);
                order_reads<S, 2 * S - 1, 2 * KO>();
            }
        }
    }

    if (!in)
        return;
    const int64_t row = mine * 32 + low;
    if (MODE == kItems && A.out) {             // the whole sum: the gradients themselves
        const float both = sum.s + other_half(sum.s), e = -held.down + (float)weight_exponent(A.weight_top);
        if (row < A.count) {
            if (A.dbias && h == 0)
                A.dbias[row] = times_power(both, e);
            typedef typename Y::t T;
            T *to = (T *)A.out + row * A.ld_out;
            if constexpr (MODE != kNll)
#pragma unroll
                for (int ko = 0; ko < KO; ++ko)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int k = 32 * ko + 8 * i + 4 * h;
                        struct alignas(4 * sizeof(T)) Quad { T v[4]; } o;
                        const f32x4 ce = Y::scaled ? column_exponents(A.col_top, k) : (f32x4)(0.0f);
#pragma unroll
                        for (int j = 0; j < 4; ++j)
                            o.v[j] = (T)times_power(acc[ko][4 * i + j] * A.scale, e + ce[j]);
                        if (A.quads && k + 4 <= A.K)
                            *(Quad *)(to + k) = o;
                        else
                            for (int j = 0; j < 4; ++j)
                                if (k + j < A.K)
                                    to[k + j] = o.v[j];
                    }
        }
        return;
    }
    store_stats(A.stats + (int64_t)sp * 3 * A.still_rows + row, A.still_rows, h, held, sum, at);
    if constexpr (MODE != kNll) {
        float *to = A.part + (sp * A.still_rows + row) * (32 * KO) + 4 * h;
#pragma unroll
        for (int ko = 0; ko < KO; ++ko)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const f32x4 o = {acc[ko][4 * i], acc[ko][4 * i + 1], acc[ko][4 * i + 2], acc[ko][4 * i + 3]};
                *(f32x4 *)(to + 32 * ko + 8 * i) = o;
            }
    }
}

// ---------------------------------------------------------------------------------------------------------------------
// Rows too wide for a wavefront's registers (k > 256): plain tiled products of packed matrices, the catalogue in chunks.  The
// statistics come from a first run over all logits; then, chunk by chunk, G is written in both operand layouts (16-bit parts,
// a chunk at a time) and multiplied with the items (dx, summed over the chunks) and with x (dw).  Rows are not cut, so a chunk is
// kChunkBytes or, from a million rows on (350k in 32 bits), the least that a workgroup takes, 256 items: 1 KB a row, 3 in 32 bits.
// Bound by the matrix instructions: 8 N V K operations.  Logits are made in 256 x 128 outputs a workgroup and 128 x 64 a wavefront,
// two workgroups a compute unit: six operands read from shared memory for eight products (four for four, 64 x 64, keep shared
// memory as busy as the matrix units).  2,048 x 50,001 of 1000 in half precision: statistics 247 us, G 252 us (0.83 and 0.81
// PFLOP/s; a third stage on its way cost 5 per cent), the products with G 192 and 290.
//   kChunkBytes  more is fewer launches and fuller last rounds, and memory: 4,096 x 50k of 600 in bf16 with 1 GB 1,572 us, with 512 MB
//                1,743, with 2 GB 1,575
// ---------------------------------------------------------------------------------------------------------------------
constexpr int64_t kChunkBytes = 1024ll << 20;

template <class Y> struct Wide {
    static constexpr int S = Y::S, KC = S == 1 ? 2 : 1, per = KC * S;   // units of the contraction a stage, of one tile
    static constexpr int stage = 12 * per * kUnit;          // 8 tiles of one matrix, 4 of the other
};
constexpr int kWideA = 8, kWideB = 4;

// For each group: the 256 x 128 product of 8 + 4 tiles over `steps` stages, handed to `done(group, acc)`.  a(group, step, tile) and
// b(group, step, tile) are a tile's KC S consecutive units.
template <class Y, class Z, class A, class B, class D>
__device__ __forceinline__ void wide_core(char *lds, int64_t groups, int steps, const A &a, const B &b, const D &done)
{
    constexpr int S = Z::S, KC = Z::KC, per = Z::per;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wa = wave >> 1, wb = wave & 1;
    int64_t ahead_g = 0;                       // the next stage to bring
    int ahead = 0, buf = 0;
    auto bring = [&](char *to) {
        if (ahead_g >= groups)
            return;
        // wavefront w brings tiles w and w + 4 of the first matrix and w of the other
        const char *pa = a(ahead_g, ahead, wave), *pc = a(ahead_g, ahead, wave + 4), *pb = b(ahead_g, ahead, wave);
#pragma unroll
        for (int u = 0; u < per; ++u) {
            stage_unit(pa + u * kUnit, to + (wave * per + u) * kUnit);
            stage_unit(pc + u * kUnit, to + ((4 + wave) * per + u) * kUnit);
            stage_unit(pb + u * kUnit, to + ((8 + wave) * per + u) * kUnit);
        }
        if (++ahead == steps) {
            ahead = 0;
            ++ahead_g;
        }
    };
    f32x16 acc[4][2];
    if (steps <= 0)
        return;
    bring(lds);
    for (int64_t g = 0; g < groups; ++g) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            for (int j = 0; j < 2; ++j)
                acc[i][j] = (f32x16)(0.0f);
        for (int step = 0; step < steps; ++step) {
            staged_barrier();                      // this stage has arrived, and the one before it has been read
            bring(lds + (buf ^ 1) * Z::stage);
            const char *at = lds + buf * Z::stage + lane * 16;
            buf ^= 1;
#pragma unroll
            for (int c = 0; c < KC; ++c) {
                Parts<Y> x[4], y[2];
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    for (int s = 0; s < S; ++s)
                        x[i].p[s] = *(const typename Y::m::v8 *)(at + ((4 * wa + i) * per + c * S + s) * kUnit);
#pragma unroll
                for (int j = 0; j < 2; ++j)
                    for (int s = 0; s < S; ++s)
                        y[j].p[s] = *(const typename Y::m::v8 *)(at + ((8 + 2 * wb + j) * per + c * S + s) * kUnit);
#pragma unroll
                for (int i = 0; i < 4; ++i)
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
    const float *bias, *reg_bias, *target_log, *away;
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
    typedef Wide<Y> Z;
    __shared__ __attribute__((aligned(1024))) char lds[2 * Z::stage];
    const int lane = threadIdx.x & 63, low = lane & 31, h = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wa = wave >> 1, wb = wave & 1;
    const int sp = blockIdx.x % A.splits;
    const int64_t n0 = (int64_t)(blockIdx.x / A.splits) * 4;
    const int64_t all = (A.v_tiles + kWideA - 1) / kWideA, g0 = all * sp / A.splits, g1 = all * (sp + 1) / A.splits;
    int target[2];
    float at[2];
    Held held[2];
    Sum sum[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const int64_t tile = n0 + 2 * wb + j;
        target[j] = tile < A.n_tiles ? A.meta[tile * 32 + low] : kNoTarget;
        held[j].begin();
        sum[j] = {0.0f, 0.0f};
        at[j] = -INFINITY;
    }
    wide_core<Y, Z>(
        lds, g1 - g0, A.CB / Z::KC,
        [&](int64_t g, int step, int tile) { return A.w + (((g0 + g) * kWideA + tile) * A.CB + step * Z::KC) * Z::S * kUnit; },
        [&](int64_t, int step, int tile) { return A.x + ((n0 + tile) * A.CB + step * Z::KC) * Z::S * kUnit; },
        [&](int64_t g, f32x16 (&acc)[4][2]) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int64_t tile = (g0 + g) * kWideA + 4 * wa + i;
                if (tile >= A.v_tiles)
                    break;
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    f32x16 &x = acc[i][j];
                    wide_bias(x, A, tile, h);
                    take_target(x, 1.0f, (int)tile, h, target[j], at[j]);
                    exponentials<Y>(x, 1.0f, held[j], sum[j], [](float) {});
                    sum[j].add(sum16(x));
                }
            }
        });
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const int64_t tile = n0 + 2 * wb + j;
        if (tile < A.n_tiles)
            store_stats(A.stats + (int64_t)(2 * sp + wa) * 3 * A.rows + tile * 32 + low, A.rows, h, held[j], sum[j], at[j]);
    }
}

// G of 4 tiles of rows against 8 tiles of items of the chunk, in both layouts, and the sums over its rows
template <class Y> __global__ __launch_bounds__(256, 2) void wide_g_kernel(WideArgs A)
{
    typedef Wide<Y> Z;
    typedef typename Y::m::e e;
    constexpr int S = Y::S;
    __shared__ __attribute__((aligned(1024))) char lds[2 * Z::stage];
    const int lane = threadIdx.x & 63, low = lane & 31, h = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wa = wave >> 1, wb = wave & 1;
    e(*const turn)[36] = (e(*)[36])(lds + wave * 2304);      // a block a wavefront, to exchange its lanes and registers: where the stages were
    const int64_t ngroups = (A.n_tiles + 3) / 4, n0 = blockIdx.x % ngroups * 4, vg = blockIdx.x / ngroups * kWideA;   // vg: within the chunk
    int meta[2];
    float down[2], tg[2], away[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const int64_t tile = n0 + 2 * wb + j;
        const bool in = tile < A.n_tiles;
        meta[j] = in ? A.meta[tile * 32 + low] : kNoTarget;
        down[j] = in ? A.reg_bias[tile * 32 + low] : -INFINITY;
        away[j] = meta[j] < 0 ? A.away[tile * 32 + low] : 0.0f;
        tg[j] = in ? A.target_log[tile * 32 + low] : 0.0f;
    }
    wide_core<Y, Z>(
        lds, 1, A.CB / Z::KC,
        [&](int64_t, int step, int tile) { return A.w + ((A.v0 + vg + tile) * A.CB + step * Z::KC) * Z::S * kUnit; },
        [&](int64_t, int step, int tile) { return A.x + ((n0 + tile) * A.CB + step * Z::KC) * Z::S * kUnit; },
        [&](int64_t, f32x16 (&acc)[4][2]) {
            __syncthreads();                   // the last stage has been read by every wavefront
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int64_t vt = vg + 4 * wa + i, tile = A.v0 + vt;
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
                    if (__any(meta[j] < 0)) {
#pragma unroll
                        for (int r = 0; r < 16; ++r)
                            x[r] = share_log((x[r] + away[j]) + down[j]);
                    } else {
#pragma unroll
                        for (int r = 0; r < 16; ++r)
                            x[r] += down[j];
                    }
                    const bool hit = __any(((meta[j] & kTarget) >> 5) == (int)tile);
                    unsigned flip = meta[j] & kNegative ? 0xFFFFu : 0u;
                    if (hit)
#pragma unroll
                        for (int r = 0; r < 16; ++r)
                            if ((meta[j] & kTarget) == (int)tile * 32 + row_of(r, h)) {
                                x[r] = tg[j];
                                flip ^= 1u << r;
                            }
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        x[r] = __builtin_amdgcn_exp2f(x[r] + (float)Y::shift);
                        x[r] = flip >> r & 1 ? -x[r] : x[r];
                    }
                    total += x;
                    Parts<Y> p[2];
#pragma unroll
                    for (int r = 0; r < 16; r += 2)
                        split2<Y>(x[r], x[r + 1], p[r >> 3], r & 7);
                    for (int s = 0; s < S; ++s) {
#pragma unroll
                        for (int t = 0; t < 2; ++t)
                            *(typename Y::m::v8 *)(A.g_rows + (((nt * A.v_count + vt) * 2 + t) * S + s) * kUnit + lane * 16) = p[t].p[s];
#pragma unroll
                        for (int r = 0; r < 16; ++r)
                            turn[low][row_of(r, h)] = p[r >> 3].p[s][r & 7];
                        // (one wavefront's own block: its accesses to shared memory are served in order)
                        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
                        for (int t = 0; t < 2; ++t) {
                            typename Y::m::v8 q;
#pragma unroll
                            for (int r = 0; r < 8; ++r)
                                q[r] = turn[16 * t + row_of(r, h)][low];
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
                            A.part_sum[((n0 / 2 + wb) * A.v_count + vt) * 32 + row_of(r, h)] = v;
                    }
                }
            }
        });
}

// c[m][k] = sum over the contraction's tiles of a (by_row units, `a_units` of them a tile) times b (by_col units)
struct ProductArgs {
    const char *a, *b;
    int64_t a_tiles, a_units, tiles;      // output tiles, units from one to the next, contraction tiles (32 each)
    int KO, splits;
    float *part;                          // [split][32 a_tiles][32 KO] sums; `more`: what is there goes in too
    int more;
    void *out;                            // or the results themselves: times scale 2^(weight_exponent - shift), `count` rows of K
    const uint32_t *weight_top;
    int64_t count, ld;
    int K;
    float scale;
};

// 256 x 256 outputs a workgroup, 128 x 128 a wavefront and one wavefront a SIMD: eight operands for sixteen products, since shared memory
// bounds smaller tiles.  Stages lie in a ring: while one is multiplied the first operands of the next are read, and the one after
// that is known to have arrived.  2,048 x 50,001 x 1000 in half precision: dx, one round of 256 workgroups
// in eight pieces, 192 us, 1.07 PFLOP/s; dw, 784 workgroups or three rounds and a bit, 290.
template <class Y> struct Ring {
    static constexpr int S = Y::S, KC = S == 1 ? 2 : 1, per = KC * S, tiles = 16;
    static constexpr int depth = S == 1 ? 4 : 3;               // 128 or 144 KB
    static constexpr int stage = tiles * per * kUnit;
    static constexpr int loads = tiles / 4 * per;              // of a wavefront, a stage
};
constexpr int kProductA = 8, kProductB = 8;                    // tiles of a workgroup

template <class Y> __global__ __launch_bounds__(256, 1) void wide_product_kernel(ProductArgs A)
{
    typedef Ring<Y> Z;
    constexpr int S = Y::S, KC = Z::KC, per = Z::per;
    __shared__ __attribute__((aligned(1024))) char lds[Z::depth * Z::stage];
    const int lane = threadIdx.x & 63, low = lane & 31, h = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wa = wave >> 1, wb = wave & 1;
    const unsigned kgroups = (A.KO + kProductB - 1) / kProductB;
    // workgroups whose ids are equal modulo 8 share a die: those of one piece of the contraction, or of one group of rows
    unsigned sp = 0, id = blockIdx.x, kg, mg;
    if (A.splits > 1) {
        sp = id % A.splits;
        id /= A.splits;
        kg = id % kgroups;
        mg = id / kgroups;
    } else {
        kg = id / 8 % kgroups;
        mg = id % 8 + id / 8 / kgroups * 8;
    }
    const int64_t m0 = (int64_t)mg * kProductA;
    const int k0 = (int)kg * kProductB;
    if (m0 >= A.a_tiles)
        return;
    const int64_t all = A.tiles * (2 / KC), s0 = all * sp / A.splits, s1 = all * (sp + 1) / A.splits;   // stages of KC units
    const int steps = (int)(s1 - s0);

    // wavefront w brings tiles w and w + 4 of each matrix
    const char *const pa = A.a + (m0 + wave) * A.a_units * S * kUnit, *const pc = A.a + (m0 + wave + 4) * A.a_units * S * kUnit;
    const int kb = k0 + wave < A.KO ? k0 + wave : A.KO - 1, kd = k0 + wave + 4 < A.KO ? k0 + wave + 4 : A.KO - 1;
    auto stage = [&](int step) {
        char *const to = lds + step % Z::depth * Z::stage;
        const int64_t u = (s0 + step) * KC, row = (u >> 1) * A.KO;
        const char *const b = A.b + ((row + kb) * 2 + (u & 1)) * S * kUnit, *const d = A.b + ((row + kd) * 2 + (u & 1)) * S * kUnit;
#pragma unroll
        for (int i = 0; i < per; ++i) {
            stage_unit(pa + (u * S + i) * kUnit, to + (wave * per + i) * kUnit);
            stage_unit(pc + (u * S + i) * kUnit, to + ((4 + wave) * per + i) * kUnit);
            stage_unit(b + i * kUnit, to + ((8 + wave) * per + i) * kUnit);
            stage_unit(d + i * kUnit, to + ((12 + wave) * per + i) * kUnit);
        }
    };
    struct Operands { Parts<Y> x[4], y[4]; };
    auto fetch = [&](int step, int c) {
        const char *const at = lds + step % Z::depth * Z::stage + lane * 16 + c * S * kUnit;
        Operands o;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            for (int s = 0; s < S; ++s) {
                o.x[i].p[s] = *(const typename Y::m::v8 *)(at + ((4 * wa + i) * per + s) * kUnit);
                o.y[i].p[s] = *(const typename Y::m::v8 *)(at + ((8 + 4 * wb + i) * per + s) * kUnit);
            }
        return o;
    };

    for (int s = 0; s < Z::depth - 1 && s < steps; ++s)
        stage(s);
    // one value of block (i, j): row row_of(r, h), column low
    auto place = [&](int i, int j, int r) { return A.part + ((sp * A.a_tiles + m0 + 4 * wa + i) * 32 + row_of(r, h)) * (int64_t)(32 * A.KO) + 32 * (k0 + 4 * wb + j) + low; };
    auto mine = [&](int i, int j) { return m0 + 4 * wa + i < A.a_tiles && k0 + 4 * wb + j < A.KO; };
    f32x16 acc[4][4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            acc[i][j] = (f32x16)(0.0f);
            if (A.more && mine(i, j))          // (all loads ahead of all stores: one by one they would wait for each other)
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    acc[i][j][r] = *place(i, j, r);
        }
    staged_barrier();
    Operands now;
    if (steps > 0)
        now = fetch(0, 0);
    for (int step = 0; step < steps; ++step) {
        // Here stages up to step + 1 have arrived for every wavefront, and all have read step - 1, whose place this one takes.
        if (step + Z::depth - 1 < steps)
            stage(step + Z::depth - 1);
#pragma unroll
        for (int c = 0; c < KC; ++c) {
            const Operands next = c + 1 < KC ? fetch(step, c + 1) : fetch(step + 1 < steps ? step + 1 : step, 0);
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    acc[i][j] = product<Y>(now.x[i], now.y[j], acc[i][j]);
            if constexpr (S == 1)
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
                    __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
                    __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
                }
            now = next;
        }
        // step + 2 has to be there before the next step reads ahead: all but the latest stage's loads, if one is on its way behind it
        if (Z::depth == 4 && step + 3 < steps)
            asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"(Z::loads) : "memory");
        else
            asm volatile("s_waitcnt vmcnt(0)\n\ts_barrier" ::: "memory");
    }

    const float f = A.out ? A.scale * __builtin_amdgcn_exp2f((float)(weight_exponent(A.weight_top) - Y::shift)) : 0.0f;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (!mine(i, j))
                continue;
            if (A.out) {
                const int k = 32 * (k0 + 4 * wb + j) + low;
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const int64_t m = (m0 + 4 * wa + i) * 32 + row_of(r, h);
                    if (m < A.count && k < A.K)
                        ((typename Y::t *)A.out)[m * A.ld + k] = (typename Y::t)(acc[i][j][r] * f);
                }
            } else {
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    *place(i, j, r) = acc[i][j][r];
            }
        }
}

// dbias of a chunk: 2^(weight_exponent - shift) times the sums of its rows' groups
static __global__ __launch_bounds__(256) void wide_sums_kernel(const float *sums, int64_t rows, int groups, const uint32_t *weight_top, int shift, int64_t count, float *dbias)
{
    const int64_t v = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (v >= count)
        return;
    float all = 0.0f;
#pragma unroll 4
    for (int s = 0; s < groups; ++s)
        all += sums[s * rows + v];
    dbias[v] = ldexpf(all, weight_exponent(weight_top) - shift);
}

// ---------------------------------------------------------------------------------------------------------------------
// Joins a row's splits: loss and lse, what the items' side needs of the row, and dx (a wavefront a row).  Bound by memory with
// gradients: 4,001 rows of 64 sums in 24 pieces, 25 MB, in 10 us; by latency without (3 us for a row, 9 for 8,192).
// ---------------------------------------------------------------------------------------------------------------------
struct FinishArgs {
    const float *stats, *part;
    const int64_t *target;
    const float *bias, *weight;
    const uint32_t *weight_top;
    const void *w;                 // items, for the target's own row
    const uint32_t *col_top;
    float *loss, *lse, *reg_bias, *target_log;
    float *away;                   // Shares come from z - lse, and what the lse adds to a large maximum would be lost in it: for such rows minus
                                   // the maximum (others: 0), and reg_bias is relative to it
    int32_t *meta;
    void *dx;
    int64_t N, V, rows, ldw, lddx;
    int K, KP, splits;
    float scale;
};

template <class Y, bool GRAD> __global__ __launch_bounds__(256) void finish_rows_kernel(FinishArgs A)
{
    const int lane = threadIdx.x & 63;
    const int64_t n = block_number() * 4 + (threadIdx.x >> 6);
    if (n >= A.rows)
        return;
    if (n >= A.N) {                // rows that only fill the last tile: no share of any sum
        if (GRAD && lane == 0) {
            A.reg_bias[n] = A.target_log[n] = -INFINITY;
            A.away[n] = 0.0f;
            A.meta[n] = kNoTarget;
        }
        return;
    }
    const int64_t t = A.target[n], item = t >= 0 && t < A.V ? t : 0;
    const float bias = A.bias ? A.bias[item] : 0.0f, given = GRAD && A.weight ? A.weight[n] : 1.0f;
    // splits over the lanes, 256 at a time: all loads first, then maxima, then sums relative to them
    float held = kNothing, at = -INFINITY, others = 0.0f;
    for (int s0 = 0; s0 < A.splits; s0 += 256) {
        float tops[4], sums[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            tops[i] = kNothing;
            sums[i] = 0.0f;
            const int s = s0 + 64 * i + lane;
            if (s < A.splits) {
                const float *const from = A.stats + 3 * s * A.rows + n;
                tops[i] = from[0];
                sums[i] = from[A.rows];
                at = larger(at, from[2 * A.rows]);
            }
        }
        const float before = held;
        held = wave_max(fmaxf(fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3])), held));
        others = times_power(others, before - held);
#pragma unroll
        for (int i = 0; i < 4; ++i)
            others += times_power(sums[i], tops[i] - held);
    }
    for (int d = 32; d; d >>= 1) {
        at = larger(at, __shfl_xor(at, d));
        others += __shfl_xor(others, d);
    }
    // `held` is below the others' largest by the shift, or (see Held) that itself; the target's own logit may be far above it
    const int shift = fabsf(held) < kFar ? Y::shift : 0;
    const float top = held + (float)shift;
    others = ldexpf(others, -shift);
    const float peak = fmaxf(top, ceilf(at));
    const float rest = times_power(others, top - peak), own = __builtin_amdgcn_exp2f(at - peak), all = rest + own;
    const float lse2 = all > 0.0f || all != all ? peak + log2f(all) : -INFINITY;
    float loss = 0.0f;
    bool alive = t >= 0;
    if (t >= A.V) {                // no such item: said in the loss, and kept out of the gradients
        loss = __builtin_nanf("");
        alive = false;
    } else if (t >= 0) {
        if ((A.bias && masks(bias)) || (!(at > kNothing) && at == at && all == all)) {   // a masked target
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
        const float weight = alive ? given : 0.0f, share = ldexpf(fabsf(weight), -weight_exponent(A.weight_top));
        if (lane == 0) {
            const bool away = alive && fabsf(lse2) > kAwayFrom;
            A.reg_bias[n] = alive ? log2f(share) - (away ? log2f(all) : lse2) : -INFINITY;
            A.away[n] = away ? -peak : 0.0f;
            A.target_log[n] = alive ? log2f(share * (rest / all)) : -INFINITY;
            A.meta[n] = alive ? (int32_t)t | (weight < 0.0f ? kNegative : 0) | (away ? kAway : 0) : kNoTarget;
        }
        if (!A.dx)
            return;
        // dx: four columns a lane, the splits over as many lanes as that leaves (KP / 4 = 8 KO lanes for a split, a power of two above)
        typedef typename Y::t T;
        T *dx = (T *)A.dx + n * A.lddx;
        const T *w = (const T *)A.w + item * A.ldw;
        const int span = A.KP <= 32 ? 8 : A.KP <= 64 ? 16 : A.KP <= 128 ? 32 : 64, k = 4 * (lane & (span - 1)), step = 64 / span;
        f32x4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
        if (alive && k < A.KP)
#pragma unroll 4
            for (int s = lane / span; s < A.splits; s += step) {
                const float down = A.stats[3 * s * A.rows + n] - held;
                const f32x4 p = *(const f32x4 *)(A.part + (s * A.rows + n) * A.KP + k);
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    sum[j] += times_power(p[j], down);
            }
        for (int d = 32; d >= span; d >>= 1)
#pragma unroll
            for (int j = 0; j < 4; ++j)
                sum[j] += __shfl_xor(sum[j], d);
        const f32x4 ce = Y::scaled && k < A.KP ? column_exponents(A.col_top, k) : (f32x4)(0.0f);
        if (lane < span)
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (k + j < A.K) {
                    const float v = times_power(sum[j], held - peak + ce[j]);
                    dx[k + j] = (T)(alive ? A.scale * weight * (v / all - rest / all * (float)w[k + j]) : 0.0f);
                }
    }
}

// ---------------------------------------------------------------------------------------------------------------------
// A few rows (up to 64) without gradients: what serving asks for.  Bound by reading the items once, so nothing is packed: a
// wavefront reads a tile of 32 items as it lies in the table, 16 bytes a lane and neighbours side by side (reading operands -- 16 bytes
// of each row -- fetched every line four times), turns it into operands through shared memory of its own, and splits it as it goes;
// the rows lie in shared memory as operands.  (Three bfloat16 parts for 32-bit matrices: they need no scale, and the matrix
// instructions have time to spare.)  61 rows, 380k items of 100 in bf16, 76 MB: 30 us, 2.5 TB/s with the launch's start and end (a
// sum of a large tensor reads 4.0 TB/s), 42 by operands; one row, 27k of 50 in 32 bits: 8 us.  Against 64 items alone they take 12 and 7.6 us:
// the last one or two tiles, their biases and the end of the rows' operands are read value by value, each waited for before the next.
// ---------------------------------------------------------------------------------------------------------------------
struct FewArgs {
    const void *x, *w;
    const int64_t *target;
    const float *bias;
    float *stats;                  // [workgroup][3][rows]
    int64_t N, V, ldx, ldw, rows, v_tiles;
    int K, groups;                 // groups: workgroups
    float c, sign;
};

// The tiles that are read 16 bytes a lane, at 32-bit offsets from the tile's start: 32 rows follow each (see `load`).  Items 2^24 values
// apart or more -- a few thousand fill the memory -- are read value by value.
__device__ __forceinline__ int64_t few_fast(const FewArgs &A) { return A.V >= 64 && A.ldw < (1 << 24) ? (A.V - 32) / 32 : 0; }

// 8 values as words
template <class T> struct Raw { uint32_t v[2 * sizeof(T)]; };
typedef uint32_t Chunk __attribute__((ext_vector_type(4)));
typedef Chunk LooseChunk __attribute__((aligned(2)));     // anywhere in a table
template <class T> __device__ __forceinline__ void zeros_from(Raw<T> &r, int left)   // `left` of the 8 are values (fewer than none: none)
{
#pragma unroll
    for (int j = 0; j < (int)(2 * sizeof(T)); ++j) {
        if (sizeof(T) == 4)
            r.v[j] = j < left ? r.v[j] : 0u;
        else
            r.v[j] &= 2 * j + 1 < left ? 0xFFFFFFFFu : 2 * j < left ? 0xFFFFu : 0u;
    }
}
template <class Y> __device__ __forceinline__ Parts<Y> parts_of(const Raw<typename Y::t> &r)
{
    Parts<Y> q;
    if constexpr (Y::S == 1) {     // as they are
        __builtin_memcpy(&q, &r, sizeof(q));
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
            split<Y>(__uint_as_float(r.v[j]), q, j);
    }
    return q;
}

// a tile's biases (base 2) as they belong to its logits' registers; `masked`: some lane's items are out, whatever their rows hold
struct FewBias {
    f32x4 b[4];
    bool masked;
};
__device__ __forceinline__ FewBias few_bias(const FewArgs &A, int64_t tile, bool whole, int h)
{
    FewBias o;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        o.b[i] = (f32x4)(0.0f);
        if (whole && A.bias) {
            __builtin_memcpy(&o.b[i], A.bias + tile * 32 + row_of(4 * i, h), 16);
            o.b[i] *= kLog2e;
        } else if (!whole) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int64_t v = tile * 32 + row_of(4 * i + j, h);
                o.b[i][j] = v >= A.V ? -INFINITY : A.bias ? A.bias[v] * kLog2e : 0.0f;
            }
        }
    }
    float least = 0.0f;
#pragma unroll
    for (int i = 0; i < 16; ++i)
        least = fminf(least, o.b[i >> 2][i & 3]);
    o.masked = __any(least <= kNothing);
    return o;
}

// 32 rows' statistics in a wavefront
struct FewRows {
    int target;
    float at;
    Held held;
    Sum sum;
    __device__ __forceinline__ void begin(const FewArgs &A, int64_t n)
    {
        const int64_t t = n < A.N ? A.target[n] : -1;
        target = t >= 0 && t < A.V ? (int)t : kNoTarget;
        held.begin();
        at = -INFINITY;
        sum = {0.0f, 0.0f};
    }
    template <class Y> __device__ __forceinline__ void add(f32x16 x, const FewArgs &A, const FewBias &o, int tile, int h)
    {
#pragma unroll
        for (int i = 0; i < 16; ++i)
            x[i] = fmaf(x[i], A.c, o.b[i >> 2][i & 3]);
        if (o.masked)
#pragma unroll
            for (int i = 0; i < 16; ++i)
                x[i] = o.b[i >> 2][i & 3] <= kNothing ? -INFINITY : x[i];
        take_target(x, 1.0f, tile, h, target, at);
        exponentials<Y>(x, 1.0f, held, sum, [](float) {});
        sum.add(sum16(x));
    }
};

// the wavefronts' pieces become the workgroup's
template <int QB, int WAVES> __device__ __forceinline__ void few_store(const FewArgs &A, const FewRows (&rows)[QB], float (&join)[WAVES][QB][3][32], int wave, int low, int h)
{
#pragma unroll
    for (int q = 0; q < QB; ++q) {
        const float both = rows[q].sum.s + other_half(rows[q].sum.s), hit = larger(rows[q].at, other_half(rows[q].at));
        if (h == 0) {
            join[wave][q][0][low] = -rows[q].held.down;
            join[wave][q][1][low] = both;
            join[wave][q][2][low] = hit;
        }
    }
    __syncthreads();
    if (threadIdx.x < 32 * QB) {
        const int q = threadIdx.x >> 5;
        float m = kNothing, all = 0.0f, hit = -INFINITY;
        for (int i = 0; i < WAVES; ++i) {
            m = fmaxf(m, join[i][q][0][low]);
            hit = larger(hit, join[i][q][2][low]);
        }
        for (int i = 0; i < WAVES; ++i)
            all += times_power(join[i][q][1][low], join[i][q][0][low] - m);
        float *to = A.stats + (int64_t)blockIdx.x * 3 * A.rows + threadIdx.x;
        to[0] = m;
        to[A.rows] = all;
        to[2 * A.rows] = hit;
    }
}

// QB: tiles of 32 rows; CB: operands of a row, K / 16 or more (of six, since each is a kernel: 64 rows, 100k items of 200 in bf16 with 13
// 42 us, with 16 48).  Eight wavefronts a workgroup where shared memory holds as many tiles beside the rows, else four; one workgroup a
// compute unit.
template <class Y, int QB, int CB> struct FewShape {
    static constexpr int chunks = CB * (int)sizeof(typename Y::t);        // of 16 bytes, a row
    static constexpr int rows_bytes = QB * CB * Y::S * kUnit, own = chunks * 512;   // the rows' operands; a wavefront's tile
    static constexpr int waves = rows_bytes + 8 * own <= 152 << 10 ? 8 : 4, bytes = rows_bytes + waves * own;
};

template <class Y, int QB, int CB> __global__ __launch_bounds__((FewShape<Y, QB, CB>::waves * 64), (FewShape<Y, QB, CB>::waves / 4)) void few_kernel(FewArgs A)
{
    typedef FewShape<Y, QB, CB> Z;
    constexpr int S = Y::S, NC = Z::chunks;
    typedef typename Y::t T;
    extern __shared__ __attribute__((aligned(1024))) char lds[];
    __shared__ float join[Z::waves][QB][3][32];
    const int lane = threadIdx.x & 63, low = lane & 31, h = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t step = (int64_t)gridDim.x * Z::waves, fast = few_fast(A);
    char *const own = lds + Z::rows_bytes + wave * Z::own;

    // chunk p = 64 i + lane of a tile: row p / NC, bytes 16 (p % NC) on.  A row's last chunks reach beyond its end: where 32 rows or more
    // follow (K > 8 CB or CB is 2: no further than that), what is there is read and zeroed later; the last one or two tiles are read
    // value by value.
    Chunk next[NC / 2];
    uint32_t from[NC / 2];                 // bytes from the tile's start
#pragma unroll
    for (int i = 0; i < NC / 2; ++i)
        from[i] = (uint32_t)((64 * i + lane) / NC) * (uint32_t)(A.ldw * sizeof(T)) + (64 * i + lane) % NC * 16;
    auto load = [&](int64_t tile) __attribute__((always_inline)) {
        const char *const start = (const char *)A.w + tile * 32 * A.ldw * (int64_t)sizeof(T);
        if (tile < fast) {
#pragma unroll
            for (int i = 0; i < NC / 2; ++i)
                next[i] = *(const LooseChunk *)(start + from[i]);
        } else {
#pragma unroll 1
            for (int i = 0; i < NC / 2; ++i) {      // through shared memory: a register cannot be chosen by i
                const int r = (64 * i + lane) / NC, k = (64 * i + lane) % NC * (16 / (int)sizeof(T));
#pragma unroll
                for (int j = 0; j < (int)(16 / sizeof(T)); ++j)
                    ((T *)(own + (64 * i + lane) * 16))[j] = tile * 32 + r < A.V && k + j < A.K ? ((const T *)A.w)[(tile * 32 + r) * A.ldw + k + j] : (T)0.0f;
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
            for (int i = 0; i < NC / 2; ++i)
                next[i] = *(const Chunk *)(own + (64 * i + lane) * 16);
        }
    };
    // where chunk c of row r lies: rows side by side, each chunk's a place further on (no two of eight neighbours on one bank, written or read)
    auto place = [&](int c, int r) { return own + c * 512 + ((r + c) & 31) * 16; };

    int64_t tile = (int64_t)blockIdx.x * Z::waves + wave;
    if (tile < A.v_tiles)
        load(tile);
    for (int u = wave; u < QB * CB; u += Z::waves) {
        const int q = u / CB, cb = u % CB;
        const int64_t n = q * 32 + low;
        Parts<Y> p;
        const T *const row = (const T *)A.x + (n < A.N ? n : 0) * A.ldx + 16 * cb + 8 * h;
        if (16 * cb + 16 <= A.K) {
            struct Eight { T v[8]; } r;
            __builtin_memcpy(&r, row, sizeof(r));
#pragma unroll
            for (int j = 0; j < 8; ++j)
                split<Y>(n < A.N ? A.sign * (float)r.v[j] : 0.0f, p, j);
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                split<Y>(n < A.N && 16 * cb + 8 * h + j < A.K ? A.sign * (float)row[j] : 0.0f, p, j);
        }
        for (int s = 0; s < S; ++s)
            *(typename Y::m::v8 *)(lds + (u * S + s) * kUnit + lane * 16) = p.p[s];
    }
    FewRows rows[QB];
#pragma unroll
    for (int q = 0; q < QB; ++q)
        rows[q].begin(A, q * 32 + low);
    __syncthreads();
    for (; tile < A.v_tiles; tile += step) {
        // (one wavefront's own memory: its accesses are served in order)
#pragma unroll
        for (int i = 0; i < NC / 2; ++i)
            *(Chunk *)place((64 * i + lane) % NC, (64 * i + lane) / NC) = next[i];
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        if (tile + step < fast)
            load(tile + step);
        const FewBias bias = few_bias(A, tile, tile < fast, h);
        f32x16 z[QB];
#pragma unroll
        for (int q = 0; q < QB; ++q)
            z[q] = (f32x16)(0.0f);
#pragma unroll
        for (int cb = 0; cb < CB; ++cb) {
            Raw<T> raw;
#pragma unroll
            for (int i = 0; i < (int)sizeof(T) / 2; ++i) {
                const Chunk c = *(const Chunk *)place((2 * cb + h) * (int)sizeof(T) / 2 + i, low);
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    raw.v[4 * i + j] = c[j];
            }
            if (16 * cb + 16 > A.K)
                zeros_from(raw, A.K - 16 * cb - 8 * h);
            const Parts<Y> a = parts_of<Y>(raw);
#pragma unroll
            for (int q = 0; q < QB; ++q) {
                Parts<Y> y;
                for (int s = 0; s < S; ++s)
                    y.p[s] = *(const typename Y::m::v8 *)(lds + ((q * CB + cb) * S + s) * kUnit + lane * 16);
                z[q] = product<Y>(a, y, z[q]);
            }
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        if (tile + step >= fast && tile + step < A.v_tiles)      // (the slow way goes through `own`: the operands have been read)
            load(tile + step);
#pragma unroll
        for (int q = 0; q < QB; ++q)
            rows[q].template add<Y>(z[q], A, bias, (int)tile, h);
    }
    few_store<QB, Z::waves>(A, rows, join, wave, low, h);
}

// The same for wider rows, 64 columns at a time; the rows, packed by a launch of their own, come from the caches.  One row, 380k items of
// 1000 in 32 bits, 1.5 GB: 395 us, 3.84 TB/s; 50k, fewer tiles than wavefronts: 100 us; 64: 66 us,
// which is the last tiles' value by value.
template <class Y, int QB> __global__ __launch_bounds__(512, 2) void few_wide_kernel(FewArgs A)
{
    typedef typename Y::t T;
    constexpr int S = Y::S, CB = 4, NC = CB * (int)sizeof(T), waves = 8, columns = 16 * CB;
    __shared__ __attribute__((aligned(1024))) char lds[waves][NC * 512];
    __shared__ float join[waves][QB][3][32];
    const int lane = threadIdx.x & 63, low = lane & 31, h = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t step = (int64_t)gridDim.x * waves, fast = few_fast(A);
    const int parts = (A.K + columns - 1) / columns;
    char *const own = lds[wave];

    Chunk next[NC / 2];
    uint32_t from[NC / 2];
#pragma unroll
    for (int i = 0; i < NC / 2; ++i)
        from[i] = (uint32_t)((64 * i + lane) / NC) * (uint32_t)(A.ldw * sizeof(T)) + (64 * i + lane) % NC * 16;
    // columns 64 c on of a tile (a row's last ones reach beyond its end by less than a row: 32 rows follow)
    auto load = [&](int64_t tile, int c) __attribute__((always_inline)) {
        const char *const start = (const char *)A.w + (tile * 32 * A.ldw + c * columns) * (int64_t)sizeof(T);
        if (tile < fast) {
#pragma unroll
            for (int i = 0; i < NC / 2; ++i)
                next[i] = *(const LooseChunk *)(start + from[i]);
        } else {
#pragma unroll 1
            for (int i = 0; i < NC / 2; ++i) {
                const int r = (64 * i + lane) / NC, k = c * columns + (64 * i + lane) % NC * (16 / (int)sizeof(T));
#pragma unroll
                for (int j = 0; j < (int)(16 / sizeof(T)); ++j)
                    ((T *)(own + (64 * i + lane) * 16))[j] = tile * 32 + r < A.V && k + j < A.K ? ((const T *)A.w)[(tile * 32 + r) * A.ldw + k + j] : (T)0.0f;
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
            for (int i = 0; i < NC / 2; ++i)
                next[i] = *(const Chunk *)(own + (64 * i + lane) * 16);
        }
    };
    auto place = [&](int c, int r) { return own + c * 512 + ((r + c) & 31) * 16; };

    int64_t tile = (int64_t)blockIdx.x * waves + wave;
    if (tile < A.v_tiles)
        load(tile, 0);
    FewRows rows[QB];
#pragma unroll
    for (int q = 0; q < QB; ++q)
        rows[q].begin(A, q * 32 + low);
    for (; tile < A.v_tiles; tile += step) {
        const FewBias bias = few_bias(A, tile, tile < fast, h);
        f32x16 z[QB];
#pragma unroll
        for (int q = 0; q < QB; ++q)
            z[q] = (f32x16)(0.0f);
#pragma unroll 1
        for (int c = 0; c < parts; ++c) {
            Parts<Y> y[QB][CB];
#pragma unroll
            for (int q = 0; q < QB; ++q)
#pragma unroll
                for (int cb = 0; cb < CB; ++cb)
                    for (int s = 0; s < S; ++s)
                        y[q][cb].p[s] = *(const typename Y::m::v8 *)((const char *)A.x + (((int64_t)(q * parts + c) * CB + cb) * S + s) * kUnit + lane * 16);
            // (one wavefront's own memory: its accesses are served in order)
#pragma unroll
            for (int i = 0; i < NC / 2; ++i)
                *(Chunk *)place((64 * i + lane) % NC, (64 * i + lane) / NC) = next[i];
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            const int64_t tile2 = c + 1 < parts ? tile : tile + step;
            const int c2 = c + 1 < parts ? c + 1 : 0;
            if (tile2 < fast)
                load(tile2, c2);
#pragma unroll
            for (int cb = 0; cb < CB; ++cb) {
                Raw<T> raw;
#pragma unroll
                for (int i = 0; i < (int)sizeof(T) / 2; ++i) {
                    const Chunk v = *(const Chunk *)place((2 * cb + h) * (int)sizeof(T) / 2 + i, low);
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        raw.v[4 * i + j] = v[j];
                }
                if (c * columns + 16 * cb + 16 > A.K)
                    zeros_from(raw, A.K - c * columns - 16 * cb - 8 * h);
                const Parts<Y> a = parts_of<Y>(raw);
#pragma unroll
                for (int q = 0; q < QB; ++q)
                    z[q] = product<Y>(a, y[q][cb], z[q]);
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            if (tile2 >= fast && tile2 < A.v_tiles)
                load(tile2, c2);
        }
#pragma unroll
        for (int q = 0; q < QB; ++q)
            rows[q].template add<Y>(z[q], A, bias, (int)tile, h);
    }
    few_store<QB, waves>(A, rows, join, wave, low, h);
}

// Joins the splits of a product with G, bound by memory (27k x 64 in three pieces, 21 MB and 7 out, in 10 us): out = scale 2^weight_exponent sum, dbias = 2^weight_exponent sum (four columns a thread)
struct JoinArgs {
    const float *part, *tops;              // tops (the passes' pieces): [split][3][rows] with the sums behind, else NULL
    const uint32_t *weight_top, *col_top;
    int64_t count, rows, ld;
    int K, KP, splits;
    float scale;
    void *out;
    float *dbias;
};

template <class Y> __global__ __launch_bounds__(256) void join_kernel(JoinArgs A)
{
    const int quads = A.KP / 4;
    const int64_t id = block_number() * 256 + threadIdx.x, v = id / quads;
    const int k = (int)(id - v * quads) * 4;
    if (v >= A.count)
        return;
    float top = A.tops ? kNothing : -(float)Y::shift;
    if (A.tops)
        for (int s = 0; s < A.splits; ++s)
            top = fmaxf(top, A.tops[3 * s * A.rows + v]);
    const float e = top + (float)weight_exponent(A.weight_top);
    f32x4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
    for (int s = 0; s < A.splits; ++s) {
        const f32x4 p = *(const f32x4 *)(A.part + (s * A.rows + v) * A.KP + k);
        const float down = A.tops ? A.tops[3 * s * A.rows + v] - top : 0.0f;
#pragma unroll
        for (int j = 0; j < 4; ++j)
            sum[j] += times_power(p[j], down);
    }
    const f32x4 ce = Y::scaled ? column_exponents(A.col_top, k) : (f32x4)(0.0f);
#pragma unroll
    for (int j = 0; j < 4; ++j)
        if (k + j < A.K)
            ((typename Y::t *)A.out)[v * A.ld + k + j] = (typename Y::t)times_power(sum[j] * A.scale, e + ce[j]);
    if (A.dbias && k == 0) {
        float all = 0.0f;
        for (int s = 0; s < A.splits; ++s)
            all += times_power(A.tops[(3 * s + 1) * A.rows + v], A.tops[3 * s * A.rows + v] - top);
        A.dbias[v] = times_power(all, e);
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
inline int64_t up(int64_t a, int64_t b) { return (a + b - 1) / b * b; }
constexpr int kMostSplits = 256;      // a row's pieces are joined by one wavefront
inline int64_t tiles_padded(int64_t tiles) { return up(tiles, kPadTiles); }

// How many pieces a contraction of so many units is cut into, for a launch of `workgroups` tiles of which `room` are resident together:
// by an estimate of its time in microseconds -- rounds of workgroups, each with its start, its units and what it writes of its
// piece, and the pieces' join.  More than eight come in eights (one a die).  (As many as fill one round instead: 2,048 x 20k of 300 in
// 32 bits 831 us against 806, 50k x 2k of 600 3,475 : 3,386.)
inline int wide_splits(int64_t workgroups, int64_t units, int64_t room, double unit_us, double start_us, double piece_us)
{
    double best = 0.0;
    int at = 0;
    for (int s = 1; s <= kMostSplits / 2 && (s == 1 || s <= units); s += s < 8 ? 1 : 8) {
        const int64_t rounds = (workgroups * s + room - 1) / room;
        const double us = rounds * (start_us + (double)((units + s - 1) / s) * unit_us) + (s > 1 ? (double)workgroups * s / room * piece_us : 0.0);
        if (!at || us < best) {
            best = us;
            at = s;
        }
    }
    return at;
}

// For the passes, by an estimate of their time in microseconds (8,192 rows, 100k items of 50, loss alone: 392 us, in one piece 2,141; 100
// rows, 1k items with gradients 46, in one piece 86): rounds of the workgroups that are resident together, each with
// its start and its stages, whose cost grows with the wavefronts that share a SIMD; and what it takes to join the pieces.  More than
// eight come in eights, so that the pieces of equal number share a die's cache.
template <class Y, int KO, int ODD, int MODE> int pass_splits(int64_t still_tiles, int64_t stream_tiles, int cus)
{
    typedef Shape<Y, KO, ODD, MODE> Z;
    const int64_t groups = (still_tiles + Z::NW - 1) / Z::NW, stages = (stream_tiles + Z::RT - 1) / Z::RT;
    const double products = (Z::CB + (MODE == kNll ? 0 : 2 * KO)) * (2 * Y::S - 1);
    const double stage_us = Z::RT * (16 * products + 700) / 2000;              // one wavefront's, with others beside it
    const double join_us = MODE == kNll ? 0.0 : 32.0 * still_tiles * 32 * KO * 8 / 4e6;   // a piece written and read again, at 4 TB/s
    const int64_t room = (int64_t)cus * Z::waves * 4 / Z::NW;
    double best = 0.0;
    int at = 0;
    for (int s = 1; s <= kMostSplits && s <= stages; s += s < 8 ? 1 : 8) {
        const int64_t all = groups * s, rounds = all / room, rest = all % room;
        const double shared = rest ? (double)((rest * Z::NW + 4 * cus - 1) / (4 * cus)) : 0.0, each = (double)((stages + s - 1) / s);
        const double us = rounds * (5 + each * (Z::waves + 1) * stage_us) + (rest ? 5 + each * (shared + 1) * stage_us : 0.0) + (s > 1 ? 3 + s * join_us : 0.0);
        if (!at || us < best) {
            best = us;
            at = s;
        }
    }
    return at;
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
    char *ws;                 // NULL: only the size is asked for
    int64_t ws_bytes;
    hipStream_t st;
};

// pieces of the workspace, one after the other
struct Space {
    char *base;
    int64_t used;
    template <class T> T *take(int64_t bytes)
    {
        T *const p = (T *)(base + used);
        used += up(bytes, 1024);
        return p;
    }
};

constexpr int64_t kOneTileMore = 64 * 4;    // staging reads 64 words for a tile's 32

template <class Y, int KO, int ODD, int MODE> int64_t workgroups(int64_t tiles)
{
    typedef Shape<Y, KO, ODD, MODE> Z;
    return (tiles + Z::NW - 1) / Z::NW;
}

template <class Y, int KO, int ODD, int MODE> void launch_pass(PassArgs &A, int64_t groups, hipStream_t st)
{
    typedef Shape<Y, KO, ODD, MODE> Z;
    const int64_t stages = (A.stream_tiles + Z::RT - 1) / Z::RT;
    A.base = (int)(stages / A.splits);
    A.more = (int)(stages % A.splits);
    pass_kernel<Y, KO, ODD, MODE><<<dim3((unsigned)A.splits, (unsigned)(groups < kGridY ? groups : kGridY), (unsigned)((groups + kGridY - 1) / kGridY)), Z::NW * 64, 0, st>>>(A);
}

inline void fill_prepare(PrepArgs &P, const Call &C, int64_t np, int64_t vp)
{
    P.target = C.target;
    P.bias = C.bias;
    P.N = C.n;
    P.V = C.v;
    P.np = np;
    P.vp = vp;
}
inline dim3 join_blocks(int64_t rows, int KP) { return blocks_of((rows * (KP / 4) + 255) / 256); }
inline unsigned prepare_blocks(const PrepArgs &P)
{
    const int64_t most = P.np > P.vp ? P.np : P.vp;
    return (unsigned)(((most > P.zeros ? most : P.zeros) + 255) / 256);
}

inline void fill_matrices(Matrix &w, Matrix &x, const Call &C)
{
    w.p = C.w;
    w.ld = C.ldw;
    w.rows = C.v;
    w.sign = 1.0f;
    x.p = C.x;
    x.ld = C.ldx;
    x.rows = C.n;
    x.sign = C.scale < 0.0f ? -1.0f : 1.0f;       // the sign of the scale, so that logits rise with the product
    x.weight = C.weight;
    x.each = !C.grad;
}

inline void fill_finish(FinishArgs &F, const Call &C)
{
    F.target = C.target;
    F.bias = C.bias;
    F.weight = C.weight;
    F.w = C.w;
    F.loss = C.loss;
    F.lse = C.lse;
    F.N = C.n;
    F.V = C.v;
    F.ldw = C.ldw;
    F.lddx = C.lddx;
    F.K = (int)C.k;
    F.scale = C.scale;
}

// Rows of up to 256 values: returns the workspace's bytes, or a negative code / launch error where there is one to launch in.
template <class Y, int KO, int ODD> int64_t run_narrow(const Call &C)
{
    typedef typename Y::t T;
    constexpr int KP = 32 * KO, CB = 2 * KO - ODD;
    const int64_t n_tiles = (C.n + 31) / 32, v_tiles = (C.v + 31) / 32, nt = tiles_padded(n_tiles), vt = tiles_padded(v_tiles), row_unit = (int64_t)CB * Y::S * kUnit, col_unit = (int64_t)2 * KO * Y::S * kUnit;
    const int64_t nr = n_tiles * 32, vr = v_tiles * 32;
    const int64_t row_groups = C.grad ? workgroups<Y, KO, ODD, kRows>(n_tiles) : workgroups<Y, KO, ODD, kNll>(n_tiles), item_groups = workgroups<Y, KO, ODD, kItems>(v_tiles);
    const int row_splits = C.grad ? pass_splits<Y, KO, ODD, kRows>(n_tiles, v_tiles, C.cus) : pass_splits<Y, KO, ODD, kNll>(n_tiles, v_tiles, C.cus);
    const int item_splits = pass_splits<Y, KO, ODD, kItems>(v_tiles, n_tiles, C.cus);
    Space W = {C.ws, 0};
    Matrix mw = {}, mx = {};
    fill_matrices(mw, mx, C);
    PrepArgs P = {};
    fill_prepare(P, C, nt * 32, vt * 32);
    mw.by_row = W.take<char>(vt * row_unit);
    mx.by_row = W.take<char>(nt * row_unit);
    P.bias2 = W.take<float>(vt * 32 * 4 + kOneTileMore);
    P.meta = W.take<int32_t>(nt * 32 * 4 + kOneTileMore);
    mw.bias2 = C.bias ? P.bias2 : nullptr;
    mx.meta = C.grad ? P.meta : nullptr;
    if (Y::scaled) {
        mw.exps = W.take<int32_t>(vt * 4);
        mx.exps = W.take<int32_t>(nt * (C.grad ? 4 : 32 * 4));
    }
    float *const stats = W.take<float>((int64_t)row_splits * 3 * nr * 4), *reg_bias = nullptr, *target_log = nullptr, *away = nullptr, *item_stats = nullptr, *part = nullptr;
    if (C.grad) {
        mw.by_col = W.take<char>(vt * col_unit);
        mx.by_col = W.take<char>(nt * col_unit);
        P.zeros = Y::scaled ? 1 + 2 * KP : 1;
        P.zero = W.take<uint32_t>(P.zeros * 4);
        mx.weight_top = P.zero + P.zeros - 1;
        if (Y::scaled) {
            mw.col_top = P.zero;
            mx.col_top = P.zero + KP;
        }
        reg_bias = W.take<float>(nt * 32 * 4 + kOneTileMore);
        target_log = W.take<float>(nt * 32 * 4 + kOneTileMore);
        away = W.take<float>(nr * 4);
        const int64_t rows_part = row_splits * nr * KP * 4, items_part = item_splits > 1 ? item_splits * vr * KP * 4 : 0;
        part = W.take<float>(rows_part > items_part ? rows_part : items_part);   // (the rows' is read before the items' is written)
        if (item_splits > 1)
            item_stats = W.take<float>((int64_t)item_splits * 3 * vr * 4);
    }
    if (!C.ws)
        return W.used;
    if (C.ws_bytes < W.used)
        return HPF_EINVAL;

    prepare_kernel<<<prepare_blocks(P), 256, 0, C.st>>>(P);
    if (Y::scaled && C.grad) {
        const int most = C.cus, wb = (int)(C.v / 128 < 1 ? 1 : C.v / 128 > most ? most : C.v / 128), xb = (int)(C.n / 128 < 1 ? 1 : C.n / 128 > most ? most : C.n / 128);
        columns_kernel<<<wb + xb, 1024, 0, C.st>>>(mw, mx, (int)C.k, wb);
    }
    pack_kernel<Y, KO><<<blocks_of(v_tiles + n_tiles), 256, 0, C.st>>>(mw, mx, (int)C.k, CB, v_tiles);

    PassArgs A = {};
    A.still = mx.by_row;
    A.by_row = mw.by_row;
    A.by_col = mw.by_col;
    A.still_exp = mx.exps;
    A.stream_exp = mw.exps;
    A.reg_bias = P.bias2;
    A.meta = P.meta;
    A.stats = stats;
    A.part = part;
    A.still_tiles = n_tiles;
    A.still_rows = nr;
    A.stream_tiles = v_tiles;
    A.c = fabsf(C.scale) * kLog2e;
    A.splits = row_splits;
    A.bias = C.bias != nullptr;
    FinishArgs F = {};
    fill_finish(F, C);
    F.stats = stats;
    F.part = part;
    F.weight_top = mx.weight_top;
    F.col_top = mw.col_top;
    F.reg_bias = reg_bias;
    F.target_log = target_log;
    F.away = away;
    F.meta = P.meta;
    F.dx = C.dx;
    F.rows = nr;
    F.KP = KP;
    F.splits = row_splits;
    if (!C.grad) {
        launch_pass<Y, KO, ODD, kNll>(A, row_groups, C.st);
        finish_rows_kernel<Y, false><<<blocks_of((nr + 3) / 4), 256, 0, C.st>>>(F);
        return (int)hipGetLastError();
    }
    launch_pass<Y, KO, ODD, kRows>(A, row_groups, C.st);
    finish_rows_kernel<Y, true><<<blocks_of((nr + 3) / 4), 256, 0, C.st>>>(F);

    A.still = mw.by_row;
    A.by_row = mx.by_row;
    A.by_col = mx.by_col;
    A.still_exp = mw.exps;
    A.stream_exp = mx.exps;
    A.reg_bias = reg_bias;
    A.lane_bias = P.bias2;
    A.target_log = target_log;
    A.away = away;
    A.stats = item_stats;
    A.still_tiles = v_tiles;
    A.still_rows = vr;
    A.stream_tiles = n_tiles;
    A.splits = item_splits;
    if (item_splits == 1) {
        A.out = C.dw;
        A.dbias = C.bias ? C.dbias : nullptr;
        A.col_top = mx.col_top;
        A.weight_top = mx.weight_top;
        A.ld_out = C.lddw;
        A.count = C.v;
        A.K = (int)C.k;
        A.quads = C.lddw % 4 == 0 && (uintptr_t)C.dw % (4 * sizeof(T)) == 0;
        A.scale = C.scale;
    }
    launch_pass<Y, KO, ODD, kItems>(A, item_groups, C.st);
    if (item_splits > 1) {
        const JoinArgs J = {part, item_stats, mx.weight_top, mx.col_top, C.v, vr, C.lddw, (int)C.k, KP, item_splits, C.scale, C.dw, C.bias ? C.dbias : nullptr};
        join_kernel<Y><<<join_blocks(C.v, KP), 256, 0, C.st>>>(J);
    }
    return (int)hipGetLastError();
}

// wider rows
template <class Y> int64_t run_wide(const Call &C)
{
    typedef typename Y::t T;
    const int KO = (int)((C.k + 31) / 32 + 1) / 2 * 2, KP = 32 * KO, CB = 2 * KO, kg = (KO + kProductB - 1) / kProductB;
    const int64_t n_tiles = (C.n + 31) / 32, v_tiles = (C.v + 31) / 32, nt = tiles_padded(n_tiles), vt = tiles_padded(v_tiles), unit = (int64_t)2 * KO * Y::S * kUnit, row_unit = (int64_t)CB * Y::S * kUnit;
    const int64_t nr = n_tiles * 32, nb = (n_tiles + kWideB - 1) / kWideB, na = nt / kProductA, room = C.cus;   // the products' workgroups that are resident
    const int products = Y::S == 1 ? 1 : 6;
    // a group's product of 256 x 128 x K on half a compute unit, at two thirds of its rate, and its exponentials
    const int row_splits = wide_splits(nb, vt / kWideA, 2 * room, 0.024 * (double)KP * products + 4.0, 5.0, 0.0);
    // tiles of items at a time: equal chunks of what kChunkBytes hold
    int64_t most = kChunkBytes / (nt * 32 * 32 * 2 * Y::S * 2) / kWideA * kWideA;
    most = most < kWideA ? kWideA : most;
    const int64_t chunks = (v_tiles + most - 1) / most, chunk = up((v_tiles + chunks - 1) / chunks, kWideA);
    // four tiles of a 256 x 256 product; 256 KB of sums written by every compute unit at once, and read again
    const double unit_us = 3.2 * products, piece_us = 32.0;
    const int dx_splits = wide_splits(na * kg, chunk / 4, room, unit_us, 5.0, piece_us);
    const auto dw_splits_of = [&](int64_t tiles) { return wide_splits((tiles + kProductA - 1) / kProductA * kg, n_tiles / 4, room, unit_us, 5.0, piece_us); };
    const int64_t last = v_tiles % chunk ? v_tiles % chunk : chunk;
    const int64_t dw_rows = 32 * (dw_splits_of(chunk) * chunk > dw_splits_of(last) * last ? dw_splits_of(chunk) * chunk : dw_splits_of(last) * last);
    Space S = {C.ws, 0};
    Matrix mw = {}, mx = {};
    fill_matrices(mw, mx, C);
    PrepArgs P = {};
    fill_prepare(P, C, nt * 32, vt * 32);
    mw.by_row = S.take<char>(vt * row_unit);
    mx.by_row = S.take<char>(nt * row_unit);
    P.bias2 = S.take<float>(vt * 32 * 4);
    P.meta = S.take<int32_t>(nt * 32 * 4);
    mw.bias2 = C.bias ? P.bias2 : nullptr;
    mx.meta = C.grad ? P.meta : nullptr;
    WideArgs A = {};
    FinishArgs F = {};
    fill_finish(F, C);
    float *dw_part = nullptr, *dx_part = nullptr;
    A.stats = S.take<float>((int64_t)2 * row_splits * 3 * nr * 4);
    if (C.grad) {
        mw.by_col = S.take<char>(vt * unit);
        mx.by_col = S.take<char>(nt * unit);
        F.reg_bias = S.take<float>(nt * 32 * 4);
        F.target_log = S.take<float>(nt * 32 * 4);
        F.away = S.take<float>(nr * 4);
        P.zeros = 1;
        P.zero = mx.weight_top = S.take<uint32_t>(4);
        dw_part = S.take<float>(dw_splits_of(chunk) > 1 || dw_splits_of(last) > 1 ? dw_rows * KP * 4 : 4);
        dx_part = S.take<float>(dx_splits * nr * KP * 4);
        A.part_sum = S.take<float>(2 * nb * chunk * 32 * 4);
        A.g_rows = S.take<char>(nt * chunk * 2 * Y::S * kUnit);
        A.g_items = S.take<char>(chunk * nt * 2 * Y::S * kUnit);
    }
    if (!C.ws)
        return S.used;
    if (C.ws_bytes < S.used)
        return HPF_EINVAL;

    prepare_kernel<<<prepare_blocks(P), 256, 0, C.st>>>(P);
    pack_wide_kernel<Y><<<dim3((unsigned)v_tiles, (unsigned)((KP + 127) / 128)), 256, 0, C.st>>>(mw, (int)C.k, CB, KO);
    pack_wide_kernel<Y><<<dim3((unsigned)n_tiles, (unsigned)((KP + 127) / 128)), 256, 0, C.st>>>(mx, (int)C.k, CB, KO);
    A.w = mw.by_row;
    A.x = mx.by_row;
    A.bias = P.bias2;
    A.meta = P.meta;
    A.n_tiles = n_tiles;
    A.v_tiles = v_tiles;
    A.rows = nr;
    A.c = fabsf(C.scale) * kLog2e;
    A.CB = CB;
    A.splits = row_splits;
    A.has_bias = C.bias != nullptr;
    wide_stats_kernel<Y><<<(unsigned)(nb * row_splits), 256, 0, C.st>>>(A);
    F.stats = A.stats;
    F.weight_top = mx.weight_top;
    F.meta = P.meta;
    F.rows = nr;
    F.splits = 2 * row_splits;
    if (!C.grad) {
        finish_rows_kernel<Y, false><<<blocks_of((nr + 3) / 4), 256, 0, C.st>>>(F);
        return (int)hipGetLastError();
    }
    finish_rows_kernel<Y, true><<<blocks_of((nr + 3) / 4), 256, 0, C.st>>>(F);
    A.reg_bias = F.reg_bias;
    A.target_log = F.target_log;
    A.away = F.away;
    for (int64_t v0 = 0; v0 < v_tiles; v0 += chunk) {
        A.v0 = v0;
        A.v_count = v_tiles - v0 < chunk ? v_tiles - v0 : chunk;
        const int dw_splits = dw_splits_of(A.v_count);
        const int64_t vg = (A.v_count + kWideA - 1) / kWideA, first = v0 * 32, count = C.v - first < A.v_count * 32 ? C.v - first : A.v_count * 32;
        wide_g_kernel<Y><<<(unsigned)(nb * vg), 256, 0, C.st>>>(A);
        ProductArgs D = {};
        D.a = A.g_rows;
        D.b = mw.by_col + v0 * unit;
        D.a_tiles = n_tiles;
        D.a_units = A.v_count * 2;
        D.tiles = A.v_count;
        D.KO = KO;
        D.splits = dx_splits;
        D.part = dx_part;
        D.more = v0 > 0;
        wide_product_kernel<Y><<<(unsigned)(up(na, 8) * kg * dx_splits), 256, 0, C.st>>>(D);
        D.a = A.g_items;
        D.b = mx.by_col;
        D.a_tiles = A.v_count;
        D.a_units = n_tiles * 2;
        D.tiles = n_tiles;
        D.splits = dw_splits;
        D.part = dw_part;
        D.more = 0;
        D.out = nullptr;
        if (dw_splits == 1) {
            D.out = (T *)C.dw + first * C.lddw;
            D.weight_top = mx.weight_top;
            D.count = count;
            D.ld = C.lddw;
            D.K = (int)C.k;
            D.scale = C.scale;
        }
        wide_product_kernel<Y><<<(unsigned)(up(vg, 8) * kg * dw_splits), 256, 0, C.st>>>(D);
        if (dw_splits > 1) {
            const JoinArgs J = {dw_part, nullptr, mx.weight_top, nullptr, count, A.v_count * 32, C.lddw, (int)C.k, KP, dw_splits, C.scale, (T *)C.dw + first * C.lddw, nullptr};
            join_kernel<Y><<<join_blocks(count, KP), 256, 0, C.st>>>(J);
        }
        if (C.bias)
            wide_sums_kernel<<<(unsigned)((count + 255) / 256), 256, 0, C.st>>>(A.part_sum, A.v_count * 32, (int)(2 * nb), mx.weight_top, Y::shift, count, C.dbias + first);
    }
    const JoinArgs J = {dx_part, nullptr, mx.weight_top, nullptr, C.n, nr, C.lddx, (int)C.k, KP, dx_splits, C.scale, C.dx, nullptr};
    join_kernel<Y><<<join_blocks(C.n, KP), 256, 0, C.st>>>(J);
    return (int)hipGetLastError();
}

// a few rows, no gradients (a choice by what the workspace's size is asked for with, so not by strides)
inline bool is_few(const Call &C) { return !C.grad && C.n <= 64; }
// of so many values shared memory has room for the rows and a tile
template <class Y> bool few_are_wide(const Call &C) { return C.k > (Y::S == 1 ? 256 : 128); }

template <class Y, int QB, int CB> void launch_few(FewArgs &A, int cus, hipStream_t st)
{
    typedef FewShape<Y, QB, CB> Z;
    const int64_t grid = (A.v_tiles + Z::waves - 1) / Z::waves;
    A.groups = (int)(grid > cus ? cus : grid);
    if (Z::bytes > 64 << 10)
        (void)hipFuncSetAttribute((const void *)few_kernel<Y, QB, CB>, hipFuncAttributeMaxDynamicSharedMemorySize, Z::bytes);
    few_kernel<Y, QB, CB><<<A.groups, Z::waves * 64, Z::bytes, st>>>(A);
}
template <class Y, int QB> void launch_few_rows(FewArgs &A, int cus, hipStream_t st)
{
    if (A.K <= 32)
        launch_few<Y, QB, 2>(A, cus, st);
    else if (A.K <= 64)
        launch_few<Y, QB, 4>(A, cus, st);
    else if (A.K <= 112)
        launch_few<Y, QB, 7>(A, cus, st);
    else if (A.K <= 128)
        launch_few<Y, QB, 8>(A, cus, st);
    else if constexpr (Y::S == 1) {
        if (A.K <= 208)
            launch_few<Y, QB, 13>(A, cus, st);
        else
            launch_few<Y, QB, 16>(A, cus, st);
    }
}

template <class Y> int64_t run_few(const Call &C)
{
    FewArgs A = {};
    A.rows = up(C.n, 32);
    A.v_tiles = (C.v + 31) / 32;
    A.K = (int)C.k;
    Space S = {C.ws, 0};
    A.stats = S.take<float>((int64_t)C.cus * 3 * A.rows * 4);
    const int parts = (int)((C.k + 63) / 64);
    char *const packed = S.take<char>(few_are_wide<Y>(C) ? A.rows / 32 * parts * 4 * Y::S * kUnit : 0);
    if (!C.ws)
        return S.used;
    if (C.ws_bytes < S.used)
        return HPF_EINVAL;
    A.x = C.x;
    A.w = C.w;
    A.target = C.target;
    A.bias = C.bias;
    A.N = C.n;
    A.V = C.v;
    A.ldx = C.ldx;
    A.ldw = C.ldw;
    A.c = fabsf(C.scale) * kLog2e;
    A.sign = C.scale < 0.0f ? -1.0f : 1.0f;
    if (few_are_wide<Y>(C)) {
        Matrix w = {}, x = {};
        fill_matrices(w, x, C);
        x.by_row = packed;
        pack_wide_kernel<Y><<<dim3((unsigned)((C.n + 31) / 32), (unsigned)((parts + 1) / 2)), 256, 0, C.st>>>(x, A.K, 4 * parts, 0);
        A.x = packed;
        A.sign = 1.0f;
        const int64_t grid = (A.v_tiles + 7) / 8;
        A.groups = (int)(grid > C.cus ? C.cus : grid);
        if (C.n <= 32)
            few_wide_kernel<Y, 1><<<A.groups, 512, 0, C.st>>>(A);
        else
            few_wide_kernel<Y, 2><<<A.groups, 512, 0, C.st>>>(A);
    } else if (C.n <= 32) {
        launch_few_rows<Y, 1>(A, C.cus, C.st);
    } else {
        launch_few_rows<Y, 2>(A, C.cus, C.st);
    }
    FinishArgs F = {};
    fill_finish(F, C);
    F.stats = A.stats;
    F.rows = A.rows;
    F.splits = A.groups;
    finish_rows_kernel<Y, false><<<(unsigned)(A.rows / 4), 256, 0, C.st>>>(F);
    return (int)hipGetLastError();
}

template <class Y, int KO> int64_t run_columns(const Call &C) { return C.k <= 32 * KO - 16 ? run_narrow<Y, KO, 1>(C) : run_narrow<Y, KO, 0>(C); }

template <class Y> int64_t run_any_narrow(const Call &C)
{
    switch ((C.k + 31) / 32) {
    case 1: return run_columns<Y, 1>(C);
    case 2: return run_columns<Y, 2>(C);
    case 3: return run_columns<Y, 3>(C);
    case 4: return run_columns<Y, 4>(C);
    case 5: return run_columns<Y, 5>(C);
    case 6: return run_columns<Y, 6>(C);
    case 7: return run_columns<Y, 7>(C);
    default: return run_columns<Y, 8>(C);
    }
}

// one source file a type (they compile side by side): the workspace's bytes, 0 for a launched call, or an error
int64_t run_f32(const Call &C);
int64_t run_bf16(const Call &C);
int64_t run_f16(const Call &C);

}  // namespace hpf_softmax
#endif  // HPF_SOFTMAX_DEV_H
