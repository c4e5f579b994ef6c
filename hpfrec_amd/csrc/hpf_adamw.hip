// hpf_adamw.hip -- one AdamW step (decoupled weight decay) over a list of tensors in one launch; moments in 32 or in 8 bits.
//
//   m <- b1 m + (1 - b1) g;   v <- b2 v + (1 - b2) g^2
//   p <- p (1 - lr wd) - (lr / (1 - b1^t)) m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// Every product and sum is rounded once, in this order (no contraction into fused operations): the 8-bit forms below round
// with random bits, and a step has to give the same codes wherever it is computed.
//
// 8-bit moments: m and r = sqrt(v) in e4m3, each times a power of two that 256 consecutive values share.  The power puts the
// block's largest finite magnitude into [128, 256), so that the division by it is exact and rounding up cannot pass 448;
// what is left spans 2^-17 of that largest value.  Rounding is STOCHASTIC: with b2 = 0.999 a moment changes by less than a
// thousandth in a step, and rounding to nearest -- 1/16 at most in e4m3 -- would never let it move.  16 random bits a
// value, a function of (seed, step, tensor, index) alone.  A root that is not zero keeps at least the smallest code, since
// a later step divides by it.
//
// Bound by memory: 28 bytes a value with 32-bit moments (p, m, v both ways, g), 16 with 8-bit ones.  One wavefront takes 256
// consecutive values at a time (4 a lane: 16-byte accesses in 32 bits, and exactly one block of an 8-bit moment, whose
// largest value is then a reduction within the wavefront), and an equal share of all blocks of the launch.  Where a large copy
// moves 4.77 TB/s: 69M values in 32 bits 397 us, 4.87 TB/s; 138M bf16 values with masters and 8-bit moments 496 us, 4.48 TB/s; 8.3M
// in 32 bits with 8-bit moments 32 us, 4.1 TB/s; 153k values 8 us, which is latency.  Four workgroups a compute unit (8.3M: 33 us, two
// 40, eight 106, since the counter's arrivals are served one by one) and two blocks of a wavefront in flight (138M: one 512 us, two
// 499, four 500; 69M in 32 bits 398, 403, 405).
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "hpf_hip.h"

#pragma clang fp contract(off)

namespace {

constexpr int kBlock = 256;              // values per wavefront pass = values per scale of an 8-bit moment
constexpr int kAtOnce = 2;               // blocks of a wavefront in flight
constexpr int kMaxTensors = 40;          // per launch: their descriptors travel in the kernel's arguments
constexpr int64_t kMaxBlocks = 0x7FFFFF00;   // per launch, and per tensor: 2^39 values, less 2^16
constexpr int kTicketShift = 40;         // the step counter's upper bits count the workgroups that are done
constexpr int kMaxGrid = 1 << 22;        // what fits there

struct Tensor {
    void *p;
    const void *g;
    void *m, *v;
    float *master, *m_scale, *v_scale;
    int64_t n;
    double wd;
    int32_t block0;                      // its first block in the launch
    int32_t number;                      // its number in the caller's list (part of the random bits' key)
    int32_t wide;                        // every pointer allows the wide accesses
};

struct Args {
    Tensor t[kMaxTensors];
    unsigned long long *step;
    const float *lr_dev;
    double lr, b1, b2, eps;
    uint64_t seed;
    int32_t ntensors, nblocks, advance;
};
static_assert(sizeof(Args) <= 4096, "kernel arguments");

template <class T> __device__ inline void load4(const T *p, bool wide, int valid, float out[4])
{
    if (wide && valid == 4) {
        struct alignas(4 * sizeof(T)) V { T x[4]; };
        const V q = *reinterpret_cast<const V *>(p);
        for (int i = 0; i < 4; ++i)
            out[i] = (float)q.x[i];
    } else {
        for (int i = 0; i < 4; ++i)
            out[i] = i < valid ? (float)p[i] : 0.0f;
    }
}

template <class T> __device__ inline void store4(T *p, bool wide, int valid, const float in[4])
{
    if (wide && valid == 4) {
        struct alignas(4 * sizeof(T)) V { T x[4]; };
        V q;
        for (int i = 0; i < 4; ++i)
            q.x[i] = (T)in[i];
        *reinterpret_cast<V *>(p) = q;
    } else {
        for (int i = 0; i < 4; ++i)
            if (i < valid)
                p[i] = (T)in[i];
    }
}

__device__ inline uint32_t load_codes(const uint8_t *p, bool wide, int valid)
{
    if (wide && valid == 4)
        return *reinterpret_cast<const uint32_t *>(p);
    uint32_t w = 0;
    for (int i = 0; i < 4; ++i)
        if (i < valid)
            w |= (uint32_t)p[i] << (8 * i);
    return w;
}

__device__ inline void store_codes(uint8_t *p, bool wide, int valid, uint32_t w)
{
    if (wide && valid == 4) {
        *reinterpret_cast<uint32_t *>(p) = w;
        return;
    }
    for (int i = 0; i < 4; ++i)
        if (i < valid)
            p[i] = (uint8_t)(w >> (8 * i));
}

__device__ inline void decode4(uint32_t w, float scale, float out[4])
{
    const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
    out[0] = lo[0] * scale;
    out[1] = lo[1] * scale;
    out[2] = hi[0] * scale;
    out[3] = hi[1] * scale;
}

constexpr uint32_t kMulA = 0x9E3779B1u, kMulB = 0x6A09E669u;   // odd: the fractions of the golden ratio and of sqrt(2)

__device__ inline uint32_t mix(uint32_t x)
{
    x ^= x >> 16;
    x *= kMulA;
    x ^= x >> 15;
    x *= kMulB;
    return x ^ (x >> 16);
}

// the power of two that puts `top` (finite, >= 0) into [128, 256); 1 for an empty block
__device__ inline float block_scale(float top)
{
    const int e = (int)(__float_as_uint(top) >> 23) - 7;        // biased; a subnormal's scale: 2^-126
    return top > 0.0f ? __uint_as_float((uint32_t)(e > 1 ? e : 1) << 23) : 1.0f;
}

// four values' codes; inv is the scale's reciprocal (exact: a power of two)
template <bool ROOT> __device__ inline uint32_t encode4(const float x[4], float inv, const uint32_t bits16[4])
{
    float q[4];
    bool lost = false;
    for (int i = 0; i < 4; ++i) {
        const float y = x[i] * inv, a = fabsf(y);
        const float low = a < 0x1p-6f ? 0x1p-6f : 0.0f;         // e4m3's subnormals: a fixed step, at the end of this sum's mantissa
        const uint32_t b = (__float_as_uint(a + low) + (bits16[i] << 4)) & 0xFFF00000u;
        float r = __uint_as_float(b) - low;
        if (ROOT)
            r = fmaxf(r, x[i] > 0.0f ? 0x1p-9f : 0.0f);         // a root above zero keeps the smallest code
        q[i] = ROOT ? r : copysignf(r, y);
        lost |= !(a < 0x1p127f);
    }
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(q[0], q[1], 0, false);
    w = __builtin_amdgcn_cvt_pk_fp8_f32(q[2], q[3], w, true);
    if (__any(lost))                                            // infinite or NaN: the one code that says so
        for (int i = 0; i < 4; ++i)
            if (!(fabsf(x[i]) < INFINITY))
                w = (int)(((uint32_t)w & ~(0xFFu << (8 * i))) | 0x7Fu << (8 * i));
    return (uint32_t)w;
}

// the wavefront's largest, by exchanges within registers (lanes' neighbours, rows of 16, halves)
template <int CTRL> __device__ inline float max_dpp(float x)
{
    return fmaxf(x, __uint_as_float((uint32_t)__builtin_amdgcn_update_dpp((int)__float_as_uint(x), (int)__float_as_uint(x), CTRL, 0xF, 0xF, true)));
}
__device__ inline float wave_max(float x)
{
    x = max_dpp<0xB1>(x);     // lanes 1 0 3 2
    x = max_dpp<0x4E>(x);     // lanes 2 3 0 1
    x = max_dpp<0x141>(x);    // mirrored within 8
    x = max_dpp<0x140>(x);    // mirrored within 16
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}

// the largest finite magnitude of the block
__device__ inline float block_top(const float x[4])
{
    float top = wave_max(fmaxf(fmaxf(fabsf(x[0]), fabsf(x[1])), fmaxf(fabsf(x[2]), fabsf(x[3]))));   // (of NaN and a number: the number)
    if (!(top < INFINITY)) {
        top = 0.0f;
        for (int i = 0; i < 4; ++i)
            top = fmaxf(top, fabsf(x[i]) < INFINITY ? fabsf(x[i]) : 0.0f);
        top = wave_max(top);
    }
    return top;
}

// the square root of x >= 2^-96, rounded to nearest: the hardware's, good to one unit, against its two neighbours
__device__ inline float root_of(float x)
{
    const float s = __builtin_amdgcn_sqrtf(x), down = __uint_as_float(__float_as_uint(s) - 1), up = __uint_as_float(__float_as_uint(s) + 1);
    const float r = fmaf(-down, s, x) <= 0.0f ? down : s;
    return fmaf(-up, s, x) > 0.0f ? up : r;
}

// b^n
__device__ inline double power(double b, unsigned long long n)
{
    double r = 1.0;
    for (; n; n >>= 1, b *= b)
        r = n & 1 ? r * b : r;
    return r;
}

template <class P, class G, int BITS> __global__ __launch_bounds__(256) void adamw_kernel(Args A)
{
    const int lane = threadIdx.x & 63;
    const unsigned long long at = __hip_atomic_load(A.step, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) & ((1ull << kTicketShift) - 1);
    const unsigned long long now = at + 1;
    const double lr = A.lr_dev ? (double)*A.lr_dev : A.lr;
    const float rate = (float)(lr / (1.0 - power(A.b1, now))), over_root = (float)(1.0 / sqrt(1.0 - power(A.b2, now))), eps = (float)A.eps;
    const float b1 = (float)A.b1, b2 = (float)A.b2, c1 = (float)(1.0 - A.b1), c2 = (float)(1.0 - A.b2);
    const uint32_t key0 = mix(mix(mix((uint32_t)A.seed) ^ (uint32_t)(A.seed >> 32)) + (uint32_t)now);

    // an equal share of consecutive blocks for each wavefront, from the tensor that holds the first one on
    const int wave = __builtin_amdgcn_readfirstlane((int)(blockIdx.x * 4 + (threadIdx.x >> 6))), waves = gridDim.x * 4;
    const int share = A.nblocks / waves, more = A.nblocks % waves;
    int done = share * wave + (wave < more ? wave : more);
    const int stop = done + share + (wave < more);
    for (int ti = 0; done < stop; ++ti) {
        const int last = ti + 1 < A.ntensors ? A.t[ti + 1].block0 : A.nblocks;     // beyond the tensor's
        if (last <= done)
            continue;
        const Tensor &t = A.t[ti];
        const float keep = (float)(1.0 - lr * t.wd);
        const bool wide = t.wide != 0;
        const uint32_t key = mix(key0 + (uint32_t)t.number);
        P *const pp = (P *)t.p;
        const G *const gp = (const G *)t.g;
        const int end = last < stop ? last : stop;
        for (; done < end; done += kAtOnce) {      // kAtOnce blocks' loads are on their way together
            float p[kAtOnce][4], g[kAtOnce][4], m[kAtOnce][4], v[kAtOnce][4];
            int valid[kAtOnce];
#pragma unroll
            for (int u = 0; u < kAtOnce; ++u) {
                const int64_t block = done + u - t.block0, i0 = block * kBlock + 4 * lane, left = done + u < end ? t.n - i0 : 0;
                valid[u] = left >= 4 ? 4 : left > 0 ? (int)left : 0;
                load4(gp + i0, wide, valid[u], g[u]);
                if constexpr (sizeof(P) == 4)
                    load4((const float *)pp + i0, wide, valid[u], p[u]);
                else
                    load4(t.master + i0, wide, valid[u], p[u]);
                if constexpr (BITS == 8) {
                    const bool in = done + u < end;
                    decode4(load_codes((const uint8_t *)t.m + i0, wide, valid[u]), in ? t.m_scale[block] : 0.0f, m[u]);
                    decode4(load_codes((const uint8_t *)t.v + i0, wide, valid[u]), in ? t.v_scale[block] : 0.0f, v[u]);
                    for (int i = 0; i < 4; ++i)
                        v[u][i] = v[u][i] * v[u][i];
                } else {
                    load4((const float *)t.m + i0, wide, valid[u], m[u]);
                    load4((const float *)t.v + i0, wide, valid[u], v[u]);
                }
            }
#pragma unroll
            for (int u = 0; u < kAtOnce; ++u) {
                const int64_t block = done + u - t.block0, i0 = block * kBlock + 4 * lane;
                float r[4];
                bool tiny = false;
                for (int i = 0; i < 4; ++i) {
                    m[u][i] = m[u][i] * b1 + g[u][i] * c1;
                    v[u][i] = v[u][i] * b2 + (g[u][i] * g[u][i]) * c2;
                    tiny |= v[u][i] < 0x1p-96f;
                }
                if (__any(tiny)) {             // whatever the size
                    for (int i = 0; i < 4; ++i) {
                        r[i] = sqrtf(v[u][i]);
                        p[u][i] = p[u][i] * keep - rate * m[u][i] / (r[i] * over_root + eps);
                    }
                } else {                       // (the hardware's reciprocal is good to one unit, which is what p needs of it)
                    for (int i = 0; i < 4; ++i) {
                        r[i] = root_of(v[u][i]);
                        p[u][i] = p[u][i] * keep - (rate * m[u][i]) * __builtin_amdgcn_rcpf(r[i] * over_root + eps);
                    }
                }
                if constexpr (sizeof(P) == 4) {
                    store4((float *)pp + i0, wide, valid[u], p[u]);
                } else {
                    store4(t.master + i0, wide, valid[u], p[u]);
                    store4(pp + i0, wide, valid[u], p[u]);
                }
                if constexpr (BITS == 8) {
                    const float ms = block_scale(block_top(m[u])), rs = block_scale(block_top(r));
                    uint32_t bm[4], br[4];
                    for (int i = 0; i < 4; ++i) {
                        const uint32_t w = mix((uint32_t)(i0 + i) + key + (uint32_t)((i0 + i) >> 32) * kMulA);
                        bm[i] = w & 0xFFFFu;
                        br[i] = w >> 16;
                    }
                    store_codes((uint8_t *)t.m + i0, wide, valid[u], encode4<false>(m[u], 1.0f / ms, bm));
                    store_codes((uint8_t *)t.v + i0, wide, valid[u], encode4<true>(r, 1.0f / rs, br));
                    if (lane == 0 && done + u < end) {
                        t.m_scale[block] = ms;
                        t.v_scale[block] = rs;
                    }
                } else {
                    store4((float *)t.m + i0, wide, valid[u], m[u]);
                    store4((float *)t.v + i0, wide, valid[u], v[u]);
                }
            }
        }
        done = end;
    }
    // The counter moves on once every workgroup has read it: the last to arrive adds the one and takes the arrivals away.
    if (A.advance) {
        __syncthreads();
        if (threadIdx.x == 0) {
            const unsigned long long one = 1ull << kTicketShift;
            const unsigned long long was = __hip_atomic_fetch_add(A.step, one, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            if ((was >> kTicketShift) == gridDim.x - 1)
                __hip_atomic_fetch_add(A.step, 1ull - gridDim.x * one, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
    }
}

template <class P, class G> int launch(const Args &A, int bits, int grid, hipStream_t st)
{
    if (bits == 8)
        adamw_kernel<P, G, 8><<<grid, 256, 0, st>>>(A);
    else
        adamw_kernel<P, G, 32><<<grid, 256, 0, st>>>(A);
    return (int)hipGetLastError();
}

template <class P> int launch_g(const Args &A, int gtype, int bits, int grid, hipStream_t st)
{
    if (gtype == HPF_F32)
        return launch<P, float>(A, bits, grid, st);
    if (gtype == HPF_BF16)
        return launch<P, __bf16>(A, bits, grid, st);
    return launch<P, _Float16>(A, bits, grid, st);
}

bool aligned(const void *p, int bytes) { return ((uintptr_t)p & (uintptr_t)(bytes - 1)) == 0; }

}  // namespace

extern "C" int hpf_hip_adamw_step(const hpf_adamw_tensor *tensors, int ntensors, int param_type, int grad_type, int state_bits,
                                  int64_t *step, int advance, const float *lr_dev, double lr, double beta1, double beta2,
                                  double eps, uint64_t seed, int grid_blocks, void *stream)
{
    if (ntensors < 0 || (ntensors > 0 && !tensors) || !step || grid_blocks <= 0)
        return HPF_EINVAL;
    if ((state_bits != 32 && state_bits != 8) || param_type < HPF_F32 || param_type > HPF_F16 || grad_type < HPF_F32 ||
        grad_type > HPF_F16)
        return HPF_EUNSUPPORTED;
    if (!(beta1 >= 0.0 && beta1 < 1.0) || !(beta2 >= 0.0 && beta2 < 1.0) || !(eps >= 0.0))
        return HPF_EINVAL;
    const int psize = param_type == HPF_F32 ? 4 : 2, gsize = grad_type == HPF_F32 ? 4 : 2, ssize = state_bits / 8;
    for (int i = 0; i < ntensors; ++i) {
        const hpf_adamw_tensor &t = tensors[i];
        if (t.n < 0)
            return HPF_EINVAL;
        if (t.n == 0)
            continue;
        if ((t.n - 1) / kBlock >= kMaxBlocks)
            return HPF_EUNSUPPORTED;           // (here, so that a refused call has changed nothing)
        if (!t.param || !t.grad || !t.m || !t.v || (param_type != HPF_F32) != (t.master != nullptr))
            return HPF_EINVAL;
        if (state_bits == 8 ? (!t.m_scale || !t.v_scale) : (t.m_scale || t.v_scale))
            return HPF_EINVAL;
        if (!aligned(t.param, psize) || !aligned(t.grad, gsize) || !aligned(t.m, ssize) || !aligned(t.v, ssize) ||
            !aligned(t.master, 4) || !aligned(t.m_scale, 4) || !aligned(t.v_scale, 4))
            return HPF_EINVAL;
    }
    int i = 0;
    do {   // as many tensors a launch as its arguments hold; at least one launch, which moves the counter on
        Args A;
        A.step = (unsigned long long *)step;
        A.lr_dev = lr_dev;
        A.lr = lr;
        A.b1 = beta1;
        A.b2 = beta2;
        A.eps = eps;
        A.seed = seed;
        A.ntensors = 0;
        int64_t blocks = 0;
        for (; i < ntensors && A.ntensors < kMaxTensors; ++i) {
            const hpf_adamw_tensor &t = tensors[i];
            if (t.n == 0)
                continue;
            const int64_t mine = (t.n + kBlock - 1) / kBlock;
            if (blocks + mine > kMaxBlocks)
                break;
            Tensor &d = A.t[A.ntensors++];
            d.p = t.param;
            d.g = t.grad;
            d.m = t.m;
            d.v = t.v;
            d.master = t.master;
            d.m_scale = t.m_scale;
            d.v_scale = t.v_scale;
            d.n = t.n;
            d.wd = t.weight_decay;
            d.block0 = (int32_t)blocks;
            d.number = t.number;
            d.wide = aligned(t.param, 4 * psize) && aligned(t.grad, 4 * gsize) && aligned(t.m, 4 * ssize) &&
                     aligned(t.v, 4 * ssize) && aligned(t.master, 16);
            blocks += mine;
        }
        A.nblocks = (int32_t)blocks;
        A.advance = i >= ntensors ? advance != 0 : 0;
        if (blocks == 0 && !A.advance)
            break;
        const int64_t want = (blocks + 7) / 8;       // four wavefronts of kAtOnce blocks
        const int most = grid_blocks < kMaxGrid ? grid_blocks : kMaxGrid, grid = (int)(want < 1 ? 1 : want < most ? want : most);
        const hipStream_t st = (hipStream_t)stream;
        const int rc = param_type == HPF_F32    ? launch_g<float>(A, grad_type, state_bits, grid, st)
                       : param_type == HPF_BF16 ? launch_g<__bf16>(A, grad_type, state_bits, grid, st)
                                                : launch_g<_Float16>(A, grad_type, state_bits, grid, st);
        if (rc)
            return rc;
    } while (i < ntensors);
    return 0;
}
