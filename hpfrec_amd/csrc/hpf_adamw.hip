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
// largest value is then a reduction within the wavefront).
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "hpf_hip.h"

#pragma clang fp contract(off)

namespace {

constexpr int kBlock = 256;              // values per wavefront pass = values per scale of an 8-bit moment
constexpr int kChunkBlocks = 16;         // blocks per workgroup pass: 4 wavefronts x 4
constexpr int kMaxTensors = 40;          // per launch: their descriptors travel in the kernel's arguments
constexpr int kTicketShift = 40;         // the step counter's upper bits count the workgroups that are done

struct Tensor {
    void *p;
    const void *g;
    void *m, *v;
    float *master, *m_scale, *v_scale;
    int64_t n;
    double wd;
    int32_t chunk0;                      // first chunk of this tensor in the launch
    int32_t number;                      // its number in the caller's list (part of the random bits' key)
    int32_t wide;                        // every pointer allows the wide accesses
};

struct Args {
    Tensor t[kMaxTensors];
    unsigned long long *step;
    const float *lr_dev;
    double lr, b1, b2, eps;
    uint64_t seed;
    int32_t ntensors, nchunks, advance;
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
    int e = 127 - 126;                                          // a subnormal's scale: 2^-126
    const int b = (int)(__float_as_uint(top) >> 23);            // biased exponent
    if (b - 7 > 1)
        e = b - 7;
    return top > 0.0f ? __uint_as_float((uint32_t)e << 23) : 1.0f;
}

// four values' codes; inv is the scale's reciprocal (exact: a power of two)
__device__ inline uint32_t encode4(const float x[4], float inv, const uint32_t bits16[4], bool least)
{
    float q[4];
    uint32_t lost = 0;
    for (int i = 0; i < 4; ++i) {
        const float y = x[i] * inv, a = fabsf(y);
        const float low = a < 0x1p-6f ? 0x1p-6f : 0.0f;         // e4m3's subnormals: a fixed step, at the end of this sum's mantissa
        const uint32_t b = (__float_as_uint(a + low) + (bits16[i] << 4)) & 0xFFF00000u;
        float r = __uint_as_float(b) - low;
        if (least && r == 0.0f && x[i] > 0.0f)
            r = 0x1p-9f;
        q[i] = copysignf(r, y);
        if (!(a < 0x1p127f))                                    // infinite or NaN: the one code that says so
            lost |= 0x7Fu << (8 * i);
    }
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(q[0], q[1], 0, false);
    w = __builtin_amdgcn_cvt_pk_fp8_f32(q[2], q[3], w, true);
    uint32_t keep = (uint32_t)w;
    for (int i = 0; i < 4; ++i)
        if (lost >> (8 * i) & 0xFF)
            keep = (keep & ~(0xFFu << (8 * i))) | 0x7Fu << (8 * i);
    return keep;
}

__device__ inline float wave_max(float x)
{
    for (int d = 32; d; d >>= 1)
        x = fmaxf(x, __shfl_xor(x, d));
    return x;
}

__device__ inline float finite_or_zero(float x) { return x < INFINITY ? x : 0.0f; }   // x >= 0 or NaN

template <class P, class G, int BITS> __global__ __launch_bounds__(256) void adamw_kernel(Args A)
{
    __shared__ double corr[2];
    __shared__ float lr_s;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const unsigned long long at = __hip_atomic_load(A.step, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) & ((1ull << kTicketShift) - 1);
    const unsigned long long now = at + 1;
    if (threadIdx.x == 0) {
        corr[0] = 1.0 - pow(A.b1, (double)now);
        corr[1] = sqrt(1.0 - pow(A.b2, (double)now));
        lr_s = A.lr_dev ? *A.lr_dev : 0.0f;
    }
    __syncthreads();
    const double lr = A.lr_dev ? (double)lr_s : A.lr;
    const float rate = (float)(lr / corr[0]), root = (float)corr[1], eps = (float)A.eps;
    const float b1 = (float)A.b1, b2 = (float)A.b2, c1 = (float)(1.0 - A.b1), c2 = (float)(1.0 - A.b2);
    const uint32_t key0 = mix(mix(mix((uint32_t)A.seed) ^ (uint32_t)(A.seed >> 32)) + (uint32_t)now);

    int ti = 0;
    for (int chunk = blockIdx.x; chunk < A.nchunks; chunk += gridDim.x) {
        while (ti + 1 < A.ntensors && A.t[ti + 1].chunk0 <= chunk)
            ++ti;
        const Tensor &t = A.t[ti];
        const float keep = (float)(1.0 - lr * t.wd);
        const bool wide = t.wide != 0;
        const uint32_t key = mix(key0 + (uint32_t)t.number);
        P *const pp = (P *)t.p;
        const G *const gp = (const G *)t.g;
        const int64_t block0 = (int64_t)(chunk - t.chunk0) * kChunkBlocks + wave;
#pragma unroll
        for (int k = 0; k < kChunkBlocks / 4; ++k) {
            const int64_t block = block0 + 4 * k, i0 = block * kBlock + 4 * lane, left = t.n - i0;
            if (block * kBlock >= t.n)
                break;
            const int valid = left >= 4 ? 4 : left > 0 ? (int)left : 0;
            float p[4], g[4], m[4], v[4];
            load4(gp + i0, wide, valid, g);
            if constexpr (sizeof(P) == 4)
                load4((const float *)pp + i0, wide, valid, p);
            else
                load4(t.master + i0, wide, valid, p);
            if constexpr (BITS == 8) {
                decode4(load_codes((const uint8_t *)t.m + i0, wide, valid), t.m_scale[block], m);
                decode4(load_codes((const uint8_t *)t.v + i0, wide, valid), t.v_scale[block], v);
                for (int i = 0; i < 4; ++i)
                    v[i] = v[i] * v[i];
            } else {
                load4((const float *)t.m + i0, wide, valid, m);
                load4((const float *)t.v + i0, wide, valid, v);
            }
            float r[4], top_m = 0.0f, top_r = 0.0f;
            for (int i = 0; i < 4; ++i) {
                m[i] = m[i] * b1 + g[i] * c1;
                v[i] = v[i] * b2 + (g[i] * g[i]) * c2;
                r[i] = sqrtf(v[i]);
                p[i] = p[i] * keep - rate * m[i] / (r[i] / root + eps);
                if constexpr (BITS == 8) {
                    top_m = fmaxf(top_m, finite_or_zero(fabsf(m[i])));
                    top_r = fmaxf(top_r, finite_or_zero(r[i]));
                }
            }
            if constexpr (sizeof(P) == 4) {
                store4((float *)pp + i0, wide, valid, p);
            } else {
                store4(t.master + i0, wide, valid, p);
                store4(pp + i0, wide, valid, p);
            }
            if constexpr (BITS == 8) {
                const float ms = block_scale(wave_max(top_m)), rs = block_scale(wave_max(top_r));
                uint32_t bm[4], br[4];
                for (int i = 0; i < 4; ++i) {
                    const uint32_t w = mix((uint32_t)(i0 + i) + key + (uint32_t)((i0 + i) >> 32) * kMulA);
                    bm[i] = w & 0xFFFFu;
                    br[i] = w >> 16;
                }
                store_codes((uint8_t *)t.m + i0, wide, valid, encode4(m, 1.0f / ms, bm, false));
                store_codes((uint8_t *)t.v + i0, wide, valid, encode4(r, 1.0f / rs, br, true));
                if (lane == 0) {
                    t.m_scale[block] = ms;
                    t.v_scale[block] = rs;
                }
            } else {
                store4((float *)t.m + i0, wide, valid, m);
                store4((float *)t.v + i0, wide, valid, v);
            }
        }
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
        int64_t chunks = 0;
        for (; i < ntensors && A.ntensors < kMaxTensors; ++i) {
            const hpf_adamw_tensor &t = tensors[i];
            if (t.n == 0)
                continue;
            const int64_t mine = (t.n + (int64_t)kBlock * kChunkBlocks - 1) / ((int64_t)kBlock * kChunkBlocks);
            if (chunks + mine > 0x7FFFFFFF) {
                if (chunks == 0)
                    return HPF_EUNSUPPORTED;   // one tensor of over 2^43 values
                break;
            }
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
            d.chunk0 = (int32_t)chunks;
            d.number = t.number;
            d.wide = aligned(t.param, 4 * psize) && aligned(t.grad, 4 * gsize) && aligned(t.m, 4 * ssize) &&
                     aligned(t.v, 4 * ssize) && aligned(t.master, 16);
            chunks += mine;
        }
        A.nchunks = (int32_t)chunks;
        A.advance = i >= ntensors ? advance != 0 : 0;
        if (chunks == 0 && !A.advance)
            break;
        const int grid = (int)(chunks < 1 ? 1 : chunks < grid_blocks ? chunks : grid_blocks);
        const hipStream_t st = (hipStream_t)stream;
        const int rc = param_type == HPF_F32    ? launch_g<float>(A, grad_type, state_bits, grid, st)
                       : param_type == HPF_BF16 ? launch_g<__bf16>(A, grad_type, state_bits, grid, st)
                                                : launch_g<_Float16>(A, grad_type, state_bits, grid, st);
        if (rc)
            return rc;
    } while (i < ntensors);
    return 0;
}
