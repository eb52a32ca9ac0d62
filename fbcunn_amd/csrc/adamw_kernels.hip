// One AdamW step over many tensors (gfx950).
//
//   m = beta1 m + (1 - beta1) g          v = beta2 v + (1 - beta2) g^2
//   p = p (1 - lr decay) - lr / (1 - beta1^t) * m / (sqrt(v) / sqrt(1 - beta2^t) + eps)
//
// in 32 bits, every operation rounded by itself (this file is compiled without contraction of a product and a sum),
// so that a plain evaluation of the formulas gives the same states bit for bit, and with 32-bit states the same parameters.
// With 8-bit states the parameter's quotient takes a root and a reciprocal that are off by up to one unit each.
//
// The step is bound by memory: 28 bytes a parameter in 32 bits, 14 with 32-bit parameters, 16-bit gradients and
// 8-bit states.  One launch takes all tensors: a table of pieces of 4096 parameters, walked by at most 2048 workgroups,
// so a network of many short tensors costs no more launches than one long tensor.
//
// 8-bit states.  256 consecutive values share a scale, the largest of them over 448, and are held as e4m3 numbers of
// value / scale.  A wavefront holds exactly one such block (64 lanes x 4 values), so its scale is one reduction over
// the wavefront.  They are rounded up or down at random, in proportion to the distance: beta2 = 0.999 moves v by a
// thousandth a step, and a rounding to the nearest of numbers an eighth apart would never let it move.  The random numbers
// are a hash of (seed, step, place), so a step can be repeated.  A positive v is never rounded to zero, where the
// step m / sqrt(v) would have no bound.
//
// Measured: 40 million parameters of 160 tensors in 32 bits 222 us (5.05 TB/s, what a large copy reaches); 250 million with 16-bit
// gradients and 8-bit states 721 us (4.88 TB/s); 25 million in bf16 with 8-bit states, unaligned, 59 us (4.28 TB/s; here
// the arithmetic counts: 62 us with the rounding in integer operations, 69 with divisions and roots rounded to half a unit too).  Non-temporal stores,
// 1024 to 4096 workgroups and 8 or 16 parameters in flight a lane are all within 3 %; a workgroup for each piece is
// slower with 8-bit states (783 us).  2.9 million of 126 tensors: 13.2 us with 8-bit states, 16.7 in 32 bits (30.7 and 32.7
// where all workgroups report their end at one address).
#include <hip/hip_runtime.h>

#include <cmath>
#include <type_traits>

#include "kernels.h"
#include "lanes.h"
#include "training.h"

namespace fbfc {

constexpr int kMaxGroups = 2048;   // 8 workgroups on each of 256 CUs
constexpr int kStretch = 4;        // vectors of 4 parameters that a lane holds at once
typedef float float4v __attribute__((ext_vector_type(4)));
typedef float float2v __attribute__((ext_vector_type(2)));
constexpr unsigned kHash1 = 0x9E3779B1u, kHash2 = 0xBB67AE85u, kHash3 = 0xB504F335u;  // fractions of the golden
                                                                                      // ratio, of the roots of 3 and 1/2, odd

// The powers of the betas are carried along by one product a step: no logarithm at the end of a step.
static __host__ __device__ AdamwClock clock_of(long t, double power1, double power2, unsigned seed)
{
    AdamwClock c;
    c.t = t;
    c.power1 = power1;
    c.power2 = power2;
    c.inv_bias1 = 1.0 / (1.0 - power1);
    c.inv_root2 = (float)(1.0 / sqrt(1.0 - power2));
    c.key = seed * kHash1 + (unsigned)(t + 1) * kHash2;
    c.done = 0;
    return c;
}

AdamwClock adamw_clock(long t, double beta1, double beta2, unsigned seed)
{
    return clock_of(t, std::pow(beta1, (double)(t + 1)), std::pow(beta2, (double)(t + 1)), seed);
}

__global__ void adamw_set_clock_kernel(AdamwClock *clock, AdamwClock to) { *clock = to; }

// Two numbers with 20 random bits on top, of the place whose product with kHash1, plus the key, is `x`.
__device__ __forceinline__ void random_pair(unsigned x, unsigned &a, unsigned &b)
{
    x ^= x >> 16;
    x *= kHash2;
    x ^= x >> 15;
    x *= kHash3;
    x ^= x >> 16;
    unsigned y = x * kHash1;
    y ^= y >> 16;
    y *= kHash2;
    a = x;
    b = y;
}

// The largest magnitude of the wavefront.  The bits of magnitudes are in the order of their values, a NaN's above all.
__device__ __forceinline__ float wave_top(const float4v &v)
{
    unsigned m[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) m[i] = __float_as_uint(v[i]) & 0x7FFFFFFFu;
    const unsigned top = max(max(m[0], m[1]), max(m[2], m[3]));
    return __uint_as_float(lanes_reduce<64>(top, [](unsigned a, unsigned b) { return max(a, b); }));
}

// Byte I of `codes` becomes the e4m3 bits of a value of at most 448, rounded with the 20 upper bits of `random`: the
// instruction adds them below the last bit that is kept, of subnormal numbers too.
template <int I>
__device__ __forceinline__ unsigned round8(float value, unsigned random, unsigned codes)
{
    return __builtin_amdgcn_cvt_sr_fp8_f32(value, (int)random, (int)codes, I);
}

// scale of a block, and its inverse; a block below 2^-100 is zero
__device__ __forceinline__ float scale8(float top, float &inverse)
{
    const float scale = top < 0x1p-100f ? 0.0f : top * (1.0f / 448.0f);
    inverse = scale > 0.0f ? 1.0f / scale : 0.0f;
    return scale;
}

__device__ __forceinline__ float4v decode8(unsigned codes, float scale)
{
    const float2v lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)codes, false);
    const float2v hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)codes, true);
    return float4v{lo[0] * scale, lo[1] * scale, hi[0] * scale, hi[1] * scale};
}

// What a lane reads for its 4 parameters.
template <typename P, typename G, int BITS>
struct Four {
    Vec<P, 4> p;
    Vec<G, 4> g;
    typename std::conditional<BITS == 32, float4v, unsigned>::type m, v;
    float ms, vs;
};

template <typename P, typename G, int BITS>
__device__ __forceinline__ void load_four(Four<P, G, BITS> &f, const AdamwArgs &a, const P *param, const G *grad, long at, long left)
{
    f.p = load_some<4>(param, left);
    f.g = load_some<4>(grad, left);
    if constexpr (BITS == 32) {
        f.m = *reinterpret_cast<const float4v *>(static_cast<const float *>(a.m) + at);
        f.v = *reinterpret_cast<const float4v *>(static_cast<const float *>(a.v) + at);
    } else {
        f.m = static_cast<const unsigned *>(a.m)[at >> 2];
        f.v = static_cast<const unsigned *>(a.v)[at >> 2];
        f.ms = a.m_scale[at >> 8];
        f.vs = a.v_scale[at >> 8];
    }
}

template <typename P, typename G, int BITS>
__device__ __forceinline__ void step_four(const Four<P, G, BITS> &f, const AdamwArgs &a, float root2, float step, unsigned key, P *param, long at,
                                          long left)
{
    float4v m, v;
    if constexpr (BITS == 32) {
        m = f.m;
        v = f.v;
    } else {
        m = decode8(f.m, f.ms);
        v = decode8(f.v, f.vs);
    }
    Vec<P, 4> out;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float g = (float)f.g[i] * a.grad_scale;
        m[i] = m[i] * a.keep1 + g * a.take1;
        v[i] = v[i] * a.keep2 + g * g * a.take2;
        float q;
        if constexpr (BITS == 32)
            q = m[i] / (sqrtf(v[i]) * root2 + a.eps);
        else  // the arithmetic, not the memory, bounds this form: root and reciprocal to one unit each
            q = m[i] * __builtin_amdgcn_rcpf(__builtin_amdgcn_sqrtf(v[i]) * root2 + a.eps);
        out[i] = (P)((float)f.p[i] * a.decay - q * step);
    }
    store_some<4>(param, out, left);
    if constexpr (BITS == 32) {
        *reinterpret_cast<float4v *>(static_cast<float *>(a.m) + at) = m;
        *reinterpret_cast<float4v *>(static_cast<float *>(a.v) + at) = v;
    } else {
        float mi, vi;
        const float ms = scale8(wave_top(m), mi), vs = scale8(wave_top(v), vi);
        const unsigned x = (unsigned)at * kHash1 + (unsigned)((unsigned long)at >> 32) * kHash3 + key;
        unsigned mc = 0, vc = 0;
        const auto round = [&](auto place) {
            constexpr int I = decltype(place)::value;
            unsigned r, q;
            random_pair(x + I * kHash1, r, q);
            mc = round8<I>(copysignf(fminf(fabsf(m[I]) * mi, 448.0f), m[I]), r, mc);
            vc = round8<I>(fmaxf(fminf(v[I] * vi, 448.0f), v[I] > 0.0f && vi > 0.0f ? 0x1p-9f : 0.0f), q, vc);  // 2^-9: the smallest
        };
        round(std::integral_constant<int, 0>{});
        round(std::integral_constant<int, 1>{});
        round(std::integral_constant<int, 2>{});
        round(std::integral_constant<int, 3>{});
        static_cast<unsigned *>(a.m)[at >> 2] = mc;
        static_cast<unsigned *>(a.v)[at >> 2] = vc;
        if ((threadIdx.x & 63) == 0) {
            a.m_scale[at >> 8] = ms;
            a.v_scale[at >> 8] = vs;
        }
    }
}

// Counts one more of `all`; whether it is the last, which leaves the count at zero for the next step.
__device__ __forceinline__ bool one_more(unsigned *count, unsigned all)
{
    if (__hip_atomic_fetch_add(count, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) != all - 1) return false;
    __hip_atomic_store(count, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    return true;
}

template <typename P, typename G, int BITS>
__global__ __launch_bounds__(256) void adamw_kernel(AdamwArgs a)
{
    const AdamwClock now = *a.clock;
    const float step = (float)(a.lr * now.inv_bias1);
    for (int k = blockIdx.x; k < a.n_pieces; k += gridDim.x) {
        const AdamwPiece piece = a.pieces[k];
        P *param = static_cast<P *>(piece.param);
        const G *grad = static_cast<const G *>(piece.grad);
        long o = threadIdx.x * 4;
        // whole stretches: the loads of all of it before the first store
        for (; o - threadIdx.x * 4 + kStretch * 1024 <= piece.n; o += kStretch * 1024) {
            Four<P, G, BITS> f[kStretch];
#pragma unroll
            for (int j = 0; j < kStretch; ++j) load_four<P, G, BITS>(f[j], a, param + o + j * 1024, grad + o + j * 1024, piece.first + o + j * 1024, 4);
#pragma unroll
            for (int j = 0; j < kStretch; ++j)
                step_four<P, G, BITS>(f[j], a, now.inv_root2, step, now.key, param + o + j * 1024, piece.first + o + j * 1024, 4);
        }
        for (; (o & ~255L) < piece.n; o += 1024) {  // whole wavefronts stay or leave
            Four<P, G, BITS> f;
            load_four<P, G, BITS>(f, a, param + o, grad + o, piece.first + o, piece.n - o);
            step_four<P, G, BITS>(f, a, now.inv_root2, step, now.key, param + o, piece.first + o, piece.n - o);
        }
    }
    // Every wavefront of this workgroup has read the clock; the last workgroup of all moves it on, so a step replayed
    // from a graph is the next step.
    __syncthreads();
    if (threadIdx.x == 0) {
        const unsigned line = blockIdx.x % kAdamwLines, lines = min(gridDim.x, (unsigned)kAdamwLines);
        if (one_more(a.ended + line * kAdamwLine, (gridDim.x - line + kAdamwLines - 1) / kAdamwLines) && one_more(&a.clock->done, lines))
            *a.clock = clock_of(now.t + 1, now.power1 * a.beta1, now.power2 * a.beta2, a.seed);
    }
}

hipError_t launch_adamw_set_clock(const AdamwArgs &a, long t, hipStream_t s)
{
    FBFC_LAUNCH(adamw_set_clock_kernel, dim3(1), dim3(1), 0, s, a.clock, adamw_clock(t, a.beta1, a.beta2, a.seed));
    return hipGetLastError();
}

template <typename P, typename G>
static hipError_t launch_typed(int bits, const AdamwArgs &a, hipStream_t s)
{
    const int groups = a.n_pieces < 1 ? 1 : a.n_pieces < kMaxGroups ? a.n_pieces : kMaxGroups;
    kernel_log_add(bits == 8 ? "adamw_kernel<8>" : "adamw_kernel<32>", (long)groups * 256);
    if (bits == 8)
        FBFC_LAUNCH((adamw_kernel<P, G, 8>), dim3(groups), dim3(256), 0, s, a);
    else
        FBFC_LAUNCH((adamw_kernel<P, G, 32>), dim3(groups), dim3(256), 0, s, a);
    return hipGetLastError();
}

template <typename P>
static hipError_t launch_grad(int grad_type, int bits, const AdamwArgs &a, hipStream_t s)
{
    return grad_type == kF32 ? launch_typed<P, float>(bits, a, s)
           : grad_type == kBF16 ? launch_typed<P, bf16>(bits, a, s) : launch_typed<P, f16>(bits, a, s);
}

hipError_t launch_adamw(int param_type, int grad_type, int state_bits, const AdamwArgs &a, hipStream_t s)
{
    return param_type == kF32 ? launch_grad<float>(grad_type, state_bits, a, s)
           : param_type == kBF16 ? launch_grad<bf16>(grad_type, state_bits, a, s)
                                 : launch_grad<f16>(grad_type, state_bits, a, s);
}

}  // namespace fbfc
