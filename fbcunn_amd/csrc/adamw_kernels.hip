// One AdamW step over many tensors (gfx950).
//
//   m = beta1 m + (1 - beta1) g          v = beta2 v + (1 - beta2) g^2
//   p = p (1 - lr decay) - lr / (1 - beta1^t) * m / (sqrt(v) / sqrt(1 - beta2^t) + eps)
//
// in 32 bits, every operation rounded by itself (this file is compiled without contraction of a product and a sum),
// so that a plain evaluation of the formulas gives the same states bit for bit.
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
#include <hip/hip_runtime.h>

#include <cmath>

#include "kernels.h"
#include "training.h"

namespace fbfc {

constexpr int kMaxGroups = 2048;   // 8 workgroups on each of 256 CUs
constexpr unsigned kHash1 = 0x9E3779B1u, kHash2 = 0xBB67AE85u, kHash3 = 0xB504F335u;  // fractions of the golden
                                                                                      // ratio, of the roots of 3 and 1/2, odd

static __host__ __device__ AdamwClock clock_at(long t, double beta1, double beta2, unsigned seed)
{
    AdamwClock c;
    const double next = (double)(t + 1);
    c.t = t;
    c.inv_bias1 = 1.0 / -expm1(next * log(beta1));
    c.inv_root2 = (float)(1.0 / sqrt(-expm1(next * log(beta2))));
    c.key = seed * kHash1 + (unsigned)(t + 1) * kHash2;
    c.done = 0;
    return c;
}

AdamwClock adamw_clock(long t, double beta1, double beta2, unsigned seed) { return clock_at(t, beta1, beta2, seed); }

__global__ void adamw_set_clock_kernel(AdamwClock *clock, long t, double beta1, double beta2, unsigned seed)
{
    *clock = clock_at(t, beta1, beta2, seed);
}

// Two 20-bit numbers in the upper bits of `a` and `b`.
__device__ __forceinline__ void random_pair(long i, unsigned key, unsigned &a, unsigned &b)
{
    unsigned x = (unsigned)i * kHash1 + (unsigned)((unsigned long)i >> 32) * kHash3 + key;
    x ^= x >> 16;
    x *= kHash2;
    x ^= x >> 15;
    x *= kHash3;
    x ^= x >> 16;
    unsigned y = x * kHash1;
    y ^= y >> 16;
    y *= kHash2;
    a = x >> 12;
    b = y >> 12;
}

// The largest value of the wavefront; NaN if one is NaN.
__device__ __forceinline__ float wave_max(float v)
{
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) {
        const float o = __shfl_xor(v, off, 64);
        v = (o > v || o != o) ? o : v;
    }
    return v;
}
__device__ __forceinline__ float max_nan(float a, float b) { return (b > a || b != b) ? b : a; }

// e4m3 bits of four magnitudes times `inverse`.  The bits of a 32-bit float of 2^-120 times the value hold an e4m3
// number on top (its smallest normal number, 2^-6, becomes the float's, 2^-126), so a 20-bit random number added below
// rounds it, subnormal numbers too.
__device__ __forceinline__ unsigned round8(float magnitude, float inverse, unsigned random)
{
    const unsigned bits = __float_as_uint(magnitude * inverse * 0x1p-120f);
    const unsigned code = (bits + random) >> 20;
    return code < 0x7Eu ? code : 0x7Eu;
}

// scale of a block, and its inverse; a block below 2^-100 is zero
__device__ __forceinline__ float scale8(float top, float &inverse)
{
    const float scale = top < 0x1p-100f ? 0.0f : top * (1.0f / 448.0f);
    inverse = scale > 0.0f ? 1.0f / scale : 0.0f;
    return scale;
}

typedef float float4v __attribute__((ext_vector_type(4)));
typedef float float2v __attribute__((ext_vector_type(2)));

__device__ __forceinline__ float4v decode8(unsigned codes)
{
    const float2v lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)codes, false);
    const float2v hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)codes, true);
    return float4v{lo[0], lo[1], hi[0], hi[1]};
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
        for (long o = threadIdx.x * 4; (o & ~255L) < piece.n; o += 1024) {  // whole wavefronts stay or leave
            const long at = piece.first + o, left = piece.n - o;
            float4v p, g, m, v;
            {
                const Vec<P, 4> pv = load_some<4>(param + o, left);
                const Vec<G, 4> gv = load_some<4>(grad + o, left);
                if (BITS == 32) {
                    m = *reinterpret_cast<const float4v *>(static_cast<const float *>(a.m) + at);
                    v = *reinterpret_cast<const float4v *>(static_cast<const float *>(a.v) + at);
                } else {
                    const unsigned mc = static_cast<const unsigned *>(a.m)[at >> 2];
                    const unsigned vc = static_cast<const unsigned *>(a.v)[at >> 2];
                    m = decode8(mc) * a.m_scale[at >> 8];
                    v = decode8(vc) * a.v_scale[at >> 8];
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    p[i] = (float)pv[i];
                    g[i] = (float)gv[i] * a.grad_scale;
                }
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                m[i] = m[i] * a.keep1 + g[i] * a.take1;
                v[i] = v[i] * a.keep2 + g[i] * g[i] * a.take2;
                const float d = sqrtf(v[i]) * now.inv_root2 + a.eps;
                p[i] = p[i] * a.decay - m[i] / d * step;
            }
            Vec<P, 4> out;
#pragma unroll
            for (int i = 0; i < 4; ++i) out[i] = (P)p[i];
            store_some<4>(param + o, out, left);
            if (BITS == 32) {
                *reinterpret_cast<float4v *>(static_cast<float *>(a.m) + at) = m;
                *reinterpret_cast<float4v *>(static_cast<float *>(a.v) + at) = v;
            } else {
                float mi, vi;
                const float ms = scale8(wave_max(max_nan(max_nan(fabsf(m[0]), fabsf(m[1])), max_nan(fabsf(m[2]), fabsf(m[3])))), mi);
                const float vs = scale8(wave_max(max_nan(max_nan(v[0], v[1]), max_nan(v[2], v[3]))), vi);
                unsigned mc = 0, vc = 0;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    unsigned r, q;
                    random_pair(at + i, now.key, r, q);
                    const unsigned c = round8(fabsf(m[i]), mi, r) | (m[i] < 0.0f ? 0x80u : 0u);
                    unsigned w = round8(v[i], vi, q);
                    w = w == 0 && v[i] > 0.0f && vi > 0.0f ? 1u : w;
                    mc |= c << (8 * i);
                    vc |= w << (8 * i);
                }
                static_cast<unsigned *>(a.m)[at >> 2] = mc;
                static_cast<unsigned *>(a.v)[at >> 2] = vc;
                if ((threadIdx.x & 63) == 0) {
                    a.m_scale[at >> 8] = ms;
                    a.v_scale[at >> 8] = vs;
                }
            }
        }
    }
    // Every wavefront of this workgroup has read the clock; the last workgroup of all moves it on, so a step replayed
    // from a graph is the next step.
    __syncthreads();
    if (threadIdx.x == 0 &&
        __hip_atomic_fetch_add(&a.clock->done, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == gridDim.x - 1)
        *a.clock = clock_at(now.t + 1, a.beta1, a.beta2, a.seed);
}

hipError_t launch_adamw_set_clock(const AdamwArgs &a, long t, hipStream_t s)
{
    FBFC_LAUNCH(adamw_set_clock_kernel, dim3(1), dim3(1), 0, s, a.clock, t, a.beta1, a.beta2, a.seed);
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
