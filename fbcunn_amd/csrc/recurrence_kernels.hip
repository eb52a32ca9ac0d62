// The gated linear recurrence (gfx950): for every sequence and channel
//
//   a_t = sigmoid(gate_t + bias)        h_t = a_t h_{t-1} + (1 - a_t) x_t        y_t = h_t
//
// and its gradients, with u_t = gy_t + a_{t+1} u_{t+1} and behind the last step the gradient of its state:
//
//   gx_t = (1 - a_t) u_t     ggate_t = u_t (h_{t-1} - x_t) a_t (1 - a_t)     gbias = sum ggate     gstate = a_1 u_1
//
// Bound by memory: forward reads two tensors and writes one, backward reads three and writes two, if each is touched
// once.  A run of steps maps a state h to A h + S, and two runs after each other to (A2 A1, A2 S1 + S2), so the
// steps can be worked on side by side: a wavefront holds 16 steps of 64 lanes' channels in registers, a workgroup
// of up to 8 wavefronts a tile of 128 steps, whose runs it joins through the LDS.  Then either one workgroup walks over the
// tiles of its channels (where there are enough channels to fill the GPU), or every tile is a workgroup of its own and
// the state goes from tile to tile through memory: a tile announces its (A, S) as soon as it has them, looks back for
// the nearest state announced by a tile before it, and applies the (A, S) of those in between, in their order, so that the
// result does not depend on how far it had to look.  Tiles are given out by a counter in the order in which they
// depend on each other, so every tile that is waited for has begun, and it announces (A, S) without waiting.
//
// Backward does the same from the last tile to the first; the states h inside a tile come from the state before it, which
// the forward pass leaves in `checkpoints` (4 bytes for 128 steps), so y is neither read nor relied on to have 32 bits.
#include <hip/hip_runtime.h>

#include "kernels.h"
#include "training.h"

namespace fbfc {

constexpr int kRun = 16;      // steps of a wavefront
constexpr int kWaves = 8;     // wavefronts of a workgroup, at most
constexpr int kLanes = 64;

// Announcements.  A word is announced once it differs from what the workspace is filled with, all ones (a NaN that
// announce() never writes), so value and flag arrive together and no fence is needed.
typedef unsigned long long word64;
constexpr unsigned kUnset = 0xFFFFFFFFu;
constexpr word64 kUnset2 = ~0ull;

__device__ __forceinline__ unsigned announced(float v) { return v != v ? 0x7FC00000u : __float_as_uint(v); }

struct Chain {
    unsigned *ticket;   // of the next tile to be given out, less one
    word64 *runs;       // (A, S) of each tile and channel
    unsigned *states;   // the state behind each tile
};

struct Shape {
    int waves, blocks;  // wavefronts of a workgroup, workgroups beside each other over the channels of a sequence
    long tiles;         // after each other
    long cols;          // batch * blocks
    bool chain;
};

__host__ __device__ __forceinline__ Shape shape_of(int batch, int channels, long steps, int v)
{
    Shape s;
    const long runs = (steps + kRun - 1) / kRun;
    s.waves = runs < kWaves ? (int)runs : kWaves;
    if (s.waves < 1) s.waves = 1;
    s.blocks = (channels + kLanes * v - 1) / (kLanes * v);
    s.tiles = (runs + s.waves - 1) / s.waves;
    s.cols = (long)batch * s.blocks;
    // 512 workgroups fill the GPU by themselves; fewer leave CUs idle, and their tiles are then spread
    s.chain = s.tiles > 1 && s.cols < 512;
    return s;
}

__device__ __forceinline__ Chain chain_of(unsigned char *workspace, const Shape &s, int v)
{
    Chain c;
    c.ticket = reinterpret_cast<unsigned *>(workspace);
    c.runs = reinterpret_cast<word64 *>(workspace + 256);
    c.states = reinterpret_cast<unsigned *>(c.runs + s.tiles * s.cols * kLanes * v);
    return c;
}
static size_t chain_bytes(const Shape &s, int v) { return 256 + (size_t)s.tiles * s.cols * kLanes * v * 12; }

__global__ __launch_bounds__(256) void recurrence_clear_kernel(uint4 *p, long n)
{
    for (long i = blockIdx.x * 256L + threadIdx.x; i < n; i += gridDim.x * 256L) p[i] = uint4{kUnset, kUnset, kUnset, kUnset};
}

// The state in front of tile `at` of column `col`, of this lane's channels; `dir` is where the tile before it lies.
template <int V>
__device__ __forceinline__ void look_back(const Chain &ch, const Shape &s, long at, long col, int dir, int lane, float (&h)[V])
{
    const long cell = kLanes * V;
    long j = at + dir;
    while (true) {
        bool state = true, run = true;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const long k = (j * s.cols + col) * cell + lane * V + i;
            const unsigned p = __hip_atomic_load(ch.states + k, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            const word64 r = __hip_atomic_load(ch.runs + k, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            h[i] = __uint_as_float(p);
            state &= p != kUnset;
            run &= r != kUnset2;
        }
        if (__all(state)) break;
        if (__all(run)) j += dir;  // the first tile announces no run, so the search ends there
        else __builtin_amdgcn_s_sleep(1);
    }
    for (j -= dir; j != at; j -= dir) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const word64 r = __hip_atomic_load(ch.runs + (j * s.cols + col) * cell + lane * V + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            h[i] = fmaf(__uint_as_float((unsigned)r), h[i], __uint_as_float((unsigned)(r >> 32)));
        }
    }
}

template <int V>
__device__ __forceinline__ void announce_run(const Chain &ch, const Shape &s, long at, long col, int lane, const float (&A)[V], const float (&S)[V])
{
#pragma unroll
    for (int i = 0; i < V; ++i)
        __hip_atomic_store(ch.runs + (at * s.cols + col) * (kLanes * V) + lane * V + i,
                           (word64)announced(S[i]) << 32 | announced(A[i]), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
template <int V>
__device__ __forceinline__ void announce_state(const Chain &ch, const Shape &s, long at, long col, int lane, const float (&h)[V])
{
#pragma unroll
    for (int i = 0; i < V; ++i)
        __hip_atomic_store(ch.states + (at * s.cols + col) * (kLanes * V) + lane * V + i, announced(h[i]), __ATOMIC_RELAXED,
                           __HIP_MEMORY_SCOPE_AGENT);
}

// V channels of this lane in one row of a tensor.  The address is moved back where the row ends inside or before it, and
// the values are moved to their places, so that no load has a condition.
template <typename T, int V>
struct LaneRow {
    const T *base;
    long st, off;
    int shift;
    __device__ LaneRow(const Steps &t, int b, int c, int channels)
    {
        base = static_cast<const T *>(t.data) + (long)b * t.sb;
        st = t.st;
        const int first = c + V <= channels ? c : channels - V;
        shift = c - first;
        off = (long)first * t.sc;
    }
    __device__ __forceinline__ Vec<T, V> load(long step) const { return load_vec<V>(base + step * st + off); }
    __device__ __forceinline__ float value(const Vec<T, V> &v, int i) const
    {
        if (V == 1) return (float)v[0];
        return (float)(i == 0 && shift == 1 ? v[1] : v[i]);
    }
};
template <typename T, int V>
__device__ __forceinline__ void store_lane(const Steps &t, int b, long step, int c, int channels, const float (&x)[V])
{
    T *p = static_cast<T *>(t.data) + (long)b * t.sb + step * t.st + (long)c * t.sc;
    Vec<T, V> o;
#pragma unroll
    for (int i = 0; i < V; ++i) o[i] = (T)x[i];
    if (c < channels) store_some<V>(p, o, channels - c);
}

template <typename T, int V>
__global__ __launch_bounds__(kLanes *kWaves) void recurrence_forward_kernel(RecArgs a)
{
    __shared__ float sA[2][kWaves][kLanes * V], sS[2][kWaves][kLanes * V], carried[kLanes * V];
    __shared__ unsigned given;
    const Shape s = shape_of(a.batch, a.channels, a.steps, V);
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const Chain ch = chain_of(a.workspace, s, V);
    long work = blockIdx.x;
    if (s.chain) {
        if (threadIdx.x == 0) given = __hip_atomic_fetch_add(ch.ticket, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) + 1u;
        __syncthreads();
        work = __builtin_amdgcn_readfirstlane(given);
    }
    const long col = work % s.cols;
    const int b = (int)(col / s.blocks), c = (int)(col % s.blocks) * kLanes * V + lane * V;
    const long first = s.chain ? work / s.cols : 0, end = s.chain ? first + 1 : s.tiles;
    long len = a.steps;
    if (a.lengths != nullptr) {
        const long n = a.lengths[b];
        len = n < 0 ? 0 : n < len ? n : len;
    }
    const LaneRow<T, V> xr(a.x, b, c, a.channels), gr(a.gate, b, c, a.channels);
    float bias[V], carry[V];  // carry: wavefront 0, the state before the tile
#pragma unroll
    for (int i = 0; i < V; ++i) {
        bias[i] = a.bias != nullptr && c + i < a.channels ? a.bias[c + i] : 0.0f;
        carry[i] = a.state_in != nullptr && c + i < a.channels ? a.state_in[(long)b * a.channels + c + i] : 0.0f;
    }
    int turn = 0;
    for (long tile = first; tile < end; ++tile, turn ^= 1) {
        const long t0 = (tile * s.waves + w) * kRun;
        float x[kRun][V], k[kRun][V], A[V], S[V];  // k: 1 - a
        if (len > 0) {
            Vec<T, V> xv[kRun], gv[kRun];
#pragma unroll
            for (int t = 0; t < kRun; ++t) {
                const long at = t0 + t < len ? t0 + t : len - 1;
                xv[t] = xr.load(at);
                gv[t] = gr.load(at);
            }
#pragma unroll
            for (int i = 0; i < V; ++i) A[i] = 1.0f, S[i] = 0.0f;
#pragma unroll
            for (int t = 0; t < kRun; ++t) {
                const bool live = t0 + t < len;
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    float keep;
                    sigmoid_pair(gr.value(gv[t], i) + bias[i], keep, k[t][i]);
                    x[t][i] = live ? xr.value(xv[t], i) : 0.0f;
                    k[t][i] = live ? k[t][i] : 0.0f;
                    A[i] *= live ? keep : 1.0f;
                    S[i] = fmaf(k[t][i], x[t][i] - S[i], S[i]);
                }
            }
        } else {
#pragma unroll
            for (int i = 0; i < V; ++i) {
                A[i] = 1.0f, S[i] = 0.0f;
#pragma unroll
                for (int t = 0; t < kRun; ++t) x[t][i] = k[t][i] = 0.0f;
            }
        }
#pragma unroll
        for (int i = 0; i < V; ++i) {
            sA[turn][w][lane * V + i] = A[i];
            sS[turn][w][lane * V + i] = S[i];
        }
        __syncthreads();
        if (w == 0) {
            for (int j = 1; j < s.waves; ++j)
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const float Aj = sA[turn][j][lane * V + i];
                    A[i] *= Aj;
                    S[i] = fmaf(Aj, S[i], sS[turn][j][lane * V + i]);
                }
            if (s.chain && tile > 0) {
                if (tile + 1 < s.tiles) announce_run<V>(ch, s, tile, col, lane, A, S);
                look_back<V>(ch, s, tile, col, -1, lane, carry);
            }
#pragma unroll
            for (int i = 0; i < V; ++i) {
                carried[lane * V + i] = carry[i];
                if (a.checkpoints != nullptr && c + i < a.channels)
                    a.checkpoints[(tile * a.batch + b) * a.channels + c + i] = carry[i];
                carry[i] = fmaf(A[i], carry[i], S[i]);
            }
            if (s.chain && tile + 1 < s.tiles) announce_state<V>(ch, s, tile, col, lane, carry);
        }
        __syncthreads();
        float h[V];
#pragma unroll
        for (int i = 0; i < V; ++i) h[i] = carried[lane * V + i];
        for (int j = 0; j < w; ++j)
#pragma unroll
            for (int i = 0; i < V; ++i) h[i] = fmaf(sA[turn][j][lane * V + i], h[i], sS[turn][j][lane * V + i]);
#pragma unroll
        for (int t = 0; t < kRun; ++t) {
            float out[V];
#pragma unroll
            for (int i = 0; i < V; ++i) {
                h[i] = fmaf(k[t][i], x[t][i] - h[i], h[i]);
                out[i] = t0 + t < len ? h[i] : 0.0f;
            }
            if (t0 + t < a.steps) store_lane<T, V>(a.y, b, t0 + t, c, a.channels, out);
        }
        if (a.state_out != nullptr && tile + 1 == s.tiles && w + 1 == s.waves)
#pragma unroll
            for (int i = 0; i < V; ++i)
                if (c + i < a.channels) a.state_out[(long)b * a.channels + c + i] = h[i];
    }
}

template <typename T, int V>
__global__ __launch_bounds__(kLanes *kWaves) void recurrence_backward_kernel(RecArgs a, float *partial)
{
    __shared__ float sA[2][kWaves][kLanes * V], sS[2][kWaves][kLanes * V], sR[2][kWaves][kLanes * V], carried[kLanes * V];
    __shared__ unsigned given;
    const Shape s = shape_of(a.batch, a.channels, a.steps, V);
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const Chain ch = chain_of(a.workspace, s, V);
    long work = blockIdx.x;
    if (s.chain) {
        if (threadIdx.x == 0) given = __hip_atomic_fetch_add(ch.ticket, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) + 1u;
        __syncthreads();
        work = __builtin_amdgcn_readfirstlane(given);
    }
    const long col = work % s.cols;
    const int b = (int)(col / s.blocks), c = (int)(col % s.blocks) * kLanes * V + lane * V;
    const long first = s.chain ? s.tiles - 1 - work / s.cols : s.tiles - 1, end = s.chain ? first : 0;
    long len = a.steps;
    if (a.lengths != nullptr) {
        const long n = a.lengths[b];
        len = n < 0 ? 0 : n < len ? n : len;
    }
    const LaneRow<T, V> xr(a.x, b, c, a.channels), gr(a.gate, b, c, a.channels), yr(a.y, b, c, a.channels);
    float bias[V], carry[V];  // carry: wavefront 0, a_{t+1} u_{t+1} behind the tile
#pragma unroll
    for (int i = 0; i < V; ++i) {
        bias[i] = a.bias != nullptr && c + i < a.channels ? a.bias[c + i] : 0.0f;
        carry[i] = a.state_in != nullptr && c + i < a.channels ? a.state_in[(long)b * a.channels + c + i] : 0.0f;
    }
    int turn = 0;
    for (long tile = first; tile >= end; --tile, turn ^= 1) {
        const long t0 = (tile * s.waves + w) * kRun;
        float x[kRun][V], k[kRun][V], keep[kRun][V], gy[kRun][V], A[V], S[V], R[V];
        float before[V];
#pragma unroll
        for (int i = 0; i < V; ++i)
            before[i] = c + i < a.channels ? a.checkpoints[(tile * a.batch + b) * a.channels + c + i] : 0.0f;
        if (len > 0) {
            Vec<T, V> xv[kRun], gv[kRun], yv[kRun];
#pragma unroll
            for (int t = 0; t < kRun; ++t) {
                const long at = t0 + t < len ? t0 + t : len - 1;
                xv[t] = xr.load(at);
                gv[t] = gr.load(at);
                yv[t] = yr.load(at);
            }
#pragma unroll
            for (int t = 0; t < kRun; ++t) {
                const bool live = t0 + t < len;
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    sigmoid_pair(gr.value(gv[t], i) + bias[i], keep[t][i], k[t][i]);
                    x[t][i] = live ? xr.value(xv[t], i) : 0.0f;
                    gy[t][i] = live ? yr.value(yv[t], i) : 0.0f;
                    k[t][i] = live ? k[t][i] : 0.0f;
                    keep[t][i] = live ? keep[t][i] : 1.0f;
                }
            }
        } else {
#pragma unroll
            for (int t = 0; t < kRun; ++t)
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    x[t][i] = k[t][i] = gy[t][i] = 0.0f;
                    keep[t][i] = 1.0f;
                }
        }
#pragma unroll
        for (int i = 0; i < V; ++i) {
            A[i] = 1.0f, S[i] = R[i] = 0.0f;
#pragma unroll
            for (int t = 0; t < kRun; ++t) {
                A[i] *= keep[t][i];
                S[i] = fmaf(k[t][i], x[t][i] - S[i], S[i]);
            }
#pragma unroll
            for (int t = kRun - 1; t >= 0; --t) R[i] = keep[t][i] * (gy[t][i] + R[i]);
            sA[turn][w][lane * V + i] = A[i];
            sS[turn][w][lane * V + i] = S[i];
            sR[turn][w][lane * V + i] = R[i];
        }
        __syncthreads();
        if (w == 0) {
            // the whole tile, from its last wavefront to its first
            float At[V], Rt[V];
#pragma unroll
            for (int i = 0; i < V; ++i) {
                At[i] = sA[turn][s.waves - 1][lane * V + i];
                Rt[i] = sR[turn][s.waves - 1][lane * V + i];
            }
            for (int j = s.waves - 2; j >= 0; --j)
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const float Aj = sA[turn][j][lane * V + i];
                    At[i] *= Aj;
                    Rt[i] = fmaf(Aj, Rt[i], sR[turn][j][lane * V + i]);
                }
            if (s.chain && tile + 1 < s.tiles) {
                if (tile > 0) announce_run<V>(ch, s, tile, col, lane, At, Rt);
                look_back<V>(ch, s, tile, col, 1, lane, carry);
            }
#pragma unroll
            for (int i = 0; i < V; ++i) {
                carried[lane * V + i] = carry[i];
                carry[i] = fmaf(At[i], carry[i], Rt[i]);
            }
            if (s.chain && tile > 0) announce_state<V>(ch, s, tile, col, lane, carry);
        }
        __syncthreads();
        float g[V], sum[V], h[kRun][V];  // h: the state before each step
#pragma unroll
        for (int i = 0; i < V; ++i) {
            g[i] = carried[lane * V + i];
            sum[i] = 0.0f;
        }
        for (int j = s.waves - 1; j > w; --j)
#pragma unroll
            for (int i = 0; i < V; ++i) g[i] = fmaf(sA[turn][j][lane * V + i], g[i], sR[turn][j][lane * V + i]);
        for (int j = 0; j < w; ++j)
#pragma unroll
            for (int i = 0; i < V; ++i) before[i] = fmaf(sA[turn][j][lane * V + i], before[i], sS[turn][j][lane * V + i]);
#pragma unroll
        for (int i = 0; i < V; ++i) {
            h[0][i] = before[i];
#pragma unroll
            for (int t = 1; t < kRun; ++t) h[t][i] = fmaf(k[t - 1][i], x[t - 1][i] - h[t - 1][i], h[t - 1][i]);
        }
#pragma unroll
        for (int t = kRun - 1; t >= 0; --t) {
            float gx[V], gz[V];
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const float u = gy[t][i] + g[i];
                gx[i] = k[t][i] * u;
                gz[i] = gx[i] * (h[t][i] - x[t][i]) * keep[t][i];
                sum[i] += gz[i];
                g[i] = keep[t][i] * u;
            }
            if (t0 + t < a.steps) {
                if (a.grad_x.data != nullptr) store_lane<T, V>(a.grad_x, b, t0 + t, c, a.channels, gx);
                if (a.grad_gate.data != nullptr) store_lane<T, V>(a.grad_gate, b, t0 + t, c, a.channels, gz);
            }
        }
        if (a.state_out != nullptr && tile == 0 && w == 0)
#pragma unroll
            for (int i = 0; i < V; ++i)
                if (c + i < a.channels) a.state_out[(long)b * a.channels + c + i] = g[i];
        if (partial != nullptr) {
            // the tile's sum of gate gradients, in the place of the runs that everybody has read after the barrier
            __syncthreads();
#pragma unroll
            for (int i = 0; i < V; ++i) sR[turn][w][lane * V + i] = sum[i];
            __syncthreads();
            if (w == 0)
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    float v = 0.0f;
                    for (int j = 0; j < s.waves; ++j) v += sR[turn][j][lane * V + i];
                    if (c + i < a.channels) partial[(tile * a.batch + b) * a.channels + c + i] = v;
                }
        }
    }
}

// One step, or none: the form of a single token.
template <typename T, int V>
__global__ __launch_bounds__(256) void recurrence_step_kernel(RecArgs a)
{
    const int per = (a.channels + V - 1) / V;
    const long i = blockIdx.x * 256L + threadIdx.x;
    if (i >= (long)a.batch * per) return;
    const int b = (int)(i / per), c = (int)(i % per) * V;
    const bool live = a.steps > 0 && (a.lengths == nullptr || a.lengths[b] > 0);
    const long left = a.channels - c, at = (long)b * a.channels + c;
    Vec<T, V> xv = {}, gv = {};
    if (live) {
        xv = load_some<V>(static_cast<const T *>(a.x.data) + b * a.x.sb + (long)c * a.x.sc, left);
        gv = load_some<V>(static_cast<const T *>(a.gate.data) + b * a.gate.sb + (long)c * a.gate.sc, left);
    }
    Vec<float, V> h = {}, bias = {};
    if (a.state_in != nullptr) h = load_some<V>(a.state_in + at, left);
    if (a.bias != nullptr) bias = load_some<V>(a.bias + c, left);
    Vec<T, V> y;
#pragma unroll
    for (int j = 0; j < V; ++j) {
        float keep, k;
        sigmoid_pair((float)gv[j] + bias[j], keep, k);
        if (live) h[j] = fmaf(k, (float)xv[j] - h[j], h[j]);
        y[j] = (T)(live ? h[j] : 0.0f);
    }
    if (a.checkpoints != nullptr && a.steps > 0) {
        Vec<float, V> h0 = {};
        if (a.state_in != nullptr) h0 = load_some<V>(a.state_in + at, left);
        store_some<V>(a.checkpoints + at, h0, left);
    }
    if (a.steps > 0) store_some<V>(static_cast<T *>(a.y.data) + b * a.y.sb + (long)c * a.y.sc, y, left);
    if (a.state_out != nullptr) store_some<V>(a.state_out + at, h, left);
}

// grad_bias: the sum of `rows` rows of sums, 16 channels and 16 slices of the rows a workgroup, in a fixed order.
__global__ __launch_bounds__(256) void recurrence_bias_kernel(const float *partial, long rows, int channels, float factor, float *out)
{
    __shared__ float part[16][17];
    const int i = threadIdx.x & 15, slice = threadIdx.x >> 4, at = blockIdx.x * 16 + i;
    float sum = 0.0f;
    if (at < channels)
        for (long r = slice; r < rows; r += 16) sum += partial[r * channels + at];
    part[slice][i] = sum;
    __syncthreads();
    if (slice != 0 || at >= channels) return;
    for (int k = 1; k < 16; ++k) sum += part[k][i];
    out[at] = sum * factor;
}

// V: channels of a lane, 2 where the channels of every tensor lie side by side
static int lane_channels(const RecArgs &a)
{
    if (a.channels < 2) return 1;
    for (const Steps *t : {&a.x, &a.gate, &a.y, &a.grad_x, &a.grad_gate})
        if (t->data != nullptr && t->sc != 1) return 1;
    return 2;
}

size_t recurrence_checkpoint_bytes(int batch, int channels, long steps)
{
    return (size_t)shape_of(batch, channels, steps, 1).tiles * batch * channels * sizeof(float);
}

size_t recurrence_workspace_bytes(int batch, int channels, long steps)
{
    size_t most = 0;
    for (int v = 1; v <= 2; ++v) {
        const Shape s = shape_of(batch, channels, steps, v);
        const size_t n = s.chain ? chain_bytes(s, v) : 0;
        most = n > most ? n : most;
    }
    most = (most + 255) / 256 * 256;
    return most + recurrence_checkpoint_bytes(batch, channels, steps);  // the sums of the gate's gradients of each tile
}

bool recurrence_fits(int batch, int channels, long steps)
{
    const Shape s = shape_of(batch, channels, steps, 1);
    return s.tiles < (1L << 31) / s.cols && (long)batch * channels < (1L << 38);
}

static hipError_t clear_chain(const RecArgs &a, const Shape &s, int v, hipStream_t stream)
{
    const long n = (long)((chain_bytes(s, v) + 15) / 16), blocks = (n + 255) / 256;
    const unsigned grid = (unsigned)(blocks < 2048 ? blocks : 2048);
    kernel_log_add("recurrence_clear_kernel", grid * 256L);
    FBFC_LAUNCH(recurrence_clear_kernel, dim3(grid), dim3(256), 0, stream, reinterpret_cast<uint4 *>(a.workspace), n);
    return hipGetLastError();
}

template <typename T>
static hipError_t forward_typed(const RecArgs &a, hipStream_t stream)
{
    const int v = lane_channels(a);
    if (a.steps <= 1) {
        const bool wide = v == 2 && a.channels >= 4;
        const long lanes = (long)a.batch * ((a.channels + (wide ? 3 : 0)) / (wide ? 4 : 1));
        const dim3 grid((unsigned)((lanes + 255) / 256));
        kernel_log_add("recurrence_step_kernel", (long)grid.x * 256);
        if (wide) FBFC_LAUNCH((recurrence_step_kernel<T, 4>), grid, dim3(256), 0, stream, a);
        else FBFC_LAUNCH((recurrence_step_kernel<T, 1>), grid, dim3(256), 0, stream, a);
        return hipGetLastError();
    }
    const Shape s = shape_of(a.batch, a.channels, a.steps, v);
    if (s.chain) {
        const hipError_t e = clear_chain(a, s, v, stream);
        if (e != hipSuccess) return e;
    }
    const dim3 grid((unsigned)(s.chain ? s.tiles * s.cols : s.cols)), block(s.waves * kLanes);
    kernel_log_add(s.chain ? "recurrence_forward_kernel<chain>" : "recurrence_forward_kernel", (long)grid.x * block.x);
    if (v == 2) FBFC_LAUNCH((recurrence_forward_kernel<T, 2>), grid, block, 0, stream, a);
    else FBFC_LAUNCH((recurrence_forward_kernel<T, 1>), grid, block, 0, stream, a);
    return hipGetLastError();
}

template <typename T>
static hipError_t backward_typed(const RecArgs &a, hipStream_t stream)
{
    const int v = lane_channels(a);
    const Shape s = shape_of(a.batch, a.channels, a.steps, v);
    float *partial = nullptr;
    if (a.grad_bias != nullptr)
        partial = reinterpret_cast<float *>(a.workspace + recurrence_workspace_bytes(a.batch, a.channels, a.steps) -
                                            recurrence_checkpoint_bytes(a.batch, a.channels, a.steps));
    if (s.chain) {
        const hipError_t e = clear_chain(a, s, v, stream);
        if (e != hipSuccess) return e;
    }
    const dim3 grid((unsigned)(s.chain ? s.tiles * s.cols : s.cols)), block(s.waves * kLanes);
    kernel_log_add(s.chain ? "recurrence_backward_kernel<chain>" : "recurrence_backward_kernel", (long)grid.x * block.x);
    if (v == 2) FBFC_LAUNCH((recurrence_backward_kernel<T, 2>), grid, block, 0, stream, a, partial);
    else FBFC_LAUNCH((recurrence_backward_kernel<T, 1>), grid, block, 0, stream, a, partial);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || partial == nullptr) return e;
    const int blocks = (a.channels + 15) / 16;
    kernel_log_add("recurrence_bias_kernel", blocks * 256L);
    FBFC_LAUNCH(recurrence_bias_kernel, dim3(blocks), dim3(256), 0, stream, partial, s.tiles * a.batch, a.channels, a.factor, a.grad_bias);
    return hipGetLastError();
}

hipError_t launch_recurrence_forward(int type, const RecArgs &a, hipStream_t s)
{
    return type == kF32 ? forward_typed<float>(a, s) : type == kBF16 ? forward_typed<bf16>(a, s) : forward_typed<f16>(a, s);
}

hipError_t launch_recurrence_backward(int type, const RecArgs &a, hipStream_t s)
{
    if (a.steps < 1 || a.batch < 1) {
        // nothing but the state's gradient, and sums over nothing
        if (a.state_out != nullptr && a.batch > 0) {
            RecArgs step = a;
            step.checkpoints = nullptr;
            step.lengths = nullptr;
            const hipError_t e = launch_recurrence_forward(type, step, s);
            if (e != hipSuccess) return e;
        }
        if (a.grad_bias == nullptr) return hipSuccess;
        kernel_log_add("recurrence_bias_kernel", (a.channels + 15) / 16 * 256L);
        FBFC_LAUNCH(recurrence_bias_kernel, dim3((a.channels + 15) / 16), dim3(256), 0, s, nullptr, 0L, a.channels, a.factor, a.grad_bias);
        return hipGetLastError();
    }
    return type == kF32 ? backward_typed<float>(a, s) : type == kBF16 ? backward_typed<bf16>(a, s) : backward_typed<f16>(a, s);
}

}  // namespace fbfc
