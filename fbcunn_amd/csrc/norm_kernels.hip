// The norms before and after a block, fused with its gate and its residual scale (gfx950).
//
//   i1 = 1 / sqrt(mean branch^2 + eps)          u  = branch i1 post scale
//   r' = residual + sigmoid(gate) u             i2 = 1 / sqrt(mean r'^2 + eps)          n = r' i2 pre
//
// and its gradients, with w = gn pre, k = sigmoid(gate), yn = branch i1, rn = r' i2:
//
//   g  = gr + i2 (w - rn mean(w rn))                   gradient of the residual and of r'
//   gpre = sum gn rn      q = sum g k yn               gpost = q scale, gscale = q post
//   gbranch = i1 (g k post scale - yn mean(g k post scale yn))          ggate = g u k (1 - k)
//
// Everything in a row is in 32 bits and rounded once where it is stored; n is the norm of r' before that rounding, and
// the backward pass computes r' again from its inputs (it would have to read r' otherwise, as many bytes).
//
// Bound by memory: a forward pass reads three rows and writes two, a backward pass reads five and writes three.  A row of
// up to 8192 channels stays in registers from its first load to its last store, with all its loads issued before the first sum.
// Longer ones take a workgroup of more than 512 threads, whose 128 registers do not hold it: forward in 32 bits, and backward in
// every type, part of it goes through scratch memory (4096 rows of 12288 channels: forward 101 us in bf16, 472 us (2.1 TB/s) in
// 32 bits; backward 644 us (1.3 TB/s) in bf16, 1033 us in 32 bits; of 8192 channels 67, 129, 149 and 227 us).  Rows of up
// to 1024 channels take 8 to 64 lanes, and longer ones a workgroup, whose wavefronts exchange their sums through
// the LDS with one barrier a sum.  The workgroups walk over the rows, so that the weights and the sums of the weights'
// gradients stay in registers too; these are then added over the workgroups in a fixed order by a second kernel.
//
// Measured: 8192 rows of 2048 channels in bf16 forward 35.9 us (4.67 TB/s; a copy of that size reaches 5.5); 65536 rows of
// 4096 in bf16 backward 871 us (4.93 TB/s, what a large copy reaches); 3001 rows of 1000 in 32 bits backward 25 us and 4.7 us
// for the sums of the weights' gradients.
#include <hip/hip_runtime.h>

#include "column_sums.h"
#include "kernels.h"
#include "lanes.h"
#include "training.h"

namespace fbfc {

// "Lanes of a row" of the kernels in which a row takes the whole workgroup: of up to 512 threads, which may have 256
// registers each, or of up to 1024 with 128 (rows of more than 8192 channels).
constexpr int kWide = 0, kWidest = -1;
constexpr int kMaxWaves = 16;

template <typename T>
constexpr int kVec = 16 / (int)sizeof(T);

// Sum over the lanes of a row.  `slot`: kMaxWaves floats of LDS for this sum alone; the barrier of the next sum (of
// another slot) stands between this one's reads and its next writes.
constexpr bool whole_group(int lanes) { return lanes <= 0; }
constexpr int most_threads(int lanes) { return lanes > 0 ? 256 : lanes == kWide ? 512 : 1024; }

template <int L>
__device__ __forceinline__ float row_sum(float v, float *slot)
{
    if constexpr (!whole_group(L)) return lanes_sum<L>(v);
    v = lanes_sum<64>(v);
    if ((threadIdx.x & 63) == 0) slot[threadIdx.x >> 6] = v;
    __syncthreads();
    float sum = 0.0f;
    for (int i = 0; i < (int)blockDim.x >> 6; ++i) sum += slot[i];
    return sum;
}

template <int L>
struct RowWalk {
    int lane, lanes;
    long row, step;
    __device__ RowWalk()
    {
        lanes = whole_group(L) ? (int)blockDim.x : L;
        const int per = whole_group(L) ? 1 : 256 / (whole_group(L) ? 1 : L);
        lane = whole_group(L) ? (int)threadIdx.x : (int)threadIdx.x % lanes;
        row = (long)blockIdx.x * per + (whole_group(L) ? 0 : (int)threadIdx.x / lanes);
        step = (long)gridDim.x * per;
    }
};

template <typename T, int E>
__device__ __forceinline__ void load_row(Vec<T, kVec<T>> (&v)[E], const Rows &t, long row, const int (&c)[E], int channels)
{
    const T *p = static_cast<const T *>(t.data) + row * t.stride;
#pragma unroll
    for (int e = 0; e < E; ++e) v[e] = load_in_row<T>(p, c[e], channels);
}

// The weights of this lane's channels: post scale, and pre; zero behind the last channel.
template <int V, int E>
__device__ __forceinline__ void load_weights(const NormArgs &a, bool branch, bool normed, const int (&c)[E], float (&post)[E * V], float (&pre)[E * V])
{
#pragma unroll
    for (int e = 0; e < E; ++e)
#pragma unroll
        for (int i = 0; i < V; i += 4) {
            const int at = c[e] + i;
            Vec<float, 4> p = {}, s = {}, q = {};
            if (branch) {
                p = load_some<4>(a.post + at, a.channels - at);
                s = load_some<4>(a.scale + at, a.channels - at);
            }
            if (normed) q = load_some<4>(a.pre + at, a.channels - at);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                post[e * V + i + j] = p[j] * s[j];
                pre[e * V + i + j] = q[j];
            }
        }
}

// Whether vector e of any lane of the wavefront passes the end of the rows.
template <int V, int E>
__device__ __forceinline__ unsigned ends_of(const int (&c)[E], int channels)
{
    unsigned ends = 0;
#pragma unroll
    for (int e = 0; e < E; ++e) ends |= __any(c[e] + V > channels) ? 1u << e : 0u;
    return ends;
}
template <typename T, int E>
__device__ __forceinline__ void end_row(Vec<T, kVec<T>> (&v)[E], unsigned ends, const int (&c)[E], int channels)
{
#pragma unroll
    for (int e = 0; e < E; ++e)
        if (ends >> e & 1) end_of_row<T>(v[e], c[e], channels);
}

template <typename T, int E>
struct ForwardRow {
    Vec<T, kVec<T>> r[E], y[E], z[E];
    __device__ __forceinline__ void load(const NormArgs &a, long row, const int (&c)[E])
    {
        load_row<T, E>(r, a.residual, row, c, a.channels);
        if (a.branch.data != nullptr) load_row<T, E>(y, a.branch, row, c, a.channels);
        if (a.gate.data != nullptr) load_row<T, E>(z, a.gate, row, c, a.channels);
    }
    __device__ __forceinline__ void end(unsigned ends, const int (&c)[E], int channels)
    {
        if (ends == 0) return;
        end_row<T, E>(r, ends, c, channels);
        end_row<T, E>(y, ends, c, channels);
        end_row<T, E>(z, ends, c, channels);
    }
};

template <typename T, int L, int E>
__global__ __launch_bounds__(most_threads(L)) void norm_forward_kernel(NormArgs a)
{
    constexpr int V = kVec<T>;
    __shared__ float slot[2][kMaxWaves];
    const RowWalk<L> walk;
    const bool branch = a.branch.data != nullptr, gated = a.gate.data != nullptr, normed = a.normed.data != nullptr;
    int c[E];
    float post[E * V], pre[E * V];
#pragma unroll
    for (int e = 0; e < E; ++e) c[e] = (walk.lane + e * walk.lanes) * V;
    const float share = 1.0f / (float)a.channels;
    const unsigned ends = ends_of<V, E>(c, a.channels);
    ForwardRow<T, E> in = {}, next = {};
    if (walk.row < a.rows) next.load(a, walk.row, c);
    load_weights<V, E>(a, branch, normed, c, post, pre);
    for (long row = walk.row; row < a.rows; row += walk.step) {
        in = next;
        if (row + walk.step < a.rows) next.load(a, row + walk.step, c);  // while this row is worked on
        in.end(ends, c, a.channels);
        const auto &rv = in.r, &yv = in.y, &zv = in.z;
        float r[E * V];
        if (branch) {
            float sum = 0.0f;
#pragma unroll
            for (int j = 0; j < E * V; ++j) sum += (float)yv[j / V][j % V] * (float)yv[j / V][j % V];
            const float i1 = rsqrtf(row_sum<L>(sum, slot[0]) * share + a.eps);
#pragma unroll
            for (int j = 0; j < E * V; ++j) {
                float u = (float)yv[j / V][j % V] * i1 * post[j];
                if (gated) {
                    float k, no;
                    sigmoid_pair((float)zv[j / V][j % V], k, no);
                    u *= k;
                }
                r[j] = (float)rv[j / V][j % V] + u;
            }
            T *out = static_cast<T *>(a.output.data) + row * a.output.stride;
#pragma unroll
            for (int e = 0; e < E; ++e) {
                Vec<T, V> o;
#pragma unroll
                for (int i = 0; i < V; ++i) o[i] = (T)r[e * V + i];
                if (c[e] < a.channels) store_some<V>(out + c[e], o, a.channels - c[e]);
            }
        } else {
#pragma unroll
            for (int j = 0; j < E * V; ++j) r[j] = (float)rv[j / V][j % V];
        }
        if (normed) {
            float sum = 0.0f;
#pragma unroll
            for (int j = 0; j < E * V; ++j) sum += r[j] * r[j];  // values behind the last channel are zero
            const float i2 = rsqrtf(row_sum<L>(sum, slot[1]) * share + a.eps);
            T *out = static_cast<T *>(a.normed.data) + row * a.normed.stride;
#pragma unroll
            for (int e = 0; e < E; ++e) {
                Vec<T, V> o;
#pragma unroll
                for (int i = 0; i < V; ++i) o[i] = (T)(r[e * V + i] * i2 * pre[e * V + i]);
                if (c[e] < a.channels) store_some<V>(out + c[e], o, a.channels - c[e]);
            }
        }
        if (whole_group(L) && !(branch && normed)) __syncthreads();  // one sum a row: nothing else parts its slot's uses
    }
}

template <typename T, int L, int E>
__global__ __launch_bounds__(most_threads(L)) void norm_backward_kernel(NormArgs a)
{
    constexpr int V = kVec<T>, N = E * V;
    __shared__ float slot[4][kMaxWaves];
    const RowWalk<L> walk;
    const bool branch = a.branch.data != nullptr, gated = a.gate.data != nullptr, normed = a.grad_normed.data != nullptr;
    // with 128 registers, which the row itself passes already, the weights are read again for each row, from the caches
    constexpr bool kKeep = L != kWidest;
    int c[E];
    float post[N], pre[N], q[N], s[N];
#pragma unroll
    for (int e = 0; e < E; ++e) c[e] = (walk.lane + e * walk.lanes) * V;
#pragma unroll
    for (int j = 0; j < N; ++j) q[j] = s[j] = 0.0f;
    const unsigned ends = ends_of<V, E>(c, a.channels);
    if (kKeep) load_weights<V, E>(a, branch, normed, c, post, pre);
    const float share = 1.0f / (float)a.channels;
    for (long row = walk.row; row < a.rows; row += walk.step) {
        if (!kKeep) load_weights<V, E>(a, branch, normed, c, post, pre);
        Vec<T, V> rv[E] = {}, yv[E] = {}, zv[E] = {}, gv[E] = {}, nv[E] = {};
        if (normed) {
            load_row<T, E>(rv, a.residual, row, c, a.channels);
            load_row<T, E>(nv, a.grad_normed, row, c, a.channels);
        }
        if (branch) load_row<T, E>(yv, a.branch, row, c, a.channels);
        if (gated) load_row<T, E>(zv, a.gate, row, c, a.channels);
        if (a.grad_output.data != nullptr) load_row<T, E>(gv, a.grad_output, row, c, a.channels);
        if (ends != 0) {
            end_row<T, E>(rv, ends, c, a.channels);
            end_row<T, E>(nv, ends, c, a.channels);
            end_row<T, E>(yv, ends, c, a.channels);
            end_row<T, E>(zv, ends, c, a.channels);
            end_row<T, E>(gv, ends, c, a.channels);
        }
        float i1 = 0.0f, k[N], g[N];
        if (branch) {
            float sum = 0.0f;
#pragma unroll
            for (int j = 0; j < N; ++j) sum += (float)yv[j / V][j % V] * (float)yv[j / V][j % V];
            i1 = rsqrtf(row_sum<L>(sum, slot[0]) * share + a.eps);
        }
#pragma unroll
        for (int j = 0; j < N; ++j) {
            float no;
            k[j] = 1.0f;
            if (gated) sigmoid_pair((float)zv[j / V][j % V], k[j], no);
            g[j] = (float)gv[j / V][j % V];
        }
        if (normed) {
            float sum = 0.0f, dot = 0.0f, r[N];
#pragma unroll
            for (int j = 0; j < N; ++j) {
                r[j] = (float)rv[j / V][j % V];
                if (branch) {
                    const float u = (float)yv[j / V][j % V] * i1 * post[j];
                    r[j] += gated ? k[j] * u : u;
                }
                sum += r[j] * r[j];
                dot += (float)nv[j / V][j % V] * pre[j] * r[j];
            }
            const float i2 = rsqrtf(row_sum<L>(sum, slot[1]) * share + a.eps);
            const float mean = row_sum<L>(dot, slot[2]) * share * i2;
#pragma unroll
            for (int j = 0; j < N; ++j) {
                const float gn = (float)nv[j / V][j % V], rn = r[j] * i2;
                g[j] += i2 * (gn * pre[j] - rn * mean);
                s[j] += gn * rn;
            }
        }
        if (a.grad_residual.data != nullptr) {
            T *out = static_cast<T *>(a.grad_residual.data) + row * a.grad_residual.stride;
#pragma unroll
            for (int e = 0; e < E; ++e) {
                Vec<T, V> o;
#pragma unroll
                for (int i = 0; i < V; ++i) o[i] = (T)g[e * V + i];
                if (c[e] < a.channels) store_some<V>(out + c[e], o, a.channels - c[e]);
            }
        }
        if (branch) {
            float dot = 0.0f;
#pragma unroll
            for (int j = 0; j < N; ++j) {
                const float yn = (float)yv[j / V][j % V] * i1, gk = g[j] * k[j];
                q[j] += gk * yn;
                dot += gk * post[j] * yn;
            }
            const float mean = row_sum<L>(dot, slot[3]) * share;
            if (a.grad_branch.data != nullptr) {
                T *out = static_cast<T *>(a.grad_branch.data) + row * a.grad_branch.stride;
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    Vec<T, V> o;
#pragma unroll
                    for (int i = 0; i < V; ++i) {
                        const int j = e * V + i;
                        const float yn = (float)yv[e][i] * i1;
                        o[i] = (T)(i1 * (g[j] * k[j] * post[j] - yn * mean));
                    }
                    if (c[e] < a.channels) store_some<V>(out + c[e], o, a.channels - c[e]);
                }
            }
            if (gated && a.grad_gate.data != nullptr) {
                T *out = static_cast<T *>(a.grad_gate.data) + row * a.grad_gate.stride;
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    Vec<T, V> o;
#pragma unroll
                    for (int i = 0; i < V; ++i) {
                        const int j = e * V + i;
                        float yes, no;  // again: cheaper than registers that hold 1 - k over the sums
                        sigmoid_pair((float)zv[e][i], yes, no);
                        o[i] = (T)(g[j] * ((float)yv[e][i] * i1 * post[j]) * yes * no);
                    }
                    if (c[e] < a.channels) store_some<V>(out + c[e], o, a.channels - c[e]);
                }
            }
        }
    }
    if (a.partial == nullptr) return;
    // The sums of this workgroup: q, then s, each one row of `channels`; narrow rows are first added over the rows
    // that the workgroup works on side by side.
    float *mine = a.partial + (long)blockIdx.x * 2 * a.channels;
    if constexpr (whole_group(L)) {
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const int at = c[j / V] + j % V;
            if (at < a.channels) {
                mine[at] = q[j];
                mine[a.channels + at] = s[j];
            }
        }
    } else {
        constexpr int per = 256 / L;
        __shared__ float both[2][256];
#pragma unroll
        for (int j = 0; j < N; ++j) {
            both[0][threadIdx.x] = q[j];
            both[1][threadIdx.x] = s[j];
            __syncthreads();
            const int at = c[j / V] + j % V;
            if (threadIdx.x < L && at < a.channels) {
                float x = 0.0f, y = 0.0f;
                for (int i = 0; i < per; ++i) {
                    x += both[0][threadIdx.x + i * L];
                    y += both[1][threadIdx.x + i * L];
                }
                mine[at] = x;
                mine[a.channels + at] = y;
            }
            __syncthreads();
        }
    }
}

// Adds the workgroups' sums.
__global__ __launch_bounds__(kSumThreads) void norm_weights_kernel(NormArgs a, int groups)
{
    __shared__ float part[2][kSumSlices][kSumColumns];
    const int at = blockIdx.x * kSumColumns + threadIdx.x % kSumColumns, slice = threadIdx.x / kSumColumns;
    float q = 0.0f, s = 0.0f;
    if (at < a.channels) {
        q = slice_sum(a.partial + at, 2L * a.channels, groups, slice);
        s = slice_sum(a.partial + a.channels + at, 2L * a.channels, groups, slice);
    }
    q = slices_sum(q, part[0]);
    s = slices_sum(s, part[1]);
    if (threadIdx.x >= kSumColumns || at >= a.channels) return;
    if (a.grad_post != nullptr) a.grad_post[at] = q * a.scale[at] * a.factor;
    if (a.grad_scale != nullptr) a.grad_scale[at] = q * a.post[at] * a.factor;
    if (a.grad_pre != nullptr) a.grad_pre[at] = s * a.factor;
}

// How a row is laid over lanes: 8 to 64 of them (several rows a workgroup of 256), or the whole workgroup (`wide`), each
// with `vectors` of 16 bytes.
struct RowShape {
    int lanes, vectors, threads;
    bool wide;
    long groups;
};

static RowShape row_shape(long rows, int channels, int type, bool backward)
{
    const int vec = type == kF32 ? 4 : 8;
    const int need = (channels + vec - 1) / vec;
    RowShape r;
    r.vectors = 1;
    // few rows: 16 bytes a lane, the shortest way through a row; many: up to 16 values a lane, and no barriers up to 1024 channels
    const bool few = rows < 512;
    r.wide = need > (few ? 64 : 1024 / vec);
    if (!r.wide) {
        r.lanes = need <= 8 ? 8 : need <= 16 ? 16 : need <= 32 ? 32 : 64;
        r.vectors = need <= 64 ? 1 : 16 / vec;
        r.threads = 256;
    } else {
        r.vectors = few && need <= 1024 ? 1 : 16 / vec;
        r.lanes = ((need + r.vectors - 1) / r.vectors + 63) / 64 * 64;
        r.threads = r.lanes;
    }
    const int side = r.wide ? 1 : 256 / r.lanes;
    const long blocks = (rows + side - 1) / side;
    // Workgroups: 1024 threads on each of 256 CUs, backward, with twice the registers, 512.  (3001 rows of 1000 channels
    // in 32 bits, backward: 512 workgroups 30.7 us, as few as share the rows evenly, 376, 35.6 us, 751 37.7 us.)
    const int held = (backward ? 512 : 1024) / r.threads;
    const long most = 256L * (held > 0 ? held : 1);
    r.groups = blocks < most ? blocks : most;
    return r;
}

size_t norm_workspace_bytes(long rows, int channels, int type)
{
    if (rows < 1) return 0;
    return (size_t)row_shape(rows, channels, type, true).groups * 2 * channels * sizeof(float);
}

template <typename T>
static hipError_t forward_typed(const NormArgs &a, const RowShape &r, hipStream_t s)
{
    constexpr int V = kVec<T>;
    const dim3 grid((unsigned)r.groups), block(r.threads);
    kernel_log_add(r.wide ? "norm_forward_kernel<wide>" : "norm_forward_kernel", r.groups * r.threads);
    if (r.wide) {
        if (r.vectors == 1) FBFC_LAUNCH((norm_forward_kernel<T, kWidest, 1>), grid, block, 0, s, a);
        else if (r.threads <= 512) FBFC_LAUNCH((norm_forward_kernel<T, kWide, 16 / V>), grid, block, 0, s, a);
        else FBFC_LAUNCH((norm_forward_kernel<T, kWidest, 16 / V>), grid, block, 0, s, a);
    } else if (r.lanes == 8) FBFC_LAUNCH((norm_forward_kernel<T, 8, 1>), grid, block, 0, s, a);
    else if (r.lanes == 16) FBFC_LAUNCH((norm_forward_kernel<T, 16, 1>), grid, block, 0, s, a);
    else if (r.lanes == 32) FBFC_LAUNCH((norm_forward_kernel<T, 32, 1>), grid, block, 0, s, a);
    else if (r.vectors == 1) FBFC_LAUNCH((norm_forward_kernel<T, 64, 1>), grid, block, 0, s, a);
    else FBFC_LAUNCH((norm_forward_kernel<T, 64, 16 / V>), grid, block, 0, s, a);
    return hipGetLastError();
}

template <typename T>
static hipError_t backward_typed(const NormArgs &a, const RowShape &r, hipStream_t s)
{
    constexpr int V = kVec<T>;
    const dim3 grid((unsigned)r.groups), block(r.threads);
    kernel_log_add(r.wide ? "norm_backward_kernel<wide>" : "norm_backward_kernel", r.groups * r.threads);
    if (r.wide) {
        if (r.vectors == 1) FBFC_LAUNCH((norm_backward_kernel<T, kWidest, 1>), grid, block, 0, s, a);
        else if (r.threads <= 512) FBFC_LAUNCH((norm_backward_kernel<T, kWide, 16 / V>), grid, block, 0, s, a);
        else FBFC_LAUNCH((norm_backward_kernel<T, kWidest, 16 / V>), grid, block, 0, s, a);
    } else if (r.lanes == 8) FBFC_LAUNCH((norm_backward_kernel<T, 8, 1>), grid, block, 0, s, a);
    else if (r.lanes == 16) FBFC_LAUNCH((norm_backward_kernel<T, 16, 1>), grid, block, 0, s, a);
    else if (r.lanes == 32) FBFC_LAUNCH((norm_backward_kernel<T, 32, 1>), grid, block, 0, s, a);
    else if (r.vectors == 1) FBFC_LAUNCH((norm_backward_kernel<T, 64, 1>), grid, block, 0, s, a);
    else FBFC_LAUNCH((norm_backward_kernel<T, 64, 16 / V>), grid, block, 0, s, a);
    return hipGetLastError();
}

hipError_t launch_norm_forward(int type, const NormArgs &a, hipStream_t s)
{
    if (a.rows < 1) return hipSuccess;
    const RowShape r = row_shape(a.rows, a.channels, type, false);
    return type == kF32 ? forward_typed<float>(a, r, s) : type == kBF16 ? forward_typed<bf16>(a, r, s) : forward_typed<f16>(a, r, s);
}

hipError_t launch_norm_backward(int type, const NormArgs &a, hipStream_t s)
{
    RowShape r = {};
    if (a.rows > 0) {
        r = row_shape(a.rows, a.channels, type, true);
        const hipError_t e = type == kF32 ? backward_typed<float>(a, r, s)
                             : type == kBF16 ? backward_typed<bf16>(a, r, s) : backward_typed<f16>(a, r, s);
        if (e != hipSuccess) return e;
    }
    if (a.grad_post == nullptr && a.grad_scale == nullptr && a.grad_pre == nullptr) return hipSuccess;
    const int blocks = (a.channels + kSumColumns - 1) / kSumColumns;
    kernel_log_add("norm_weights_kernel", (long)blocks * kSumThreads);
    FBFC_LAUNCH(norm_weights_kernel, dim3(blocks), dim3(kSumThreads), 0, s, a, (int)r.groups);
    return hipGetLastError();
}

}  // namespace fbfc
