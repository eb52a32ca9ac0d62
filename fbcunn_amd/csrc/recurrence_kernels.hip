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
// tiles of its channels (where there are enough channels to fill the GPU, or two tiles), or every tile is a workgroup of its own and
// the state goes from tile to tile through memory: a tile announces its (A, S) as soon as it has them, looks back for
// the nearest state announced by a tile before it, and applies the (A, S) of those in between, in their order, so that the
// result does not depend on how far it had to look.  Tiles are given out by a counter in the order in which they
// depend on each other, so every tile that is waited for has begun, and it announces (A, S) without waiting.
//
// Backward does the same from the last tile to the first; the states h inside a tile come from the state before it, which
// the forward pass leaves in `checkpoints` (4 bytes for 128 steps), so y is neither read nor relied on to have 32 bits.
//
// Measured: 131072 steps of 2048 channels in bf16, forward 384 us (4.2 TB/s), backward 661 us (4.1 TB/s; a large copy
// reaches 5.0 TB/s); without the walk back the forward pass took 287 us where it takes 372 with it.  8 sequences of 2048 steps x
// 1024 channels in bf16 forward 28 us (3.6 TB/s) and 2 to 4.6 us for clearing: its 1024 workgroups begin in step and read and write by turns.
#include <hip/hip_runtime.h>

#include <type_traits>

#include "column_sums.h"
#include "kernels.h"
#include "training.h"

namespace fbfc {

constexpr int kRun = 16;     // steps of a wavefront
constexpr int kWaves = 8;     // wavefronts of a workgroup, at most
constexpr int kLanes = 64;
// Columns (a sequence's block of channels) from which on one workgroup walks over all tiles of its column: with one on
// each CU, handing the state from tile to tile gains nothing (256 columns of 12 tiles in 32 bits: 60 us walked over, 64
// handed on; 4 tiles 21 and 28).  Below, tiles are worked on side by side where there are enough to make up for clearing the
// announcements: 3 or more (16 columns in 32 bits: 2 tiles 7.4 us walked over and 10.8 handed on, 4 tiles 11.8 and 10.3, 12
// tiles 31 and 10), or, with half of the CUs at work anyway, 5 (128 columns in bf16: 3 tiles 14.9 and 17.5, 4 tiles
// 20.3 and 19.8, 12 tiles 54 and 39).
constexpr int kGroups = 256;
constexpr int kXcds = 8, kCounterLine = 32, kFew = 2048;  // see draw()
constexpr int kHead = kXcds * kCounterLine * (int)sizeof(unsigned);  // bytes of the workspace before the announcements
constexpr float kLog2e = 1.44269504088896340736f;

// Announcements.  A word is announced once it differs from what the workspace is filled with, all ones (a NaN that
// announced() never gives), so value and flag arrive together and no fence is needed.
typedef unsigned long long word64;
constexpr unsigned kUnset = 0xFFFFFFFFu;
constexpr word64 kUnset2 = ~0ull;

__device__ __forceinline__ unsigned announced(float v) { return v != v ? 0x7FC00000u : __float_as_uint(v); }

struct Chain {
    unsigned *tickets;  // of the next tile that each counter gives out, less one
    word64 *runs;       // (A, S) of each tile and channel
    unsigned *states;   // the state behind each tile
};

struct Shape {
    int waves, blocks;  // wavefronts of a workgroup, workgroups beside each other over the channels of a sequence
    int tiles;          // after each other
    int cols;           // batch * blocks
    bool chain;
};

__host__ __device__ __forceinline__ Shape shape_of(int batch, int channels, long steps, int v)
{
    Shape s;
    const long runs = (steps + kRun - 1) / kRun;
    s.waves = runs < kWaves ? (int)runs : kWaves;
    if (s.waves < 1) s.waves = 1;
    s.blocks = (channels + kLanes * v - 1) / (kLanes * v);
    s.tiles = (int)((runs + s.waves - 1) / s.waves);  // recurrence_fits()
    s.cols = batch * s.blocks;
    s.chain = s.cols < kGroups && s.tiles > (s.cols < kGroups / 2 ? 2 : 4);
    return s;
}

__device__ __forceinline__ Chain chain_of(unsigned char *workspace, const Shape &s, int v)
{
    Chain c;
    c.tickets = reinterpret_cast<unsigned *>(workspace);
    c.runs = reinterpret_cast<word64 *>(workspace + kHead);
    c.states = reinterpret_cast<unsigned *>(c.runs + (long)s.tiles * s.cols * kLanes * v);
    return c;
}
static size_t chain_bytes(const Shape &s, int v) { return kHead + (size_t)s.tiles * s.cols * kLanes * v * 12; }

__global__ __launch_bounds__(256) void recurrence_clear_kernel(uint4 *p, long n)
{
    for (long i = blockIdx.x * 256L + threadIdx.x; i < n; i += gridDim.x * 256L) p[i] = uint4{kUnset, kUnset, kUnset, kUnset};
}

template <int V>
__device__ __forceinline__ void fold(float (&h)[V], const word64 (&run)[V])
{
#pragma unroll
    for (int i = 0; i < V; ++i) h[i] = fmaf(__uint_as_float((unsigned)run[i]), h[i], __uint_as_float((unsigned)(run[i] >> 32)));
}

// The state in front of tile `at` of column `col`, of this lane's channels; `dir` is where the tile before it lies.  Four
// tiles are asked at once, since an answer takes about a microsecond (8 sequences of 2048 steps x 1024 channels in bf16 forward:
// one at a time 33.5 us, two 33.8, four 30.9).
constexpr int kAsk = 4;
template <int V>
__device__ __forceinline__ void look_back(const Chain &ch, const Shape &s, int at, int col, int dir, int lane, float (&h)[V])
{
    const long cell = (long)kLanes * V, row = (long)s.cols * cell;
    const unsigned *states = ch.states + col * cell;
    const word64 *runs = ch.runs + col * cell;
    const unsigned own = lane * V;
    int j = at + dir;  // the nearest of the tiles that are asked
    while (true) {
        unsigned state[kAsk][V];
        word64 run[kAsk][V];
#pragma unroll
        for (int q = 0; q < kAsk; ++q) {
            int k = j + dir * q;
            k = k < 0 ? 0 : k < s.tiles ? k : s.tiles - 1;
#pragma unroll
            for (int i = 0; i < V; ++i) {
                state[q][i] = __hip_atomic_load(states + k * row + (own + i), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                run[q][i] = __hip_atomic_load(runs + k * row + (own + i), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            }
        }
        int hit = -1, known = 0;  // the tile whose state is announced; how many before it have announced their runs
#pragma unroll
        for (int q = 0; q < kAsk; ++q) {
            bool has_state = true, has_run = true;
#pragma unroll
            for (int i = 0; i < V; ++i) {
                has_state &= state[q][i] != kUnset;
                has_run &= run[q][i] != kUnset2;
            }
            if (hit < 0 && known == q) {
                if (__all(has_state)) {
                    hit = q;
#pragma unroll
                    for (int i = 0; i < V; ++i) h[i] = __uint_as_float(state[q][i]);
                } else if (__all(has_run)) {
                    ++known;  // never the first tile, which announces no run: the walk ends there
                }
            }
        }
        if (hit >= 0) {
#pragma unroll
            for (int q = kAsk - 1; q >= 0; --q)
                if (q < hit) fold<V>(h, run[q]);
            break;
        }
        if (known == kAsk) j += dir * kAsk;
        else __builtin_amdgcn_s_sleep(1);
    }
    // the tiles that earlier rounds passed over
    for (j -= dir; j != at; j -= dir) {
        word64 run[V];
#pragma unroll
        for (int i = 0; i < V; ++i) run[i] = __hip_atomic_load(runs + j * row + (own + i), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        fold<V>(h, run);
    }
}

template <int V>
__device__ __forceinline__ void announce_run(const Chain &ch, const Shape &s, int at, int col, int lane, const float (&A)[V], const float (&S)[V])
{
#pragma unroll
    for (int i = 0; i < V; ++i)
        __hip_atomic_store(ch.runs + (long)(at * s.cols + col) * (kLanes * V) + lane * V + i,
                           (word64)announced(S[i]) << 32 | announced(A[i]), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
template <int V>
__device__ __forceinline__ void announce_state(const Chain &ch, const Shape &s, int at, int col, int lane, const float (&h)[V])
{
#pragma unroll
    for (int i = 0; i < V; ++i)
        __hip_atomic_store(ch.states + (long)(at * s.cols + col) * (kLanes * V) + lane * V + i, announced(h[i]), __ATOMIC_RELAXED,
                           __HIP_MEMORY_SCOPE_AGENT);
}

// A tensor's rows as a lane reads and writes them: V channels from c on.  Where the last block of channels ends inside
// or before a lane, its loads are moved back to end with the row, so that no load has a condition, and an odd last channel
// is then moved to its place.  Orders of memory: kDense, channels side by side, with an offset that fits 32 bits, so that the
// row's address stays in scalar registers; kPlanes, steps side by side, as a convolution leaves them: each lane reads its 16
// steps in vectors of 16 bytes (8 sequences of 2048 steps x 1024 channels in 32 bits, input and gate in planes, forward 43 us so, 76
// one step at a time; 38 with the channels side by side; in bf16 29, 77 and 29); kAny.
//
// Forward, a lane has 4 bytes of each row, two channels in 16 bits.  Backward it has one: with two, a wavefront needs 178
// registers instead of 113, and one workgroup fits a CU where two do (131072 steps of 2048 channels in bf16: 752 us with two
// channels, 662 with one; forward 393 with two and 425 with one).
enum Order { kAny, kDense, kPlanes };
template <typename T, Order IN>
constexpr int kLaneChannels = IN == kDense && sizeof(T) == 2 ? 2 : 1;
constexpr Order kOut(Order in) { return in == kAny ? kAny : kDense; }  // of what is written

template <typename T, Order ORDER, int V>
struct LaneRows {
    typedef typename std::conditional<ORDER == kDense, unsigned, long>::type Offset;
    const char *base;
    long st;             // bytes from row to row
    Offset off;          // of this lane's loads in a row, in bytes
    __device__ LaneRows(const Steps &t, int b, int c, int channels)
    {
        base = static_cast<const char *>(t.data) + (long)b * t.sb * (long)sizeof(T);
        st = t.st * (long)sizeof(T);
        const int first = c + V <= channels ? c : channels - V;
        off = (Offset)(ORDER == kDense ? (long)first * (long)sizeof(T) : first * t.sc * (long)sizeof(T));
    }
    __device__ __forceinline__ const char *row(long step) const
    {
        const unsigned long at = (unsigned long)(base + step * st);
        const unsigned lo = __builtin_amdgcn_readfirstlane((unsigned)at), hi = __builtin_amdgcn_readfirstlane((unsigned)(at >> 32));
        return reinterpret_cast<const char *>((unsigned long)hi << 32 | lo);
    }
    // Where the lane's values lie in a row.  The row's address is kept by itself, in scalar registers: it would else be
    // added up in two registers of every lane for each row.
    __device__ __forceinline__ T *place(const char *row) const
    {
        Offset o = off;
        if constexpr (ORDER == kDense) asm("" : "+s"(row), "+v"(o));
        return reinterpret_cast<T *>(const_cast<char *>(row) + o);
    }
    // 16 rows from step t0 on, of which `n` are the sequence's; the others repeat its last one (there is one).  FULL: all are
    // the sequence's, and all lanes have V channels.
    template <bool FULL>
    __device__ __forceinline__ void load(Vec<T, V> (&v)[kRun], long t0, int n, long len, int c, int channels) const
    {
        const char *r = row(FULL || n > 0 ? t0 : len - 1);
        if constexpr (ORDER == kPlanes) {
            static_assert(V == 1, "a lane walks along one line");
            if (FULL || n == kRun) {
                constexpr int N = 16 / (int)sizeof(T);
                const T *p = place(r);
                Vec<T, N> w[kRun / N];
#pragma unroll
                for (int j = 0; j < kRun / N; ++j) w[j] = load_vec<N>(p + j * N);
#pragma unroll
                for (int t = 0; t < kRun; ++t) v[t][0] = w[t / N][t % N];
                return;
            }
        }
#pragma unroll
        for (int t = 0; t < kRun; ++t) {
            v[t] = load_vec<V>(place(r));
            r += FULL || t + 1 < n ? st : 0;
        }
        if (FULL) return;
        if constexpr (V == 2)
            if (__any(c + 1 == channels))
#pragma unroll
                for (int t = 0; t < kRun; ++t) v[t][0] = c + 1 == channels ? v[t][1] : v[t][0];
    }
    template <bool FULL>
    __device__ __forceinline__ void store(const char *row, int c, int channels, const float (&x)[V]) const
    {
        T *p = place(row);
        Vec<T, V> o;
#pragma unroll
        for (int i = 0; i < V; ++i) o[i] = (T)x[i];
        if (FULL || c + V <= channels) store_vec<V>(p, o);
        else if (V == 2 && c < channels) store_vec<1>(p + 1, Vec<T, 1>{o[0]});  // its address was moved back by one
    }
};

// The same value, of which the compiler knows nothing: what was computed from it before is not kept in registers for what
// follows.
template <typename T, int V>
__device__ __forceinline__ void forget(Vec<T, V> &v)
{
    if constexpr (sizeof(T) * V == 4) {
        unsigned u = __builtin_bit_cast(unsigned, v);
        asm("" : "+v"(u));
        v = __builtin_bit_cast(Vec<T, V>, u);
    }
}

// A gate as it is kept: 1 - a, or -a where a is the smaller, so that the smaller of the two, e^-|z| / (1 + e^-|z|), has its full
// precision.  The sign bit tells them apart, not the value: for a gate below -87 e^z underflows, and -a is -0.
__device__ __forceinline__ float gate_of(float gate, float bias2)
{
    const float z = fmaf(gate, kLog2e, bias2), e = __builtin_amdgcn_exp2f(-fabsf(z));
    return copysignf(e * __builtin_amdgcn_rcpf(1.0f + e), z);
}
__device__ __forceinline__ bool holds_a(float m) { return __float_as_int(m) < 0; }
__device__ __forceinline__ float closed_of(float m) { return holds_a(m) ? 1.0f + m : m; }
__device__ __forceinline__ float open_of(float m) { return holds_a(m) ? -m : 1.0f - m; }
// v a, rounded once
__device__ __forceinline__ float kept(float m, float v) { return fmaf(-m, v, holds_a(m) ? 0.0f : v); }
// The state after h and x, which are `d` = x - h apart, from the side of the larger weight: h + (1 - a) d or x - a d.  So behind a
// closed gate it is x, with no rounding of the size of h.  (With h + (1 - a) d alone, and a (1 - (1 - a)) in products: 8 sequences of
// 2048 steps x 1024 channels in bf16 forward 28.7 us, 29.7 so; 131072 steps x 2048 channels 1047 us in training, 1055 so.)
__device__ __forceinline__ float moved(float m, float h, float x, float d) { return fmaf(m, d, holds_a(m) ? x : h); }

// Tickets count the tiles of all columns (sequences and blocks of channels) in the order in which they depend on each
// other, those of different columns side by side: what is worked on at one time lies in the same rows of memory.  Other ways
// of giving out tiles, on the forward pass over 131072 steps of 2048 channels in bf16 (385 us so): a counter for each column, 399
// us; that with the columns kept to one XCD, 454 us; workgroups that stay and draw their next tile ahead, 417 us.
//
// Additions to one address follow each other about 10 ns apart, which the first 512 workgroups of a launch wait for.  Where
// there are few, 8 counters give out the tiles of an eighth of the columns each (5 sequences of 1537 steps x 515
// channels in 32 bits: 585 workgroups, a training step 50.1 us with one counter, 45.6 so; 4 x 3219 x 714 in fp16, up to
// 1248: 75 and 65).  Where there are many, columns that drift apart cost more than the start (a training step of 1 x 30000 x
// 2048 in bf16, up to 7520: 264 us with one counter, 274 with 8; of the long sequence above, 32768: 1049 and 1139).
//
// Workgroups go to the 8 XCDs in turn, so every eighth one takes columns beside each other: where rows do not begin on a line
// of memory, two columns share lines, which one L2 cache then reads and writes once (64 sequences of 128 steps x 1001
// channels in 32 bits: a training step 84 us with columns in turn, 69 so; 37 x 287 x 1723 171 and 149, with 1728 channels 131 and
// 134).
__device__ __forceinline__ unsigned column_of(unsigned i, unsigned cols)
{
    const unsigned xcd = i % kXcds, more = cols % kXcds;
    return xcd * (cols / kXcds) + (xcd < more ? xcd : more) + i / kXcds;
}
__device__ __forceinline__ unsigned draw(const Chain &ch, const Shape &s)
{
    const unsigned cols = s.cols, few = s.tiles * s.cols <= kFew, counter = few ? blockIdx.x % cols % kXcds : 0;
    const unsigned n = __hip_atomic_fetch_add(ch.tickets + counter * kCounterLine, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) + 1u;
    if (!few) return n;
    const unsigned columns = (cols - counter + kXcds - 1) / kXcds;
    return n / columns * cols + column_of(n % columns * kXcds + counter, cols);
}
__device__ __forceinline__ long length_of(const int *lengths, int b, long steps)
{
    if (lengths == nullptr) return steps;
    const long n = __builtin_amdgcn_readfirstlane(lengths[b]);
    return n < 0 ? 0 : n < steps ? n : steps;
}

// How many of the 16 steps from t0 on lie before `end`.
__device__ __forceinline__ int steps_before(long t0, long end) { return (int)(end - t0 < 0 ? 0 : end - t0 < kRun ? end - t0 : kRun); }

// Zero in the steps behind the end.
template <typename T, int V>
__device__ __forceinline__ void cut_run(Vec<T, V> (&v)[kRun], int n)
{
#pragma unroll
    for (int t = 0; t < kRun; ++t)
        if (t >= n) v[t] = Vec<T, V>{};
}

// The runs of wavefronts 0 to count - 1, as one; and of wavefronts from to kWaves - 1, the last of them first.  Those that
// the workgroup does not have hold identities, so that every read has a fixed place and none waits for another.
template <int V>
__device__ __forceinline__ void join(float (&A)[V], float (&S)[V], const float (*a)[kLanes * V], const float (*s)[kLanes * V], int count, int lane)
{
#pragma unroll
    for (int i = 0; i < V; ++i) A[i] = 1.0f, S[i] = 0.0f;
#pragma unroll
    for (int j = 0; j < kWaves; ++j)
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const float Aj = a[j][lane * V + i], Sj = s[j][lane * V + i];
            A[i] = j < count ? A[i] * Aj : A[i];
            S[i] = j < count ? fmaf(Aj, S[i], Sj) : S[i];
        }
}
template <int V>
__device__ __forceinline__ void join_back(float (&A)[V], float (&R)[V], const float (*a)[kLanes * V], const float (*r)[kLanes * V], int from, int lane)
{
#pragma unroll
    for (int i = 0; i < V; ++i) A[i] = 1.0f, R[i] = 0.0f;
#pragma unroll
    for (int j = kWaves - 1; j >= 0; --j)
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const float Aj = a[j][lane * V + i], Rj = r[j][lane * V + i];
            A[i] = j >= from ? A[i] * Aj : A[i];
            R[i] = j >= from ? fmaf(Aj, R[i], Rj) : R[i];
        }
}
template <int V>
__device__ __forceinline__ void fill_runs(float (*to)[kWaves][kLanes * V], int waves, float v)
{
    for (int j = waves; j < kWaves; ++j)
        for (int i = threadIdx.x; i < kLanes * V; i += blockDim.x) to[0][j][i] = to[1][j][i] = v;
}

template <typename T, Order IN>
__global__ __launch_bounds__(kLanes *kWaves, 4) void recurrence_forward_kernel(RecArgs a)
{
    constexpr int V = kLaneChannels<T, IN>;
    __shared__ float sA[2][kWaves][kLanes * V], sS[2][kWaves][kLanes * V], carried[kLanes * V];
    __shared__ unsigned given;
    const long steps = a.steps;
    const Shape s = shape_of(a.batch, a.channels, steps, V);
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const Chain ch = chain_of(a.workspace, s, V);
    unsigned long ticket = s.chain ? 0 : column_of(blockIdx.x, s.cols);
    const unsigned long all = (unsigned long)s.tiles * s.cols;
    if (s.chain) {
        if (threadIdx.x == 0) given = draw(ch, s);
        __syncthreads();
        ticket = __builtin_amdgcn_readfirstlane(given);
    }
    fill_runs<V>(sA, s.waves, 1.0f);
    fill_runs<V>(sS, s.waves, 0.0f);
    float carry[V];  // in the first wavefront: the state before the tile
    for (int turn = 0; ticket < all; turn ^= 1, ticket = s.chain ? all : ticket + s.cols) {
        const int order = (int)(ticket / (unsigned)s.cols), col = (int)(ticket % (unsigned)s.cols), tile = order;
        const int b = col / s.blocks, c = col % s.blocks * kLanes * V + lane * V;
        const long len = length_of(a.lengths, b, steps);
        const LaneRows<T, IN, V> xr(a.x, b, c, a.channels), gr(a.gate, b, c, a.channels);
        const LaneRows<T, kOut(IN), V> yr(a.y, b, c, a.channels);
        const bool whole = __all(c + V <= a.channels);
        float bias2[V];
#pragma unroll
        for (int i = 0; i < V; ++i) {
            bias2[i] = a.bias != nullptr && c + i < a.channels ? a.bias[c + i] * kLog2e : 0.0f;
            if (order == 0) carry[i] = a.state_in != nullptr && c + i < a.channels ? a.state_in[(long)b * a.channels + c + i] : 0.0f;
        }
        const long t0 = ((long)__builtin_amdgcn_readfirstlane(tile) * s.waves + w) * kRun;
        const int n = steps_before(t0, len), n_all = steps_before(t0, steps);
        const bool full = n == kRun && whole;
        // The runs from the wavefront's first step to each of its steps, so that one operation a step is left once the state
        // before them is known (131072 steps of 2048 channels in bf16: 384 us so, 391 with the gates kept in their place).
        float A[kRun][V], S[kRun][V];
        auto read = [&](auto all) {
            constexpr bool FULL = decltype(all)::value;
            Vec<T, V> x[kRun], gate[kRun];
            xr.template load<FULL>(x, t0, n, len, c, a.channels);
            gr.template load<FULL>(gate, t0, n, len, c, a.channels);
#pragma unroll
            for (int t = 0; t < kRun; ++t) {
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const float a = t > 0 ? A[t > 0 ? t - 1 : 0][i] : 1.0f, h = t > 0 ? S[t > 0 ? t - 1 : 0][i] : 0.0f;
                    const float m = gate_of((float)gate[t][i], bias2[i]), xt = (float)x[t][i];
                    A[t][i] = FULL || t < n ? kept(m, a) : a;
                    S[t][i] = FULL || t < n ? moved(m, h, xt, xt - h) : h;
                }
                if (t % 2 == 1) __builtin_amdgcn_sched_barrier(0);
            }
        };
        if (full) read(std::true_type{});
        else if (len > 0) read(std::false_type{});
        else
#pragma unroll
            for (int t = 0; t < kRun; ++t)
#pragma unroll
                for (int i = 0; i < V; ++i) A[t][i] = 1.0f, S[t][i] = 0.0f;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            sA[turn][w][lane * V + i] = A[kRun - 1][i];
            sS[turn][w][lane * V + i] = S[kRun - 1][i];
        }
        __syncthreads();
        // the runs of the wavefronts before this one, as one; of the whole tile in the first wavefront
        float Ap[V], Sp[V];
        join<V>(Ap, Sp, sA[turn], sS[turn], w == 0 ? kWaves : w, lane);
        if (w == 0) {
            if (s.chain && tile > 0) {
                if (tile + 1 < s.tiles) announce_run<V>(ch, s, tile, col, lane, Ap, Sp);
                look_back<V>(ch, s, tile, col, -1, lane, carry);
            }
            float after[V];
#pragma unroll
            for (int i = 0; i < V; ++i) after[i] = fmaf(Ap[i], carry[i], Sp[i]);
            if (s.chain && tile + 1 < s.tiles) announce_state<V>(ch, s, tile, col, lane, after);
#pragma unroll
            for (int i = 0; i < V; ++i) {
                carried[lane * V + i] = carry[i];
                if (a.checkpoints != nullptr && c + i < a.channels)
                    a.checkpoints[((long)tile * a.batch + b) * a.channels + c + i] = carry[i];
                carry[i] = after[i];
                Ap[i] = 1.0f;
                Sp[i] = 0.0f;
            }
        }
        __syncthreads();
        float h[V];  // the state before the wavefront's steps
#pragma unroll
        for (int i = 0; i < V; ++i) h[i] = fmaf(Ap[i], carried[lane * V + i], Sp[i]);
        auto write = [&](auto all) {
            constexpr bool FULL = decltype(all)::value;
            const char *to = yr.row(t0);
#pragma unroll
            for (int t = 0; t < kRun; ++t, to += yr.st) {
                float out[V];
#pragma unroll
                for (int i = 0; i < V; ++i) out[i] = FULL || t < n ? fmaf(A[t][i], h[i], S[t][i]) : 0.0f;
                if (FULL || t < n_all) yr.template store<FULL>(to, c, a.channels, out);
                if (t % 2 == 1) __builtin_amdgcn_sched_barrier(0);
            }
        };
        if (full) write(std::true_type{});
        else write(std::false_type{});
        if (a.state_out != nullptr && tile + 1 == s.tiles && w + 1 == s.waves)
#pragma unroll
            for (int i = 0; i < V; ++i)
                if (c + i < a.channels) a.state_out[(long)b * a.channels + c + i] = fmaf(A[kRun - 1][i], h[i], S[kRun - 1][i]);
    }
}

template <typename T, Order IN, Order GRAD>
__global__ __launch_bounds__(kLanes *kWaves, 4) void recurrence_backward_kernel(RecArgs a, float *partial)
{
    constexpr int V = 1;
    __shared__ float sA[2][kWaves][kLanes * V], sS[2][kWaves][kLanes * V], sR[2][kWaves][kLanes * V], carried[kLanes * V];
    __shared__ unsigned given;
    const long steps = a.steps;
    const Shape s = shape_of(a.batch, a.channels, steps, V);
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const Chain ch = chain_of(a.workspace, s, V);
    unsigned long ticket = s.chain ? 0 : column_of(blockIdx.x, s.cols);
    const unsigned long all = (unsigned long)s.tiles * s.cols;
    if (s.chain) {
        if (threadIdx.x == 0) given = draw(ch, s);
        __syncthreads();
        ticket = __builtin_amdgcn_readfirstlane(given);
    }
    fill_runs<V>(sA, s.waves, 1.0f);
    fill_runs<V>(sS, s.waves, 0.0f);
    fill_runs<V>(sR, s.waves, 0.0f);
    float carry[V];  // in the first wavefront: a_{t+1} u_{t+1} behind the tile
    for (int turn = 0; ticket < all; turn ^= 1, ticket = s.chain ? all : ticket + s.cols) {
        const int order = (int)(ticket / (unsigned)s.cols), col = (int)(ticket % (unsigned)s.cols), tile = s.tiles - 1 - order;
        const int b = col / s.blocks, c = col % s.blocks * kLanes * V + lane * V;
        const long len = length_of(a.lengths, b, steps);
        const LaneRows<T, IN, V> xr(a.x, b, c, a.channels), gr(a.gate, b, c, a.channels);
        const LaneRows<T, GRAD, V> yr(a.y, b, c, a.channels);
        const LaneRows<T, kOut(IN), V> gxr(a.grad_x, b, c, a.channels), ggr(a.grad_gate, b, c, a.channels);
        const bool whole = __all(c + V <= a.channels);
        float bias2[V];
#pragma unroll
        for (int i = 0; i < V; ++i) {
            bias2[i] = a.bias != nullptr && c + i < a.channels ? a.bias[c + i] * kLog2e : 0.0f;
            if (order == 0) carry[i] = a.state_in != nullptr && c + i < a.channels ? a.state_in[(long)b * a.channels + c + i] : 0.0f;
        }
        const long t0 = ((long)__builtin_amdgcn_readfirstlane(tile) * s.waves + w) * kRun;
        const int n = steps_before(t0, len), n_all = steps_before(t0, steps);
        const bool full = n == kRun && whole;
        Vec<T, V> x[kRun], gy[kRun];
        float m[kRun][V], before[V];  // m: the gates
        float A[V], S[V], R[V];       // product of the a, state behind these steps, a u of the first of them, from zero
#pragma unroll
        for (int i = 0; i < V; ++i)
            before[i] = c + i < a.channels ? a.checkpoints[((long)tile * a.batch + b) * a.channels + c + i] : 0.0f;
        auto read = [&](auto all) {
            constexpr bool FULL = decltype(all)::value;
            Vec<T, V> gate[kRun];
            xr.template load<FULL>(x, t0, n, len, c, a.channels);
            gr.template load<FULL>(gate, t0, n, len, c, a.channels);
            yr.template load<FULL>(gy, t0, n, len, c, a.channels);
            if (!FULL && n < kRun) {
                cut_run<T, V>(x, n);
                cut_run<T, V>(gy, n);
            }
#pragma unroll
            for (int i = 0; i < V; ++i) {
                A[i] = 1.0f;
                S[i] = R[i] = 0.0f;
            }
#pragma unroll
            for (int t = 0; t < kRun; ++t) {
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    m[t][i] = FULL || t < n ? gate_of((float)gate[t][i], bias2[i]) : 0.0f;
                    A[i] = kept(m[t][i], A[i]);
                    S[i] = moved(m[t][i], S[i], (float)x[t][i], (float)x[t][i] - S[i]);
                    R[i] = fmaf(A[i], (float)gy[t][i], R[i]);
                }
                if (t % 4 == 3) __builtin_amdgcn_sched_barrier(0);  // few steps at a time, or their parts fill the registers
            }
        };
        if (full) {
            read(std::true_type{});
        } else if (len > 0) {
            read(std::false_type{});
        } else {
#pragma unroll
            for (int t = 0; t < kRun; ++t) {
                x[t] = gy[t] = Vec<T, V>{};
#pragma unroll
                for (int i = 0; i < V; ++i) m[t][i] = 0.0f;
            }
#pragma unroll
            for (int i = 0; i < V; ++i) {
                A[i] = 1.0f;
                S[i] = R[i] = 0.0f;
            }
        }
#pragma unroll
        for (int i = 0; i < V; ++i) {
            sA[turn][w][lane * V + i] = A[i];
            sS[turn][w][lane * V + i] = S[i];
            sR[turn][w][lane * V + i] = R[i];
        }
        __syncthreads();
        // The runs of the wavefronts behind this one, as one; of the whole tile in the first wavefront, which announces them.
        float Aq[V], Rq[V];
        join_back<V>(Aq, Rq, sA[turn], sR[turn], w == 0 ? 0 : w + 1, lane);
        if (w == 0 && s.chain && tile > 0 && tile + 1 < s.tiles) announce_run<V>(ch, s, tile, col, lane, Aq, Rq);
        // the states inside this wavefront's steps, from the one before the tile
        {
            float Ap[V], Sp[V];
            join<V>(Ap, Sp, sA[turn], sS[turn], w, lane);
#pragma unroll
            for (int i = 0; i < V; ++i) before[i] = fmaf(Ap[i], before[i], Sp[i]);
        }
        float d[kRun][V];  // the state before each step, less x
#pragma unroll
        for (int t = 0; t < kRun; ++t) {
            forget<T, V>(x[t]);
#pragma unroll
            for (int i = 0; i < V; ++i) {
                d[t][i] = before[i] - (float)x[t][i];
                before[i] = moved(m[t][i], before[i], (float)x[t][i], -d[t][i]);
            }
            if (t % 4 == 3) __builtin_amdgcn_sched_barrier(0);
        }
        if (w == 0) {
            if (s.chain && tile + 1 < s.tiles) look_back<V>(ch, s, tile, col, 1, lane, carry);
            float after[V];
#pragma unroll
            for (int i = 0; i < V; ++i) after[i] = fmaf(Aq[i], carry[i], Rq[i]);
            if (s.chain && tile > 0) announce_state<V>(ch, s, tile, col, lane, after);
#pragma unroll
            for (int i = 0; i < V; ++i) {
                carried[lane * V + i] = carry[i];
                carry[i] = after[i];
            }
            join_back<V>(Aq, Rq, sA[turn], sR[turn], 1, lane);
        }
        __syncthreads();
        float g[V], sum[V];
#pragma unroll
        for (int i = 0; i < V; ++i) {
            g[i] = fmaf(Aq[i], carried[lane * V + i], Rq[i]);
            sum[i] = 0.0f;
        }
#pragma unroll
        for (int t = 0; t < kRun; ++t) forget<T, V>(gy[t]);
        auto write = [&](auto all) {
            constexpr bool FULL = decltype(all)::value;
            const char *to_x = gxr.row(t0 + kRun - 1), *to_gate = ggr.row(t0 + kRun - 1);
#pragma unroll
            for (int t = kRun - 1; t >= 0; --t, to_x -= gxr.st, to_gate -= ggr.st) {
                float gx[V], gz[V];
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const float k = closed_of(m[t][i]), keep = open_of(m[t][i]);
                    const float u = (float)gy[t][i] + g[i];
                    gx[i] = k * u;
                    g[i] = keep * u;
                    gz[i] = k * d[t][i] * g[i];
                    sum[i] += gz[i];
                }
                if (FULL || t < n_all) {
                    if (a.grad_x.data != nullptr) gxr.template store<FULL>(to_x, c, a.channels, gx);
                    if (a.grad_gate.data != nullptr) ggr.template store<FULL>(to_gate, c, a.channels, gz);
                }
                if (t % 4 == 0) __builtin_amdgcn_sched_barrier(0);
            }
        };
        if (full) write(std::true_type{});
        else write(std::false_type{});
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
                    if (c + i < a.channels) partial[((long)tile * a.batch + b) * a.channels + c + i] = v;
                }
        }
    }
}

// One step, or none: the form of a single token.
template <typename T, int V>
__global__ __launch_bounds__(256) void recurrence_step_kernel(RecArgs a)
{
    const unsigned per = (a.channels + V - 1) / V, i = blockIdx.x * 256u + threadIdx.x;  // recurrence_fits(): below 2^31
    if (i >= a.batch * per) return;
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
        const float z = (float)gv[j] + bias[j], x = (float)xv[j], d = x - h[j];
        sigmoid_pair(z, keep, k);
        if (live) h[j] = z < 0.0f ? fmaf(-keep, d, x) : fmaf(k, d, h[j]);  // as moved()
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

// grad_bias: the sum of `rows` rows of sums.
__global__ __launch_bounds__(kSumThreads) void recurrence_bias_kernel(const float *partial, long rows, int channels, float factor, float *out)
{
    __shared__ float part[kSumSlices][kSumColumns];
    const int at = blockIdx.x * kSumColumns + threadIdx.x % kSumColumns;
    const float sum = slices_sum(at < channels ? slice_sum(partial + at, channels, rows, threadIdx.x / kSumColumns) : 0.0f, part);
    if (threadIdx.x < kSumColumns && at < channels) out[at] = sum * factor;
}

static hipError_t launch_bias(const float *partial, long rows, const RecArgs &a, hipStream_t s)
{
    const int blocks = (a.channels + kSumColumns - 1) / kSumColumns;
    kernel_log_add("recurrence_bias_kernel", (long)blocks * kSumThreads);
    FBFC_LAUNCH(recurrence_bias_kernel, dim3(blocks), dim3(kSumThreads), 0, s, partial, rows, a.channels, a.factor, a.grad_bias);
    return hipGetLastError();
}

// The order of a tensor's memory; rows of dense ones are within the reach of 32 bits.
static Order order_of(int type, const Steps &t, const RecArgs &a)
{
    if (t.sc == 1 && a.channels >= (type == kF32 ? 1 : 2) && a.channels <= 1 << 29) return kDense;
    return t.st == 1 ? kPlanes : kAny;
}
static bool dense(int type, const Steps &t, const RecArgs &a) { return t.data == nullptr || order_of(type, t, a) == kDense; }

size_t recurrence_checkpoint_bytes(int batch, int channels, long steps)
{
    return (size_t)shape_of(batch, channels, steps, 1).tiles * (size_t)batch * channels * sizeof(float);
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

// One launch has fewer than 2^32 threads, of up to 512 in a workgroup; the kernel that adds up the bias's gradient has 64 for
// each channel.
bool recurrence_fits(int batch, int channels, long steps)
{
    const long tiles = (steps + kRun * kWaves - 1) / (kRun * kWaves) + 1, most = 1L << 23;
    if (channels > 1 << 25 || (long)batch * channels >= 1L << 31 || tiles >= 1L << 31) return false;
    for (int v = 1; v <= 2; ++v) {
        const long cols = (channels + kLanes * v - 1L) / (kLanes * v) * batch;
        if (cols >= most || (cols > 0 && cols < kGroups && tiles >= most / cols)) return false;  // a workgroup a column, or a tile
    }
    return true;
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
static hipError_t forward_typed(int type, const RecArgs &a, hipStream_t stream)
{
    const bool out = dense(type, a.y, a);
    const Order x = order_of(type, a.x, a), in = out && x == order_of(type, a.gate, a) ? x : kAny;
    const int v = in == kDense ? kLaneChannels<T, kDense> : 1;
    if (a.steps <= 1) {
        const bool wide = in == kDense && a.channels >= 4;
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
    const dim3 grid(s.chain ? s.tiles * s.cols : s.cols), block(s.waves * kLanes);
    kernel_log_add(s.chain ? "recurrence_forward_kernel<chain>" : "recurrence_forward_kernel", (long)grid.x * block.x);
    if (in == kDense) FBFC_LAUNCH((recurrence_forward_kernel<T, kDense>), grid, block, 0, stream, a);
    else if (in == kPlanes) FBFC_LAUNCH((recurrence_forward_kernel<T, kPlanes>), grid, block, 0, stream, a);
    else FBFC_LAUNCH((recurrence_forward_kernel<T, kAny>), grid, block, 0, stream, a);
    return hipGetLastError();
}

template <typename T>
static hipError_t backward_typed(int type, const RecArgs &a, hipStream_t stream)
{
    const bool out = dense(type, a.grad_x, a) && dense(type, a.grad_gate, a);
    const Order x = order_of(type, a.x, a), grad = order_of(type, a.y, a);
    const Order in = out && grad != kAny && x == order_of(type, a.gate, a) ? x : kAny;
    const Shape s = shape_of(a.batch, a.channels, a.steps, 1);
    float *partial = nullptr;
    if (a.grad_bias != nullptr)
        partial = reinterpret_cast<float *>(a.workspace + recurrence_workspace_bytes(a.batch, a.channels, a.steps) -
                                            recurrence_checkpoint_bytes(a.batch, a.channels, a.steps));
    if (s.chain) {
        const hipError_t e = clear_chain(a, s, 1, stream);
        if (e != hipSuccess) return e;
    }
    const dim3 grid(s.chain ? s.tiles * s.cols : s.cols), block(s.waves * kLanes);
    kernel_log_add(s.chain ? "recurrence_backward_kernel<chain>" : "recurrence_backward_kernel", (long)grid.x * block.x);
    if (in == kDense && grad == kDense) FBFC_LAUNCH((recurrence_backward_kernel<T, kDense, kDense>), grid, block, 0, stream, a, partial);
    else if (in == kDense) FBFC_LAUNCH((recurrence_backward_kernel<T, kDense, kPlanes>), grid, block, 0, stream, a, partial);
    else if (in == kPlanes && grad == kDense) FBFC_LAUNCH((recurrence_backward_kernel<T, kPlanes, kDense>), grid, block, 0, stream, a, partial);
    else if (in == kPlanes) FBFC_LAUNCH((recurrence_backward_kernel<T, kPlanes, kPlanes>), grid, block, 0, stream, a, partial);
    else FBFC_LAUNCH((recurrence_backward_kernel<T, kAny, kAny>), grid, block, 0, stream, a, partial);
    const hipError_t e = hipGetLastError();
    return e != hipSuccess || partial == nullptr ? e : launch_bias(partial, (long)s.tiles * a.batch, a, stream);
}

hipError_t launch_recurrence_forward(int type, const RecArgs &a, hipStream_t s)
{
    return type == kF32 ? forward_typed<float>(type, a, s) : type == kBF16 ? forward_typed<bf16>(type, a, s) : forward_typed<f16>(type, a, s);
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
        return a.grad_bias == nullptr ? hipSuccess : launch_bias(nullptr, 0, a, s);
    }
    return type == kF32 ? backward_typed<float>(type, a, s) : type == kBF16 ? backward_typed<bf16>(type, a, s) : backward_typed<f16>(type, a, s);
}

}  // namespace fbfc
