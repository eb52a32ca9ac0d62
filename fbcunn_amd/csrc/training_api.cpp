// C ABI of the training and serving operators: argument checking and launches.  Every argument is checked before the
// first call of the HIP runtime, so refusals need no GPU.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <cstdio>
#include <cstring>
#include <new>
#include <vector>

#include "../../include/fbfftconv.h"
#include "errors.h"
#include "kernels.h"
#include "training.h"

using fbfc::fail;

static_assert(FBFC_F32 == fbfc::kF32 && FBFC_BF16 == fbfc::kBF16 && FBFC_F16 == fbfc::kF16, "one set of values");

namespace {

bool type_ok(int t) { return t == FBFC_F32 || t == FBFC_BF16 || t == FBFC_F16; }
size_t type_bytes(int t) { return t == FBFC_F32 ? 4 : 2; }
bool aligned(const void *p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

// Whether every pointer of 32-bit values is aligned to them (a null one is).
template <typename... P>
bool aligned32(const P *...p)
{
    return (aligned(p, 4) && ...);
}

// A stretch of memory that a call reads or writes.
struct Range {
    uintptr_t begin, end;
    bool written;
};

// Whether something that is written shares memory with anything else.
bool ranges_overlap(std::vector<Range> &r)
{
    std::sort(r.begin(), r.end(), [](const Range &a, const Range &b) { return a.begin < b.begin; });
    uintptr_t any = 0, written = 0;
    for (const Range &x : r) {
        if (x.begin == x.end) continue;
        if (x.begin < (x.written ? any : written)) return true;
        any = std::max(any, x.end);
        if (x.written) written = std::max(written, x.end);
    }
    return false;
}

}  // namespace

struct fbfc_adamw {
    int device;
    fbfc_adamw_config config;
    void *memory;  // the clock, the counts of workgroups, the table of pieces
    fbfc::AdamwArgs args;
};

extern "C" {

// ---- AdamW ---------------------------------------------------------------------------------------
long fbfc_adamw_state_elements(const fbfc_adamw_tensor *tensors, int count)
{
    if (tensors == nullptr || count < 1) return 0;
    long n = 0;
    for (int i = 0; i < count; ++i) {
        if (tensors[i].n < 0 || tensors[i].n > (1L << 40)) return 0;
        n += (tensors[i].n + fbfc::kAdamwBlock - 1) / fbfc::kAdamwBlock * fbfc::kAdamwBlock;
    }
    return n;
}

static int adamw_check(const fbfc_adamw_config *c, const fbfc_adamw_tensor *tensors, int count, const void *m,
                       const void *v, const float *m_scale, const float *v_scale)
{
    if (c == nullptr || tensors == nullptr) return fail(FBFC_ERR_INVALID_ARGUMENT, "null argument");
    if (count < 1) return fail(FBFC_ERR_INVALID_ARGUMENT, "at least one tensor is needed");
    bool empty = true;  // no parameter at all, and so no states
    for (int i = 0; i < count; ++i) empty = empty && tensors[i].n == 0;
    if (!empty && (m == nullptr || v == nullptr)) return fail(FBFC_ERR_INVALID_ARGUMENT, "null argument");
    if (!type_ok(c->param_type) || !type_ok(c->grad_type)) return fail(FBFC_ERR_INVALID_ARGUMENT, "unknown type");
    if (c->state_bits != 8 && c->state_bits != 32)
        return fail(FBFC_ERR_INVALID_ARGUMENT, "states have 8 or 32 bits");
    if (!(c->beta1 >= 0 && c->beta1 < 1 && c->beta2 >= 0 && c->beta2 < 1))
        return fail(FBFC_ERR_INVALID_ARGUMENT, "betas must be in [0, 1)");
    if (!(c->eps > 0 && std::isfinite(c->eps) && (float)c->eps > 0.0f))
        return fail(FBFC_ERR_INVALID_ARGUMENT, "eps must be positive");
    if (c->state_bits == 8 && !empty && (m_scale == nullptr || v_scale == nullptr))
        return fail(FBFC_ERR_INVALID_ARGUMENT, "states of 8 bits need their scales");
    if (!aligned(m, 16) || !aligned(v, 16)) return fail(FBFC_ERR_INVALID_ARGUMENT, "states must be 16-byte aligned");
    if (c->state_bits == 8 && (!aligned(m_scale, 4) || !aligned(v_scale, 4)))
        return fail(FBFC_ERR_INVALID_ARGUMENT, "scales must be 4-byte aligned");
    const size_t pb = type_bytes(c->param_type), gb = type_bytes(c->grad_type), sb = c->state_bits / 8;
    long pieces = 0;
    for (int i = 0; i < count; ++i) {
        const fbfc_adamw_tensor &t = tensors[i];
        if (t.n < 0) return fail(FBFC_ERR_INVALID_ARGUMENT, "sizes must not be negative");
        if (t.n > (1L << 40)) return fail(FBFC_ERR_UNSUPPORTED_SIZE, "a tensor of more than 2^40 parameters");
        if (t.n > 0 && (t.param == nullptr || t.grad == nullptr)) return fail(FBFC_ERR_INVALID_ARGUMENT, "null tensor");
        if (!aligned(t.param, pb) || !aligned(t.grad, gb))
            return fail(FBFC_ERR_INVALID_ARGUMENT, "tensors must be aligned to their type");
        pieces += (t.n + fbfc::kAdamwSmallPiece - 1) / fbfc::kAdamwSmallPiece;
    }
    if (pieces > INT32_MAX) return fail(FBFC_ERR_UNSUPPORTED_SIZE, "too many parameters for one optimizer");
    const size_t n = (size_t)fbfc_adamw_state_elements(tensors, count);
    std::vector<Range> r;
    r.reserve(2 * (size_t)count + 4);
    auto add = [&r](const void *p, size_t bytes, bool written) {
        r.push_back({reinterpret_cast<uintptr_t>(p), reinterpret_cast<uintptr_t>(p) + bytes, written});
    };
    for (int i = 0; i < count; ++i) {
        add(tensors[i].param, tensors[i].n * pb, true);
        add(tensors[i].grad, tensors[i].n * gb, false);
    }
    add(m, n * sb, true);
    add(v, n * sb, true);
    if (c->state_bits == 8) {
        add(m_scale, n / fbfc::kAdamwBlock * 4, true);
        add(v_scale, n / fbfc::kAdamwBlock * 4, true);
    }
    if (ranges_overlap(r))
        return fail(FBFC_ERR_INVALID_ARGUMENT, "a parameter or a state shares memory with another tensor");
    return FBFC_OK;
}

static int adamw_create(const fbfc_adamw_config *c, const fbfc_adamw_tensor *tensors, int count, void *m, void *v,
                        float *m_scale, float *v_scale, fbfc_adamw **out)
{
    const int rc = adamw_check(c, tensors, count, m, v, m_scale, v_scale);
    if (rc != FBFC_OK) return rc;
    std::vector<fbfc::AdamwPiece> pieces;
    const size_t pb = type_bytes(c->param_type), gb = type_bytes(c->grad_type);
    long first = 0, n = 0;
    for (int i = 0; i < count; ++i) n += tensors[i].n;
    const long size = n < 2048L * fbfc::kAdamwPiece ? fbfc::kAdamwSmallPiece : fbfc::kAdamwPiece;
    for (int i = 0; i < count; ++i) {
        const fbfc_adamw_tensor &t = tensors[i];
        for (long o = 0; o < t.n; o += size)
            pieces.push_back({static_cast<char *>(t.param) + o * pb, static_cast<const char *>(t.grad) + o * gb, first + o,
                              std::min(t.n - o, size)});
        first += (t.n + fbfc::kAdamwBlock - 1) / fbfc::kAdamwBlock * fbfc::kAdamwBlock;
    }
    fbfc_adamw *p = new (std::nothrow) fbfc_adamw();
    if (p == nullptr) return fail(FBFC_ERR_OUT_OF_MEMORY, "host allocation failed");
    p->config = *c;
    constexpr size_t counts = 256, head = counts + fbfc::kAdamwLines * fbfc::kAdamwLine * sizeof(unsigned);
    static_assert(sizeof(fbfc::AdamwClock) <= counts, "the clock has a line of its own");
    unsigned char begin[head] = {};
    const fbfc::AdamwClock clock = fbfc::adamw_clock(0, c->beta1, c->beta2, c->seed);
    std::memcpy(begin, &clock, sizeof clock);
    hipError_t e = hipGetDevice(&p->device);
    if (e == hipSuccess) e = hipMalloc(&p->memory, head + pieces.size() * sizeof(fbfc::AdamwPiece));
    if (e == hipSuccess) e = hipMemcpy(p->memory, begin, sizeof begin, hipMemcpyHostToDevice);
    if (e == hipSuccess && !pieces.empty())
        e = hipMemcpy(static_cast<char *>(p->memory) + head, pieces.data(), pieces.size() * sizeof(fbfc::AdamwPiece),
                      hipMemcpyHostToDevice);
    if (e != hipSuccess) {
        (void)hipGetLastError();
        fbfc_adamw_destroy(p);
        if (e == hipErrorOutOfMemory) return fail(FBFC_ERR_OUT_OF_MEMORY, "no memory for the optimizer's table");
        return fbfc::fail_hip(e, "optimizer allocation");
    }
    fbfc::AdamwArgs &a = p->args;
    a.pieces = reinterpret_cast<const fbfc::AdamwPiece *>(static_cast<char *>(p->memory) + head);
    a.n_pieces = (int)pieces.size();
    a.clock = static_cast<fbfc::AdamwClock *>(p->memory);
    a.ended = reinterpret_cast<unsigned *>(static_cast<char *>(p->memory) + counts);
    a.m = m;
    a.v = v;
    a.m_scale = m_scale;
    a.v_scale = v_scale;
    a.beta1 = c->beta1;
    a.beta2 = c->beta2;
    a.seed = c->seed;
    a.keep1 = (float)c->beta1;
    a.take1 = (float)(1 - c->beta1);
    a.keep2 = (float)c->beta2;
    a.take2 = (float)(1 - c->beta2);
    a.eps = (float)c->eps;
    *out = p;
    return FBFC_OK;
}

int fbfc_adamw_create(const fbfc_adamw_config *config, const fbfc_adamw_tensor *tensors, int count, void *m, void *v,
                      float *m_scale, float *v_scale, fbfc_adamw **opt)
{
    if (opt == nullptr) return fail(FBFC_ERR_INVALID_ARGUMENT, "null argument");
    *opt = nullptr;
    try {
        return adamw_create(config, tensors, count, m, v, m_scale, v_scale, opt);
    } catch (const std::bad_alloc &) {
        return fail(FBFC_ERR_OUT_OF_MEMORY, "host allocation failed");
    }
}

int fbfc_adamw_destroy(fbfc_adamw *p)
{
    if (p == nullptr) return FBFC_OK;
    if (p->memory) (void)hipFree(p->memory);
    delete p;
    return FBFC_OK;
}

static int adamw_device(const fbfc_adamw *p)
{
    int device = -1;
    FBFC_TRY(hipGetDevice(&device), "hipGetDevice");
    if (device != p->device)
        return fail(FBFC_ERR_INVALID_ARGUMENT, "the optimizer was made on another device than the current one");
    return FBFC_OK;
}

int fbfc_adamw_set_step(fbfc_adamw *p, long t, void *stream)
{
    if (p == nullptr) return fail(FBFC_ERR_INVALID_ARGUMENT, "null argument");
    if (t < 0) return fail(FBFC_ERR_INVALID_ARGUMENT, "the number of steps must not be negative");
    const int rc = adamw_device(p);
    if (rc != FBFC_OK) return rc;
    FBFC_TRY(fbfc::launch_adamw_set_clock(p->args, t, static_cast<hipStream_t>(stream)), "AdamW clock");
    return FBFC_OK;
}

int fbfc_adamw_get_step(fbfc_adamw *p, long *t, void *stream)
{
    if (p == nullptr || t == nullptr) return fail(FBFC_ERR_INVALID_ARGUMENT, "null argument");
    const int rc = adamw_device(p);
    if (rc != FBFC_OK) return rc;
    hipStream_t s = static_cast<hipStream_t>(stream);
    FBFC_TRY(hipMemcpyAsync(t, &p->args.clock->t, sizeof *t, hipMemcpyDeviceToHost, s), "AdamW step count");
    FBFC_TRY(hipStreamSynchronize(s), "hipStreamSynchronize");
    return FBFC_OK;
}

int fbfc_adamw_step(fbfc_adamw *p, double lr, double weight_decay, float grad_scale, void *stream)
{
    if (p == nullptr) return fail(FBFC_ERR_INVALID_ARGUMENT, "null argument");
    if (!std::isfinite(lr) || !std::isfinite(weight_decay))
        return fail(FBFC_ERR_INVALID_ARGUMENT, "the learning rate and the weight decay must be finite");
    const int rc = adamw_device(p);
    if (rc != FBFC_OK) return rc;
    fbfc::kernel_log_clear();
    fbfc::AdamwArgs a = p->args;
    a.lr = lr;
    a.decay = (float)(1 - lr * weight_decay);
    a.grad_scale = grad_scale;
    FBFC_TRY(fbfc::launch_adamw(p->config.param_type, p->config.grad_type, p->config.state_bits, a,
                                static_cast<hipStream_t>(stream)), "AdamW step");
    return FBFC_OK;
}

// ---- norms around a block --------------------------------------------------------------------------
static fbfc::Rows rows_of(const fbfc_rows *r)
{
    return r == nullptr || r->data == nullptr ? fbfc::Rows{nullptr, 0} : fbfc::Rows{r->data, r->stride};
}

static int norm_check_desc(const fbfc_residual_norm_desc *d)
{
    if (d == nullptr) return fail(FBFC_ERR_INVALID_ARGUMENT, "null argument");
    if (!type_ok(d->type)) return fail(FBFC_ERR_INVALID_ARGUMENT, "unknown type");
    if (d->rows < 0 || d->channels < 1) return fail(FBFC_ERR_INVALID_ARGUMENT, "sizes must be positive");
    if (d->channels > fbfc::kNormMaxChannels) {
        char buf[96];
        std::snprintf(buf, sizeof buf, "rows of %d channels: up to %d are supported", d->channels, fbfc::kNormMaxChannels);
        return fail(FBFC_ERR_UNSUPPORTED_SIZE, buf);
    }
    if (!(d->eps > 0 && std::isfinite(d->eps))) return fail(FBFC_ERR_INVALID_ARGUMENT, "eps must be positive");
    return FBFC_OK;
}

// Alignment, and that the rows of a tensor that is written do not overlap.
static int norm_check_rows(const fbfc_residual_norm_desc *d, const fbfc::Rows &r, bool written)
{
    if (r.data == nullptr) return FBFC_OK;
    if (!aligned(r.data, type_bytes(d->type))) return fail(FBFC_ERR_INVALID_ARGUMENT, "rows must be aligned to their type");
    if (r.stride < 0 || (written && d->rows > 1 && r.stride < d->channels))
        return fail(FBFC_ERR_INVALID_ARGUMENT, "rows that are written must not overlap");
    return FBFC_OK;
}

static int norm_check_weights(const fbfc::NormArgs &a, bool normed)
{
    if (a.gate.data != nullptr && a.branch.data == nullptr) return fail(FBFC_ERR_INVALID_ARGUMENT, "a gate needs a branch");
    if (a.branch.data != nullptr && (a.post == nullptr || a.scale == nullptr))
        return fail(FBFC_ERR_INVALID_ARGUMENT, "a branch needs its norm's weight and its scale");
    if (normed && a.pre == nullptr) return fail(FBFC_ERR_INVALID_ARGUMENT, "the norm behind the block needs its weight");
    if (!aligned32(a.post, a.scale, a.pre, a.grad_post, a.grad_scale, a.grad_pre))
        return fail(FBFC_ERR_INVALID_ARGUMENT, "weights must be aligned to 4 bytes");
    return FBFC_OK;
}

int fbfc_residual_norm_forward(const fbfc_residual_norm_desc *d, const fbfc_rows *residual, const fbfc_rows *branch,
                               const fbfc_rows *gate, const float *post_weight, const float *scale,
                               const float *pre_weight, const fbfc_rows *output, const fbfc_rows *normed, void *stream)
{
    int rc = norm_check_desc(d);
    if (rc != FBFC_OK) return rc;
    fbfc::NormArgs a = {};
    a.rows = d->rows;
    a.channels = d->channels;
    a.eps = d->eps;
    a.residual = rows_of(residual);
    a.branch = rows_of(branch);
    a.gate = rows_of(gate);
    a.post = post_weight;
    a.scale = scale;
    a.pre = pre_weight;
    a.output = rows_of(output);
    a.normed = rows_of(normed);
    if (d->rows == 0) return FBFC_OK;
    if (a.residual.data == nullptr) return fail(FBFC_ERR_INVALID_ARGUMENT, "null residual");
    if ((a.branch.data == nullptr) != (a.output.data == nullptr))
        return fail(FBFC_ERR_INVALID_ARGUMENT, "the output goes with the branch: without one it is the residual itself");
    if (a.output.data == nullptr && a.normed.data == nullptr) return fail(FBFC_ERR_INVALID_ARGUMENT, "nothing to compute");
    rc = norm_check_weights(a, a.normed.data != nullptr);
    if (rc != FBFC_OK) return rc;
    for (const fbfc::Rows *r : {&a.residual, &a.branch, &a.gate})
        if ((rc = norm_check_rows(d, *r, false)) != FBFC_OK) return rc;
    for (const fbfc::Rows *r : {&a.output, &a.normed})
        if ((rc = norm_check_rows(d, *r, true)) != FBFC_OK) return rc;
    fbfc::kernel_log_clear();
    FBFC_TRY(fbfc::launch_norm_forward(d->type, a, static_cast<hipStream_t>(stream)), "residual norm");
    return FBFC_OK;
}

size_t fbfc_residual_norm_workspace_bytes(const fbfc_residual_norm_desc *d)
{
    if (d == nullptr || !type_ok(d->type) || d->rows < 1 || d->channels < 1 || d->channels > fbfc::kNormMaxChannels) return 0;
    return fbfc::norm_workspace_bytes(d->rows, d->channels, d->type);
}

int fbfc_residual_norm_backward(const fbfc_residual_norm_desc *d, const fbfc_rows *residual, const fbfc_rows *branch,
                                const fbfc_rows *gate, const float *post_weight, const float *scale,
                                const float *pre_weight, const fbfc_rows *grad_output, const fbfc_rows *grad_normed,
                                const fbfc_rows *grad_residual, const fbfc_rows *grad_branch, const fbfc_rows *grad_gate,
                                float *grad_post_weight, float *grad_scale, float *grad_pre_weight, float factor,
                                void *workspace, void *stream)
{
    int rc = norm_check_desc(d);
    if (rc != FBFC_OK) return rc;
    fbfc::NormArgs a = {};
    a.rows = d->rows;
    a.channels = d->channels;
    a.eps = d->eps;
    a.residual = rows_of(residual);
    a.branch = rows_of(branch);
    a.gate = rows_of(gate);
    a.post = post_weight;
    a.scale = scale;
    a.pre = pre_weight;
    a.grad_output = rows_of(grad_output);
    a.grad_normed = rows_of(grad_normed);
    a.grad_residual = rows_of(grad_residual);
    a.grad_branch = rows_of(grad_branch);
    a.grad_gate = rows_of(grad_gate);
    a.grad_post = grad_post_weight;
    a.grad_scale = grad_scale;
    a.grad_pre = grad_pre_weight;
    a.factor = factor;
    const bool weights = grad_post_weight != nullptr || grad_scale != nullptr || grad_pre_weight != nullptr;
    if (d->rows > 0) {
        if (a.residual.data == nullptr) return fail(FBFC_ERR_INVALID_ARGUMENT, "null residual");
        if (a.grad_output.data == nullptr && a.grad_normed.data == nullptr)
            return fail(FBFC_ERR_INVALID_ARGUMENT, "a gradient of the output or of the norm behind it is needed");
        if (a.branch.data == nullptr && (a.grad_branch.data != nullptr || grad_post_weight != nullptr || grad_scale != nullptr))
            return fail(FBFC_ERR_INVALID_ARGUMENT, "there is no branch to have a gradient");
        if (a.gate.data == nullptr && a.grad_gate.data != nullptr)
            return fail(FBFC_ERR_INVALID_ARGUMENT, "there is no gate to have a gradient");
        rc = norm_check_weights(a, a.grad_normed.data != nullptr);
        if (rc != FBFC_OK) return rc;
        for (const fbfc::Rows *r : {&a.residual, &a.branch, &a.gate, &a.grad_output, &a.grad_normed})
            if ((rc = norm_check_rows(d, *r, false)) != FBFC_OK) return rc;
        for (const fbfc::Rows *r : {&a.grad_residual, &a.grad_branch, &a.grad_gate})
            if ((rc = norm_check_rows(d, *r, true)) != FBFC_OK) return rc;
        if (weights && (workspace == nullptr || !aligned(workspace, 4)))
            return fail(FBFC_ERR_INVALID_ARGUMENT, "the gradients of the weights need the workspace");
    } else if ((grad_post_weight != nullptr && scale == nullptr) || (grad_scale != nullptr && post_weight == nullptr)) {
        return fail(FBFC_ERR_INVALID_ARGUMENT, "a branch needs its norm's weight and its scale");
    }
    a.partial = weights ? static_cast<float *>(workspace) : nullptr;
    fbfc::kernel_log_clear();
    FBFC_TRY(fbfc::launch_norm_backward(d->type, a, static_cast<hipStream_t>(stream)), "residual norm gradients");
    return FBFC_OK;
}

// ---- gated linear recurrence -----------------------------------------------------------------------
static fbfc::Steps steps_of(const fbfc_steps *t)
{
    return t == nullptr || t->data == nullptr ? fbfc::Steps{nullptr, 0, 0, 0}
                                              : fbfc::Steps{t->data, t->stride_batch, t->stride_step, t->stride_channel};
}

static int recurrence_check_desc(const fbfc_recurrence_desc *d)
{
    if (d == nullptr) return fail(FBFC_ERR_INVALID_ARGUMENT, "null argument");
    if (!type_ok(d->type)) return fail(FBFC_ERR_INVALID_ARGUMENT, "unknown type");
    if (d->batch < 0 || d->steps < 0 || d->channels < 1) return fail(FBFC_ERR_INVALID_ARGUMENT, "sizes must be positive");
    if (d->steps > (1L << 40) || !fbfc::recurrence_fits(d->batch, d->channels, d->steps))
        return fail(FBFC_ERR_UNSUPPORTED_SIZE, "more sequences, channels and steps than one launch can take");
    return FBFC_OK;
}

static int recurrence_check_steps(const fbfc_recurrence_desc *d, const fbfc::Steps &t, bool written)
{
    if (t.data == nullptr) return FBFC_OK;
    if (!aligned(t.data, type_bytes(d->type))) return fail(FBFC_ERR_INVALID_ARGUMENT, "tensors must be aligned to their type");
    if (!written) return FBFC_OK;
    // the places of a tensor that is written must differ: with its dimensions ordered by stride, each stride passes
    // over all that the smaller ones reach
    struct Dim {
        long n, stride;
    } dims[3] = {{d->batch, t.sb}, {d->steps, t.st}, {d->channels, t.sc}};
    std::sort(dims, dims + 3, [](const Dim &x, const Dim &y) { return x.stride < y.stride; });
    long reach = 0;  // of the smaller strides
    for (const Dim &x : dims) {
        if (x.n < 2) continue;
        if (x.stride <= reach || x.stride > (1L << 60) / x.n)
            return fail(FBFC_ERR_INVALID_ARGUMENT, "strides of a tensor that is written must not overlap or be negative");
        reach += x.stride * (x.n - 1);
    }
    return FBFC_OK;
}

size_t fbfc_recurrence_checkpoint_bytes(const fbfc_recurrence_desc *d)
{
    if (d == nullptr || d->batch < 1 || d->steps < 1 || d->channels < 1) return 0;
    return fbfc::recurrence_checkpoint_bytes(d->batch, d->channels, d->steps);
}

size_t fbfc_recurrence_workspace_bytes(const fbfc_recurrence_desc *d)
{
    if (d == nullptr || d->batch < 1 || d->steps < 1 || d->channels < 1) return 0;
    return fbfc::recurrence_workspace_bytes(d->batch, d->channels, d->steps);
}

int fbfc_recurrence_forward(const fbfc_recurrence_desc *d, const fbfc_steps *input, const fbfc_steps *gate,
                            const float *gate_bias, const float *state_in, const int *lengths, const fbfc_steps *output,
                            float *state_out, float *checkpoints, void *workspace, void *stream)
{
    int rc = recurrence_check_desc(d);
    if (rc != FBFC_OK) return rc;
    fbfc::RecArgs a = {};
    a.batch = d->batch;
    a.channels = d->channels;
    a.steps = d->steps;
    a.x = steps_of(input);
    a.gate = steps_of(gate);
    a.y = steps_of(output);
    a.bias = gate_bias;
    a.state_in = state_in;
    a.lengths = lengths;
    a.state_out = state_out;
    a.checkpoints = checkpoints;
    a.workspace = static_cast<unsigned char *>(workspace);
    if (d->batch == 0) return FBFC_OK;
    if (!aligned32(gate_bias, state_in, lengths, state_out, checkpoints))
        return fail(FBFC_ERR_INVALID_ARGUMENT, "states, lengths and the bias must be aligned to 4 bytes");
    if (d->steps > 0) {
        if (a.x.data == nullptr || a.gate.data == nullptr || a.y.data == nullptr)
            return fail(FBFC_ERR_INVALID_ARGUMENT, "input, gate and output are needed");
        for (const fbfc::Steps *t : {&a.x, &a.gate, &a.y})
            if ((rc = recurrence_check_steps(d, *t, t == &a.y)) != FBFC_OK) return rc;
        if (d->steps > 1 && (workspace == nullptr || !aligned(workspace, 16)))
            return fail(FBFC_ERR_INVALID_ARGUMENT, "a workspace aligned to 16 bytes is needed");
    }
    fbfc::kernel_log_clear();
    FBFC_TRY(fbfc::launch_recurrence_forward(d->type, a, static_cast<hipStream_t>(stream)), "recurrence");
    return FBFC_OK;
}

int fbfc_recurrence_backward(const fbfc_recurrence_desc *d, const fbfc_steps *input, const fbfc_steps *gate,
                             const float *gate_bias, const int *lengths, const float *checkpoints,
                             const fbfc_steps *grad_output, const float *grad_state_out, const fbfc_steps *grad_input,
                             const fbfc_steps *grad_gate, float *grad_gate_bias, float factor, float *grad_state_in,
                             void *workspace, void *stream)
{
    int rc = recurrence_check_desc(d);
    if (rc != FBFC_OK) return rc;
    fbfc::RecArgs a = {};
    a.batch = d->batch;
    a.channels = d->channels;
    a.steps = d->steps;
    a.x = steps_of(input);
    a.gate = steps_of(gate);
    a.y = steps_of(grad_output);
    a.grad_x = steps_of(grad_input);
    a.grad_gate = steps_of(grad_gate);
    a.bias = gate_bias;
    a.state_in = grad_state_out;
    a.lengths = lengths;
    a.state_out = grad_state_in;
    a.checkpoints = const_cast<float *>(checkpoints);
    a.grad_bias = grad_gate_bias;
    a.factor = factor;
    a.workspace = static_cast<unsigned char *>(workspace);
    if (!aligned32(gate_bias, lengths, checkpoints, grad_state_out, grad_gate_bias, grad_state_in))
        return fail(FBFC_ERR_INVALID_ARGUMENT, "states, lengths and the bias must be aligned to 4 bytes");
    if (d->batch > 0 && d->steps > 0) {
        if (a.x.data == nullptr || a.gate.data == nullptr || a.y.data == nullptr || checkpoints == nullptr)
            return fail(FBFC_ERR_INVALID_ARGUMENT, "input, gate, the output's gradient and the checkpoints are needed");
        for (const fbfc::Steps *t : {&a.x, &a.gate, &a.y, &a.grad_x, &a.grad_gate})
            if ((rc = recurrence_check_steps(d, *t, t == &a.grad_x || t == &a.grad_gate)) != FBFC_OK) return rc;
        if (workspace == nullptr || !aligned(workspace, 16))
            return fail(FBFC_ERR_INVALID_ARGUMENT, "a workspace aligned to 16 bytes is needed");
    }
    fbfc::kernel_log_clear();
    FBFC_TRY(fbfc::launch_recurrence_backward(d->type, a, static_cast<hipStream_t>(stream)), "recurrence gradients");
    return FBFC_OK;
}

}  // extern "C"
