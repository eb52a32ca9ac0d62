// Internal launch interface of the training and serving operators (training_api.cpp and their kernels).
#pragma once
#include <hip/hip_runtime.h>

#include "act.h"

namespace fbfc {

// adamw_kernels.hip ----------------------------------------------------------------
// A piece of one tensor: n parameters and gradients, whose states begin at `first` (a multiple of 256).
struct AdamwPiece {
    void *param;
    const void *grad;
    long first;
    long n;
};
// Parameters of a piece: enough for a workgroup to hold all its loads in flight, or, where that leaves CUs
// without a piece (below 2048 pieces), as few as one load each.
constexpr int kAdamwPiece = 4096, kAdamwSmallPiece = 1024;
constexpr int kAdamwBlock = 256;    // 8-bit states: values that share a scale
// What a step takes from the number of steps before it; on the device, brought up to date by the last workgroup.
struct AdamwClock {
    long t;             // steps taken
    double power1, power2;  // beta1^(t + 1), beta2^(t + 1)
    double inv_bias1;   // 1 / (1 - beta1^(t + 1))
    float inv_root2;    // 1 / sqrt(1 - beta2^(t + 1))
    unsigned key;       // of the random numbers of step t + 1
    unsigned done;      // lines of AdamwArgs::ended that are complete
};
// Workgroups of the running step that have ended, counted on lines of their own: additions to one address follow each
// other 10 ns apart, and 2048 of them would take longer than a short step.
constexpr int kAdamwLines = 32, kAdamwLine = 16;   // values of a line
struct AdamwArgs {
    const AdamwPiece *pieces;
    int n_pieces;
    AdamwClock *clock;
    unsigned *ended;   // kAdamwLines lines, all zero between steps
    void *m, *v;
    float *m_scale, *v_scale;
    double beta1, beta2;
    unsigned seed;
    float keep1, take1, keep2, take2;  // beta1, 1 - beta1, beta2, 1 - beta2
    float eps;
    double lr;
    float decay;       // 1 - lr * weight_decay
    float grad_scale;
};
AdamwClock adamw_clock(long t, double beta1, double beta2, unsigned seed);
hipError_t launch_adamw(int param_type, int grad_type, int state_bits, const AdamwArgs &a, hipStream_t s);
hipError_t launch_adamw_set_clock(const AdamwArgs &a, long t, hipStream_t s);

// norm_kernels.hip ------------------------------------------------------------------
// Rows of one activation tensor: element (r, c) lies r * stride + c values from `data`; absent where data is null.
struct Rows {
    void *data;
    long stride;
};
struct NormArgs {
    long rows;
    int channels;
    float eps;
    Rows residual, branch, gate;
    const float *post, *scale, *pre;      // with a branch: the first two; with a norm behind it: the last
    Rows output, normed;                  // forward
    Rows grad_output, grad_normed;        // backward
    Rows grad_residual, grad_branch, grad_gate;
    float *grad_post, *grad_scale, *grad_pre;
    float factor;                         // of the three gradients above
    float *partial;                       // norm_workspace_bytes
};
constexpr int kNormMaxChannels = 16384;
size_t norm_workspace_bytes(long rows, int channels, int type);
hipError_t launch_norm_forward(int type, const NormArgs &a, hipStream_t s);
hipError_t launch_norm_backward(int type, const NormArgs &a, hipStream_t s);

// recurrence_kernels.hip -------------------------------------------------------------
// One activation tensor over (batch, step, channel), strides in values; absent where data is null.
struct Steps {
    void *data;
    long sb, st, sc;
};
struct RecArgs {
    int batch, channels;
    long steps;
    Steps x, gate, y;              // y: the output, or the gradient of the output
    Steps grad_x, grad_gate;
    const float *bias;
    const int *lengths;
    const float *state_in;         // backward: the gradient of the state behind the last step
    float *state_out;              // backward: the gradient of the state before the first step
    float *checkpoints;            // the state before each tile of steps: (tiles, batch, channels)
    float *grad_bias;
    float factor;                  // of grad_bias
    unsigned char *workspace;
};
size_t recurrence_checkpoint_bytes(int batch, int channels, long steps);
size_t recurrence_workspace_bytes(int batch, int channels, long steps);
bool recurrence_fits(int batch, int channels, long steps);
hipError_t launch_recurrence_forward(int type, const RecArgs &a, hipStream_t s);
hipError_t launch_recurrence_backward(int type, const RecArgs &a, hipStream_t s);

}  // namespace fbfc
