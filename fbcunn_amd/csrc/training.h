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
constexpr int kAdamwPiece = 4096;   // parameters of a piece
constexpr int kAdamwBlock = 256;    // 8-bit states: values that share a scale
// What a step takes from the number of steps before it; on the device, brought up to date by the last workgroup.
struct AdamwClock {
    long t;             // steps taken
    double inv_bias1;   // 1 / (1 - beta1^(t + 1))
    float inv_root2;    // 1 / sqrt(1 - beta2^(t + 1))
    unsigned key;       // of the random numbers of step t + 1
    unsigned done;      // workgroups of the running step that have ended
};
struct AdamwArgs {
    const AdamwPiece *pieces;
    int n_pieces;
    AdamwClock *clock;
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

}  // namespace fbfc
