// Error reporting of the C entry points: every failure leaves its message in the calling thread's
// fbfc_last_error() and returns its code (api.cpp).
#pragma once
#include <hip/hip_runtime.h>

#include <string>

namespace fbfc {

int fail(int code, const std::string &msg);
int fail_hip(hipError_t e, const char *what);

}  // namespace fbfc

#define FBFC_TRY(expr, what)                                   \
    do {                                                       \
        hipError_t e_ = (expr);                                \
        if (e_ != hipSuccess) return fbfc::fail_hip(e_, what); \
    } while (0)
