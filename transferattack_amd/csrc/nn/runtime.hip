// Error reporting and ABI bookkeeping of libta_nn.so.
#include <stdarg.h>
#include <stdio.h>
#include "ta_nn_common.h"

namespace ta_nn {

static thread_local char g_error[512] = "";

void set_error(const char* fmt, ...) {
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(g_error, sizeof(g_error), fmt, ap);
    va_end(ap);
}

int check_launch(const char* what) {
    const hipError_t err = hipGetLastError();
    if (err != hipSuccess) {
        set_error("%s: %s", what, hipGetErrorString(err));
        return static_cast<int>(err);
    }
    return 0;
}

}  // namespace ta_nn

extern "C" int ta_nn_abi_version(void) { return TA_NN_ABI_VERSION; }
extern "C" const char* ta_nn_last_error(void) { return ta_nn::g_error; }
