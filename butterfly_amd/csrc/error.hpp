// The thread's last error message, shared by the entry points of all files.
#pragma once

namespace bf {

// Stores the message for bf_last_error() and returns `code`.
int fail(int code, const char *fmt, ...) __attribute__((format(printf, 2, 3)));

}  // namespace bf

#define BF_HIP_CHECK(expr)                                                              \
    do {                                                                                \
        hipError_t e_ = (expr);                                                         \
        if (e_ != hipSuccess)                                                           \
            return bf::fail(BF_ERR_HIP, "%s failed: %s", #expr, hipGetErrorString(e_)); \
    } while (0)
