// host.h -- what the library's source files share on the host: the error text of spanqr_last_error and the check of a
// HIP runtime call.
#ifndef SPANQR_HOST_H
#define SPANQR_HOST_H

#include <hip/hip_runtime.h>

#include <stdarg.h>
#include <stdio.h>

#include "../../include/spanqr.h"

namespace spanqr_host {

// keeps `text` for spanqr_last_error of this thread and returns `code`; defined in spanqr.hip
__attribute__((visibility("hidden"))) int set_error(int code, const char* text) noexcept;

__attribute__((format(printf, 2, 3))) inline int error(int code, const char* fmt, ...) noexcept {
    char buf[512];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(buf, sizeof buf, fmt, ap);
    va_end(ap);
    return set_error(code, buf);
}

// the launches before it are enqueued; a launch that was refused shows here
inline int launched(const char* what) noexcept {
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? SPANQR_OK : error(SPANQR_EHIP, "%s: %s", what, hipGetErrorString(e));
}

}  // namespace spanqr_host

#endif  // SPANQR_HOST_H
