// runtime.hip -- dkz_internal.hpp's plumbing for libdkz_dense.so: the stream
// and the sync-after-launch switch are libdkz.so's, read through its public
// entry points; the error context is this library's own.
#include <stdarg.h>
#include <stdio.h>

#include "dense_internal.hpp"

namespace dkz {
namespace {
thread_local char g_context[512] = "";
}

hipStream_t current_stream() { return static_cast<hipStream_t>(dkz_get_stream()); }

bool sync_after_launch() { return dkz_get_sync_after_launch() != 0; }

void set_error_context(const char *fmt, ...) {
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(g_context, sizeof g_context, fmt, ap);
    va_end(ap);
}

int after_launch(const char *name, dim3 grid, dim3 block, hipStream_t stream) {
    hipError_t e = hipGetLastError();
    const char *what = "launching";
    if (e == hipSuccess && sync_after_launch()) {
        e = hipStreamSynchronize(stream);
        what = "running";
    }
    if (e != hipSuccess)
        set_error_context("HIP: %s %s <<<(%u,%u),(%u,%u)>>> failed: %s", what, name, grid.x, grid.y, block.x, block.y,
                          hipGetErrorString(e));
    return (int)e;
}

}  // namespace dkz

extern "C" const char *dkz_dense_last_error_context(void) { return dkz::g_context; }
