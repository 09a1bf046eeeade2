// dkz_dense.hpp -- the fused dense operators of libdkz_dense (include/dkz_dense.h) in
// dkz_gpu.hpp's manner: the names and argument order of darknet_zig_amd/gpu.py,
// sizes checked into int, a failing call throws dkz::gpu::Error. Header only,
// C++17; link with -ldkz_dense -ldkz.
//
// A bf16 tensor of n elements is a Buf of (n + 1) / 2 four-byte elements.
// Workspaces are the caller's, of the bytes that the *Workspace functions say.
#pragma once

#include "dkz_dense.h"
#include "dkz_gpu.hpp"

namespace dkz {
namespace gpu {

inline void mustDense(int err, const char *what) {
    if (err == 0) return;
    std::string msg = std::string(backend_label) + ": " + what + " failed: " + dkz_error_string(err);
    const char *ctx = dkz_dense_last_error_context();
    if (ctx && ctx[0]) msg += std::string(" (") + ctx + ")";
    throw Error(err, msg);
}

// What any call needs, and what the fastest way takes, in bytes.
struct Workspaces {
    size_t least, best;
};

inline void seededDropout(size_t n, int x_type, Buf x, Buf residual, float prob, float scale, unsigned seed, unsigned long long first,
                          int y_type, Buf y) {
    mustDense(dkz_seeded_dropout(ci(n), x_type, x.ptr, residual.ptr, prob, scale, seed, first, y_type, y.ptr), "seeded_dropout");
}

inline size_t linearForwardWorkspace(int type, size_t rows, size_t inputs, size_t outputs) {
    size_t need = 0;
    mustDense(dkz_linear_forward_workspace(type, ci(rows), ci(inputs), ci(outputs), &need), "linear_forward_workspace");
    return need;
}

inline void linearForward(int type, size_t rows, size_t inputs, size_t outputs, int activation, float prob, float scale, unsigned seed,
                          unsigned long long first, Buf input, Buf weights, Buf biases, Buf residual, Buf activated, Buf output,
                          Buf workspace) {
    mustDense(dkz_linear_forward(type, ci(rows), ci(inputs), ci(outputs), activation, prob, scale, seed, first, input.ptr, weights.ptr,
                                 biases.f(), residual.ptr, activated.ptr, output.ptr, workspace.ptr, 4 * workspace.len),
              "linear_forward");
}

inline size_t linearBackwardWorkspace(int type, size_t rows, size_t inputs, size_t outputs) {
    size_t need = 0;
    mustDense(dkz_linear_backward_workspace(type, ci(rows), ci(inputs), ci(outputs), &need), "linear_backward_workspace");
    return need;
}

inline void linearBackward(int type, size_t rows, size_t inputs, size_t outputs, int activation, float prob, float scale, unsigned seed,
                           unsigned long long first, Buf input, Buf weights, Buf activated, Buf delta, Buf input_residual, float beta,
                           Buf bias_updates, Buf weight_updates, Buf input_delta, Buf workspace) {
    mustDense(dkz_linear_backward(type, ci(rows), ci(inputs), ci(outputs), activation, prob, scale, seed, first, input.ptr, weights.ptr,
                                  activated.ptr, delta.ptr, input_residual.ptr, beta, bias_updates.f(), weight_updates.ptr,
                                  input_delta.ptr, workspace.ptr, 4 * workspace.len),
              "linear_backward");
}

inline Workspaces linearCrossEntropyForwardWorkspace(int type, size_t rows, size_t inputs, size_t classes) {
    Workspaces need{0, 0};
    mustDense(dkz_linear_cross_entropy_forward_workspace(type, ci(rows), ci(inputs), ci(classes), &need.least, &need.best),
              "linear_cross_entropy_forward_workspace");
    return need;
}

inline void linearCrossEntropyForward(int type, size_t rows, size_t inputs, size_t classes, Buf input, Buf weights, Buf biases,
                                      Buf targets, Buf loss, Buf lse, Buf workspace) {
    mustDense(dkz_linear_cross_entropy_forward(type, ci(rows), ci(inputs), ci(classes), input.ptr, weights.ptr, biases.f(),
                                               static_cast<const int *>(targets.ptr), loss.f(), lse.f(), workspace.ptr,
                                               4 * workspace.len),
              "linear_cross_entropy_forward");
}

inline Workspaces linearCrossEntropyBackwardWorkspace(int type, size_t rows, size_t inputs, size_t classes) {
    Workspaces need{0, 0};
    mustDense(dkz_linear_cross_entropy_backward_workspace(type, ci(rows), ci(inputs), ci(classes), &need.least, &need.best),
              "linear_cross_entropy_backward_workspace");
    return need;
}

inline void linearCrossEntropyBackward(int type, size_t rows, size_t inputs, size_t classes, Buf input, Buf weights, Buf biases,
                                       Buf targets, Buf lse, Buf row_scales, float scale, float beta, Buf bias_updates,
                                       Buf weight_updates, Buf input_delta, Buf workspace) {
    mustDense(dkz_linear_cross_entropy_backward(type, ci(rows), ci(inputs), ci(classes), input.ptr, weights.ptr, biases.f(),
                                                static_cast<const int *>(targets.ptr), lse.f(), row_scales.f(), scale, beta,
                                                bias_updates.f(), weight_updates.ptr, input_delta.ptr, workspace.ptr,
                                                4 * workspace.len),
              "linear_cross_entropy_backward");
}

}  // namespace gpu
}  // namespace dkz
