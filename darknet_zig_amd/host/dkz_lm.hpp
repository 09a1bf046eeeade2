// dkz_lm.hpp -- a token model's operators of libdkz_lm (include/dkz_lm.h) in
// dkz_dense.hpp's manner: the names and argument order of darknet_zig_amd/gpu.py, sizes
// checked into int, a failing call throws dkz::gpu::Error. Header only, C++17; link with
// -ldkz_lm -ldkz. Tensors and workspaces are dkz_dense.hpp's.
#pragma once

#include "dkz_gpu.hpp"
#include "dkz_lm.h"

namespace dkz {
namespace gpu {

inline void mustLm(int err, const char *what) {
    if (err == 0) return;
    std::string msg = std::string(backend_label) + ": " + what + " failed: " + dkz_error_string(err);
    const char *ctx = dkz_lm_last_error_context();
    if (ctx && ctx[0]) msg += std::string(" (") + ctx + ")";
    throw Error(err, msg);
}

inline size_t gatedForwardWorkspace(int type, size_t rows, size_t inputs, size_t hidden) {
    size_t need = 0;
    mustLm(dkz_gated_forward_workspace(type, ci(rows), ci(inputs), ci(hidden), &need), "gated_forward_workspace");
    return need;
}

inline void gatedForward(int type, size_t rows, size_t inputs, size_t hidden, int activation, Buf input, Buf weights, Buf biases, Buf sums,
                         Buf output, Buf workspace) {
    mustLm(dkz_gated_forward(type, ci(rows), ci(inputs), ci(hidden), activation, input.ptr, weights.ptr, biases.f(), sums.ptr, output.ptr,
                             workspace.ptr, 4 * workspace.len),
           "gated_forward");
}

inline size_t gatedBackwardWorkspace(int type, size_t rows, size_t inputs, size_t hidden) {
    size_t need = 0;
    mustLm(dkz_gated_backward_workspace(type, ci(rows), ci(inputs), ci(hidden), &need), "gated_backward_workspace");
    return need;
}

inline void gatedBackward(int type, size_t rows, size_t inputs, size_t hidden, int activation, Buf input, Buf weights, Buf sums, Buf delta,
                          Buf input_residual, float beta, Buf bias_updates, Buf weight_updates, Buf input_delta, Buf workspace) {
    mustLm(dkz_gated_backward(type, ci(rows), ci(inputs), ci(hidden), activation, input.ptr, weights.ptr, sums.ptr, delta.ptr, input_residual.ptr,
                              beta, bias_updates.f(), weight_updates.ptr, input_delta.ptr, workspace.ptr, 4 * workspace.len),
           "gated_backward");
}

inline size_t tokenLogProbsWorkspace(int type, size_t rows, size_t classes, size_t top) {
    size_t need = 0;
    mustLm(dkz_token_log_probs_workspace(type, ci(rows), ci(classes), ci(top), &need), "token_log_probs_workspace");
    return need;
}

inline void tokenLogProbs(int type, size_t rows, size_t classes, size_t pitch, Buf logits, float temperature, size_t given, Buf tokens, size_t top,
                          Buf log_probs, Buf entropy, Buf stats, Buf top_tokens, Buf top_log_probs, Buf workspace) {
    mustLm(dkz_token_log_probs(type, ci(rows), ci(classes), ci(pitch), logits.ptr, temperature, ci(given), static_cast<const int *>(tokens.ptr),
                               ci(top), log_probs.f(), entropy.f(), stats.f(), static_cast<int *>(top_tokens.ptr), top_log_probs.f(),
                               workspace.ptr, 4 * workspace.len),
           "token_log_probs");
}

inline void tokenLogProbsBackward(int type, size_t rows, size_t classes, size_t pitch, Buf logits, float temperature, size_t given, Buf tokens,
                                  Buf stats, Buf entropy, Buf log_prob_deltas, Buf entropy_deltas, float beta, Buf logits_delta) {
    mustLm(dkz_token_log_probs_backward(type, ci(rows), ci(classes), ci(pitch), logits.ptr, temperature, ci(given),
                                        static_cast<const int *>(tokens.ptr), stats.f(), entropy.f(), log_prob_deltas.f(), entropy_deltas.f(),
                                        beta, logits_delta.ptr),
           "token_log_probs_backward");
}

inline size_t distillationWorkspace(int type, size_t rows, size_t classes) {
    size_t need = 0;
    mustLm(dkz_distillation_workspace(type, ci(rows), ci(classes), &need), "distillation_workspace");
    return need;
}

inline void distillation(int type, size_t rows, size_t classes, size_t pitch, Buf logits, float temperature, size_t top, Buf teacher_tokens,
                         Buf teacher_logits, Buf row_scales, float scale, Buf loss, Buf logits_delta, Buf workspace) {
    mustLm(dkz_distillation(type, ci(rows), ci(classes), ci(pitch), logits.ptr, temperature, ci(top),
                            static_cast<const int *>(teacher_tokens.ptr), teacher_logits.f(), row_scales.f(), scale, loss.f(),
                            logits_delta.ptr, workspace.ptr, 4 * workspace.len),
           "distillation");
}

}  // namespace gpu
}  // namespace dkz
