//! dkz_lm.zig -- the C ABI of libdkz_lm.so (include/dkz_lm.h) as Zig `extern fn`
//! declarations, every entry point in the header's order, and one wrapper each in
//! gpu.zig's manner: a token model's operators beside dkz_dense.zig's (gated
//! feed-forward blocks, log probabilities of tokens with the entropy and the top
//! alternatives, distillation). No counterpart in the reference's gpu.zig.
//!
//! Types, tensors and workspaces are dkz_dense.zig's.
//!
//! Link: exe.linkSystemLibrary("dkz_lm") beside "dkz", both in one directory.
const std = @import("std");
const gpu = @import("gpu.zig");

/// hipError_t: 0 on success.
pub const Status = c_int;

/// enum dkz_gate: a gate's activations beside logistic, relu and linear.
pub const silu: c_int = 14;
pub const gelu: c_int = 15;

pub extern fn dkz_lm_last_error_context() [*:0]const u8;
pub extern fn dkz_gated_forward_workspace(type: c_int, rows: c_int, inputs: c_int, hidden: c_int, bytes: *usize) Status;
pub extern fn dkz_gated_forward(type: c_int, rows: c_int, inputs: c_int, hidden: c_int, activation: c_int, input: ?*anyopaque, weights: ?*anyopaque, biases: ?*anyopaque, sums: ?*anyopaque, output: ?*anyopaque, workspace: ?*anyopaque, workspace_bytes: usize) Status;
pub extern fn dkz_gated_backward_workspace(type: c_int, rows: c_int, inputs: c_int, hidden: c_int, bytes: *usize) Status;
pub extern fn dkz_gated_backward(type: c_int, rows: c_int, inputs: c_int, hidden: c_int, activation: c_int, input: ?*anyopaque, weights: ?*anyopaque, sums: ?*anyopaque, delta: ?*anyopaque, input_residual: ?*anyopaque, beta: f32, bias_updates: ?*anyopaque, weight_updates: ?*anyopaque, input_delta: ?*anyopaque, workspace: ?*anyopaque, workspace_bytes: usize) Status;
pub extern fn dkz_token_log_probs_workspace(type: c_int, rows: c_int, classes: c_int, top: c_int, bytes: *usize) Status;
pub extern fn dkz_token_log_probs(type: c_int, rows: c_int, classes: c_int, pitch: c_int, logits: ?*anyopaque, temperature: f32, given: c_int, tokens: ?*anyopaque, top: c_int, log_probs: ?*anyopaque, entropy: ?*anyopaque, stats: ?*anyopaque, top_tokens: ?*anyopaque, top_log_probs: ?*anyopaque, workspace: ?*anyopaque, workspace_bytes: usize) Status;
pub extern fn dkz_token_log_probs_backward(type: c_int, rows: c_int, classes: c_int, pitch: c_int, logits: ?*anyopaque, temperature: f32, given: c_int, tokens: ?*anyopaque, stats: ?*anyopaque, entropy: ?*anyopaque, log_prob_deltas: ?*anyopaque, entropy_deltas: ?*anyopaque, beta: f32, logits_delta: ?*anyopaque) Status;
pub extern fn dkz_distillation_workspace(type: c_int, rows: c_int, classes: c_int, bytes: *usize) Status;
pub extern fn dkz_distillation(type: c_int, rows: c_int, classes: c_int, pitch: c_int, logits: ?*anyopaque, temperature: f32, top: c_int, teacher_tokens: ?*anyopaque, teacher_logits: ?*anyopaque, row_scales: ?*anyopaque, scale: f32, loss: ?*anyopaque, logits_delta: ?*anyopaque, workspace: ?*anyopaque, workspace_bytes: usize) Status;

fn must(err: Status, what: []const u8) void {
    if (err != 0) std.debug.panic("{s}: {s} failed ({d}): {s}", .{ gpu.backend_label, what, err, dkz_lm_last_error_context() });
}

inline fn ci(x: usize) c_int {
    return @intCast(x);
}

/// Bytes of a workspace, in the unit that the ABI counts.
inline fn bytes(b: gpu.Buf) usize {
    return 4 * b.len;
}

pub fn gatedForwardWorkspace(type_code: c_int, rows: usize, inputs: usize, hidden: usize) usize {
    if (!gpu.enabled) unreachable;
    var need: usize = 0;
    must(dkz_gated_forward_workspace(type_code, ci(rows), ci(inputs), ci(hidden), &need), "gated_forward_workspace");
    return need;
}

pub fn gatedForward(type_code: c_int, rows: usize, inputs: usize, hidden: usize, activation: c_int, input: gpu.Buf, weights: gpu.Buf, biases: gpu.Buf, sums: gpu.Buf, output: gpu.Buf, workspace: gpu.Buf) void {
    if (!gpu.enabled) unreachable;
    must(dkz_gated_forward(type_code, ci(rows), ci(inputs), ci(hidden), activation, input.ptr, weights.ptr, biases.ptr, sums.ptr, output.ptr, workspace.ptr, bytes(workspace)), "gated_forward");
}

pub fn gatedBackwardWorkspace(type_code: c_int, rows: usize, inputs: usize, hidden: usize) usize {
    if (!gpu.enabled) unreachable;
    var need: usize = 0;
    must(dkz_gated_backward_workspace(type_code, ci(rows), ci(inputs), ci(hidden), &need), "gated_backward_workspace");
    return need;
}

pub fn gatedBackward(type_code: c_int, rows: usize, inputs: usize, hidden: usize, activation: c_int, input: gpu.Buf, weights: gpu.Buf, sums: gpu.Buf, delta: gpu.Buf, input_residual: gpu.Buf, beta: f32, bias_updates: gpu.Buf, weight_updates: gpu.Buf, input_delta: gpu.Buf, workspace: gpu.Buf) void {
    if (!gpu.enabled) unreachable;
    must(dkz_gated_backward(type_code, ci(rows), ci(inputs), ci(hidden), activation, input.ptr, weights.ptr, sums.ptr, delta.ptr, input_residual.ptr, beta, bias_updates.ptr, weight_updates.ptr, input_delta.ptr, workspace.ptr, bytes(workspace)), "gated_backward");
}

pub fn tokenLogProbsWorkspace(type_code: c_int, rows: usize, classes: usize, top: usize) usize {
    if (!gpu.enabled) unreachable;
    var need: usize = 0;
    must(dkz_token_log_probs_workspace(type_code, ci(rows), ci(classes), ci(top), &need), "token_log_probs_workspace");
    return need;
}

pub fn tokenLogProbs(type_code: c_int, rows: usize, classes: usize, pitch: usize, logits: gpu.Buf, temperature: f32, given: usize, tokens: gpu.Buf, top: usize, log_probs: gpu.Buf, entropy: gpu.Buf, stats: gpu.Buf, top_tokens: gpu.Buf, top_log_probs: gpu.Buf, workspace: gpu.Buf) void {
    if (!gpu.enabled) unreachable;
    must(dkz_token_log_probs(type_code, ci(rows), ci(classes), ci(pitch), logits.ptr, temperature, ci(given), tokens.ptr, ci(top), log_probs.ptr, entropy.ptr, stats.ptr, top_tokens.ptr, top_log_probs.ptr, workspace.ptr, bytes(workspace)), "token_log_probs");
}

pub fn tokenLogProbsBackward(type_code: c_int, rows: usize, classes: usize, pitch: usize, logits: gpu.Buf, temperature: f32, given: usize, tokens: gpu.Buf, stats: gpu.Buf, entropy: gpu.Buf, log_prob_deltas: gpu.Buf, entropy_deltas: gpu.Buf, beta: f32, logits_delta: gpu.Buf) void {
    if (!gpu.enabled) unreachable;
    must(dkz_token_log_probs_backward(type_code, ci(rows), ci(classes), ci(pitch), logits.ptr, temperature, ci(given), tokens.ptr, stats.ptr, entropy.ptr, log_prob_deltas.ptr, entropy_deltas.ptr, beta, logits_delta.ptr), "token_log_probs_backward");
}

pub fn distillationWorkspace(type_code: c_int, rows: usize, classes: usize) usize {
    if (!gpu.enabled) unreachable;
    var need: usize = 0;
    must(dkz_distillation_workspace(type_code, ci(rows), ci(classes), &need), "distillation_workspace");
    return need;
}

pub fn distillation(type_code: c_int, rows: usize, classes: usize, pitch: usize, logits: gpu.Buf, temperature: f32, top: usize, teacher_tokens: gpu.Buf, teacher_logits: gpu.Buf, row_scales: gpu.Buf, scale: f32, loss: gpu.Buf, logits_delta: gpu.Buf, workspace: gpu.Buf) void {
    if (!gpu.enabled) unreachable;
    must(dkz_distillation(type_code, ci(rows), ci(classes), ci(pitch), logits.ptr, temperature, ci(top), teacher_tokens.ptr, teacher_logits.ptr, row_scales.ptr, scale, loss.ptr, logits_delta.ptr, workspace.ptr, bytes(workspace)), "distillation");
}
