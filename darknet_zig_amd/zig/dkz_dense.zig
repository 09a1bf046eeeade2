//! dkz_dense.zig -- the C ABI of libdkz_dense.so (include/dkz_dense.h) as Zig
//! `extern fn` declarations, every entry point in the header's order, and one
//! wrapper each in gpu.zig's manner: the fused dense operators (connected layers
//! with bias, activation, dropout and residual; dropout without a stored mask;
//! softmax cross-entropy without stored logits), beside gpu.zig's own ops. No
//! counterpart in the reference's gpu.zig.
//!
//! Types follow dkz.zig's rules (int -> c_int, float -> f32, device buffers ->
//! ?*anyopaque; unsigned long long -> c_ulonglong). A bf16 tensor of n elements is a
//! Buf of (n + 1) / 2 four-byte elements. Workspaces are the caller's, of the
//! bytes that the *Workspace functions say.
//!
//! Link: exe.linkSystemLibrary("dkz_dense") beside "dkz", both in one directory.
const std = @import("std");
const gpu = @import("gpu.zig");

/// hipError_t: 0 on success.
pub const Status = c_int;

/// enum dkz_type.
pub const f32_type: c_int = 0;
pub const bf16_type: c_int = 1;

pub extern fn dkz_dense_last_error_context() [*:0]const u8;
pub extern fn dkz_seeded_dropout(n: c_int, x_type: c_int, x: ?*anyopaque, residual: ?*anyopaque, prob: f32, scale: f32, seed: c_uint, first: c_ulonglong, y_type: c_int, y: ?*anyopaque) Status;
pub extern fn dkz_linear_forward_workspace(type: c_int, rows: c_int, inputs: c_int, outputs: c_int, bytes: *usize) Status;
pub extern fn dkz_linear_forward(type: c_int, rows: c_int, inputs: c_int, outputs: c_int, activation: c_int, prob: f32, scale: f32, seed: c_uint, first: c_ulonglong, input: ?*anyopaque, weights: ?*anyopaque, biases: ?*anyopaque, residual: ?*anyopaque, activated: ?*anyopaque, output: ?*anyopaque, workspace: ?*anyopaque, workspace_bytes: usize) Status;
pub extern fn dkz_linear_backward_workspace(type: c_int, rows: c_int, inputs: c_int, outputs: c_int, bytes: *usize) Status;
pub extern fn dkz_linear_backward(type: c_int, rows: c_int, inputs: c_int, outputs: c_int, activation: c_int, prob: f32, scale: f32, seed: c_uint, first: c_ulonglong, input: ?*anyopaque, weights: ?*anyopaque, activated: ?*anyopaque, delta: ?*anyopaque, input_residual: ?*anyopaque, beta: f32, bias_updates: ?*anyopaque, weight_updates: ?*anyopaque, input_delta: ?*anyopaque, workspace: ?*anyopaque, workspace_bytes: usize) Status;
pub extern fn dkz_linear_cross_entropy_forward_workspace(type: c_int, rows: c_int, inputs: c_int, classes: c_int, least: *usize, best: *usize) Status;
pub extern fn dkz_linear_cross_entropy_forward(type: c_int, rows: c_int, inputs: c_int, classes: c_int, input: ?*anyopaque, weights: ?*anyopaque, biases: ?*anyopaque, targets: ?*anyopaque, loss: ?*anyopaque, lse: ?*anyopaque, workspace: ?*anyopaque, workspace_bytes: usize) Status;
pub extern fn dkz_linear_cross_entropy_backward_workspace(type: c_int, rows: c_int, inputs: c_int, classes: c_int, least: *usize, best: *usize) Status;
pub extern fn dkz_linear_cross_entropy_backward(type: c_int, rows: c_int, inputs: c_int, classes: c_int, input: ?*anyopaque, weights: ?*anyopaque, biases: ?*anyopaque, targets: ?*anyopaque, lse: ?*anyopaque, row_scales: ?*anyopaque, scale: f32, beta: f32, bias_updates: ?*anyopaque, weight_updates: ?*anyopaque, input_delta: ?*anyopaque, workspace: ?*anyopaque, workspace_bytes: usize) Status;

fn must(err: Status, what: []const u8) void {
    if (err != 0) std.debug.panic("{s}: {s} failed ({d}): {s}", .{ gpu.backend_label, what, err, dkz_dense_last_error_context() });
}

inline fn ci(x: usize) c_int {
    return @intCast(x);
}

/// Bytes of a workspace, in the unit that the ABI counts.
inline fn bytes(b: gpu.Buf) usize {
    return 4 * b.len;
}

/// What any call needs, and what the fastest way takes, in bytes.
pub const Workspaces = struct { least: usize, best: usize };

pub fn seededDropout(n: usize, x_type: c_int, x: gpu.Buf, residual: gpu.Buf, prob: f32, scale: f32, seed: u32, first: u64, y_type: c_int, y: gpu.Buf) void {
    if (!gpu.enabled) unreachable;
    must(dkz_seeded_dropout(ci(n), x_type, x.ptr, residual.ptr, prob, scale, seed, first, y_type, y.ptr), "seeded_dropout");
}

pub fn linearForwardWorkspace(type_code: c_int, rows: usize, inputs: usize, outputs: usize) usize {
    if (!gpu.enabled) unreachable;
    var need: usize = 0;
    must(dkz_linear_forward_workspace(type_code, ci(rows), ci(inputs), ci(outputs), &need), "linear_forward_workspace");
    return need;
}

pub fn linearForward(type_code: c_int, rows: usize, inputs: usize, outputs: usize, activation: c_int, prob: f32, scale: f32, seed: u32, first: u64, input: gpu.Buf, weights: gpu.Buf, biases: gpu.Buf, residual: gpu.Buf, activated: gpu.Buf, output: gpu.Buf, workspace: gpu.Buf) void {
    if (!gpu.enabled) unreachable;
    must(dkz_linear_forward(type_code, ci(rows), ci(inputs), ci(outputs), activation, prob, scale, seed, first, input.ptr, weights.ptr, biases.ptr, residual.ptr, activated.ptr, output.ptr, workspace.ptr, bytes(workspace)), "linear_forward");
}

pub fn linearBackwardWorkspace(type_code: c_int, rows: usize, inputs: usize, outputs: usize) usize {
    if (!gpu.enabled) unreachable;
    var need: usize = 0;
    must(dkz_linear_backward_workspace(type_code, ci(rows), ci(inputs), ci(outputs), &need), "linear_backward_workspace");
    return need;
}

pub fn linearBackward(type_code: c_int, rows: usize, inputs: usize, outputs: usize, activation: c_int, prob: f32, scale: f32, seed: u32, first: u64, input: gpu.Buf, weights: gpu.Buf, activated: gpu.Buf, delta: gpu.Buf, input_residual: gpu.Buf, beta: f32, bias_updates: gpu.Buf, weight_updates: gpu.Buf, input_delta: gpu.Buf, workspace: gpu.Buf) void {
    if (!gpu.enabled) unreachable;
    must(dkz_linear_backward(type_code, ci(rows), ci(inputs), ci(outputs), activation, prob, scale, seed, first, input.ptr, weights.ptr, activated.ptr, delta.ptr, input_residual.ptr, beta, bias_updates.ptr, weight_updates.ptr, input_delta.ptr, workspace.ptr, bytes(workspace)), "linear_backward");
}

pub fn linearCrossEntropyForwardWorkspace(type_code: c_int, rows: usize, inputs: usize, classes: usize) Workspaces {
    if (!gpu.enabled) unreachable;
    var need = Workspaces{ .least = 0, .best = 0 };
    must(dkz_linear_cross_entropy_forward_workspace(type_code, ci(rows), ci(inputs), ci(classes), &need.least, &need.best), "linear_cross_entropy_forward_workspace");
    return need;
}

pub fn linearCrossEntropyForward(type_code: c_int, rows: usize, inputs: usize, classes: usize, input: gpu.Buf, weights: gpu.Buf, biases: gpu.Buf, targets: gpu.Buf, loss: gpu.Buf, lse: gpu.Buf, workspace: gpu.Buf) void {
    if (!gpu.enabled) unreachable;
    must(dkz_linear_cross_entropy_forward(type_code, ci(rows), ci(inputs), ci(classes), input.ptr, weights.ptr, biases.ptr, targets.ptr, loss.ptr, lse.ptr, workspace.ptr, bytes(workspace)), "linear_cross_entropy_forward");
}

pub fn linearCrossEntropyBackwardWorkspace(type_code: c_int, rows: usize, inputs: usize, classes: usize) Workspaces {
    if (!gpu.enabled) unreachable;
    var need = Workspaces{ .least = 0, .best = 0 };
    must(dkz_linear_cross_entropy_backward_workspace(type_code, ci(rows), ci(inputs), ci(classes), &need.least, &need.best), "linear_cross_entropy_backward_workspace");
    return need;
}

pub fn linearCrossEntropyBackward(type_code: c_int, rows: usize, inputs: usize, classes: usize, input: gpu.Buf, weights: gpu.Buf, biases: gpu.Buf, targets: gpu.Buf, lse: gpu.Buf, row_scales: gpu.Buf, scale: f32, beta: f32, bias_updates: gpu.Buf, weight_updates: gpu.Buf, input_delta: gpu.Buf, workspace: gpu.Buf) void {
    if (!gpu.enabled) unreachable;
    must(dkz_linear_cross_entropy_backward(type_code, ci(rows), ci(inputs), ci(classes), input.ptr, weights.ptr, biases.ptr, targets.ptr, lse.ptr, row_scales.ptr, scale, beta, bias_updates.ptr, weight_updates.ptr, input_delta.ptr, workspace.ptr, bytes(workspace)), "linear_cross_entropy_backward");
}
