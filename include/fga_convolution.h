/*
 * fga_convolution.h - C ABI of the encoder convolution-module entry points of
 * libfga_attention.so (B200, sm_100a): the two depthwise convolutions, and, further down,
 * the group norm with activation and the gated linear recurrence with their backward
 * passes, which have no reference plugin.
 *
 * Each convolution entry point replaces the body of the `enqueue` method of one of the reference's
 * two depthwise-convolution TensorRT plugins, with the same tensor descriptors, binding
 * order, raw device pointers and stream, and the conventions of fga_attention.h (types,
 * status codes, no allocation, one stream, re-validation on every call, a pending CUDA
 * error reported without launching).
 *
 * inputs[0] x             [N, T, C] f32|f16|bf16   (NTC activations after the GLU)
 * inputs[1] valid_lengths [N]       int32          (clamped to [0, T])
 * inputs[2] weight        [K, C]    same type      (depthwise taps, K odd)
 * inputs[3] bias          [C]       same type
 * outputs[0] output       [N, T, C] same type
 *
 * output[n,t,c] = act(bias[c] + sum_k weight[k,c] * x[n, t+k-K/2, c]), where frames at or
 * past the valid length and outside [0, T) contribute zero. Output frames past the valid
 * length are written, not re-masked. f16/bf16 accumulate in the storage type (one fused
 * multiply-add per tap, in tap order, each rounded) and apply the activation in fp32 to the
 * rounded sum; fp32 accumulates in fp32. C must be a multiple of 4 (fp32) or 2 (f16/bf16),
 * and every buffer aligned to two elements (fp32: 8 bytes) - allocations are - else
 * FGA_ERROR_UNSUPPORTED. No workspace (the queries return 0).
 */
#ifndef FGA_CONVOLUTION_H
#define FGA_CONVOLUTION_H

#include "fga_attention.h"

#ifdef __cplusplus
extern "C" {
#endif

/* --------------------------------------------------------------------------------
 * parakeet_conformer_convolution: masked depthwise convolution, BatchNorm folded into
 * weight and bias by the exporter, then SiLU: act(v) = v / (1 + exp(-v)).
 *
 * Replaces ParakeetConvolutionPlugin::enqueue,
 *   src/fast_gpu_asr/tensorrt_plugins/parakeet_convolution_plugin.cu:552-625,
 * with the shape contract of haveValidShapes (same file :85-103) and the type checks of
 * configurePlugin (:403-441). The plugin has no fields.
 * -------------------------------------------------------------------------------- */
FGA_API int32_t fga_parakeet_conformer_convolution_check(const fga_tensor_desc* input_descs,
    int32_t nb_inputs, const fga_tensor_desc* output_descs, int32_t nb_outputs);
FGA_API size_t fga_parakeet_conformer_convolution_workspace_size(
    const fga_tensor_desc* input_descs, int32_t nb_inputs);
FGA_API int32_t fga_parakeet_conformer_convolution_enqueue(const fga_tensor_desc* input_descs,
    const fga_tensor_desc* output_descs, const void* const* inputs, void* const* outputs,
    void* workspace, size_t workspace_bytes, void* stream);

/* --------------------------------------------------------------------------------
 * zipformer_convolution: masked depthwise convolution, then Swoosh-R:
 * act(v) = softplus(v - 1) - 0.08 v - 0.313261687.
 *
 * Replaces ZipformerConvolutionPlugin::enqueue,
 *   src/fast_gpu_asr/tensorrt_plugins/zipformer_convolution_plugin.cu:757-846,
 * with the shape contract of haveValidShapes (same file :130-150). The reference's tactic
 * (block size and frames per thread) does not change results; this entry point takes none.
 * -------------------------------------------------------------------------------- */
FGA_API int32_t fga_zipformer_convolution_check(const fga_tensor_desc* input_descs,
    int32_t nb_inputs, const fga_tensor_desc* output_descs, int32_t nb_outputs);
FGA_API size_t fga_zipformer_convolution_workspace_size(const fga_tensor_desc* input_descs,
    int32_t nb_inputs);
FGA_API int32_t fga_zipformer_convolution_enqueue(const fga_tensor_desc* input_descs,
    const fga_tensor_desc* output_descs, const void* const* inputs, void* const* outputs,
    void* workspace, size_t workspace_bytes, void* stream);

/* --------------------------------------------------------------------------------
 * Group norm with activation, and the gated linear recurrence: no reference plugin.
 *
 * Both work on [N, T, C] activations with the convolutions' valid_lengths (clamped to
 * [0, T]): what padded frames hold is never used (a word of memory that one shares with a
 * valid frame may be read), and every output's padded frames are written as zeros. Conventions that all four entry points share:
 * - "type" is f32, f16 or bf16; arithmetic, statistics, sums and states are fp32, each
 *   output is rounded once.
 * - T is at most 2^30, C at most 2^18, N*T and N*C at most INT32_MAX (N*T*C may be
 *   larger), else FGA_ERROR_OVERFLOW.
 * - Buffers are aligned to their element size and outputs overlap neither inputs nor one
 *   another (one exception is named below), else FGA_ERROR_UNSUPPORTED. 16-byte aligned
 *   buffers with C a multiple of 16 bytes are the fast case.
 * - An optional binding keeps its descriptor; its pointer may be null.
 * - The workspace (bytes from the query, 16-byte aligned) needs no initialisation; a
 *   query of 0 needs none. Two calls in flight at once need two.
 * - Results do not depend on timing: repeated calls give the same bits.
 * -------------------------------------------------------------------------------- */
enum fga_activation {
    FGA_ACTIVATION_NONE = 0,
    FGA_ACTIVATION_SILU = 1,     /* v / (1 + exp(-v)) */
    FGA_ACTIVATION_SWOOSH_R = 2, /* softplus(v - 1) - 0.08 v - 0.313261687 */
};

/* --------------------------------------------------------------------------------
 * group_norm_activation: for convolution modules whose norm takes its statistics from the
 * utterance itself and so cannot be folded into the convolution's weights.
 *
 * inputs[0] x             [N, T, C] type
 * inputs[1] valid_lengths [N]       int32
 * inputs[2] weight        [C]       type
 * inputs[3] bias          [C]       type
 * outputs[0] out          [N, T, C] type
 * outputs[1] mean         [N, G]    f32   (optional)
 * outputs[2] rstd         [N, G]    f32   (optional)
 *
 * Over the valid frames of an utterance and the C/G channels of a group: mean, biased
 * variance, rstd = (variance + eps)^-1/2; out = act((x - mean) rstd weight + bias). An
 * utterance without valid frames has mean 0 and variance 0. num_groups divides C; eps is
 * finite and > 0. Biases may be any number; an infinite or NaN bias and a NaN weight show as
 * the formulas have it. |weight| rstd and |weight (x - mean) rstd| from 2^126 count as
 * infinite.
 * -------------------------------------------------------------------------------- */
FGA_API int32_t fga_group_norm_activation_check(const fga_tensor_desc* input_descs,
    int32_t nb_inputs, const fga_tensor_desc* output_descs, int32_t nb_outputs,
    int32_t num_groups, float eps, int32_t activation);
FGA_API size_t fga_group_norm_activation_workspace_size(const fga_tensor_desc* input_descs,
    int32_t nb_inputs, int32_t num_groups);
FGA_API int32_t fga_group_norm_activation_enqueue(const fga_tensor_desc* input_descs,
    const fga_tensor_desc* output_descs, const void* const* inputs, void* const* outputs,
    int32_t num_groups, float eps, int32_t activation, void* workspace, size_t workspace_bytes,
    void* stream);

/* --------------------------------------------------------------------------------
 * group_norm_activation_backward: the gradients of group_norm_activation.
 *
 * inputs[0] grad_out      [N, T, C] type
 * inputs[1] x             [N, T, C] type
 * inputs[2] valid_lengths [N]       int32
 * inputs[3] weight        [C]       type
 * inputs[4] bias          [C]       type
 * inputs[5] mean          [N, G]    f32   (the forward call's)
 * inputs[6] rstd          [N, G]    f32   (the forward call's)
 * outputs[0] grad_x       [N, T, C] type
 * outputs[1] grad_weight  [C]       type
 * outputs[2] grad_bias    [C]       type
 *
 * grad_weight and grad_bias are the sums over this call's batch (not accumulated).
 * -------------------------------------------------------------------------------- */
FGA_API int32_t fga_group_norm_activation_backward_check(const fga_tensor_desc* input_descs,
    int32_t nb_inputs, const fga_tensor_desc* output_descs, int32_t nb_outputs,
    int32_t activation);
FGA_API size_t fga_group_norm_activation_backward_workspace_size(
    const fga_tensor_desc* input_descs, int32_t nb_inputs);
FGA_API int32_t fga_group_norm_activation_backward_enqueue(const fga_tensor_desc* input_descs,
    const fga_tensor_desc* output_descs, const void* const* inputs, void* const* outputs,
    int32_t activation, void* workspace, size_t workspace_bytes, void* stream);

/* Frames between two states that gated_linear_recurrence saves for its backward pass. */
#define FGA_RECURRENCE_STATE_FRAMES 64

/* --------------------------------------------------------------------------------
 * gated_linear_recurrence: a time mixer with unbounded left context and a constant state.
 *
 * inputs[0] x             [N, T, C] type
 * inputs[1] gate          [N, T, C] type  (logits)
 * inputs[2] valid_lengths [N]       int32
 * inputs[3] initial_state [N, C]    f32   (optional: null is zero)
 * outputs[0] out          [N, T, C] type
 * outputs[1] final_state  [N, C]    f32   (may be the initial_state buffer itself)
 * outputs[2] states       [N, ceil(T/64), C] f32 (optional)
 *
 * f = sigmoid(gate), h[t] = f[t] h[t-1] + (1 - f[t]) x[t], h[-1] = initial_state;
 * out[t] = h[t] on valid frames; final_state is h after the last of them (initial_state
 * when there is none). states[n, j] is h before frame 64 j where that frame is valid, else
 * zero. T = 1 is the streaming step. f is at least 2^-126, which gates below -87.3 reach; the
 * smaller of f and 1 - f is relatively off by up to |gate| 2^-24 on top of some roundings.
 * -------------------------------------------------------------------------------- */
FGA_API int32_t fga_gated_linear_recurrence_check(const fga_tensor_desc* input_descs,
    int32_t nb_inputs, const fga_tensor_desc* output_descs, int32_t nb_outputs);
FGA_API size_t fga_gated_linear_recurrence_workspace_size(const fga_tensor_desc* input_descs,
    int32_t nb_inputs);
FGA_API int32_t fga_gated_linear_recurrence_enqueue(const fga_tensor_desc* input_descs,
    const fga_tensor_desc* output_descs, const void* const* inputs, void* const* outputs,
    void* workspace, size_t workspace_bytes, void* stream);

/* --------------------------------------------------------------------------------
 * gated_linear_recurrence_backward: the gradients of gated_linear_recurrence.
 *
 * inputs[0] grad_out         [N, T, C] type
 * inputs[1] x                [N, T, C] type
 * inputs[2] gate             [N, T, C] type
 * inputs[3] valid_lengths    [N]       int32
 * inputs[4] states           [N, ceil(T/64), C] f32 (the forward call's)
 * inputs[5] grad_final_state [N, C]    f32  (optional: null is zero)
 * outputs[0] grad_x             [N, T, C] type
 * outputs[1] grad_gate          [N, T, C] type
 * outputs[2] grad_initial_state [N, C]    f32
 * -------------------------------------------------------------------------------- */
FGA_API int32_t fga_gated_linear_recurrence_backward_check(const fga_tensor_desc* input_descs,
    int32_t nb_inputs, const fga_tensor_desc* output_descs, int32_t nb_outputs);
FGA_API size_t fga_gated_linear_recurrence_backward_workspace_size(
    const fga_tensor_desc* input_descs, int32_t nb_inputs);
FGA_API int32_t fga_gated_linear_recurrence_backward_enqueue(const fga_tensor_desc* input_descs,
    const fga_tensor_desc* output_descs, const void* const* inputs, void* const* outputs,
    void* workspace, size_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* FGA_CONVOLUTION_H */
