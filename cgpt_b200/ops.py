"""Host-side mirror of CGPT's operator API for the training hot path.

Each function has the name, argument order (outputs first, then inputs, then ``stream``, then the
options object) and error behaviour of the C++ function it stands for; ``ValueError`` plays the role
of ``std::invalid_argument``. Tensors are ``torch`` CUDA tensors used purely as device-memory handles;
all arithmetic happens in ``libcgpt_b200.so`` through the C ABI.

Reference declarations: ``include/ops/backward/*.h``, ``include/ops/{rmsnorm,rope,swiglu,embedding,
cross_entropy,cut_cross_entropy}.h``. The operators of the pre-norm block (dropout, layer norm, the two fused with the residual
add, scaled embedding) have no counterpart there and follow the same conventions.
"""
from __future__ import annotations

from dataclasses import dataclass

import torch

from . import _lib
from ._lib import check, dtype_code, lib, ptr, stream_ptr


@dataclass
class RopeOptions:
    """include/ops/rope.h:6-11"""
    rotary_dim: int = 0
    position_offset: int = 0


@dataclass
class SwiGLUBackwardOptions:
    """include/ops/backward/swiglu_backward.h:6-13"""
    accumulate_gate: bool = False
    accumulate_up: bool = False
    accumulate_gate_up: bool = False


@dataclass
class EmbeddingBackwardOptions:
    """include/ops/backward/embedding_backward.h:6-14"""
    block_size: int = 0
    bounds_check: bool = True
    accumulate_weight: bool = False


def _require(cond: bool, message: str) -> None:
    if not cond:
        raise _lib.CgptInvalidArgument(message)


def _same_cuda_dtype(name: str, *tensors: torch.Tensor) -> None:
    first = tensors[0]
    for t in tensors:
        _require(t.is_cuda, f"{name}: all tensors must be CUDA tensors")
        _require(t.dtype == first.dtype, f"{name}: all tensors must share one dtype")
        _require(t.is_contiguous(), f"{name}: tensors must be contiguous")


def _ids(t: torch.Tensor, count: int, name: str) -> torch.Tensor:
    _require(t is not None and t.is_cuda, f"{name}: token ids must be a CUDA buffer")
    _require(t.dtype in (torch.int32, torch.uint32), f"{name}: token ids must be 32-bit")
    _require(t.numel() >= count, f"{name}: token id buffer too small")
    return t


# ---------------------------------------------------------------------------------------------- Linear
@dataclass
class LinearBackwardOptions:
    """include/ops/backward/linear_backward.h:10-21 (compute_type / workspace_bytes are accepted and
    ignored: accumulation is always fp32 and scratch comes from the library's arena)."""
    compute_type: str = "F32"
    workspace_bytes: int = 32 * 1024 * 1024
    accumulate_input: bool = False
    accumulate_weight: bool = False
    accumulate_bias: bool = False


def linear_forward(output, input, weight, cublas_lt_context=None, stream=None, options=None):
    """linear_forward(output, input, weight, context, stream, options): Y = X W^T (include/ops/linear.h)."""
    _same_cuda_dtype("linear_forward", output, input, weight)
    _require(weight.dim() == 2 and input.shape[-1] == weight.shape[1] and output.shape[-1] == weight.shape[0]
             and output.numel() // weight.shape[0] == input.numel() // weight.shape[1],
             "linear_forward: incompatible shapes")
    rows = input.numel() // weight.shape[1]
    check(lib.cgpt_linear_forward(ptr(output), ptr(input), ptr(weight), rows, weight.shape[1], weight.shape[0],
                                  dtype_code(input), stream_ptr(stream)), "linear_forward")


def linear_backward(grad_input, grad_weight, grad_bias, grad_output, input, weight, cublas_lt_context=None,
                    stream=None, options: LinearBackwardOptions | None = None):
    """linear_backward (include/ops/backward/linear_backward.h:36-46). Any of grad_input / grad_weight /
    grad_bias may be None to skip that product (extension; the reference always computes all three)."""
    o = options or LinearBackwardOptions()
    outs = [t for t in (grad_input, grad_weight, grad_bias) if t is not None]
    _same_cuda_dtype("linear_backward", grad_output, input, weight, *outs)
    out_f, in_f = weight.shape
    rows = input.numel() // in_f
    _require(weight.dim() == 2 and input.shape[-1] == in_f and grad_output.shape[-1] == out_f
             and grad_output.numel() == rows * out_f, "linear_backward: incompatible shapes")
    _require(grad_input is None or grad_input.shape == input.shape, "linear_backward: grad_input shape")
    _require(grad_weight is None or grad_weight.shape == weight.shape, "linear_backward: grad_weight shape")
    _require(grad_bias is None or tuple(grad_bias.shape) == (out_f,), "linear_backward: grad_bias shape")
    check(lib.cgpt_linear_backward(ptr(grad_input), ptr(grad_weight), ptr(grad_bias), ptr(grad_output), ptr(input),
                                   ptr(weight), rows, in_f, out_f, int(o.accumulate_input), int(o.accumulate_weight),
                                   int(o.accumulate_bias), dtype_code(input), stream_ptr(stream)), "linear_backward")


def linear_forward_fused(outputs, input, weights, stream=None):
    """outputs[i] = input @ weights[i].T for up to three projections of one input, as one launch
    (cgpt_linear_forward_fused; the reference calls linear_forward once per projection)."""
    import ctypes as C
    n = len(outputs)
    _require(1 <= n <= 3 and len(weights) == n, "linear_forward_fused: 1..3 projections")
    _same_cuda_dtype("linear_forward_fused", input, *outputs, *weights)
    in_f = input.shape[-1]
    rows = input.numel() // in_f
    for y, w in zip(outputs, weights):
        _require(w.dim() == 2 and w.shape[1] == in_f and y.shape[-1] == w.shape[0] and y.numel() == rows * w.shape[0],
                 "linear_forward_fused: incompatible shapes")
    ys = (C.c_void_p * n)(*[ptr(t) for t in outputs])
    ws = (C.c_void_p * n)(*[ptr(t) for t in weights])
    outs = (C.c_size_t * n)(*[w.shape[0] for w in weights])
    check(lib.cgpt_linear_forward_fused(ys, ptr(input), ws, outs, n, rows, in_f, dtype_code(input), stream_ptr(stream)),
          "linear_forward_fused")


def linear_backward_weight_fused(grad_weights, grad_outputs, input, stream=None, accumulate_weight: bool = False):
    """grad_weights[i] (+)= grad_outputs[i].T @ input for up to three projections of one input, as one launch
    (cgpt_linear_backward_weight_fused; the reference runs one linear_backward per projection)."""
    import ctypes as C
    n = len(grad_weights)
    _require(1 <= n <= 3 and len(grad_outputs) == n, "linear_backward_weight_fused: 1..3 projections")
    _same_cuda_dtype("linear_backward_weight_fused", input, *grad_weights, *grad_outputs)
    in_f = input.shape[-1]
    rows = input.numel() // in_f
    for gw, dy in zip(grad_weights, grad_outputs):
        _require(gw.dim() == 2 and gw.shape[1] == in_f and dy.shape[-1] == gw.shape[0] and dy.numel() == rows * gw.shape[0],
                 "linear_backward_weight_fused: incompatible shapes")
    gws = (C.c_void_p * n)(*[ptr(t) for t in grad_weights])
    dys = (C.c_void_p * n)(*[ptr(t) for t in grad_outputs])
    outs = (C.c_size_t * n)(*[gw.shape[0] for gw in grad_weights])
    check(lib.cgpt_linear_backward_weight_fused(gws, dys, ptr(input), outs, n, rows, in_f, int(accumulate_weight),
                                                dtype_code(input), stream_ptr(stream)), "linear_backward_weight_fused")


def linear_swiglu_forward(gate, up, activated, input, gate_weight, up_weight, stream=None):
    """gate = input @ gate_weight.T, up = input @ up_weight.T, activated = swiglu(gate, up) in one launch
    (cgpt_linear_swiglu_forward; the reference's block forward calls linear_forward twice and swiglu_forward)."""
    _same_cuda_dtype("linear_swiglu_forward", gate, up, activated, input, gate_weight, up_weight)
    inter, in_f = gate_weight.shape
    rows = input.numel() // in_f
    _require(up_weight.shape == gate_weight.shape and input.shape[-1] == in_f
             and all(t.numel() == rows * inter and t.shape[-1] == inter for t in (gate, up, activated)),
             "linear_swiglu_forward: incompatible shapes")
    check(lib.cgpt_linear_swiglu_forward(ptr(gate), ptr(up), ptr(activated), ptr(input), ptr(gate_weight), ptr(up_weight),
                                         rows, in_f, inter, dtype_code(input), stream_ptr(stream)), "linear_swiglu_forward")


def linear_backward_input_fused(grad_input, grad_outputs, weights, stream=None, accumulate_input: bool = False):
    """grad_input (+)= sum_i grad_outputs[i] @ weights[i] for up to three projections of the same input, in one
    pass (cgpt_linear_backward_input_fused; the reference runs one accumulating linear_backward per projection)."""
    import ctypes as C
    n = len(grad_outputs)
    _require(1 <= n <= 3 and len(weights) == n, "linear_backward_input_fused: 1..3 projections")
    _same_cuda_dtype("linear_backward_input_fused", grad_input, *grad_outputs, *weights)
    in_f = grad_input.shape[-1]
    rows = grad_input.numel() // in_f
    for dy, w in zip(grad_outputs, weights):
        _require(w.dim() == 2 and w.shape[1] == in_f and dy.shape[-1] == w.shape[0] and dy.numel() == rows * w.shape[0],
                 "linear_backward_input_fused: incompatible shapes")
    dys = (C.c_void_p * n)(*[ptr(t) for t in grad_outputs])
    ws = (C.c_void_p * n)(*[ptr(t) for t in weights])
    outs = (C.c_size_t * n)(*[w.shape[0] for w in weights])
    check(lib.cgpt_linear_backward_input_fused(ptr(grad_input), dys, ws, outs, n, rows, in_f, int(accumulate_input),
                                               dtype_code(grad_input), stream_ptr(stream)), "linear_backward_input_fused")


def linear_forward_sum(output, inputs, weights, residual=None, stream=None):
    """output = residual + sum_i inputs[i] @ weights[i].T for up to three projections into the same output, in one pass
    (cgpt_linear_forward_sum; the end of the reference's parallel-residual block is two projections and two adds)."""
    import ctypes as C
    n = len(inputs)
    _require(1 <= n <= 3 and len(weights) == n, "linear_forward_sum: 1..3 projections")
    _same_cuda_dtype("linear_forward_sum", output, *inputs, *weights, *([residual] if residual is not None else []))
    out_f = output.shape[-1]
    rows = output.numel() // out_f
    for x, w in zip(inputs, weights):
        _require(w.dim() == 2 and w.shape[0] == out_f and x.shape[-1] == w.shape[1] and x.numel() == rows * w.shape[1],
                 "linear_forward_sum: incompatible shapes")
    _require(residual is None or residual.shape == output.shape, "linear_forward_sum: residual must have the output's shape")
    xs = (C.c_void_p * n)(*[ptr(t) for t in inputs])
    ws = (C.c_void_p * n)(*[ptr(t) for t in weights])
    ins = (C.c_size_t * n)(*[w.shape[1] for w in weights])
    check(lib.cgpt_linear_forward_sum(ptr(output), xs, ws, ins, n, rows, out_f, ptr(residual) if residual is not None else None,
                                      dtype_code(output), stream_ptr(stream)), "linear_forward_sum")


def gemm(c, a, b, m, n, k, a_layout=0, b_layout=0, accumulate=False, force_simt=False, stream=None):
    """Raw contraction C[m,n] (+)= A B of the library (see cgpt_gemm in include/cgpt_b200.h)."""
    _same_cuda_dtype("gemm", c, a, b)
    check(lib.cgpt_gemm(ptr(c), ptr(a), ptr(b), m, n, k, a_layout, b_layout, int(accumulate), dtype_code(c),
                        int(force_simt), stream_ptr(stream)), "gemm")


# ------------------------------------------------------------------------------------------- Attention
@dataclass
class FlashAttentionOptions:
    """include/ops/attention.h:8-32 (key_tile_size, block_size and use_tensor_cores are accepted and
    ignored by the backward, as in the reference)."""
    num_query_heads: int = 0
    num_kv_heads: int = 0
    head_dim: int = 0
    attention_scale: float = 0.0
    causal: bool = True
    query_position_offset: int = 0
    key_tile_size: int = 16
    block_size: int = 128
    use_tensor_cores: bool = True


def _attn_check(name, q, k, v, o: FlashAttentionOptions, *same_as_q, same_as_k=()):
    _same_cuda_dtype(name, q, k, v, *same_as_q, *same_as_k)
    _require(q.dim() == 4 and k.dim() == 4 and v.shape == k.shape and all(t.shape == q.shape for t in same_as_q)
             and all(t.shape == k.shape for t in same_as_k), f"{name}: invalid gradient or operand shape")
    _require(o.num_query_heads > 0 and o.num_kv_heads > 0 and o.head_dim > 0
             and o.num_query_heads % o.num_kv_heads == 0 and q.shape[2] == o.num_query_heads
             and k.shape[2] == o.num_kv_heads and q.shape[3] == o.head_dim and k.shape[3] == o.head_dim
             and q.shape[0] == k.shape[0], f"{name}: invalid attention configuration")
    _require(o.attention_scale >= 0 and o.attention_scale == o.attention_scale
             and not (o.causal and o.query_position_offset + q.shape[1] > k.shape[1]),
             f"{name}: invalid scale or causal range")


def flash_gqa_attention_forward_with_lse(output, logsumexp, query, key, value, stream=None,
                                         options: FlashAttentionOptions | None = None, force_generic=False):
    """flash_gqa_attention_forward_with_lse (include/ops/attention.h:60-81)."""
    o = options or FlashAttentionOptions()
    _attn_check("flash_gqa_attention_forward", query, key, value, o, output)
    _require(logsumexp is None or (logsumexp.dtype == torch.float32 and logsumexp.is_cuda
                                   and tuple(logsumexp.shape) == tuple(query.shape[:3])),
             "flash_gqa_attention_forward: logsumexp must be F32 [batch, seq, heads]")
    b, sq, hq, d = query.shape
    check(lib.cgpt_attention_forward(ptr(output), ptr(logsumexp), ptr(query), ptr(key), ptr(value), b, sq, key.shape[1],
                                     hq, key.shape[2], d, float(o.attention_scale), int(o.causal),
                                     o.query_position_offset, dtype_code(query), int(force_generic),
                                     stream_ptr(stream)), "flash_gqa_attention_forward_with_lse")


def flash_gqa_attention_backward_with_lse(grad_query, grad_key, grad_value, grad_output, output, logsumexp, query,
                                          key, value, stream=None, options: FlashAttentionOptions | None = None,
                                          accumulate_grads=False, force_generic=False):
    """flash_gqa_attention_backward_with_lse (include/ops/backward/attention_backward.h:57-70)."""
    o = options or FlashAttentionOptions()
    _attn_check("flash_gqa_attention_backward", query, key, value, o, grad_query, grad_output, output,
                same_as_k=(grad_key, grad_value))
    _require(logsumexp.dtype == torch.float32 and tuple(logsumexp.shape) == tuple(query.shape[:3]),
             "flash_gqa_attention_backward: logsumexp must be F32 [batch, seq, heads]")
    b, sq, hq, d = query.shape
    check(lib.cgpt_attention_backward(ptr(grad_query), ptr(grad_key), ptr(grad_value), ptr(grad_output), ptr(output),
                                      ptr(logsumexp), ptr(query), ptr(key), ptr(value), b, sq, key.shape[1], hq,
                                      key.shape[2], d, float(o.attention_scale), int(o.causal),
                                      o.query_position_offset, int(accumulate_grads), dtype_code(query),
                                      int(force_generic), stream_ptr(stream)), "flash_gqa_attention_backward_with_lse")


def flash_gqa_attention_backward(grad_query, grad_key, grad_value, grad_output, query, key, value, stream=None,
                                 options: FlashAttentionOptions | None = None, accumulate_grads=False):
    """flash_gqa_attention_backward without saved statistics (attention_backward.h:24-35)."""
    o = options or FlashAttentionOptions()
    _attn_check("flash_gqa_attention_backward", query, key, value, o, grad_query, grad_output,
                same_as_k=(grad_key, grad_value))
    b, sq, hq, d = query.shape
    check(lib.cgpt_attention_backward(ptr(grad_query), ptr(grad_key), ptr(grad_value), ptr(grad_output), None, None,
                                      ptr(query), ptr(key), ptr(value), b, sq, key.shape[1], hq, key.shape[2], d,
                                      float(o.attention_scale), int(o.causal), o.query_position_offset,
                                      int(accumulate_grads), dtype_code(query), 1, stream_ptr(stream)),
          "flash_gqa_attention_backward")


# --------------------------------------------------------------------------------------------- RMSNorm
def rmsnorm_forward(output, input, weight, epsilon, stream=None):
    """rmsnorm_forward(Tensor& output, const Tensor& input, const Tensor& weight, float eps, stream)."""
    _same_cuda_dtype("rmsnorm_forward", output, input, weight)
    _require(input.dim() == 2 and output.shape == input.shape and weight.dim() == 1
             and weight.shape[0] == input.shape[1], "rmsnorm_forward: incompatible shapes")
    check(lib.cgpt_rmsnorm_forward(ptr(output), ptr(input), ptr(weight), input.shape[0], input.shape[1],
                                   float(epsilon), dtype_code(input), stream_ptr(stream)), "rmsnorm_forward")


def rmsnorm_backward(grad_input, grad_weight, grad_output, input, weight, epsilon, stream=None,
                     residual_a=None, residual_b=None):
    """rmsnorm_backward (include/ops/backward/rmsnorm_backward.h:21-29). ``residual_a/b`` are this
    library's extension: tensors added to grad_input inside the kernel."""
    extra = [t for t in (residual_a, residual_b) if t is not None]
    _same_cuda_dtype("rmsnorm_backward", grad_input, grad_weight, grad_output, input, weight, *extra)
    _require(input.dim() == 2 and grad_output.shape == input.shape and grad_input.shape == input.shape
             and weight.dim() == 1 and weight.shape[0] == input.shape[1] and grad_weight.shape == weight.shape
             and all(t.shape == input.shape for t in extra), "rmsnorm_backward: incompatible shapes")
    check(lib.cgpt_rmsnorm_backward(ptr(grad_input), ptr(grad_weight), ptr(grad_output), ptr(input), ptr(weight),
                                    ptr(residual_a), ptr(residual_b), input.shape[0], input.shape[1],
                                    float(epsilon), dtype_code(input), stream_ptr(stream)), "rmsnorm_backward")


def rmsnorm_forward_dual(output_a, output_b, input, weight_a, weight_b, epsilon, stream=None):
    """Both RMSNorms of a parallel-residual block's input in one pass over it (cgpt_rmsnorm_forward_dual)."""
    _same_cuda_dtype("rmsnorm_forward_dual", output_a, output_b, input, weight_a, weight_b)
    _require(input.dim() == 2 and output_a.shape == input.shape and output_b.shape == input.shape and weight_a.dim() == 1
             and weight_a.shape[0] == input.shape[1] and weight_b.shape == weight_a.shape, "rmsnorm_forward_dual: incompatible shapes")
    check(lib.cgpt_rmsnorm_forward_dual(ptr(output_a), ptr(output_b), ptr(input), ptr(weight_a), ptr(weight_b), input.shape[0],
                                        input.shape[1], float(epsilon), dtype_code(input), stream_ptr(stream)), "rmsnorm_forward_dual")


def rmsnorm_backward_dual(grad_input, grad_weight_a, grad_weight_b, grad_output_a, grad_output_b, input, weight_a, weight_b,
                          epsilon, residual=None, stream=None):
    """grad_input = residual + the input gradients of both norms of the same input, and both weight gradients, in one
    pass (cgpt_rmsnorm_backward_dual)."""
    extra = [residual] if residual is not None else []
    _same_cuda_dtype("rmsnorm_backward_dual", grad_input, grad_weight_a, grad_weight_b, grad_output_a, grad_output_b, input,
                     weight_a, weight_b, *extra)
    _require(input.dim() == 2 and all(t.shape == input.shape for t in (grad_input, grad_output_a, grad_output_b, *extra))
             and weight_a.dim() == 1 and weight_a.shape[0] == input.shape[1]
             and all(t.shape == weight_a.shape for t in (weight_b, grad_weight_a, grad_weight_b)),
             "rmsnorm_backward_dual: incompatible shapes")
    check(lib.cgpt_rmsnorm_backward_dual(ptr(grad_input), ptr(grad_weight_a), ptr(grad_weight_b), ptr(grad_output_a),
                                         ptr(grad_output_b), ptr(input), ptr(weight_a), ptr(weight_b), ptr(residual),
                                         input.shape[0], input.shape[1], float(epsilon), dtype_code(input), stream_ptr(stream)),
          "rmsnorm_backward_dual")


# ------------------------------------------------------------------------------------------------ RoPE
def _rope_dims(q, k, cos_cache, sin_cache, opts, name):
    _require(q.dim() == 4 and k.dim() == 4 and q.shape[0] == k.shape[0] and q.shape[1] == k.shape[1]
             and q.shape[3] == k.shape[3], f"{name}: query/key must be [batch, seq, heads, head_dim]")
    rotary = opts.rotary_dim or q.shape[3]
    _require(rotary <= q.shape[3] and rotary % 2 == 0, f"{name}: invalid rotary_dim")
    _require(cos_cache.dim() == 2 and sin_cache.shape == cos_cache.shape and cos_cache.shape[1] == rotary // 2,
             f"{name}: caches must be [max_seq, rotary_dim/2]")
    _require(opts.position_offset + q.shape[1] <= cos_cache.shape[0], f"{name}: position exceeds cache")
    return rotary


def rope_forward(query, key, cos_cache, sin_cache, stream=None, rope_options: RopeOptions | None = None):
    """rope_forward: rotates query and key in place (include/ops/rope.h:13-39)."""
    opts = rope_options or RopeOptions()
    _same_cuda_dtype("rope_forward", query, key, cos_cache, sin_cache)
    rotary = _rope_dims(query, key, cos_cache, sin_cache, opts, "rope_forward")
    b, s, hq, d = query.shape
    check(lib.cgpt_rope_forward(ptr(query), ptr(key), ptr(cos_cache), ptr(sin_cache), b, s, hq, key.shape[2], d,
                                rotary, opts.position_offset, cos_cache.shape[0], dtype_code(query),
                                stream_ptr(stream)), "rope_forward")


def rope_backward(grad_query, grad_key, grad_rotated_query, grad_rotated_key, cos_cache, sin_cache, stream=None,
                  rope_options: RopeOptions | None = None):
    """rope_backward (include/ops/backward/rope_backward.h:22-31)."""
    opts = rope_options or RopeOptions()
    _same_cuda_dtype("rope_backward", grad_query, grad_key, grad_rotated_query, grad_rotated_key, cos_cache,
                     sin_cache)
    _require(grad_query.shape == grad_rotated_query.shape and grad_key.shape == grad_rotated_key.shape,
             "rope_backward: gradient shapes differ")
    rotary = _rope_dims(grad_query, grad_key, cos_cache, sin_cache, opts, "rope_backward")
    b, s, hq, d = grad_query.shape
    check(lib.cgpt_rope_backward(ptr(grad_query), ptr(grad_key), ptr(grad_rotated_query), ptr(grad_rotated_key),
                                 ptr(cos_cache), ptr(sin_cache), b, s, hq, grad_key.shape[2], d, rotary,
                                 opts.position_offset, cos_cache.shape[0], dtype_code(grad_query),
                                 stream_ptr(stream)), "rope_backward")


# ---------------------------------------------------------------------------------------------- SwiGLU
def swiglu_forward(output, gate, up, stream=None):
    _same_cuda_dtype("swiglu_forward", output, gate, up)
    _require(output.shape == gate.shape == up.shape, "swiglu_forward: shapes differ")
    check(lib.cgpt_swiglu_forward(ptr(output), ptr(gate), ptr(up), gate.numel(), dtype_code(gate),
                                  stream_ptr(stream)), "swiglu_forward")


def swiglu_backward(grad_gate, grad_up, grad_output, gate, up, stream=None,
                    options: SwiGLUBackwardOptions | None = None):
    """swiglu_backward, separate gate/up layout (include/ops/backward/swiglu_backward.h:29-37)."""
    o = options or SwiGLUBackwardOptions()
    _same_cuda_dtype("swiglu_backward", grad_gate, grad_up, grad_output, gate, up)
    _require(grad_gate.shape == grad_up.shape == grad_output.shape == gate.shape == up.shape,
             "swiglu_backward: shapes differ")
    check(lib.cgpt_swiglu_backward(ptr(grad_gate), ptr(grad_up), ptr(grad_output), ptr(gate), ptr(up), gate.numel(),
                                   int(o.accumulate_gate), int(o.accumulate_up), dtype_code(gate),
                                   stream_ptr(stream)), "swiglu_backward")


# ------------------------------------------------------------------------------------------- Embedding
def embedding_forward(output, device_token_ids, token_count, weight, stream=None):
    _same_cuda_dtype("embedding_forward", output, weight)
    _ids(device_token_ids, token_count, "embedding_forward")
    _require(weight.dim() == 2 and output.numel() == token_count * weight.shape[1],
             "embedding_forward: output must hold token_count * hidden elements")
    check(lib.cgpt_embedding_forward(ptr(output), ptr(device_token_ids), ptr(weight), token_count, weight.shape[0],
                                     weight.shape[1], dtype_code(weight), stream_ptr(stream)), "embedding_forward")


def embedding_backward(grad_weight, grad_output, device_token_ids, token_count, stream=None,
                       options: EmbeddingBackwardOptions | None = None):
    """embedding_backward (include/ops/backward/embedding_backward.h:35-42)."""
    o = options or EmbeddingBackwardOptions()
    _same_cuda_dtype("embedding_backward", grad_weight, grad_output)
    _ids(device_token_ids, token_count, "embedding_backward")
    _require(grad_weight.dim() == 2 and grad_output.numel() == token_count * grad_weight.shape[1],
             "embedding_backward: grad_output must hold token_count * hidden elements")
    check(lib.cgpt_embedding_backward(ptr(grad_weight), ptr(grad_output), ptr(device_token_ids), token_count,
                                      grad_weight.shape[0], grad_weight.shape[1], int(o.bounds_check),
                                      int(o.accumulate_weight), dtype_code(grad_weight), stream_ptr(stream)),
          "embedding_backward")


# --------------------------------------------------------------------------------------- Residual adds
def add_tensors(output, a, b, stream=None, c=None):
    """add_tensors / add_inplace of src/core/transformer_block.cu:161-215,261-288 (output may alias a)."""
    extra = [c] if c is not None else []
    _same_cuda_dtype("add_tensors", output, a, b, *extra)
    _require(output.shape == a.shape == b.shape, "add_tensors: shapes differ")
    check(lib.cgpt_add(ptr(output), ptr(a), ptr(b), ptr(c), a.numel(), dtype_code(a), stream_ptr(stream)),
          "add_tensors")


# ----------------------------------------------------------- Dropout, layer norm, scaled embedding (pre-norm block)
@dataclass
class DropoutOptions:
    """``probability`` of dropping an element, realised in steps of 2^-16; 0 switches dropout off (the state may then be None).
    ``site`` tells the dropouts of one step apart: give every call of a step that must draw its own mask another number, and a
    backward call the number of its forward call."""
    probability: float = 0.0
    site: int = 0


@dataclass
class ScaledEmbeddingOptions:
    """``scale`` multiplies every looked-up row (sqrt(hidden) in many models); tokens whose id is ``padding_id`` take no part in
    the gradient; ``accumulate_weight`` adds to the gradient table instead of overwriting it."""
    scale: float = 1.0
    padding_id: int | None = None
    dropout: DropoutOptions | None = None
    accumulate_weight: bool = False


_NO_DROPOUT = DropoutOptions()
_STATE_DTYPES = (torch.int64, torch.uint64)


def make_dropout_state(seed: int, step: int = 0, device=None) -> torch.Tensor:
    """The generator state that the dropout calls of a model share: {seed, step}, two 64-bit words on the device."""
    signed = lambda v: (v & 0xffffffffffffffff) - ((v & 0x8000000000000000) << 1)
    return torch.tensor([signed(seed), signed(step)], dtype=torch.int64, device="cuda" if device is None else device)


def dropout_advance(state, steps: int = 1, stream=None):
    """step += steps on the device, after a training step's backward (capturable: replays of a graph that holds this call draw new
    masks every time)."""
    _require(steps >= 0, "dropout_advance: steps must not be negative")
    device = _state_check("dropout_advance", state)
    check(lib.cgpt_dropout_advance(state.data_ptr(), steps, _stream_on("dropout_advance", device, stream)), "dropout_advance")


def _state_check(name, state, device=None):
    if (state is None or state.dtype not in _STATE_DTYPES or state.numel() != 2 or not state.is_contiguous()
            or (not state.is_cuda if device is None else state.get_device() != device)):
        _require(False, f"{name}: state must be two 64-bit words on the tensors' device")
    return state.get_device()


def _dropout_options(name, options, state, device):
    """(probability, state pointer, site) of a call."""
    o = options or _NO_DROPOUT
    if not (0.0 <= o.probability < 1.0 and 0 <= o.site <= 0xffffffff):
        _require(False, f"{name}: probability must be in [0, 1) and site must fit 32 bits")
    if o.probability == 0.0:
        return 0.0, None, o.site
    _state_check(name, state, device)
    return o.probability, state.data_ptr(), o.site


# These calls take a few microseconds of host time on a small tensor, most of it here: the checks below read each property once,
# build no message unless they fail, and take the current stream's pointer directly where torch gives it (0.2 us; through
# torch.cuda.Stream 3.6 us). A torch without CUDA has no such function: the module is imported there all the same.
_current_device = torch.cuda.current_device
_current_stream = getattr(torch._C, "_cuda_getCurrentRawStream", lambda device: torch.cuda.current_stream(device).cuda_stream)


def _stream_on(name, device, stream):
    """Stream pointer of a call whose tensors are on `device`, which has to be the current device and the stream's."""
    if device != _current_device() or (stream is not None and stream.device_index != device):
        _require(False, f"{name}: tensors and stream must be on the current device")
    return _current_stream(device) if stream is None else stream.cuda_stream


def _one_device(name, *tensors):
    """Device index of contiguous CUDA tensors of one dtype (None is skipped)."""
    first = tensors[0]
    device, dtype = first.get_device(), first.dtype      # -1: not a CUDA tensor
    for t in tensors:
        if t is not None and (t.dtype != dtype or t.get_device() != device or device < 0 or not t.is_contiguous()):
            _same_cuda_dtype(name, *[u for u in tensors if u is not None])
            _require(False, f"{name}: all tensors must be on one device")
    return device


def _ptr(t):
    return None if t is None else t.data_ptr()


def _workspace(name, workspace, size, device, stream):
    """The caller's workspace, or one allocated on the call's stream. (pointer, bytes, the tensor to keep alive)"""
    if workspace is None:
        if stream is None:
            workspace = torch.empty(size, dtype=torch.uint8, device=device)
        else:
            with torch.cuda.stream(stream):   # its memory is handed on in this stream's order
                workspace = torch.empty(size, dtype=torch.uint8, device=device)
        return workspace.data_ptr(), size, workspace
    have = workspace.numel() * workspace.element_size()
    _require(workspace.is_cuda and workspace.get_device() == device and workspace.is_contiguous() and have >= size,
             f"{name}: workspace must be a contiguous CUDA buffer of at least {size} bytes on the tensors' device")
    return workspace.data_ptr(), have, workspace


def dropout_forward(output, input, state, stream=None, options: DropoutOptions | None = None, residual=None):
    """output = [residual +] dropout(input), any shape. output may be input or residual itself."""
    device = _one_device("dropout_forward", output, input, residual)
    _require(output.shape == input.shape and (residual is None or residual.shape == input.shape), "dropout_forward: shapes differ")
    p, state_ptr, site = _dropout_options("dropout_forward", options, state, device)
    check(lib.cgpt_dropout_forward(output.data_ptr(), input.data_ptr(), _ptr(residual), input.numel(), p, state_ptr, site,
                                   dtype_code(input), _stream_on("dropout_forward", device, stream)), "dropout_forward")


def dropout_backward(grad_input, grad_output, state, stream=None, options: DropoutOptions | None = None,
                     accumulate_input: bool = False):
    """grad_input = [grad_input +] the dropout map of grad_output; the forward's state, unadvanced, and its options."""
    device = _one_device("dropout_backward", grad_input, grad_output)
    _require(grad_input.shape == grad_output.shape, "dropout_backward: shapes differ")
    p, state_ptr, site = _dropout_options("dropout_backward", options, state, device)
    check(lib.cgpt_dropout_backward(grad_input.data_ptr(), grad_output.data_ptr(), grad_output.numel(), p, state_ptr, site,
                                    int(accumulate_input), dtype_code(grad_output), _stream_on("dropout_backward", device, stream)),
          "dropout_backward")


def _norm_shapes(name, x, weight, rows_like, vectors):
    shape, vector = x.shape, weight.shape
    good = len(shape) == 2 and len(vector) == 1 and vector[0] == shape[1]
    for t in rows_like:
        good = good and (t is None or t.shape == shape)
    for t in vectors:
        good = good and (t is None or t.shape == vector)
    if not good:
        _require(False, f"{name}: incompatible shapes")


def layernorm_forward(output, input, weight, bias, epsilon, stream=None):
    """output = (input - mean) / sqrt(var + epsilon) * weight + bias over rows of a matrix; bias may be None."""
    device = _one_device("layernorm_forward", output, input, weight, bias)
    _norm_shapes("layernorm_forward", input, weight, (output,), (bias,))
    check(lib.cgpt_layernorm_forward(output.data_ptr(), input.data_ptr(), weight.data_ptr(), _ptr(bias), input.shape[0], input.shape[1],
                                     epsilon, dtype_code(input), _stream_on("layernorm_forward", device, stream)), "layernorm_forward")


def layernorm_backward(grad_input, grad_weight, grad_bias, grad_output, input, weight, epsilon, stream=None, residual=None,
                       workspace=None):
    """Gradients of layernorm_forward (statistics are recomputed from input). grad_bias may be None; ``residual`` is added to
    grad_input inside the kernel. ``workspace``: a buffer of layernorm_backward_workspace_bytes(rows, hidden) bytes, allocated
    on the call's stream when None."""
    device = _one_device("layernorm_backward", grad_input, grad_weight, grad_bias, grad_output, input, weight, residual)
    _norm_shapes("layernorm_backward", input, weight, (grad_input, grad_output, residual), (grad_weight, grad_bias))
    rows, hidden = input.shape
    s = _stream_on("layernorm_backward", device, stream)
    at, size, keep = _workspace("layernorm_backward", workspace, layernorm_backward_workspace_bytes(rows, hidden), device, stream)
    check(lib.cgpt_layernorm_backward(grad_input.data_ptr(), grad_weight.data_ptr(), _ptr(grad_bias), grad_output.data_ptr(),
                                      input.data_ptr(), weight.data_ptr(), _ptr(residual), at, size, rows, hidden, epsilon,
                                      dtype_code(input), s), "layernorm_backward")


def layernorm_backward_workspace_bytes(rows: int, hidden: int) -> int:
    """Workspace of layernorm_backward and dropout_add_layernorm_backward; enough for fewer rows of this width too."""
    return lib.cgpt_layernorm_backward_workspace_bytes(rows, hidden)


def dropout_add_layernorm_forward(output, sum, input, residual, weight, bias, epsilon, state, stream=None,
                                  options: DropoutOptions | None = None):
    """sum = residual + dropout(input); output = layernorm(sum), in one pass. sum may be input or residual itself."""
    name = "dropout_add_layernorm_forward"
    device = _one_device(name, output, sum, input, residual, weight, bias)
    _norm_shapes(name, input, weight, (output, sum, residual), (bias,))
    p, state_ptr, site = _dropout_options(name, options, state, device)
    check(lib.cgpt_dropout_add_layernorm_forward(output.data_ptr(), sum.data_ptr(), input.data_ptr(), residual.data_ptr(),
                                                 weight.data_ptr(), _ptr(bias), input.shape[0], input.shape[1], epsilon, p, state_ptr,
                                                 site, dtype_code(input), _stream_on(name, device, stream)), name)


def dropout_add_layernorm_backward(grad_input, grad_residual, grad_weight, grad_bias, grad_output, grad_sum, sum, weight, epsilon,
                                   state, stream=None, options: DropoutOptions | None = None, workspace=None):
    """Gradients of dropout_add_layernorm_forward from those of its output and (None: zero) of its sum. grad_residual may be
    grad_sum itself; grad_bias may be None. ``workspace`` as in layernorm_backward."""
    name = "dropout_add_layernorm_backward"
    device = _one_device(name, grad_input, grad_residual, grad_weight, grad_bias, grad_output, grad_sum, sum, weight)
    _norm_shapes(name, sum, weight, (grad_input, grad_residual, grad_output, grad_sum), (grad_weight, grad_bias))
    rows, hidden = sum.shape
    p, state_ptr, site = _dropout_options(name, options, state, device)
    s = _stream_on(name, device, stream)
    at, size, keep = _workspace(name, workspace, layernorm_backward_workspace_bytes(rows, hidden), device, stream)
    check(lib.cgpt_dropout_add_layernorm_backward(grad_input.data_ptr(), grad_residual.data_ptr(), grad_weight.data_ptr(), _ptr(grad_bias),
                                                  grad_output.data_ptr(), _ptr(grad_sum), sum.data_ptr(), weight.data_ptr(), at, size,
                                                  rows, hidden, epsilon, p, state_ptr, site, dtype_code(sum), s), name)


_NO_EMBEDDING_OPTIONS = ScaledEmbeddingOptions()


def _embedding_check(name, table, activations, ids, token_count, options, state):
    device = _one_device(name, table, activations)
    _ids(ids, token_count, name)
    _require(ids.get_device() == device and ids.is_contiguous(), f"{name}: token ids must be contiguous and on the tensors' device")
    _require(table.dim() == 2 and token_count > 0 and activations.numel() == token_count * table.shape[1],
             f"{name}: activations must hold token_count * hidden elements")
    return device, _dropout_options(name, options.dropout, state, device)


def scaled_embedding_forward(output, device_token_ids, token_count, weight, state=None, stream=None,
                             options: ScaledEmbeddingOptions | None = None):
    """output[t] = dropout(scale * weight[ids[t]]); ids outside the table give zero rows."""
    o = options or _NO_EMBEDDING_OPTIONS
    device, (p, state_ptr, site) = _embedding_check("scaled_embedding_forward", weight, output, device_token_ids, token_count, o, state)
    check(lib.cgpt_scaled_embedding_forward(output.data_ptr(), device_token_ids.data_ptr(), weight.data_ptr(), token_count, weight.shape[0],
                                            weight.shape[1], o.scale, p, state_ptr, site, dtype_code(weight),
                                            _stream_on("scaled_embedding_forward", device, stream)), "scaled_embedding_forward")


def scaled_embedding_backward(grad_weight, grad_output, device_token_ids, token_count, state=None, stream=None,
                              options: ScaledEmbeddingOptions | None = None, workspace=None):
    """grad_weight[v] (+)= scale * the sum of the dropout map of grad_output over the tokens with id v. ``workspace``: a buffer of
    scaled_embedding_backward_workspace_bytes(token_count, hidden) bytes, allocated on the call's stream when None."""
    name = "scaled_embedding_backward"
    o = options or _NO_EMBEDDING_OPTIONS
    device, (p, state_ptr, site) = _embedding_check(name, grad_weight, grad_output, device_token_ids, token_count, o, state)
    _require(o.padding_id is None or 0 <= o.padding_id < grad_weight.shape[0], f"{name}: padding_id must be a row of the table")
    vocab, hidden = grad_weight.shape
    s = _stream_on(name, device, stream)
    at, size, keep = _workspace(name, workspace, scaled_embedding_backward_workspace_bytes(token_count, hidden), device, stream)
    check(lib.cgpt_scaled_embedding_backward(grad_weight.data_ptr(), grad_output.data_ptr(), device_token_ids.data_ptr(), at, size,
                                             token_count, vocab, hidden, o.scale, 0xffffffff if o.padding_id is None else o.padding_id,
                                             p, state_ptr, site, int(o.accumulate_weight), dtype_code(grad_weight), s), name)


def scaled_embedding_backward_workspace_bytes(token_count: int, hidden: int) -> int:
    """Workspace of scaled_embedding_backward; enough for fewer tokens of this width too."""
    return lib.cgpt_scaled_embedding_backward_workspace_bytes(token_count, hidden)


# --------------------------------------------------------------------------------------- Cross entropy
def _ce_check(loss, logits, targets, target_count, name):
    _require(loss.is_cuda and loss.dtype == torch.float32 and tuple(loss.shape) == (1,),
             f"{name}: loss must be a CUDA F32 tensor with shape [1]")
    _require(logits.is_cuda and logits.dim() == 2 and logits.shape[0] > 0 and logits.shape[1] > 0,
             f"{name}: logits must be a non-empty CUDA matrix")
    _require(target_count == logits.shape[0], f"{name}: target count must equal logits rows")
    _ids(targets, target_count, name)


def cross_entropy_forward_backward(loss, gradient, logits, device_targets, target_count, stream=None,
                                   gradient_scale: float = 1.0):
    """cross_entropy_forward_backward (include/ops/cross_entropy.h:25-32)."""
    _ce_check(loss, logits, device_targets, target_count, "cross_entropy")
    _same_cuda_dtype("cross_entropy", gradient, logits)
    _require(gradient.shape == logits.shape, "cross_entropy: gradient shape must match logits")
    check(lib.cgpt_cross_entropy(ptr(loss), ptr(gradient), ptr(logits), ptr(device_targets), logits.shape[0],
                                 logits.shape[1], float(gradient_scale), dtype_code(logits), stream_ptr(stream)),
          "cross_entropy_forward_backward")


def cross_entropy_forward(loss, logits, device_targets, target_count, stream=None):
    """cross_entropy_forward (include/ops/cross_entropy.h:37-42)."""
    _ce_check(loss, logits, device_targets, target_count, "cross_entropy")
    check(lib.cgpt_cross_entropy(ptr(loss), None, ptr(logits), ptr(device_targets), logits.shape[0], logits.shape[1],
                                 1.0, dtype_code(logits), stream_ptr(stream)), "cross_entropy_forward")
