"""``torch.library`` registration of the operators.

The reference exposes a raw pybind function (csrc/hadamard_transform.cpp:72-81);
callers that trace or compile their model need real dispatcher ops with
fake-tensor (meta) functions, and training code needs a backward.  Registered
under the ``b200ht`` namespace:

* ``torch.ops.b200ht.hadamard_transform(x, scale)``  — out of place; autograd:
  H is symmetric, so the gradient is the same transform of the incoming gradient.
* ``torch.ops.b200ht.fused_ht_gemm(X, W, scale, token_major, out_bf16)``
* ``torch.ops.b200ht.fused_ht_gemv(W, X, scale, out_bf16)``
* ``torch.ops.b200ht.rotary_qk(q, k, positions, inv_freq, sections, axis_order, interleaved, hadamard, inverse)``
  — autograd: the inverse call on the incoming gradients; a backward that needs one of inv_freq is refused, here and below.
  Keys are required (``q[:, :0]`` without any).
* ``torch.ops.b200ht.norm_rotary_qk(q, k, q_weight, k_weight, positions, inv_freq, eps, sections, axis_order,
  interleaved, hadamard)`` — autograd: gradients of q, k and both weights.
* ``torch.ops.b200ht.lora_ht_gemm(X, W, A, B, index, scaling, scale, token_major, out_bf16)`` and
  ``torch.ops.b200ht.lora_ht_gemv(W, X, A, B, index, scaling, scale, out_bf16)`` — serving operators, no gradient.

All run the CUDA library; there is no CPU kernel behind them.
"""
from __future__ import annotations

from typing import Optional, Sequence, Tuple

import torch

from . import heads, lora, ops


@torch.library.custom_op("b200ht::hadamard_transform", mutates_args=(), device_types="cuda")
def hadamard_transform_op(x: torch.Tensor, scale: float) -> torch.Tensor:
    return ops.hadamard_transform(x, inplace=False, scale=scale)


@hadamard_transform_op.register_fake
def _(x, scale):
    return torch.empty_like(x, memory_format=torch.contiguous_format)


def _ht_backward(ctx, grad):
    return torch.ops.b200ht.hadamard_transform(grad.contiguous(), ctx.scale), None


def _ht_setup(ctx, inputs, output):
    ctx.scale = inputs[1]


hadamard_transform_op.register_autograd(_ht_backward, setup_context=_ht_setup)


@torch.library.custom_op("b200ht::fused_ht_gemm", mutates_args=(), device_types="cuda")
def fused_ht_gemm_op(X: torch.Tensor, W: torch.Tensor, scale: float, token_major: bool, out_bf16: bool) -> torch.Tensor:
    return ops.fused_ht_gemm(X, W, scale=scale, out_layout="nm" if token_major else "mn",
                             out_dtype=torch.bfloat16 if out_bf16 else torch.float32)


@fused_ht_gemm_op.register_fake
def _(X, W, scale, token_major, out_bf16):
    n, m = X.shape[0], W.shape[0]
    return X.new_empty((n, m) if token_major else (m, n), dtype=torch.bfloat16 if out_bf16 else torch.float32)


@torch.library.custom_op("b200ht::fused_ht_gemv", mutates_args=(), device_types="cuda")
def fused_ht_gemv_op(W: torch.Tensor, X: torch.Tensor, scale: float, out_bf16: bool) -> torch.Tensor:
    return ops.fused_ht_gemv(W, X, scale=scale, out_dtype=torch.bfloat16 if out_bf16 else torch.float32)


@fused_ht_gemv_op.register_fake
def _(W, X, scale, out_bf16):
    return W.new_empty((W.shape[0], X.shape[1]), dtype=torch.bfloat16 if out_bf16 else torch.float32)


def _heads_like(x):
    return torch.empty(x.shape, dtype=x.dtype, device=x.device)


def _some(grad, x):
    """A missing gradient is zero."""
    return torch.zeros(x.shape, dtype=x.dtype, device=x.device) if grad is None else grad


def _no_gradient(needed, what):
    if needed:
        raise RuntimeError(f"{what}: inv_freq has no gradient here; detach it")


@torch.library.custom_op("b200ht::rotary_qk", mutates_args=(), device_types="cuda")
def rotary_qk_op(q: torch.Tensor, k: torch.Tensor, positions: torch.Tensor, inv_freq: torch.Tensor,
                 sections: Optional[Sequence[int]] = None, axis_order: str = "blocks", interleaved: bool = False,
                 hadamard: bool = False, inverse: bool = False) -> Tuple[torch.Tensor, torch.Tensor]:
    return heads.rotary_qk(q, k, positions, inv_freq, sections=sections, axis_order=axis_order, interleaved=interleaved,
                           hadamard=hadamard, inverse=inverse)


@rotary_qk_op.register_fake
def _(q, k, positions, inv_freq, sections=None, axis_order="blocks", interleaved=False, hadamard=False, inverse=False):
    return _heads_like(q), _heads_like(k)


def _rotary_setup(ctx, inputs, output):
    q, k, positions, inv_freq, *ctx.how, ctx.inverse = inputs
    ctx.save_for_backward(positions, inv_freq)
    ctx.like = (q.shape, k.shape, q.dtype, q.device)


def _rotary_backward(ctx, dq, dk):
    _no_gradient(ctx.needs_input_grad[3], "rotary_qk")
    positions, inv_freq = ctx.saved_tensors
    qs, ks, dtype, device = ctx.like
    dq = torch.zeros(qs, dtype=dtype, device=device) if dq is None else dq
    dk = torch.zeros(ks, dtype=dtype, device=device) if dk is None else dk
    dq, dk = torch.ops.b200ht.rotary_qk(dq, dk, positions, inv_freq, *ctx.how, not ctx.inverse)
    return dq, dk, None, None, None, None, None, None, None


rotary_qk_op.register_autograd(_rotary_backward, setup_context=_rotary_setup)


@torch.library.custom_op("b200ht::norm_rotary_qk", mutates_args=(), device_types="cuda")
def norm_rotary_qk_op(q: torch.Tensor, k: torch.Tensor, q_weight: torch.Tensor, k_weight: torch.Tensor,
                      positions: torch.Tensor, inv_freq: torch.Tensor, eps: float = 1e-6,
                      sections: Optional[Sequence[int]] = None, axis_order: str = "blocks", interleaved: bool = False,
                      hadamard: bool = False) -> Tuple[torch.Tensor, torch.Tensor]:
    return heads.norm_rotary_qk(q, k, q_weight, k_weight, positions, inv_freq, eps=eps, sections=sections,
                                axis_order=axis_order, interleaved=interleaved, hadamard=hadamard)


@norm_rotary_qk_op.register_fake
def _(q, k, q_weight, k_weight, positions, inv_freq, eps=1e-6, sections=None, axis_order="blocks", interleaved=False,
      hadamard=False):
    return _heads_like(q), _heads_like(k)


@torch.library.custom_op("b200ht::norm_rotary_qk_backward", mutates_args=(), device_types="cuda")
def norm_rotary_qk_backward_op(dq: torch.Tensor, dk: torch.Tensor, q: torch.Tensor, k: torch.Tensor,
                               q_weight: torch.Tensor, k_weight: torch.Tensor, positions: torch.Tensor,
                               inv_freq: torch.Tensor, eps: float = 1e-6, sections: Optional[Sequence[int]] = None,
                               axis_order: str = "blocks", interleaved: bool = False, hadamard: bool = False
                               ) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    return heads.norm_rotary_qk_backward(dq, dk, q, k, q_weight, k_weight, positions, inv_freq, eps=eps,
                                         sections=sections, axis_order=axis_order, interleaved=interleaved,
                                         hadamard=hadamard)


@norm_rotary_qk_backward_op.register_fake
def _(dq, dk, q, k, q_weight, k_weight, positions, inv_freq, eps=1e-6, sections=None, axis_order="blocks",
      interleaved=False, hadamard=False):
    return _heads_like(q), _heads_like(k), torch.empty_like(q_weight), torch.empty_like(k_weight)


def _norm_rotary_setup(ctx, inputs, output):
    ctx.how = inputs[6:]
    ctx.save_for_backward(*inputs[:6])


def _norm_rotary_backward(ctx, dq, dk):
    _no_gradient(ctx.needs_input_grad[5], "norm_rotary_qk")
    q, k, *rest = ctx.saved_tensors
    grads = torch.ops.b200ht.norm_rotary_qk_backward(_some(dq, q), _some(dk, k), q, k, *rest, *ctx.how)
    return (*grads, None, None, None, None, None, None, None)


norm_rotary_qk_op.register_autograd(_norm_rotary_backward, setup_context=_norm_rotary_setup)


@torch.library.custom_op("b200ht::lora_ht_gemm", mutates_args=(), device_types="cuda")
def lora_ht_gemm_op(X: torch.Tensor, W: torch.Tensor, A: torch.Tensor, B: torch.Tensor, index: torch.Tensor,
                    scaling: Optional[torch.Tensor], scale: float, token_major: bool, out_bf16: bool) -> torch.Tensor:
    return lora.lora_ht_gemm(X, W, A, B, index, scaling=scaling, scale=scale, out_layout="nm" if token_major else "mn",
                             out_dtype=torch.bfloat16 if out_bf16 else torch.float32)


@lora_ht_gemm_op.register_fake
def _(X, W, A, B, index, scaling, scale, token_major, out_bf16):
    n, m = X.shape[0], W.shape[0]
    return X.new_empty((n, m) if token_major else (m, n), dtype=torch.bfloat16 if out_bf16 else torch.float32)


@torch.library.custom_op("b200ht::lora_ht_gemv", mutates_args=(), device_types="cuda")
def lora_ht_gemv_op(W: torch.Tensor, X: torch.Tensor, A: torch.Tensor, B: torch.Tensor, index: torch.Tensor,
                    scaling: Optional[torch.Tensor], scale: float, out_bf16: bool) -> torch.Tensor:
    return lora.lora_ht_gemv(W, X, A, B, index, scaling=scaling, scale=scale,
                             out_dtype=torch.bfloat16 if out_bf16 else torch.float32)


@lora_ht_gemv_op.register_fake
def _(W, X, A, B, index, scaling, scale, out_bf16):
    return W.new_empty((W.shape[0], X.shape[1] if X.dim() == 2 else 1), dtype=torch.bfloat16 if out_bf16 else torch.float32)
