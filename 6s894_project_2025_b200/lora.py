"""W . H(X) with low-rank adapters of many requests beside the shared projection.

One batch holds tokens of many requests, each with its own adapter or none; they share the weight W.  The adapters are
stacked: A (adapters, rank, K) and B (adapters, M, rank), token t has adapter ``index[t]``, and its output gains
``scaling[a] * B[a] @ (A[a] @ x_t)``.  The adapter sees the token as given, without H, as it was trained beside the
unrotated weight.  These are serving operators: W and the adapters get no gradient.  The reference has no counterpart.

All arithmetic happens in libb200ht.so, bf16 operands with fp32 sums; there is no CPU path.
"""
from __future__ import annotations

import math

import torch

from . import _lib
from .ops import _DT, _check_overwrite, _is_pow2, _on_device, _overwritten, _stream_ptr, sign_mask

_MAX_COLUMNS = 64   # columns of one decoding call; more go through the contraction
# Beyond N = 8192 the GEMV takes four columns a pass over W (one at 32768), the contraction all.  Microseconds a call, GEMV
# and contraction, 16384 x 16384: 3 columns 184 / 207, 4: 255 / 119, 16: 991 / 129, 64: 4599 / 138; M = 4096, N = 16384: 3
# columns 95 / 43, 4: 128 / 43; N = 32768: 3 columns 416 / 71, 64: 9883 / 109.  Up to three columns W . H(X) keeps the bits
# of fused_ht_gemv.
_LONG, _LONG_COLUMNS = 8192, 3


def _check(what: str, X, W, A, B, index, scaling, tokens: int, K: int, out_dtype):
    """Checks shared by both entries; returns (M, adapters, rank, A, B, index, scaling)."""
    bf16, device = torch.bfloat16, X.device
    if X.dtype != bf16 or W.dtype != bf16 or A.dtype != bf16 or B.dtype != bf16:
        raise RuntimeError(f"{what}: X, W, A and B must be bfloat16")
    if not X.is_cuda or W.device != device or A.device != device or B.device != device or index.device != device:
        raise RuntimeError(f"{what}: all tensors must be on one CUDA device")
    if not _is_pow2(K) or K < 64 or K > (1 << 15):
        raise RuntimeError(f"{what}: the Hadamard size must be a power of two from 64 to 2^15, got {K}")
    M = W.shape[0]
    if A.dim() != 3 or B.dim() != 3 or A.shape[2] != K or B.shape[1] != M or A.shape[0] != B.shape[0] or A.shape[1] != B.shape[2]:
        raise RuntimeError(f"{what}: expected A (adapters, rank, {K}) and B (adapters, {M}, rank)")
    adapters, rank = A.shape[0], A.shape[1]
    if adapters < 1 or rank < 8 or rank > 128 or rank % 8:
        raise RuntimeError(f"{what}: the rank must be a multiple of 8 up to 128 (pad with zeros) of at least one adapter, got "
                           f"{adapters} of rank {rank}")
    if max(tokens, M, adapters) >= 1 << 31:
        raise RuntimeError(f"{what}: at most 2^31 - 1 tokens, rows and adapters")
    if index.dtype != torch.int32 or index.dim() != 1 or index.shape[0] != tokens:
        raise RuntimeError(f"{what}: index must be {tokens} int32 entries")
    if scaling is not None:
        if scaling.dtype != torch.float32 or scaling.dim() != 1 or scaling.shape[0] != adapters or scaling.device != device:
            raise RuntimeError(f"{what}: scaling must be {adapters} float32 entries on the tokens' device")
        scaling = scaling.contiguous()
    if out_dtype not in (torch.float32, bf16):
        raise RuntimeError(f"{what}: out_dtype must be float32 or bfloat16")
    return M, adapters, rank, _rows(A), _rows(B), index.contiguous(), scaling


def _rows(x: torch.Tensor) -> torch.Tensor:
    """x contiguous and on a 16-byte boundary."""
    x = x.contiguous()
    return x if x.data_ptr() % 16 == 0 else x.clone()


def _out(what, out, shape, dtype, like):
    if out is None:
        return like.new_empty(shape, dtype=dtype)
    if tuple(out.shape) != shape or out.dtype != dtype or not out.is_contiguous() or out.device != like.device or out.data_ptr() % 16:
        raise RuntimeError(f"{what}: out has the wrong shape, dtype, strides, device or alignment")
    _check_overwrite(what, out)
    _overwritten(out)
    return out


def lora_ht_gemm(X: torch.Tensor, W: torch.Tensor, A: torch.Tensor, B: torch.Tensor, index: torch.Tensor, *,
                 scaling: torch.Tensor | None = None, scale: float | None = None, out_dtype: torch.dtype | None = None,
                 out_layout: str = "mn", out: torch.Tensor | None = None, signs: torch.Tensor | None = None) -> torch.Tensor:
    """``fused_ht_gemm(X, W)`` plus the adapter of each token, in one contraction.

    ``X`` (N tokens, K), ``W`` (M, K), ``A`` (adapters, rank, K) and ``B`` (adapters, M, rank) are bf16; ``index`` (N
    int32 entries) names the adapter of each token, any value outside 0 .. adapters - 1 (-1, say) none; ``scaling``
    (float32, one per adapter) defaults to 1.  The rank is a multiple of 8 up to 128.  ``scale``, ``signs``,
    ``out_dtype`` (float32 by default), ``out_layout`` and ``out`` as in ``fused_ht_gemm``; scale and signs belong to the
    transform and do not touch the adapters.  Tokens may come in any order; tokens of one adapter next to each other cost
    least.  The low-rank vectors are rounded to bf16, as H(X) is, the sums are fp32 and C is rounded once.

    Infinities and NaN in an adapter reach its own tokens only; a call with such an adapter among others in a group of 16
    tokens (16 i .. 16 i + 15) is much slower, as these results are computed again.  Adapters that no token names are not
    read.
    """
    if X.dim() != 2 or W.dim() != 2 or X.shape[1] != W.shape[1]:
        raise RuntimeError("lora_ht_gemm: expected X (N, K) and W (M, K)")
    N, K = X.shape
    if out_layout not in ("mn", "nm"):
        raise RuntimeError("lora_ht_gemm: out_layout must be 'mn' or 'nm'")
    out_dtype = out_dtype or torch.float32
    M, adapters, rank, A, B, index, scaling = _check("lora_ht_gemm", X, W, A, B, index, scaling, N, K, out_dtype)
    X, W = _rows(X), _rows(W)
    out = _out("lora_ht_gemm", out, (M, N) if out_layout == "mn" else (N, M), out_dtype, X)
    if M == 0 or N == 0:
        return out
    lib = _lib.load()
    mask = None if signs is None else sign_mask(signs, K, X.device)
    size = lib.b200ht_lora_gemm_workspace_bytes(M, N, K, rank)
    ws = X.new_empty(size // 2)   # cheaper than a tensor of bytes
    with _on_device(X.device):
        rc = lib.b200ht_lora_gemm(X.data_ptr(), W.data_ptr(), out.data_ptr(), A.data_ptr(), B.data_ptr(), index.data_ptr(),
                                  None if scaling is None else scaling.data_ptr(), M, N, K, adapters, rank, _DT[out_dtype],
                                  _lib.OUT_MN if out_layout == "mn" else _lib.OUT_NM,
                                  math.sqrt(1.0 / K) if scale is None else float(scale),
                                  None if mask is None else mask.data_ptr(), ws.data_ptr(), size, _stream_ptr(X.device))
    _lib.check(rc, "b200ht_lora_gemm")
    return out


def lora_ht_gemv(W: torch.Tensor, X: torch.Tensor, A: torch.Tensor, B: torch.Tensor, index: torch.Tensor, *,
                 scaling: torch.Tensor | None = None, scale: float | None = None, out_dtype: torch.dtype | None = None,
                 out: torch.Tensor | None = None) -> torch.Tensor:
    """``fused_ht_gemv(W, X)`` plus the adapter of each column: one token of every request of a decoding batch.

    ``W`` is (M, N), ``X`` (N, columns) with the columns fastest (or a vector, one column), the result (M, columns);
    ``A`` (adapters, rank, N), ``B`` (adapters, M, rank), ``index`` (columns int32 entries) and ``scaling`` as in
    :func:`lora_ht_gemm`.  The low-rank vectors stay fp32 and Y is rounded once.  Beyond the batch that
    ``fused_ht_gemv`` serves with one pass over W (16 columns at N = 4096; three for N above 8192, which are a pass at 16384
    and three at 32768) the call goes through :func:`lora_ht_gemm`.
    """
    if X.dim() == 1:
        X = X[:, None]
    if X.dim() != 2 or W.dim() != 2 or X.shape[0] != W.shape[1]:
        raise RuntimeError("lora_ht_gemv: expected W (M, N) and X (N, B)")
    N, columns = X.shape
    if columns < 1:
        raise RuntimeError("lora_ht_gemv: batch must be at least 1, got 0")
    out_dtype = out_dtype or torch.float32
    lib = _lib.load()
    once = lib.b200ht_fused_gemv_max_batch(N, _lib.BF16)   # columns served by one pass over W
    if columns > _MAX_COLUMNS or (once and columns > once) or (N > _LONG and columns > _LONG_COLUMNS):
        return lora_ht_gemm(X.t(), W, A, B, index, scaling=scaling, scale=scale, out_dtype=out_dtype, out=out)
    M, adapters, rank, A, B, index, scaling = _check("lora_ht_gemv", X, W, A, B, index, scaling, columns, N, out_dtype)
    X, W = _rows(X), _rows(W)
    out = _out("lora_ht_gemv", out, (M, columns), out_dtype, X)
    if M == 0:
        return out
    size = lib.b200ht_lora_gemv_workspace_bytes(M, N, columns, rank)
    ws = X.new_empty(size // 2)   # cheaper than a tensor of bytes
    with _on_device(X.device):
        rc = lib.b200ht_lora_gemv(W.data_ptr(), X.data_ptr(), out.data_ptr(), A.data_ptr(), B.data_ptr(), index.data_ptr(),
                                  None if scaling is None else scaling.data_ptr(), M, N, columns, adapters, rank,
                                  _DT[out_dtype], math.sqrt(1.0 / N) if scale is None else float(scale), ws.data_ptr(),
                                  size, _stream_ptr(X.device))
    _lib.check(rc, "b200ht_lora_gemv")
    return out
