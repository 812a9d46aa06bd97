"""Queries and keys after a projection: position rotation, RMS norm and Hadamard rotation of every head in one pass.

A model whose caches are quantised rotates the heads of its queries and keys with a Hadamard matrix.  That rotation has
to follow the position rotation, so it cannot be folded into a weight; here it costs no pass of its own.  The reference
has no counterpart: its users would run the position rotation elsewhere and csrc.hadamard_transform behind it
(csrc/hadamard_transform.cpp:12-70).

Tensors are (tokens, heads, head_dim); views of one packed projection are taken as they are.  All arithmetic happens in
libb200ht.so (fp32, angles reduced in fp64, one rounding on the store); there is no CPU path.  These
functions record no graph; ``torch.ops.b200ht.rotary_qk`` and ``norm_rotary_qk`` are the forms that differentiate.
"""
from __future__ import annotations

import functools
import struct

import torch

from . import _lib
from .ops import _DT, _check_overwrite, _is_pow2, _on_device, _overwritten, _stream_ptr

_INTS = (torch.int32, torch.int64)
_strides8 = struct.Struct("8q").pack
_strides12 = struct.Struct("12q").pack


@functools.lru_cache(maxsize=64)
def axis_table(sections: tuple[int, ...], axis_order: str, pairs: int) -> bytes:
    """The position axis of each pair, one byte per pair.

    ``"blocks"``: the first sections[0] pairs belong to axis 0, the next sections[1] to axis 1, ...
    ``"cycle"``: the axes take turns pair by pair while they have pairs left; a pair whose turn falls on a used-up
    axis belongs to axis 0.
    """
    if not 1 <= len(sections) <= 4 or any(s < 0 for s in sections) or sum(sections) != pairs:
        raise RuntimeError(f"rotary: sections must be one to four counts that add up to {pairs} pairs, got {sections}")
    if axis_order == "blocks":
        return b"".join(bytes([a]) * n for a, n in enumerate(sections))
    if axis_order != "cycle":
        raise RuntimeError("rotary: axis_order must be 'blocks' or 'cycle'")
    n = len(sections)
    table = bytes(i % n if i < n * sections[i % n] else 0 for i in range(pairs))
    if any(table.count(a) != s for a, s in enumerate(sections)):
        raise RuntimeError(f"rotary: sections {sections} cannot take turns over {pairs} pairs")
    return table


def _check_heads(x: torch.Tensor, like: torch.Tensor, what: str) -> torch.Tensor:
    sx, sl = x.shape, like.shape
    if len(sx) != 3 or sx[0] != sl[0] or sx[2] != sl[2]:
        raise RuntimeError(f"rotary: expected {what} of shape (tokens, heads, head_dim) like the queries")
    if sx[1] >= 1 << 30:
        raise RuntimeError("rotary: fewer than 2^30 tokens and heads")
    if x.dtype != like.dtype or x.device != like.device:
        raise RuntimeError(f"rotary: {what} must have the queries' dtype and device")
    return x if x.stride(2) == 1 else x.contiguous()


def _check_common(q, positions, inv_freq, sections, axis_order, hadamard):
    """Checks shared by all entry points; returns (head_dim, tokens, pairs, flags, axis table, n_axes, pos strides)."""
    device = q.device
    if q.dtype not in _DT:
        raise RuntimeError("rotary: only fp16, bf16 and fp32 are supported")
    if not q.is_cuda:
        raise RuntimeError("rotary: queries and keys must be CUDA tensors")
    if q.dim() != 3:
        raise RuntimeError("rotary: expected queries of shape (tokens, heads, head_dim)")
    tokens, heads, D = q.shape
    if tokens >= 1 << 30 or heads >= 1 << 30:
        raise RuntimeError("rotary: fewer than 2^30 tokens and heads")
    if D < 2 or D > 256 or D % 2:
        raise RuntimeError(f"rotary: head_dim must be even and at most 256, got {D}")
    if hadamard and not _is_pow2(D):
        raise RuntimeError(f"rotary: the Hadamard rotation needs a head_dim that is a power of two, got {D}")
    if inv_freq.dtype != torch.float32 or inv_freq.dim() != 1 or inv_freq.device != device:
        raise RuntimeError("rotary: inv_freq must be a float32 vector on the queries' device")
    pairs = inv_freq.shape[0]
    if pairs < 1 or 2 * pairs > D:
        raise RuntimeError(f"rotary: inv_freq must have 1 to head_dim / 2 entries, got {pairs}")
    if positions.dtype not in _INTS or positions.device != device:
        raise RuntimeError("rotary: positions must be int32 or int64 on the queries' device")
    if sections is None:
        table, n_axes = None, 1
        if positions.dim() != 1 or positions.shape[0] != tokens:
            raise RuntimeError(f"rotary: positions must be a vector of {tokens} entries")
        axis_stride, token_stride = 0, positions.stride(0)
    else:
        table = axis_table(tuple(int(s) for s in sections), axis_order, pairs)
        n_axes = len(sections)
        if positions.dim() != 2 or tuple(positions.shape) != (n_axes, tokens):
            raise RuntimeError(f"rotary: positions must have shape ({n_axes}, {tokens})")
        axis_stride, token_stride = positions.stride()
    flags = (_lib.ROT_HADAMARD if hadamard else 0) | (_lib.ROT_POS64 if positions.dtype == torch.int64 else 0)
    return D, tokens, pairs, flags, table, n_axes, axis_stride, token_stride


def _check_weights(q, q_weight, k_weight, D):
    if q_weight is None or k_weight is None:
        raise RuntimeError("norm_rotary_qk: both weights are required, also without keys (any vector like q_weight will do)")
    device, dtype = q.device, q_weight.dtype
    for w in (q_weight, k_weight):
        if tuple(w.shape) != (D,) or w.device != device:
            raise RuntimeError(f"norm_rotary_qk: the weights must be vectors of {D} entries on the queries' device")
    if k_weight.dtype != dtype or dtype != q.dtype and dtype != torch.float32:
        raise RuntimeError("norm_rotary_qk: the weights must both have the queries' dtype, or both be float32")


def _own_memory(x: torch.Tensor) -> bool:
    """True when no two elements of x (tokens, heads, head_dim) share memory."""
    dims = sorted((st, n) for n, st in zip(x.shape, x.stride()) if n > 1)
    reach = 1
    for st, n in dims:
        if st < reach:
            return False
        reach = st * (n - 1) + reach
    return True


def _apart(q: torch.Tensor, k: torch.Tensor) -> bool:
    """True when q and k, each without overlaps of its own, are known to share no memory: they lie one behind the
    other, or are disjoint groups of heads of one packed tensor."""
    if not q.numel() or not k.numel():
        return True
    size = q.element_size()

    def reach(x):
        return sum(st * (n - 1) for n, st in zip(x.shape, x.stride())) + 1

    gap = k.data_ptr() - q.data_ptr()
    if gap >= reach(q) * size or -gap >= reach(k) * size:
        return True
    row = q.stride(0)
    if row != k.stride(0) or gap % size or row == 0:   # 0: one token, seen through expand
        return False
    # within one row of the packed tensor: q's heads at 0, the keys' at `at`
    at = gap // size % row
    return at >= reach(q[0]) and at + reach(k[0]) <= row


def _run(q, k, norm, q_weight, k_weight, eps, positions, inv_freq, sections, axis_order, interleaved, hadamard, inverse, inplace):
    D, tokens, pairs, flags, table, n_axes, pa, pt = _check_common(q, positions, inv_freq, sections, axis_order, hadamard)
    q_in, k_in = q, k
    if q.stride(2) != 1:
        q = q.contiguous()
    if k is not None:
        k = _check_heads(k, q, "keys")
    if norm:
        _check_weights(q, q_weight, k_weight, D)
        q_weight, k_weight = q_weight.contiguous(), k_weight.contiguous()
        if q_weight.dtype == torch.float32:
            flags |= _lib.ROT_WEIGHT_F32
    if inplace:
        if q is not q_in or k is not k_in:
            raise RuntimeError("rotary: the last dimension must be contiguous to work in place")
        _check_overwrite("rotary", q)
        if k is not None:
            _check_overwrite("rotary", k)
        if not _own_memory(q) or (k is not None and not (_own_memory(k) and _apart(q, k))):
            raise RuntimeError("rotary: in place, queries and keys must not share memory with themselves or each other")
        qo, ko = q, k
    else:
        qo = torch.empty_like(q, memory_format=torch.contiguous_format)
        ko = None if k is None else torch.empty_like(k, memory_format=torch.contiguous_format)
    if interleaved:
        flags |= _lib.ROT_INTERLEAVED
    if inverse:
        flags |= _lib.ROT_INVERSE
    inv_freq = inv_freq.contiguous()
    hk = 0 if k is None else k.shape[1]
    if tokens and q.shape[1] + hk:
        kk, kko = (q, qo) if k is None else (k, ko)   # no keys: the pointers of no head are never read
        with _on_device(q.device):
            rc = _lib.load().b200ht_rotary_qk(
                q.data_ptr(), kk.data_ptr(), qo.data_ptr(), kko.data_ptr(),
                None if q_weight is None else q_weight.data_ptr(), None if k_weight is None else k_weight.data_ptr(), eps,
                tokens, q.shape[1], hk, D, _strides8(*q.stride()[:2], *kk.stride()[:2], *qo.stride()[:2], *kko.stride()[:2]),
                _DT[q.dtype], positions.data_ptr(), pa, pt, n_axes, table, inv_freq.data_ptr(), pairs, flags,
                _stream_ptr(q.device))
        _lib.check(rc, "b200ht_rotary_qk")
        if inplace:
            _overwritten(q)
            if k is not None:
                _overwritten(k)
    return qo, ko


def rotary_qk(q: torch.Tensor, k: torch.Tensor | None, positions: torch.Tensor, inv_freq: torch.Tensor, *,
              sections: tuple[int, ...] | None = None, axis_order: str = "blocks", interleaved: bool = False,
              hadamard: bool = False, inverse: bool = False, inplace: bool = False):
    """Rotate queries and keys by their positions; returns ``(q', k')`` (``k'`` is None without keys).

    ``q`` is (tokens, q_heads, head_dim) and ``k`` (tokens, k_heads, head_dim), fp16, bf16 or fp32 with a contiguous
    last dimension and any other strides.  ``inv_freq`` (float32, 1 .. head_dim / 2 entries) holds the radians per unit
    of position of each pair of dimensions: pair i is (i, i + pairs), with ``interleaved`` (2i, 2i + 1); dimensions
    behind the pairs are left alone.  ``positions`` (int32 or int64, any sign) has one entry per token.  With
    ``sections`` there are several axes (time, height, width): positions is (axes, tokens) and sections[a] pairs turn by
    axis a, in blocks or (``axis_order="cycle"``) in turn, see :func:`axis_table`.  The angle is
    ``positions * inv_freq`` as given, without the loss of fp32 at far positions.

    ``hadamard`` multiplies every rotated head by H / sqrt(head_dim) (Sylvester order, as ``hadamard_transform``).
    ``inverse`` undoes the call without it, which is also its gradient: H first, then the rotation by the negative
    angles.  ``inplace`` overwrites q and k and returns them; tensors that overlap themselves or each other are refused, and
    while a graph is recorded those that require grad.
    """
    return _run(q, k, False, None, None, 0.0, positions, inv_freq, sections, axis_order, interleaved, hadamard, inverse, inplace)


def norm_rotary_qk(q: torch.Tensor, k: torch.Tensor | None, q_weight: torch.Tensor, k_weight: torch.Tensor,
                   positions: torch.Tensor, inv_freq: torch.Tensor, *, eps: float = 1e-6,
                   sections: tuple[int, ...] | None = None, axis_order: str = "blocks", interleaved: bool = False,
                   hadamard: bool = False, inplace: bool = False):
    """``rotary_qk`` behind an RMS norm of every head: ``x * rsqrt(mean(x^2) + eps) * weight``, one pass, one rounding.

    ``q_weight`` and ``k_weight`` (head_dim entries) both have the queries' dtype, or both are float32.  Everything else
    as :func:`rotary_qk` (without keys both weights are needed all the same); the gradients are
    :func:`norm_rotary_qk_backward`.
    """
    return _run(q, k, True, q_weight, k_weight, float(eps), positions, inv_freq, sections, axis_order, interleaved, hadamard,
                False, inplace)


def norm_rotary_qk_backward(dq_out: torch.Tensor, dk_out: torch.Tensor, q: torch.Tensor, k: torch.Tensor,
                            q_weight: torch.Tensor, k_weight: torch.Tensor, positions: torch.Tensor,
                            inv_freq: torch.Tensor, *, eps: float = 1e-6, sections: tuple[int, ...] | None = None,
                            axis_order: str = "blocks", interleaved: bool = False, hadamard: bool = False):
    """Gradients of :func:`norm_rotary_qk`: returns ``(dq, dk, dq_weight, dk_weight)``.

    ``dq_out`` and ``dk_out`` are the gradients of its results, the other arguments those of the call (``q`` and ``k``
    before it: a call in place has lost them).  Without keys pass tensors of none, ``q[:, :0]``.  The weights' gradients are sums over all tokens and heads, in fp32 and
    in an order that depends on the sizes, the type and the layout (strides, alignment, order of the pairs) alone.
    """
    D, tokens, pairs, flags, table, n_axes, pa, pt = _check_common(q, positions, inv_freq, sections, axis_order, hadamard)
    if k is None or dk_out is None:
        raise RuntimeError("norm_rotary_qk_backward: keys and their gradients are required; without keys pass q[:, :0] for both")
    k = _check_heads(k, q, "keys")
    if q.stride(2) != 1:
        q = q.contiguous()
    _check_weights(q, q_weight, k_weight, D)
    if dq_out.shape != q.shape or dk_out.shape != k.shape:
        raise RuntimeError("norm_rotary_qk_backward: the gradients must have the shapes of q and k")
    dq_out, dk_out = _check_heads(dq_out, q, "gradients"), _check_heads(dk_out, q, "gradients")
    q_weight, k_weight = q_weight.contiguous(), k_weight.contiguous()
    if q_weight.dtype == torch.float32:
        flags |= _lib.ROT_WEIGHT_F32
    if interleaved:
        flags |= _lib.ROT_INTERLEAVED
    inv_freq = inv_freq.contiguous()
    dq = torch.empty_like(q, memory_format=torch.contiguous_format)
    dk = torch.empty_like(k, memory_format=torch.contiguous_format)
    dqw, dkw = torch.empty_like(q_weight), torch.empty_like(k_weight)
    strides = _strides12(*dq_out.stride()[:2], *dk_out.stride()[:2], *q.stride()[:2], *k.stride()[:2], *dq.stride()[:2],
                         *dk.stride()[:2])
    lib = _lib.load()
    size = lib.b200ht_norm_rotary_qk_backward_workspace_bytes(D)
    ws = q.new_empty(size // q.element_size())   # cheaper than a tensor of bytes
    with _on_device(q.device):
        rc = lib.b200ht_norm_rotary_qk_backward(
            dq_out.data_ptr(), dk_out.data_ptr(), q.data_ptr(), k.data_ptr(), q_weight.data_ptr(), k_weight.data_ptr(),
            float(eps), dq.data_ptr(), dk.data_ptr(), dqw.data_ptr(), dkw.data_ptr(), tokens, q.shape[1], k.shape[1], D,
            strides, _DT[q.dtype], positions.data_ptr(), pa, pt, n_axes, table, inv_freq.data_ptr(), pairs, flags,
            ws.data_ptr(), size, _stream_ptr(q.device))
    _lib.check(rc, "b200ht_norm_rotary_qk_backward")
    return dq, dk, dqw, dkw
