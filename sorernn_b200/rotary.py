"""The norm of query and key heads with the rotary rotation in the same pass, and the rotation's table.

* :func:`rotary_table` — cosines and sines per position and pair, kept by the model;
* :func:`qk_norm_rope` — ``RMSNorm`` of every q and k head, then the rotation of its first features by the token's
  position, one kernel for both, forward and (under autograd) backward. soreRNN's attention mixer does the same two
  steps on its q and k (sore/model/attention.py, sore/model/rope.py).

Thin calls into the C ABI (include/gdn_b200.h, ``gdn_qk_norm_rope_*``) on the current stream, CUDA tensors only.
"""
from __future__ import annotations

import ctypes
from typing import Optional, Sequence

import torch
from torch import Tensor

from . import _lib
from .gated_delta_rule import _DT
from .linear_attention import _at, _call, _refuse_tangents


def rotary_table(max_positions: int, rotary_dim: int, theta: float = 10000.0,
                 device: Optional[torch.device] = None) -> Tensor:
    """fp32 ``[max_positions, rotary_dim]``: the cosines of the ``rotary_dim / 2`` pairs, then their sines, at angle
    ``position * theta^(-2 i / rotary_dim)`` for pair i (angles in fp64: exact to fp32 at any length)."""
    if rotary_dim <= 0 or rotary_dim % 2:
        raise ValueError(f"rotary_dim must be positive and even, got {rotary_dim}")
    freq = theta ** (-torch.arange(0, rotary_dim, 2, dtype=torch.float64, device=device) / rotary_dim)
    angle = torch.arange(max_positions, dtype=torch.float64, device=device)[:, None] * freq
    return torch.cat([angle.cos(), angle.sin()], -1).float()


def _problem(q, k, q_weight, table, positions, sections, interleaved, eps) -> _lib.QkNormRopeProblem:
    B, T, HQ, D = q.shape
    n_pos, R = table.shape
    return _lib.QkNormRopeProblem(B, T, HQ, k.shape[2], D, R, n_pos, q.stride()[:3], k.stride()[:3],
                                  tuple(sections), len(sections) or 1, positions.dtype == torch.int64, interleaved,
                                  _DT[q.dtype], _DT[q_weight.dtype], eps)


def _fwd(q, k, q_weight, k_weight, table, positions, sections, interleaved, eps):
    p = _problem(q, k, q_weight, table, positions, sections, interleaved, eps)
    yq = torch.empty_like(q, memory_format=torch.contiguous_format)
    yk = torch.empty_like(k, memory_format=torch.contiguous_format)
    _call(q.device, _lib.lib().gdn_qk_norm_rope_fwd, "gdn_qk_norm_rope_fwd", ctypes.byref(p), _at(q), _at(k),
          _at(q_weight), _at(k_weight), _at(table), _at(positions), _at(yq), _at(yk))
    return yq, yk


@torch.library.custom_op("sorernn_b200::qk_norm_rope_fwd", mutates_args=())
def qk_norm_rope_fwd(q: Tensor, k: Tensor, q_weight: Tensor, k_weight: Tensor, table: Tensor, positions: Tensor,
                     sections: Sequence[int], interleaved: bool, eps: float) -> tuple[Tensor, Tensor]:
    return _fwd(q, k, q_weight, k_weight, table, positions, sections, interleaved, eps)


@qk_norm_rope_fwd.register_fake
def _(q, k, q_weight, k_weight, table, positions, sections, interleaved, eps):
    return q.new_empty(q.shape), k.new_empty(k.shape)


def _bwd(q, k, q_weight, k_weight, table, positions, sections, interleaved, eps, dyq, dyk):
    L = _lib.lib()
    p = _problem(q, k, q_weight, table, positions, sections, interleaved, eps)
    dyq, dyk = dyq.contiguous(), dyk.contiguous()
    dq = torch.empty_like(q, memory_format=torch.contiguous_format)
    dk = torch.empty_like(k, memory_format=torch.contiguous_format)
    dwq, dwk = (q.new_empty(p.D, dtype=torch.float32) for _ in range(2))
    ref = ctypes.byref(p)
    n = L.gdn_qk_norm_rope_bwd_workspace_size(ref)
    ws = q.new_empty(n, dtype=torch.uint8)
    _call(q.device, L.gdn_qk_norm_rope_bwd, "gdn_qk_norm_rope_bwd", ref, _at(q), _at(k), _at(q_weight), _at(k_weight),
          _at(table), _at(positions), _at(dyq), _at(dyk), _at(dq), _at(dk), _at(dwq), _at(dwk), _at(ws), n)
    return dq, dk, dwq, dwk


@torch.library.custom_op("sorernn_b200::qk_norm_rope_bwd", mutates_args=())
def qk_norm_rope_bwd(q: Tensor, k: Tensor, q_weight: Tensor, k_weight: Tensor, table: Tensor, positions: Tensor,
                     sections: Sequence[int], interleaved: bool, eps: float, dyq: Tensor,
                     dyk: Tensor) -> tuple[Tensor, Tensor, Tensor, Tensor]:
    """Returns ``(dq, dk, dq_weight, dk_weight)``, the weights' in fp32."""
    return _bwd(q, k, q_weight, k_weight, table, positions, sections, interleaved, eps, dyq, dyk)


@qk_norm_rope_bwd.register_fake
def _(q, k, q_weight, k_weight, table, positions, sections, interleaved, eps, dyq, dyk):
    D = q.shape[-1]
    return (q.new_empty(q.shape), k.new_empty(k.shape), q.new_empty(D, dtype=torch.float32),
            q.new_empty(D, dtype=torch.float32))


def _setup_context(ctx, inputs, output):
    q, k, q_weight, k_weight, table, positions, sections, interleaved, eps = inputs
    ctx.save_for_backward(q, k, q_weight, k_weight, table, positions)
    ctx.args = (sections, interleaved, eps)


def _backward(ctx, dyq, dyk, bwd=qk_norm_rope_bwd):
    q, k, q_weight, k_weight, table, positions = ctx.saved_tensors
    dq, dk, dwq, dwk = bwd(q, k, q_weight, k_weight, table, positions, *ctx.args, dyq, dyk)
    return dq, dk, dwq.to(q_weight.dtype), dwk.to(k_weight.dtype), None, None, None, None, None


torch.library.register_autograd("sorernn_b200::qk_norm_rope_fwd", _backward, setup_context=_setup_context)


class _QkNormRope(torch.autograd.Function):
    """The eager form of the custom op pair, which spends more on dispatch than a small call on the GPU."""

    @staticmethod
    def forward(ctx, *inputs):
        _setup_context(ctx, inputs, None)
        return _fwd(*inputs)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dyq, dyk):
        return _backward(ctx, dyq, dyk, _bwd)


def qk_norm_rope(q: Tensor, k: Tensor, q_weight: Tensor, k_weight: Tensor, table: Tensor, positions: Tensor,
                 sections: Optional[Sequence[int]] = None, interleaved: bool = False,
                 eps: float = 1e-6) -> tuple[Tensor, Tensor]:
    """``q [B,T,HQ,D]`` and ``k [B,T,HK,D]``, each head's row normalised (``x / sqrt(mean(x^2) + eps) * weight``, the
    weights ``[D]``) and its first R features rotated; returns contiguous ``(q, k)`` in their dtype. fp32 arithmetic
    with one rounding.

    ``table`` (:func:`rotary_table`) is fp32 ``[P, R]`` with R even, at most D; ``positions`` (int64 or int32) holds
    rows of it: ``[B,T]``, or with ``sections`` (pairs per position axis, e.g. time, height, width; at most four, adding
    up to R/2) ``[len(sections),B,T]``: the first ``sections[0]`` pairs turn by axis 0, and so on. Pairs are
    ``(i, i + R/2)``, or ``(2i, 2i + 1)`` when ``interleaved``. A position outside the table makes its rotated features
    NaN. q and k may be strided views (features contiguous), such as slices of one projection's output. Gradients
    reach q, k and the weights; a table that requires one is refused.
    """
    if not q.is_cuda:
        raise RuntimeError("sorernn_b200 runs on CUDA tensors only (no CPU fallback)")
    q_shape, k_shape, dtype, w_dtype, device = q.shape, k.shape, q.dtype, q_weight.dtype, q.device
    if len(q_shape) != 4 or len(k_shape) != 4 or q_shape[:2] != k_shape[:2] or q_shape[3] != k_shape[3]:
        raise ValueError(f"q must be [B,T,HQ,D] and k [B,T,HK,D], got {tuple(q_shape)} and {tuple(k_shape)}")
    B, T, _, D = q_shape
    if not 1 <= D <= 512:
        raise ValueError(f"head size must be 1 .. 512, got {D}")
    if dtype != k.dtype or dtype not in _DT:
        raise ValueError(f"q and k must share one of bf16, fp16, fp32, got {dtype} and {k.dtype}")
    if q_weight.shape != (D,) or k_weight.shape != (D,) or w_dtype != k_weight.dtype or w_dtype not in _DT:
        raise ValueError(f"q_weight and k_weight must be [{D}] of one dtype, got {w_dtype} "
                         f"{tuple(q_weight.shape)} and {k_weight.dtype} {tuple(k_weight.shape)}")
    t_shape = table.shape
    if len(t_shape) != 2 or table.dtype != torch.float32 or t_shape[1] % 2 or not 0 < t_shape[1] <= D:
        raise ValueError(f"table must be fp32 [P,R] with R even and at most {D}, got {table.dtype} "
                         f"{tuple(t_shape)}")
    if table.requires_grad and torch.is_grad_enabled():
        raise ValueError("table takes no gradient: the angles are a constant of the model")
    sections = [int(n) for n in sections] if sections else []
    if sections and (len(sections) > 4 or min(sections) < 0 or 2 * sum(sections) != t_shape[1]):
        raise ValueError(f"sections must be at most four counts adding up to R/2 = {t_shape[1] // 2}, got "
                         f"{sections}")
    want = (len(sections), B, T) if sections else (B, T)
    if positions.shape != want or positions.dtype not in (torch.int64, torch.int32):
        raise ValueError(f"positions must be int64 or int32 {want}, got {positions.dtype} {tuple(positions.shape)}")
    if k.device != device or q_weight.device != device or k_weight.device != device or table.device != device \
            or positions.device != device:
        raise ValueError("all tensors must be on one device")
    q = q if q.stride(3) == 1 else q.contiguous()
    k = k if k.stride(3) == 1 else k.contiguous()
    q_weight, k_weight = q_weight.contiguous(), k_weight.contiguous()
    args = (q, k, q_weight, k_weight, table.contiguous(), positions.contiguous(), sections, bool(interleaved),
            float(eps))
    if torch.compiler.is_compiling():
        return qk_norm_rope_fwd(*args)
    _refuse_tangents("qk_norm_rope", q, k, q_weight, k_weight)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or q_weight.requires_grad or
                                    k_weight.requires_grad):
        return _QkNormRope.apply(*args)
    return _fwd(*args)
