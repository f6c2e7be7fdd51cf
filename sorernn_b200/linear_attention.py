"""Linear attention with a fixed decay per head: the mixer without the delta rule, chunked and by the token.

Per sequence and value head h, with ``a_h = exp(log_decay[h])`` and state S ``[K, V]``::

    S_t = a_h S_(t-1) + k_t v_t^T        o_t = scale S_t^T q_t

* :func:`chunk_linear_attention` — whole sequences, forward and (under autograd) backward; layouts, grouped value
  heads, ``cu_seqlens`` and states as in :func:`sorernn_b200.chunk_gated_delta_rule`;
* :func:`linear_attention_step` — one decode token on a resident fp32 state (optionally a pool of slots), in place.

The backward needs nothing from the forward but its inputs. Both are thin calls into the C ABI
(include/gdn_b200.h, ``gdn_linear_attn_*``) on the current stream; there is no CPU fallback. ``torch.compile``
traces the custom ops ``sorernn_b200::linear_attn_fwd`` / ``linear_attn_bwd``; eager calls go to the library directly.
"""
from __future__ import annotations

import ctypes
from typing import Optional

import torch
from torch import Tensor
from torch.autograd import forward_ad

from . import _lib
from .gated_delta_rule import _DT


def _at(t: Optional[Tensor]):
    return None if t is None else t.data_ptr()


def _aligned(t: Optional[Tensor]) -> Optional[Tensor]:
    """``t`` (contiguous), or a copy where its memory starts off the library's 16-byte grid, as that of a slice may;
    autograd hands such slices over as gradients, of a concatenation for instance."""
    return t if t is None or t.data_ptr() % 16 == 0 else t.clone()


def _refuse_tangents(name: str, *tensors: Optional[Tensor]) -> None:
    """The kernels have no forward-mode derivative, and read the primal values alone."""
    if getattr(forward_ad, "_current_level", -1) >= 0 and any(
            t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise NotImplementedError(f"{name} has no forward-mode derivative")


def _call(device: torch.device, fn, name: str, *args) -> None:
    """One library call on ``device``'s current stream (the last argument of every entry point)."""
    index = device.index
    stream = torch._C._cuda_getCurrentRawStream(index)  # the handle alone: no Stream object per call
    if index != torch._C._cuda_getDevice():
        with torch.cuda.device(device):
            status = fn(*args, stream)
    else:
        status = fn(*args, stream)
    if status != 0:
        _lib.check(status, name)


def _problem(q: Tensor, v: Tensor, cu_seqlens: Optional[Tensor], scale: float,
             max_seqlen: int) -> _lib.LinearAttnProblem:
    B, T, H, K = q.shape
    _, _, HV, V = v.shape
    return _lib.LinearAttnProblem(B, T, H, HV, K, V, B if cu_seqlens is None else cu_seqlens.shape[0] - 1,
                                  _at(cu_seqlens), max_seqlen, scale, _DT[q.dtype])


def _fwd(q, k, v, log_decay, initial_state, cu_seqlens, scale, max_seqlen, want_state):
    L = _lib.lib()
    p = _problem(q, v, cu_seqlens, scale, max_seqlen)
    q, k, v, initial_state = _aligned(q), _aligned(k), _aligned(v), _aligned(initial_state)
    o = torch.empty_like(v)
    final = q.new_empty((p.N, p.HV, p.DK, p.DV), dtype=torch.float32) if want_state else None
    ref = ctypes.byref(p)
    n = L.gdn_linear_attn_fwd_workspace_size(ref)
    ws = q.new_empty(n, dtype=torch.uint8) if n else None
    _call(q.device, L.gdn_linear_attn_fwd, "gdn_linear_attn_fwd", ref, _at(q), _at(k), _at(v), _at(log_decay),
          _at(initial_state), _at(o), _at(final), _at(ws), n)
    return o, final


@torch.library.custom_op("sorernn_b200::linear_attn_fwd", mutates_args=())
def linear_attn_fwd(q: Tensor, k: Tensor, v: Tensor, log_decay: Tensor, initial_state: Optional[Tensor],
                    cu_seqlens: Optional[Tensor], scale: float, max_seqlen: int,
                    want_state: bool) -> tuple[Tensor, Tensor]:
    """Returns ``(o, final_state)``; ``final_state`` is empty unless ``want_state``."""
    o, final = _fwd(q, k, v, log_decay, initial_state, cu_seqlens, scale, max_seqlen, want_state)
    return o, q.new_empty(0, dtype=torch.float32) if final is None else final


@linear_attn_fwd.register_fake
def _(q, k, v, log_decay, initial_state, cu_seqlens, scale, max_seqlen, want_state):
    N = q.shape[0] if cu_seqlens is None else cu_seqlens.shape[0] - 1
    shape = (N, v.shape[2], q.shape[3], v.shape[3]) if want_state else (0,)
    return torch.empty_like(v), q.new_empty(shape, dtype=torch.float32)


def _bwd(q, k, v, log_decay, initial_state, do, dht, cu_seqlens, scale, max_seqlen, want_dh0):
    L = _lib.lib()
    p = _problem(q, v, cu_seqlens, scale, max_seqlen)
    dq, dk, dv = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)
    dh0 = q.new_empty((p.N, p.HV, p.DK, p.DV), dtype=torch.float32) if want_dh0 else None
    q, k, v, initial_state = _aligned(q), _aligned(k), _aligned(v), _aligned(initial_state)
    do = _aligned(do.contiguous())
    dht = None if dht is None else _aligned(dht.float().contiguous())
    ref = ctypes.byref(p)
    n = L.gdn_linear_attn_bwd_workspace_size(ref)
    ws = q.new_empty(n, dtype=torch.uint8) if n else None
    _call(q.device, L.gdn_linear_attn_bwd, "gdn_linear_attn_bwd", ref, _at(q), _at(k), _at(v), _at(log_decay),
          _at(initial_state), _at(do), _at(dht), _at(dq), _at(dk), _at(dv), _at(dh0), _at(ws), n)
    return dq, dk, dv, dh0


@torch.library.custom_op("sorernn_b200::linear_attn_bwd", mutates_args=())
def linear_attn_bwd(q: Tensor, k: Tensor, v: Tensor, log_decay: Tensor, initial_state: Optional[Tensor], do: Tensor,
                    dht: Optional[Tensor], cu_seqlens: Optional[Tensor], scale: float, max_seqlen: int,
                    want_dh0: bool) -> tuple[Tensor, Tensor, Tensor, Tensor]:
    """Returns ``(dq, dk, dv, dh0)``; ``dh0`` (fp32) is empty unless ``want_dh0``."""
    dq, dk, dv, dh0 = _bwd(q, k, v, log_decay, initial_state, do, dht, cu_seqlens, scale, max_seqlen, want_dh0)
    return dq, dk, dv, q.new_empty(0, dtype=torch.float32) if dh0 is None else dh0


@linear_attn_bwd.register_fake
def _(q, k, v, log_decay, initial_state, do, dht, cu_seqlens, scale, max_seqlen, want_dh0):
    N = q.shape[0] if cu_seqlens is None else cu_seqlens.shape[0] - 1
    shape = (N, v.shape[2], q.shape[3], v.shape[3]) if want_dh0 else (0,)
    return torch.empty_like(q), torch.empty_like(k), torch.empty_like(v), q.new_empty(shape, dtype=torch.float32)


def _setup_context(ctx, inputs, output):
    q, k, v, log_decay, initial_state, cu_seqlens, scale, max_seqlen, want_state = inputs
    ctx.save_for_backward(q, k, v, log_decay, initial_state, cu_seqlens)
    ctx.args = (scale, max_seqlen)
    ctx.set_materialize_grads(False)


def _backward(ctx, do, dht, bwd=linear_attn_bwd):
    q, k, v, log_decay, initial_state, cu_seqlens = ctx.saved_tensors
    scale, max_seqlen = ctx.args
    if do is None:  # only the final state reaches the loss
        if dht is None:
            return (None,) * 9
        do = torch.zeros_like(v)
    want_dh0 = initial_state is not None and ctx.needs_input_grad[4]
    dq, dk, dv, dh0 = bwd(q, k, v, log_decay, initial_state, do, dht if dht is not None and dht.numel() else None,
                          cu_seqlens, scale, max_seqlen, want_dh0)
    return dq, dk, dv, None, (dh0 if want_dh0 else None), None, None, None, None


torch.library.register_autograd("sorernn_b200::linear_attn_fwd", _backward, setup_context=_setup_context)


class _LinearAttn(torch.autograd.Function):
    """The eager form of the custom op pair, which spends more on dispatch than a small call on the GPU."""

    @staticmethod
    def forward(ctx, *inputs):
        out = _fwd(*inputs)
        _setup_context(ctx, inputs, out)
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, do, dht):
        return _backward(ctx, do, dht, _bwd)


def _check_log_decay(log_decay: Tensor, HV: int, device: torch.device) -> Tensor:
    if log_decay.shape != (HV,) or log_decay.dtype != torch.float32 or log_decay.device != device:
        raise ValueError(f"log_decay must be fp32 [HV] = [{HV}] on {device}, got {log_decay.dtype} "
                         f"{tuple(log_decay.shape)} on {log_decay.device}")
    if log_decay.requires_grad:
        raise ValueError("log_decay takes no gradient: a head's decay is a constant of the model")
    return log_decay.contiguous()


def chunk_linear_attention(q: Tensor, k: Tensor, v: Tensor, log_decay: Tensor, scale: Optional[float] = None,
                           initial_state: Optional[Tensor] = None, output_final_state: bool = False,
                           cu_seqlens: Optional[Tensor] = None, cu_seqlens_cpu: Optional[Tensor] = None):
    """Linear attention over whole sequences: q, k ``[B,T,H,K]``, v ``[B,T,HV,V]`` (HV a multiple of H: value head i
    uses q/k head ``i // (HV // H)``), ``log_decay`` fp32 ``[HV]`` (<= 0; no gradient), ``initial_state``
    ``[N,HV,K,V]``. K and V are at most 128; bf16 with K, V in {64, 128} runs on the tensor cores. Returns
    ``(o [B,T,HV,V], final_state [N,HV,K,V] fp32 or None)``; gradients reach q, k, v and ``initial_state``.

    ``cu_seqlens`` (int64 ``[N+1]``, B == 1) restarts the state at every document; ``cu_seqlens_cpu`` (the same values
    on the host) is read only to size the work, never to synchronise. A NaN or infinity stays within its own document
    (before its token, it can reach the outputs of the same 128-token chunk).
    """
    if not q.is_cuda:
        raise RuntimeError("sorernn_b200 runs on CUDA tensors only (no CPU fallback)")
    if q.shape != k.shape or q.dim() != 4:
        raise ValueError(f"q and k must be [B,T,H,K] with equal shapes, got {tuple(q.shape)} and {tuple(k.shape)}")
    B, T, H, K = q.shape
    if v.dim() != 4 or v.shape[:2] != (B, T) or H == 0 or v.shape[2] == 0 or v.shape[2] % H:
        raise ValueError(f"v must be [B,T,HV,V] with HV a multiple of H, got {tuple(v.shape)}")
    HV, V = v.shape[2], v.shape[3]
    if not 1 <= K <= 128 or not 1 <= V <= 128:
        raise ValueError(f"head sizes must be 1 .. 128, got K = {K}, V = {V}")
    if q.dtype != k.dtype or q.dtype != v.dtype or q.dtype not in _DT:
        raise ValueError(f"q, k and v must share one of bf16, fp16, fp32, got {q.dtype}, {k.dtype}, {v.dtype}")
    if k.device != q.device or v.device != q.device:
        raise ValueError("q, k and v must be on one device")
    log_decay = _check_log_decay(log_decay, HV, q.device)
    N, max_seqlen = B, T
    if cu_seqlens is not None:
        if B != 1:
            raise ValueError(f"cu_seqlens requires B == 1, got B = {B}")
        if cu_seqlens.dim() != 1 or cu_seqlens.shape[0] < 1:
            raise ValueError(f"cu_seqlens must be [N+1], got {tuple(cu_seqlens.shape)}")
        if cu_seqlens.dtype != torch.int64 or cu_seqlens.device != q.device or not cu_seqlens.is_contiguous():
            cu_seqlens = cu_seqlens.to(device=q.device, dtype=torch.int64).contiguous()
        N = cu_seqlens.shape[0] - 1
        if cu_seqlens_cpu is not None:
            if cu_seqlens_cpu.shape != cu_seqlens.shape:
                raise ValueError(f"cu_seqlens_cpu must have cu_seqlens' shape, got {tuple(cu_seqlens_cpu.shape)}")
            max_seqlen = int((cu_seqlens_cpu[1:] - cu_seqlens_cpu[:-1]).max()) if N else 0
    if initial_state is not None:
        if initial_state.shape != (N, HV, K, V) or initial_state.device != q.device:
            raise ValueError(f"initial_state must be {(N, HV, K, V)} on {q.device}, got "
                             f"{tuple(initial_state.shape)} on {initial_state.device}")
        initial_state = initial_state.float().contiguous()
    scale = K ** -0.5 if scale is None else float(scale)
    q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
    args = (q, k, v, log_decay, initial_state, cu_seqlens, scale, max_seqlen, output_final_state)
    if torch.compiler.is_compiling():
        o, final = linear_attn_fwd(*args)
        return o, (final if output_final_state else None)
    _refuse_tangents("chunk_linear_attention", q, k, v, initial_state)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad or
                                      initial_state is not None and initial_state.requires_grad):
        o, final = _LinearAttn.apply(*args)
    else:
        o, final = _fwd(*args)
    return o, (final if output_final_state else None)


def _step(N, H, HV, K, V, scale, act_dtype, q, k, v, log_decay, state, slots, state_indices, out):
    _call(q.device, _lib.lib().gdn_linear_attn_step, "gdn_linear_attn_step", N, H, HV, K, V, scale, act_dtype,
          _at(q), _at(k), _at(v), _at(log_decay), _at(state), slots, _at(state_indices), _at(out))
    torch.autograd.graph.increment_version((state, out))  # written in place: autograd may have saved them
    return out


class _Step(torch.autograd.Function):
    """The step where autograd records: a backward through it says that there is none, instead of losing gradients."""

    @staticmethod
    def forward(ctx, args, *recorded):  # `out` in the tuple: an output, not an input, to autograd
        return _step(*args)

    @staticmethod
    def backward(ctx, do):
        raise RuntimeError("linear_attention_step has no backward (it updates its state in place): train through "
                           "chunk_linear_attention")


def linear_attention_step(q: Tensor, k: Tensor, v: Tensor, log_decay: Tensor, state: Tensor,
                          scale: Optional[float] = None, state_indices: Optional[Tensor] = None,
                          out: Optional[Tensor] = None) -> Tensor:
    """One decode token per request: ``q, k [N,H,K]``, ``v [N,HV,V]``, ``log_decay`` fp32 ``[HV]``, ``state`` fp32,
    updated in place. Returns ``o [N,HV,V]`` in v's dtype (written into ``out`` if given).

    Without ``state_indices``, ``state`` is ``[N,HV,K,V]``. With ``state_indices`` (int32 ``[N]`` on the device, no two
    alike), ``state`` is a pool ``[slots,HV,K,V]`` and request n uses ``state[state_indices[n]]``; a negative index is
    an idle request (its output is zero, no state changes) and an index past the pool gives NaN and touches nothing.
    Where V is a multiple of 4 the state's memory has to start on a 16-byte boundary. For decoding: there is no backward.
    """
    if not q.is_cuda:
        raise RuntimeError("sorernn_b200 runs on CUDA tensors only (no CPU fallback)")
    q_shape, v_shape, dtype, device = q.shape, v.shape, q.dtype, q.device
    if len(q_shape) != 3 or k.shape != q_shape:
        raise ValueError(f"q and k must be [N,H,K] with equal shapes, got {tuple(q_shape)} and {tuple(k.shape)}")
    N, H, K = q_shape
    if len(v_shape) != 3 or v_shape[0] != N or H == 0 or v_shape[1] == 0 or v_shape[1] % H:
        raise ValueError(f"v must be [N,HV,V] with HV a multiple of H, got {tuple(v_shape)}")
    _, HV, V = v_shape
    if not 1 <= K <= 128 or not 1 <= V <= 128:
        raise ValueError(f"head sizes must be 1 .. 128, got K = {K}, V = {V}")
    if dtype != k.dtype or dtype != v.dtype or dtype not in _DT:
        raise ValueError(f"q, k and v must share one of bf16, fp16, fp32, got {dtype}, {k.dtype}, {v.dtype}")
    if state.dtype != torch.float32 or not state.is_contiguous() or k.device != device or v.device != device \
            or state.device != device:
        raise ValueError("state must be a contiguous fp32 tensor on q's device")
    s_shape = state.shape
    if len(s_shape) != 4 or s_shape[1:] != (HV, K, V) or (state_indices is None and s_shape[0] != N):
        raise ValueError(f"state must be {(N if state_indices is None else 'slots', HV, K, V)}, got "
                         f"{tuple(s_shape)}")
    if state_indices is not None:
        if state_indices.shape != (N,) or state_indices.dtype != torch.int32 or state_indices.device != device:
            raise ValueError(f"state_indices must be int32 [{N}] on {device}, got {state_indices.dtype} "
                             f"{tuple(state_indices.shape)} on {state_indices.device}")
        state_indices = state_indices.contiguous()
    log_decay = _check_log_decay(log_decay, HV, device)
    if out is None:
        out = torch.empty_like(v, memory_format=torch.contiguous_format)
    elif out.shape != v_shape or out.dtype != dtype or out.device != device or not out.is_contiguous():
        raise ValueError(f"out must be a contiguous {dtype} tensor {tuple(v_shape)} on {device}")
    scale = K ** -0.5 if scale is None else float(scale)
    args = (N, H, HV, K, V, scale, _DT[dtype], q.contiguous(), k.contiguous(), v.contiguous(), log_decay, state,
            s_shape[0], state_indices, out)
    _refuse_tangents("linear_attention_step", q, k, v, state)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad or state.requires_grad):
        return _Step.apply(args, q, k, v, state)
    return _step(*args)
