"""Token-mixer layers on this package's CUDA ops: :class:`GatedDeltaNet`, a drop-in for soreRNN's
``sore.model.gdn.GatedDeltaNet`` (sore/model/gdn.py:92-206) at the layer boundary, and :class:`LinearAttention`, its
sibling without the delta rule (fixed decay per head, normed and rotated queries and keys).

GatedDeltaNet:

``o_proj(RMSNorm(o) * silu(g_proj(x)))`` with ``o`` the gated delta rule over the q/k/v projections after
a short causal convolution + SiLU. The parameters carry the reference layer's names and shapes, so its
``state_dict`` loads unchanged (and back). Every step between the projections is one of this package's
kernels: the convolution (``layer_ops.causal_conv1d``, per-document resets from ``cu_seqlens``), the gate
and beta activations (with ``kernel_gate``: ``-exp(A_log) softplus(a + dt_bias)`` and ``sigmoid(b)`` as
fused kernels with their backward), the gated delta rule with the in-kernel q/k L2 norm and native
grouped value heads (``chunk_gated_delta_rule``), and, with ``fused_norm_gate``, RMSNorm(o)·silu(gate) in one
kernel (``layer_ops.rms_norm_gated``). The projections are plain ``nn.Linear`` (library GEMMs).
"""
from __future__ import annotations

import math
from typing import Optional, Sequence

import torch
import torch.nn.functional as F
from torch import Tensor, nn

from .gated_delta_rule import chunk_gated_delta_rule
from .layer_ops import causal_conv1d, rms_norm_gated
from .linear_attention import chunk_linear_attention, linear_attention_step
from .rotary import qk_norm_rope, rotary_table


class _RMSNormWeight(nn.Module):
    """The output norm's weight (state_dict key ``o_norm.weight``) and its eps; unfused path in fp32."""

    def __init__(self, dim: int, eps: float) -> None:
        super().__init__()
        self.eps = eps
        self.weight = nn.Parameter(torch.ones(dim))

    def forward(self, x: Tensor) -> Tensor:
        xf = x.float()
        return (xf * torch.rsqrt(xf.pow(2).mean(-1, keepdim=True) + self.eps) * self.weight.float()).to(x.dtype)


class GatedDeltaNet(nn.Module):
    """``GatedDeltaNet(d_model, qk_heads, v_heads, head_dim=128, conv_kernel=4, norm_eps=1e-6,
    kernel_gate=True, fused_norm_gate=True)``; ``forward(x [B,T,d_model], cu_seqlens=None,
    cu_seqlens_cpu=None)``: with ``cu_seqlens`` (int64 ``[S+1]``, B == 1) the convolution and the recurrent
    state restart at every document; without it every batch row is a document. ``cu_seqlens_cpu`` (the same
    values on the host) only sizes buffers; nothing synchronises the host."""

    def __init__(self, d_model: int, qk_heads: int, v_heads: int, head_dim: int = 128, conv_kernel: int = 4,
                 norm_eps: float = 1e-6, kernel_gate: bool = True, fused_norm_gate: bool = True) -> None:
        super().__init__()
        if v_heads % qk_heads:
            raise ValueError(f"v_heads = {v_heads} must be a multiple of qk_heads = {qk_heads}")
        self.qk_heads, self.v_heads, self.head_dim = qk_heads, v_heads, head_dim
        self.kernel_gate, self.fused_norm_gate = kernel_gate, fused_norm_gate
        qk, vd = qk_heads * head_dim, v_heads * head_dim
        self.q_proj = nn.Linear(d_model, qk, bias=False)
        self.k_proj = nn.Linear(d_model, qk, bias=False)
        self.v_proj = nn.Linear(d_model, vd, bias=False)
        self.g_proj = nn.Linear(d_model, vd, bias=False)
        self.a_proj = nn.Linear(d_model, v_heads, bias=False)
        self.b_proj = nn.Linear(d_model, v_heads, bias=False)
        bound = conv_kernel ** -0.5
        self.conv_q = nn.Parameter(torch.empty(qk, conv_kernel).uniform_(-bound, bound))
        self.conv_k = nn.Parameter(torch.empty(qk, conv_kernel).uniform_(-bound, bound))
        self.conv_v = nn.Parameter(torch.empty(vd, conv_kernel).uniform_(-bound, bound))
        self.A_log = nn.Parameter(torch.empty(v_heads).uniform_(1, 16).log())
        log_dt = torch.rand(v_heads) * (math.log(1e-1) - math.log(1e-3)) + math.log(1e-3)
        dt = log_dt.exp()
        self.dt_bias = nn.Parameter(dt + torch.log(-torch.expm1(-dt)))
        self.o_norm = _RMSNormWeight(head_dim, norm_eps)
        self.o_proj = nn.Linear(vd, d_model, bias=False)

    def forward(self, x: Tensor, cu_seqlens: Optional[Tensor] = None,
                cu_seqlens_cpu: Optional[Tensor] = None) -> Tensor:
        b, t, _ = x.shape

        def conv(h: Tensor, w: Tensor) -> Tensor:
            return causal_conv1d(h, w, activation="silu", cu_seqlens=cu_seqlens, cu_seqlens_cpu=cu_seqlens_cpu)[0]

        q = conv(self.q_proj(x), self.conv_q).view(b, t, self.qk_heads, self.head_dim)
        k = conv(self.k_proj(x), self.conv_k).view(b, t, self.qk_heads, self.head_dim)
        v = conv(self.v_proj(x), self.conv_v).view(b, t, self.v_heads, self.head_dim)
        if self.kernel_gate:  # raw a/b projections; the activations run as fused kernels
            gate_kw = dict(use_gate_in_kernel=True, A_log=self.A_log, dt_bias=self.dt_bias,
                           use_beta_sigmoid_in_kernel=True)
            g, beta = self.a_proj(x), self.b_proj(x)
        else:
            gate_kw = {}
            g = -self.A_log.float().exp() * F.softplus(self.a_proj(x).float() + self.dt_bias.float())
            beta = self.b_proj(x).sigmoid()
        o, _ = chunk_gated_delta_rule(q, k, v, g, beta, scale=self.head_dim ** -0.5, cu_seqlens=cu_seqlens,
                                      cu_seqlens_cpu=cu_seqlens_cpu, use_qk_l2norm_in_kernel=True, **gate_kw)
        gate = self.g_proj(x).view(b, t, self.v_heads, self.head_dim)
        if self.fused_norm_gate:
            o = rms_norm_gated(o, gate, self.o_norm.weight, None, activation="swish", eps=self.o_norm.eps)
        else:
            o = self.o_norm(o) * F.silu(gate)
        return self.o_proj(o.flatten(-2))


class LinearAttention(nn.Module):
    """Linear attention with a fixed decay per head: ``o_proj(RMSNorm(o) * silu(g_proj(x)))`` with ``o`` the scan
    ``S <- a_h S + k v^T, o = S^T q / sqrt(head_dim)`` over queries and keys that are normed per head and rotated by
    their position in one pass (``qk_norm_rope``).

    ``LinearAttention(d_model, qk_heads, v_heads, head_dim=128, rotary_dim=None, max_positions=4096, theta=1e4,
    sections=None, log_decay=None, norm_eps=1e-6)``: ``rotary_dim`` features of each head turn (default: a quarter), with
    ``sections`` by several position axes; ``log_decay`` (``[v_heads]``, <= 0; default slopes from half-lives of one
    token to 180, spread geometrically) is a constant of the layer, kept in fp32 like the rotation's table whatever the
    parameters' dtype.

    ``forward(x [B,T,d_model], positions=None, cu_seqlens=None, cu_seqlens_cpu=None, initial_state=None,
    output_final_state=False)`` runs whole sequences (training, prefill): every batch row is a document, or with
    ``cu_seqlens`` (int64 ``[N+1]``, B == 1) every packed span; positions default to the token's place in its document,
    counted from 0 also where ``initial_state`` continues one (give ``positions`` there). A document that is known on the
    host to pass ``max_positions`` is refused; a position outside the table otherwise makes its outputs NaN.
    Returns y, or ``(y, state [N,v_heads,head_dim,head_dim])`` with ``output_final_state``.
    ``step(x [N,d_model], positions [N], state, state_indices=None)`` continues N requests by one token each on their
    fp32 states, updated in place (``linear_attention_step``); positions ``[axes,N]`` with ``sections``.
    """

    def __init__(self, d_model: int, qk_heads: int, v_heads: int, head_dim: int = 128,
                 rotary_dim: Optional[int] = None, max_positions: int = 4096, theta: float = 1e4,
                 sections: Optional[Sequence[int]] = None, log_decay: Optional[Sequence[float]] = None,
                 norm_eps: float = 1e-6) -> None:
        super().__init__()
        if v_heads % qk_heads:
            raise ValueError(f"v_heads = {v_heads} must be a multiple of qk_heads = {qk_heads}")
        self.qk_heads, self.v_heads, self.head_dim, self.norm_eps = qk_heads, v_heads, head_dim, norm_eps
        self.sections = list(sections) if sections else None
        qk, vd = qk_heads * head_dim, v_heads * head_dim
        self.q_proj = nn.Linear(d_model, qk, bias=False)
        self.k_proj = nn.Linear(d_model, qk, bias=False)
        self.v_proj = nn.Linear(d_model, vd, bias=False)
        self.g_proj = nn.Linear(d_model, vd, bias=False)
        self.q_norm = _RMSNormWeight(head_dim, norm_eps)
        self.k_norm = _RMSNormWeight(head_dim, norm_eps)
        self.o_norm = _RMSNormWeight(head_dim, norm_eps)
        self.o_proj = nn.Linear(vd, d_model, bias=False)
        if log_decay is None:
            log_decay = [-2.0 ** (-8.0 * (h + 1) / v_heads) for h in range(v_heads)]
        if len(log_decay) != v_heads or max(log_decay) > 0:
            raise ValueError(f"log_decay must be v_heads = {v_heads} values <= 0")
        self._log_decay = [float(x) for x in log_decay]
        self._table_args = (max_positions, head_dim // 4 if rotary_dim is None else rotary_dim, theta)
        for name, value in zip(("log_decay", "table"), self._constants(None)):
            self.register_buffer(name, value, persistent=False)

    def _constants(self, device: Optional[torch.device]) -> tuple[Tensor, Tensor]:
        return (torch.tensor(self._log_decay, dtype=torch.float32, device=device),
                rotary_table(*self._table_args, device=device))

    def _apply(self, fn, recurse: bool = True):
        before = self.log_decay, self.table
        super()._apply(fn, recurse)
        if self.table is not before[1]:  # moved, cast or emptied, as after construction on the meta device: the
            # constants keep their values, in fp32, and no checkpoint holds them
            device = self.table.device
            kept = self._constants(torch.device("cpu")) if before[1].is_meta else before
            self.log_decay, self.table = (t.to(device) for t in kept)
        return self

    def _qkv(self, x: Tensor, positions: Tensor) -> tuple[Tensor, Tensor, Tensor]:
        q = self.q_proj(x).unflatten(-1, (self.qk_heads, self.head_dim))
        k = self.k_proj(x).unflatten(-1, (self.qk_heads, self.head_dim))
        q, k = qk_norm_rope(q, k, self.q_norm.weight, self.k_norm.weight, self.table, positions,
                            sections=self.sections, eps=self.norm_eps)
        return q, k, self.v_proj(x).unflatten(-1, (self.v_heads, self.head_dim))

    def _out(self, x: Tensor, o: Tensor) -> Tensor:
        gate = self.g_proj(x).unflatten(-1, (self.v_heads, self.head_dim))
        o = rms_norm_gated(o, gate, self.o_norm.weight, None, activation="swish", eps=self.norm_eps)
        return self.o_proj(o.flatten(-2))

    def forward(self, x: Tensor, positions: Optional[Tensor] = None, cu_seqlens: Optional[Tensor] = None,
                cu_seqlens_cpu: Optional[Tensor] = None, initial_state: Optional[Tensor] = None,
                output_final_state: bool = False):
        b, t, _ = x.shape
        if positions is None:
            longest = t
            if cu_seqlens is not None:  # known on the host if the lengths are
                lengths = None if cu_seqlens_cpu is None else cu_seqlens_cpu[1:] - cu_seqlens_cpu[:-1]
                longest = int(lengths.max()) if lengths is not None and lengths.numel() else 0
            if longest > self.table.shape[0]:  # its rotated features would be NaN, and every token's after them
                raise ValueError(f"a document of {longest} tokens is longer than max_positions = {self.table.shape[0]}")
            positions = torch.arange(t, device=x.device)
            if cu_seqlens is not None:  # the place in the document, without reading the lengths on the host
                cu = cu_seqlens.to(x.device)
                positions = positions - cu[torch.searchsorted(cu, positions, right=True) - 1]
            positions = positions.expand(b, t)
            if self.sections:
                positions = positions.expand(len(self.sections), b, t)
        q, k, v = self._qkv(x, positions)
        o, state = chunk_linear_attention(q, k, v, self.log_decay, initial_state=initial_state,
                                          output_final_state=output_final_state, cu_seqlens=cu_seqlens,
                                          cu_seqlens_cpu=cu_seqlens_cpu)
        y = self._out(x, o)
        return (y, state) if output_final_state else y

    def step(self, x: Tensor, positions: Tensor, state: Tensor, state_indices: Optional[Tensor] = None) -> Tensor:
        q, k, v = self._qkv(x[:, None], positions[..., None])
        o = linear_attention_step(q[:, 0], k[:, 0], v[:, 0], self.log_decay, state, state_indices=state_indices)
        return self._out(x, o)
