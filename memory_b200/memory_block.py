"""The memory step of the reference's ``MemoryTransformerBlock`` (memory_transformer/memory_block.py:468-487,
549-558): ``h + memory_attn(memory_layernorm(h), memory)``, with the submodule and parameter names of that
block so the matching slice of its state dict loads unchanged.  Self-attention and the MLPs of the block are
not part of this package."""
from __future__ import annotations

from typing import Optional

import torch
import torch.nn as nn

from . import functional as F_moc
from . import ops
from .memory_attention import MemoryCrossAttention


class _Norm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, kind, eps):
        shape = x.shape
        x2 = x.reshape(-1, shape[-1]).float()
        y, stats = ops.norm_fwd(x2, weight.float(), None if bias is None else bias.float(), kind, eps,
                                torch.float32)
        ctx.save_for_backward(x2, weight.float(), stats)
        ctx.cfg = (kind, bias is not None, shape, x.dtype, weight.dtype)
        return y.view(shape).to(x.dtype)

    @staticmethod
    def backward(ctx, g):
        x2, w, stats = ctx.saved_tensors
        kind, has_bias, shape, x_dtype, w_dtype = ctx.cfg
        dx, dw, db = ops.norm_bwd(g.reshape(-1, shape[-1]).float(), x2, w, stats, None, kind, has_bias)
        return dx.view(shape).to(x_dtype), dw.to(w_dtype), None if db is None else db.to(w_dtype), None, None


class RMSNorm(nn.Module):
    """x / sqrt(mean(x^2) + eps) * weight (memory_block.py:18-28), on the GPU."""

    def __init__(self, dim: int, eps: float = 1e-6):
        super().__init__()
        self.eps = eps
        self.weight = nn.Parameter(torch.ones(dim))

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return _Norm.apply(x, self.weight, None, "rms", self.eps)


class MemorySubBlock(nn.Module):
    """``forward(hidden_states, memory) -> hidden_states + memory_attn(memory_layernorm(hidden_states), memory)``.

    The normalisation writes the query projection's operand directly and the residual is added in the
    output projection's epilogue, so neither costs a pass over (B, L, d) of its own.  With ``post_norm`` the block is
    ``residual_scale * hidden_states + gate * post_norm(memory_attn(...))`` (:func:`memory_b200.gated_residual_norm`).
    """

    def __init__(self, hidden_dim: int, num_heads: int, num_kv_heads: Optional[int] = None,
                 memory_dim: Optional[int] = None, use_rms_norm: bool = True, norm_eps: float = 1e-6,
                 wo_init_zero: bool = True, compute_dtype: Optional[torch.dtype] = None, post_norm: bool = False,
                 gate: bool = False, residual_scale: float = 1.0):
        super().__init__()
        if (gate or residual_scale != 1.0) and not post_norm:
            raise ValueError("gate and residual_scale go with post_norm")
        self.use_rms_norm = use_rms_norm
        self.norm_eps = norm_eps
        self.memory_layernorm = RMSNorm(hidden_dim, eps=norm_eps) if use_rms_norm else nn.LayerNorm(hidden_dim,
                                                                                                    eps=norm_eps)
        self.memory_attn = MemoryCrossAttention(hidden_dim, num_heads, num_kv_heads=num_kv_heads,
                                                memory_dim=memory_dim, wo_init_zero=wo_init_zero,
                                                compute_dtype=compute_dtype)
        self.residual_scale = float(residual_scale)
        self.post_norm = None
        if post_norm:
            self.post_norm = RMSNorm(hidden_dim, eps=norm_eps) if use_rms_norm else nn.LayerNorm(hidden_dim, eps=norm_eps)
        self.gate = nn.Parameter(torch.ones(hidden_dim)) if gate else None

    def __setstate__(self, state):
        """Modules that were saved whole before there was a norm behind the block have none."""
        super().__setstate__(state)
        for name, value, kept in (("residual_scale", 1.0, {}), ("post_norm", None, self._modules), ("gate", None, self._parameters)):
            if name not in kept:
                self.__dict__.setdefault(name, value)

    def forward(self, hidden_states: torch.Tensor, memory: torch.Tensor, *, gate: Optional[torch.Tensor] = None,
                next_norm: Optional[nn.Module] = None):
        """``gate`` [B, d]: a gate for every sequence instead of the module's own; ``next_norm``: the norm in front of the block that
        follows (of this module's kind), whose result is returned beside the new hidden states.  Both go with ``post_norm``."""
        if memory is None:
            raise ValueError("memory must be provided")
        a = self.memory_attn
        if self.post_norm is not None:
            if next_norm is not None and (type(next_norm) is not type(self.post_norm) or next_norm.weight is None):
                raise ValueError("next_norm must be a norm of this module's kind, with a weight")
            branch = F_moc.cross_attention(
                hidden_states, memory, a.q_proj.weight, a.k_proj.weight, a.v_proj.weight, a.o_proj.weight,
                a.num_heads, a.num_kv_heads, a._compute_dtype(hidden_states),
                pre_norm="rms" if self.use_rms_norm else "layernorm", norm_weight=self.memory_layernorm.weight,
                norm_bias=getattr(self.memory_layernorm, "bias", None), norm_eps=self.norm_eps, add_residual=False)
            # states of another type than the kernels take go through fp32, as they go through the compute type in front of the block
            dtype = hidden_states.dtype
            if dtype not in F_moc._KERNEL_DTYPES:
                hidden_states, branch = hidden_states.float(), branch.float()
            got = F_moc.gated_residual_norm(
                hidden_states, branch, self.post_norm.weight, getattr(self.post_norm, "bias", None),
                norm_type="rms" if self.use_rms_norm else "layernorm", eps=self.norm_eps,
                gate=self.gate if gate is None else gate, residual_scale=self.residual_scale,
                next_weight=None if next_norm is None else next_norm.weight, next_bias=getattr(next_norm, "bias", None),
                next_eps=None if next_norm is None else next_norm.eps)
            if hidden_states.dtype == dtype:
                return got
            return got.to(dtype) if next_norm is None else (got[0].to(dtype), got[1].to(dtype))
        if gate is not None or next_norm is not None:
            raise ValueError("gate and next_norm go with post_norm")
        return F_moc.cross_attention(
            hidden_states, memory, a.q_proj.weight, a.k_proj.weight, a.v_proj.weight, a.o_proj.weight,
            a.num_heads, a.num_kv_heads, a._compute_dtype(hidden_states),
            pre_norm="rms" if self.use_rms_norm else "layernorm", norm_weight=self.memory_layernorm.weight,
            norm_bias=getattr(self.memory_layernorm, "bias", None), norm_eps=self.norm_eps, add_residual=True)
