"""Optimizer step of the memory bank from the compact gradient the backward pass produces.

The reference hands the bank to ``torch.optim.AdamW`` as its own parameter group (training/trainer.py:338-347,
372-378) and feeds it the dense 262,208 x 768 gradient of ``torch.gather``'s backward.  ``SparseBankAdamW`` applies
the identical update -- every row, bias-corrected moments, decoupled weight decay -- straight from a
``SparseBankGrad`` (chapter ids + rows), in one kernel pass, and can refresh the bf16 working copy of the bank in
the same pass.  ``clip_grad_norm_`` is the clipping in front of it (training/trainer.py:876-880), over dense gradients and
compact ones, without a host round trip.
"""
from __future__ import annotations

from operator import attrgetter
from typing import Iterable, NamedTuple, Optional, Sequence, Tuple, Union

import torch
from torch.autograd.graph import increment_version

from . import ops
from .functional import SparseBankGrad


class SparseBankAdamW:
    """AdamW for one bank parameter ([rows, d] fp32) driven by compact gradients.

    ``step(grad)`` takes the ``SparseBankGrad`` a backward pass (or ``GradReducer``) filled; its ``scale`` and the
    optional ``grad_scale`` (a number, or a tensor of one: the coefficient ``clip_grad_norm_`` left on the device, or one formed by hand, in
    any type and on any device) multiply the gradient.  ``state_dict`` / ``load_state_dict``
    use torch.optim.AdamW's per-parameter keys (``step``, ``exp_avg``, ``exp_avg_sq``), so optimizer state moves
    between the two."""

    def __init__(self, param: torch.Tensor, tokens_per_chapter: int, lr: float = 1e-4,
                 betas: Tuple[float, float] = (0.9, 0.95), eps: float = 1e-8, weight_decay: float = 0.01,
                 shadow: Optional[torch.Tensor] = None):
        if param.dtype != torch.float32 or param.dim() != 2 or not param.is_contiguous():
            raise TypeError("the bank parameter must be a contiguous fp32 [rows, d] tensor")
        if param.shape[0] % int(tokens_per_chapter) != 0:
            raise ValueError("bank rows must be a whole number of chapters")
        self.param = param
        self.t = int(tokens_per_chapter)
        self.lr, self.betas, self.eps, self.weight_decay = float(lr), tuple(betas), float(eps), float(weight_decay)
        self.exp_avg = torch.zeros_like(param, memory_format=torch.contiguous_format)
        self.exp_avg_sq = torch.zeros_like(param, memory_format=torch.contiguous_format)
        self.step_count = 0
        self.shadow = shadow       # bf16 [rows, d] refreshed by every step, or None
        self._ws = None

    @torch.no_grad()
    def step(self, grad: SparseBankGrad, grad_scale: Union[float, torch.Tensor] = 1.0, lr: Optional[float] = None) -> None:
        if len(grad.entries) != 1:
            raise NotImplementedError(
                "one compact entry per step: sum several layers' entries first (ops.bank_grad_merge)")
        uniq, num_unique, rows, t = grad.entries[0]
        if t != self.t:
            raise ValueError("gradient rows were produced with a different chapter size")
        on_device = torch.is_tensor(grad_scale) and grad_scale.is_cuda
        if on_device:
            grad_scale = _device_scale(grad_scale, self.param.device)
        self.step_count += 1
        if self._ws is None:
            self._ws = torch.empty(4 * (self.param.shape[0] // self.t), dtype=torch.uint8, device=self.param.device)
        ops.bank_adamw_step(self.param.data, self.exp_avg, self.exp_avg_sq, uniq, num_unique,
                            rows if rows.dtype == torch.float32 else rows.float(), self.t,
                            lr=self.lr if lr is None else lr, betas=self.betas, eps=self.eps,
                            weight_decay=self.weight_decay, step=self.step_count,
                            grad_scale=float(grad.scale) * (1.0 if on_device else float(grad_scale)), shadow=self.shadow,
                            workspace=self._ws, device_scale=grad_scale if on_device else None)

    def grad_sqnorm(self, grad: SparseBankGrad) -> torch.Tensor:
        """Squared L2 norm of the (scaled) bank gradient as a [1] tensor: the bank's term of a global clip norm."""
        uniq, num_unique, rows, t = grad.entries[0]
        return ops.rows_sqnorm(rows if rows.dtype == torch.float32 else rows.float(), num_unique, t) * (grad.scale ** 2)

    def state_dict(self):
        return {"step": torch.tensor(float(self.step_count)), "exp_avg": self.exp_avg, "exp_avg_sq": self.exp_avg_sq}

    def load_state_dict(self, state) -> None:
        self.step_count = int(state["step"])
        self.exp_avg.copy_(state["exp_avg"])
        self.exp_avg_sq.copy_(state["exp_avg_sq"])


def _device_scale(scale: torch.Tensor, device: torch.device) -> torch.Tensor:
    """One number of any type on a GPU as fp32 on ``device``, without a host round trip."""
    if scale.numel() != 1 or scale.is_complex() or (scale.dim() > 0 and scale.dtype == torch.float64):
        raise TypeError("a gradient scale on the device must be one number: a 0-d tensor, or one element of at most 32 bits")
    return scale.detach().to(device=device, dtype=torch.float32)


class GradClip(NamedTuple):
    """Result of :func:`clip_grad_norm_`, both 0-d fp32 on the device: the global norm before clipping, and the factor
    min(1, max_norm / (norm + eps)) that the gradients were multiplied by (pass it to ``SparseBankAdamW.step`` as
    ``grad_scale`` for the bank)."""
    total_norm: torch.Tensor
    coefficient: torch.Tensor


def clip_grad_norm_(parameters: Union[torch.Tensor, Iterable[torch.Tensor]], max_norm: float, *,
                    bank_grads: Sequence[SparseBankGrad] = (), out: Optional[Sequence[torch.Tensor]] = None,
                    eps: float = 1e-6) -> GradClip:
    """Clips gradients by their global norm in two kernel launches, without a host synchronisation.

    ``parameters``: leaves with a gradient (their ``.grad`` is clipped; those without one are passed over), or gradient tensors
    themselves, fp32, bf16 or fp16 in any mix, all on one device.  ``bank_grads``: compact bank gradients (at most one entry
    each, with their ``scale``) that count in the norm; their rows are left as they are -- give the coefficient to the optimizer
    step.  ``out``: one tensor per gradient (same shape, any of the three types) that receives the clipped values instead of the gradients.

    As with ``torch.nn.utils.clip_grad_norm_`` a norm that is NaN makes every gradient NaN and an infinite one gives the coefficient 0.
    Squares are summed in 64 bits.  A tensor listed twice counts once; dense tensors that overlap otherwise are refused,
    and so are more than 4096 tensors."""
    if not max_norm >= 0:
        raise ValueError(f"max_norm must not be negative, got {max_norm}")
    if not eps >= 0:
        raise ValueError(f"eps must not be negative, got {eps}")
    listed = (parameters,) if torch.is_tensor(parameters) else parameters
    found = [p if type(p) is torch.Tensor and not p.requires_grad else _gradient(p) for p in listed]
    grads = [g for g in found if g is not None]
    outs = grads
    if out is not None:
        outs = list(out)
        if len(outs) != len(found):
            raise ValueError(f"out must have one tensor per gradient: {len(outs)} vs {len(found)}")
        outs = [o for g, o in zip(found, outs) if g is not None]
    banks = []
    for sink in bank_grads:
        if len(sink.entries) > 1:
            raise NotImplementedError("one compact entry per bank: sum several layers' entries first (ops.bank_grad_merge)")
        for _, count, rows, t in sink.entries:
            banks.append((ops._contig(rows), count, t * rows.shape[1], float(sink.scale)))
    if not grads and not banks:
        raise ValueError("no gradients to clip")
    device = grads[0].device if grads else banks[0][0].device
    tensors = grads if outs is grads else [*grads, *outs]
    where = set(map(torch.Tensor.get_device, tensors))
    for rows, count, _, _ in banks:
        where |= {rows.get_device(), count.get_device()}
    if device.type != "cuda" or len(where) != 1 or any(map(_is_sparse, tensors)):
        raise ValueError("gradients must be dense CUDA tensors on one device")
    if outs is not grads and list(map(_shape, outs)) != list(map(_shape, grads)):
        raise ValueError("out must match the gradients in shape")
    copies: list = []
    ptrs = list(map(torch.Tensor.data_ptr, grads))
    if len(set(ptrs)) < len(ptrs) or not all(map(torch.Tensor.is_contiguous, tensors)):
        grads, outs, copies = _distinct_and_dense(grads, outs)
        ptrs = list(map(torch.Tensor.data_ptr, grads))
    result = ops.grad_clip(grads, ptrs, outs, banks, max_norm, eps, device)
    increment_version(outs)          # (written behind autograd's back: a graph that saved one of them has to notice)
    if copies:
        with torch.no_grad():
            for o, dense in copies:
                o.copy_(dense)
    return GradClip(result.as_strided((), (), 0), result.as_strided((), (), 1))


_shape, _is_sparse = attrgetter("shape"), attrgetter("is_sparse")


def _gradient(p: torch.Tensor) -> Optional[torch.Tensor]:
    return p.grad if isinstance(p, torch.nn.Parameter) or p.is_leaf else p.detach()


def _distinct_and_dense(grads: list, outs: list):
    """The same lists without a gradient's second mention, with dense copies in the place of other layouts: (gradients, outputs,
    (tensor, dense copy) pairs to copy back)."""
    in_place, seen, src, dst, copies = outs is grads, set(), [], [], []
    for g, o in zip(grads, outs):
        key = (g.data_ptr(), g.shape, g.stride(), g.dtype)
        if g.numel() == 0:
            continue
        if key in seen:
            if in_place:
                continue
            raise ValueError("a gradient is listed twice with an out of its own")
        seen.add(key)
        src.append(g.contiguous())
        dst.append(src[-1] if in_place else o if o.is_contiguous() else torch.empty(o.shape, dtype=o.dtype, device=o.device))
        if dst[-1] is not o:
            copies.append((o, dst[-1]))
    return src, src if in_place else dst, copies
