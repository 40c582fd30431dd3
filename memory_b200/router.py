"""``ChapterRouter`` with the reference's constructor, attributes and return contract
(memory_transformer/router.py:15-340), computed by the CUDA router kernels."""
from __future__ import annotations

from typing import Dict, Optional, Tuple

import torch
import torch.nn as nn

from . import functional as F_moc


class ChapterRouter(nn.Module):
    """Top-k chapter selection with load-balance / auxiliary / z losses.

    Same surface as the reference module: ``.router`` is an ``nn.Linear(hidden_dim, num_chapters)``
    (weight N(0, 0.02), zero bias), ``.top_k`` and ``.routing_strategy`` may be changed by the
    caller between calls, ``forward`` returns ``(indices int64, weights, losses)``.
    Selection order is (weight descending, chapter id ascending).

    Beyond the reference: ``score="sigmoid"``, ``balance_bias=True`` (a buffer that :meth:`update_balance` moves towards equal
    load; it counts in the selection alone), ``num_groups`` / ``top_groups`` / ``group_score`` (group-limited selection over the chapters
    behind the excluded prefix) and ``renormalize=False`` select by :func:`memory_b200.select_chapters`.  Such a router returns no loss terms (an empty
    dict): the bias takes the place of the balance loss.  ``last_load`` holds the latest call's count of rows per chapter
    (rows that give it a weight).
    """

    def __init__(self, hidden_dim: int, num_chapters: int, top_k: int = 1, routing_strategy: str = "sequence", *,
                 score: str = "softmax", balance_bias: bool = False, num_groups: int = 1, top_groups: Optional[int] = None,
                 group_score: str = "max", renormalize: bool = True):
        super().__init__()
        if num_chapters <= 0:
            raise ValueError(f"num_chapters must be > 0, got {num_chapters}")
        if top_k <= 0:
            raise ValueError(f"top_k must be > 0, got {top_k}")
        if top_k > num_chapters:
            raise ValueError(f"top_k ({top_k}) must be <= num_chapters ({num_chapters})")
        self.hidden_dim = hidden_dim
        self.num_chapters = num_chapters
        self.top_k = top_k
        self.routing_strategy = routing_strategy
        self.router = nn.Linear(hidden_dim, num_chapters, bias=True)
        nn.init.normal_(self.router.weight, mean=0.0, std=0.02)
        nn.init.zeros_(self.router.bias)
        if score not in ("softmax", "sigmoid"):
            raise ValueError(f"score must be 'softmax' or 'sigmoid', got {score!r}")
        if group_score not in ("max", "top2"):
            raise ValueError(f"group_score must be 'max' or 'top2', got {group_score!r}")
        if num_groups < 1 or not 1 <= (num_groups if top_groups is None else top_groups) <= num_groups:
            raise ValueError(f"top_groups must be in 1..num_groups, got {top_groups} of {num_groups}")
        self.selection = {"score": score, "num_groups": num_groups, "top_groups": top_groups, "group_score": group_score,
                          "renormalize": renormalize}
        self.by_logits = (score, renormalize) != ("softmax", True) or balance_bias or top_groups not in (None, num_groups)
        self.last_load: Optional[torch.Tensor] = None
        self._last_shared = 0
        self.register_buffer("balance_bias", torch.zeros(num_chapters) if balance_bias else None)

    def __setstate__(self, state):
        """Modules that were saved whole before there were other rules than the reference's follow those."""
        super().__setstate__(state)
        rules = {"score": "softmax", "num_groups": 1, "top_groups": None, "group_score": "max", "renormalize": True}
        for name, value in (("selection", rules), ("by_logits", False), ("last_load", None), ("_last_shared", 0)):
            self.__dict__.setdefault(name, value)
        self._buffers.setdefault("balance_bias", None)

    def _apply(self, fn, recurse=True):
        """Casts and moves of the module; the balance bias moves along and stays fp32 (steps of 0.001 vanish beside 0.3 in bf16)."""
        bias = self._buffers.get("balance_bias")
        super()._apply(fn, recurse)
        cast = self._buffers.get("balance_bias")
        if bias is not None and cast.dtype != bias.dtype:
            self._buffers["balance_bias"] = bias.to(cast.device)
        return self

    def select(self, logits: torch.Tensor, num_shared: int, routed_scale: float = 1.0) -> F_moc.ChapterSelection:
        """This router's selection from logits [rows, num_chapters].  Rows and chapters may be masked; places of weight 0 do not count in
        the load, so padding does not move the balance bias."""
        got = F_moc.select_chapters(logits, self.top_k, balance_bias=self.balance_bias, num_shared=num_shared,
                                    routed_scale=routed_scale, count_filled=False, **self.selection)
        self.last_load, self._last_shared = got.load, num_shared
        return got

    def update_balance(self, rate: float = 1e-3, load: Optional[torch.Tensor] = None,
                       num_shared: Optional[int] = None) -> None:
        """Moves the balance bias of every chapter behind the shared ones by ``rate`` towards the mean load: up where fewer rows
        chose it, down where more did (and up at every step where a mask keeps all rows away).  ``load`` [C] int32: the counts of a step (summed over ranks, say); they and ``num_shared`` are
        the latest call's by default."""
        if self.balance_bias is None:
            raise ValueError("this router has no balance bias")
        load = self.last_load if load is None else load
        if load is None:
            raise ValueError("no load yet: route first, or pass the counts")
        F_moc.ops.balance_bias_step(self.balance_bias, load, self._last_shared if num_shared is None else num_shared, rate)

    def forward(self, hidden_states: torch.Tensor, return_losses: bool = True, exclude_prefix_chapters: int = 0,
                rolling_window_size: Optional[int] = None
                ) -> Tuple[torch.Tensor, torch.Tensor, Dict[str, torch.Tensor]]:
        pos_weight = None
        if self.routing_strategy in ("sequence-rolling", "sequence_rolling"):
            # router.py:100-105, 159-195: the mean over t of the rolling-window means is one coefficient per position
            if hidden_states.dim() != 3:
                raise ValueError(f"hidden_states must be 3D (B, T, D), got shape {tuple(hidden_states.shape)}")
            pos_weight = self._rolling_coefficients(hidden_states.shape[1], rolling_window_size, hidden_states.device)
        elif self.routing_strategy == "token":
            # router.py:106-110 projects every token and averages the logits; the projection is linear, so this is
            # the router applied to the mean state (equal up to rounding)
            pass
        elif self.routing_strategy != "sequence":
            raise ValueError(f"Unknown routing_strategy: {self.routing_strategy}")
        if exclude_prefix_chapters < 0 or exclude_prefix_chapters > self.num_chapters:
            raise ValueError(
                f"exclude_prefix_chapters must be in [0, {self.num_chapters}], got {exclude_prefix_chapters}")
        if self.by_logits:
            got = self.select(self._pooled_logits(hidden_states, pos_weight), exclude_prefix_chapters)
            return got.indices, got.weights, {}
        idx, w, _, _, losses = F_moc.route(hidden_states, self.router.weight, self.router.bias, self.top_k,
                                           exclude_prefix_chapters, 1.0, return_losses, pos_weight=pos_weight)
        return idx, w, losses

    def _pooled_logits(self, hidden_states: torch.Tensor, pos_weight: Optional[torch.Tensor]) -> torch.Tensor:
        if hidden_states.dim() != 3:
            raise ValueError(f"hidden_states must be 3D (B, T, D), got shape {tuple(hidden_states.shape)}")
        if pos_weight is None:          # the mean is the window that spans the sequence: one coefficient, 1 / L
            pos_weight = torch.full((hidden_states.shape[1],), 1.0 / max(1, hidden_states.shape[1]), device=hidden_states.device)
        return F_moc.router_logits(hidden_states, self.router.weight, self.router.bias, pos_weight)

    def _rolling_coefficients(self, seq: int, window: Optional[int], device) -> torch.Tensor:
        key = (int(seq), None if window is None else int(window), str(device))
        cache = self.__dict__.setdefault("_rolling_cache", {})
        if key not in cache:
            if len(cache) > 16:
                cache.clear()
            cache[key] = F_moc.ops.rolling_pool_coefficients(seq, window).to(device)
        return cache[key]

    def route_token_level(self, hidden_states: torch.Tensor, return_losses: bool = True,
                          exclude_prefix_chapters: int = 0
                          ) -> Tuple[torch.Tensor, torch.Tensor, Dict[str, torch.Tensor]]:
        """Every token selects its own chapters (router.py:262-340).  Returns (global chapter ids int64
        [B, L, k'], weights [B, L, k'] renormalised over the selection, losses over all B*L routing rows);
        k' = min(top_k, num_chapters - exclude_prefix_chapters), empty tensors when k' <= 0."""
        if hidden_states.dim() != 3:
            raise ValueError(f"hidden_states must be 3D (B, T, D), got shape {tuple(hidden_states.shape)}")
        if exclude_prefix_chapters < 0 or exclude_prefix_chapters > self.num_chapters:
            raise ValueError(
                f"exclude_prefix_chapters must be in [0, {self.num_chapters}], got {exclude_prefix_chapters}")
        if self.by_logits:
            b, l, _ = hidden_states.shape
            got = self.select(F_moc.router_logits(hidden_states, self.router.weight, self.router.bias), exclude_prefix_chapters)
            return got.indices.view(b, l, -1), got.weights.view(b, l, -1), {}
        return F_moc.route_tokens(hidden_states, self.router.weight, self.router.bias, self.top_k,
                                  exclude_prefix_chapters, return_losses)

    def route_with_shared(self, hidden_states: torch.Tensor, num_shared_chapters: int,
                          routed_scaling_factor: float, return_losses: bool = True):
        """Router plus the model-side shared-prefix step (model.py:356-391) in one launch sequence.
        Returns (indices, weights, combined_indices int32, combined_weights, losses)."""
        if self.by_logits:
            got = self.select(self._pooled_logits(hidden_states, None), num_shared_chapters, routed_scaling_factor)
            return got.indices, got.weights, got.combined_indices, got.combined_weights, {}
        return F_moc.route(hidden_states, self.router.weight, self.router.bias, self.top_k,
                           num_shared_chapters, routed_scaling_factor, return_losses)


def compute_total_router_loss(losses: Dict[str, torch.Tensor], load_balance_coef: float = 0.01,
                              auxiliary_coef: float = 0.0, z_loss_coef: float = 0.0,
                              reference_tensor: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Weighted sum of the router losses (router.py:490-527); empty dicts give a zero scalar."""
    if not losses:
        return reference_tensor.new_tensor(0.0) if reference_tensor is not None else torch.tensor(0.0)
    if getattr(losses, "vector", None) is not None:
        return F_moc.weighted_losses(losses, load_balance=load_balance_coef, auxiliary=auxiliary_coef, z_loss=z_loss_coef)
    total = next(iter(losses.values())).new_tensor(0.0)
    for key, coef in (("load_balance", load_balance_coef), ("auxiliary", auxiliary_coef), ("z_loss", z_loss_coef)):
        if key in losses and coef > 0:
            total = total + coef * losses[key]
    return total
