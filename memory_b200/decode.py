"""Decode-time memory layer: cached projected bank rows and the rolling routing state.

The reference's generation loop (inference/generate.py:189-274) calls the model once per token; every memory
layer then routes on a pooled state, re-gathers (S+k)*T bank rows per sequence and re-projects them with Wk / Wv
(model.py:624-692, memory_attention.py:241-243).  While decoding, bank and projections are constant, so

``ProjectedBankCache``  holds ``norm(M) [Wk; Wv]^T`` in bf16 ([C*T, 2*HK*D], 805 MB for the 262,208-row bank), or in 8 bits
                        with a scale for each block of rows, KV head, and K or V (403 MB, half the bytes of a step);
``RoutingWindow``       is the ``rolling`` / ``hybrid`` routing state of model.py:630-660 (last
                        ``routing_window_size`` layer-input states; prefill pools the whole prompt);
``MemoryDecoder``       runs one step: router on the window -> shared prefix -> query projection -> attention
                        over gathered cache rows scaled by the chapter weight -> output projection.

Results equal ``memory_layer`` on the same inputs up to bf16 rounding of the cached rows.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch
from torch.autograd import forward_ad

from . import _lib as L
from . import ops


class ProjectedBankCache:
    """K/V projections of every bank row, built once per weight state."""

    def __init__(self, bank: torch.Tensor, wk: torch.Tensor, wv: torch.Tensor, tokens_per_chapter: int,
                 num_shared_chapters: int = 1, norm_type: Optional[str] = None, norm_eps: float = 1e-5,
                 chapters_per_pass: int = 512, cache_dtype: torch.dtype = torch.bfloat16, scale_rows: Optional[int] = None,
                 head_dim: int = 64):
        """``cache_dtype`` torch.float8_e4m3fn: 8 bits, with a scale for every ``scale_rows`` rows (a chapter's by default)."""
        t = int(tokens_per_chapter)
        rows, d = bank.shape
        if rows % t != 0:
            raise ValueError("bank rows must be a multiple of tokens_per_chapter")
        self.tokens_per_chapter = t
        self.num_chapters = rows // t
        self.kv_dim = wk.shape[0]
        self._allocate(rows, 2 * self.kv_dim, head_dim, cache_dtype, scale_rows, bank.device)
        # the reference normalises rows only when a shared and a routed slice both exist (model.py:413-418)
        norm = norm_type if 0 < num_shared_chapters < self.num_chapters else None
        cd = torch.bfloat16
        wkv = ops.cast(torch.cat([wk, wv], dim=0).contiguous(), cd)
        with torch.no_grad():
            for c0 in range(0, self.num_chapters, chapters_per_pass):
                c1 = min(self.num_chapters, c0 + chapters_per_pass)
                idx = torch.arange(c0, c1, dtype=torch.int32, device=bank.device).view(1, -1)
                rows_c, _ = ops.gather_rows_fwd(bank, t, idx, None, norm, norm_eps, cd)     # [1, n*T, d], normalised
                if self.kv_scale is None:
                    ops.gemm(rows_c.view(-1, d), wkv, out=self.kv_bank[c0 * t:c1 * t], tag="kv_cache")
                else:
                    self._write(c0 * t, ops.gemm(rows_c.view(-1, d), wkv, out_dtype=cd, tag="kv_cache"))

    def _allocate(self, rows: int, width: int, head_dim: int, cache_dtype: torch.dtype, scale_rows: Optional[int], device) -> None:
        if cache_dtype not in (torch.bfloat16, torch.float8_e4m3fn):
            raise TypeError(f"the cache is held in bfloat16 or float8_e4m3fn, not {cache_dtype}")
        t = self.tokens_per_chapter
        self.head_dim = int(head_dim)
        self.kv_bank = torch.empty(rows, width, dtype=cache_dtype, device=device)
        self.kv_scale: Optional[torch.Tensor] = None
        self.scale_rows = 0
        if cache_dtype == torch.bfloat16:
            if scale_rows is not None:
                raise ValueError("a bf16 cache has no scales")
            return
        self.scale_rows = t if scale_rows is None else int(scale_rows)
        if self.scale_rows <= 0 or t % self.scale_rows != 0:
            raise ValueError(f"a chapter of {t} rows must be whole blocks of scale_rows ({self.scale_rows})")
        if self.head_dim != 64 or width % 128 != 0:
            raise ValueError("the 8-bit cache needs head_dim 64")
        self.kv_scale = torch.empty(rows // self.scale_rows, width // self.head_dim, dtype=torch.float32, device=device)

    def _write(self, first: int, rows: torch.Tensor) -> None:
        n, b = rows.shape[0], self.scale_rows
        ops.quantize_rows(rows, b, self.head_dim, self.kv_bank[first:first + n], self.kv_scale[first // b:(first + n) // b])

    @classmethod
    def _bare(cls, kv_bank: torch.Tensor, tokens_per_chapter: int) -> "ProjectedBankCache":
        t = int(tokens_per_chapter)
        if kv_bank.dim() != 2 or t <= 0 or kv_bank.shape[0] % t != 0 or kv_bank.shape[1] % 2 != 0 or kv_bank.shape[0] == 0:
            raise ValueError(f"the cache must be [rows, 2 * num_kv_heads * head_dim] with whole chapters of {t} rows, "
                             f"got {tuple(kv_bank.shape)}")
        self = cls.__new__(cls)
        self.tokens_per_chapter, self.num_chapters, self.kv_dim = t, kv_bank.shape[0] // t, kv_bank.shape[1] // 2
        return self

    @classmethod
    def from_rows(cls, kv_rows: torch.Tensor, tokens_per_chapter: int, head_dim: int = 64,
                  cache_dtype: torch.dtype = torch.bfloat16, scale_rows: Optional[int] = None) -> "ProjectedBankCache":
        """A cache of rows that are projected already ([C*T, 2*HK*D] bf16, K heads then V heads); a bf16 cache keeps the tensor itself."""
        L.require_cuda(kv_rows)
        if kv_rows.dtype != torch.bfloat16:
            raise TypeError("projected rows must be bf16")
        self = cls._bare(kv_rows, tokens_per_chapter)
        if cache_dtype == torch.bfloat16:
            if scale_rows is not None:
                raise ValueError("a bf16 cache has no scales")
            self.kv_bank, self.kv_scale, self.scale_rows, self.head_dim = ops._contig(kv_rows), None, 0, int(head_dim)
            return self
        self._allocate(*kv_rows.shape, head_dim, cache_dtype, scale_rows, kv_rows.device)
        self._write(0, kv_rows.detach())
        return self

    @classmethod
    def from_quantized(cls, values: torch.Tensor, scales: torch.Tensor, tokens_per_chapter: int,
                       scale_rows: Optional[int] = None) -> "ProjectedBankCache":
        """A cache around e4m3 ``values`` [C*T, 2*HK*64] and fp32 ``scales`` [C*T / scale_rows, 2*HK] as another cache holds them (a
        loaded file, say); the tensors themselves are kept."""
        L.require_cuda(values, scales)
        self = cls._bare(values, tokens_per_chapter)
        self.head_dim, self.scale_rows = 64, self.tokens_per_chapter if scale_rows is None else int(scale_rows)
        self.kv_bank, self.kv_scale = ops._contig(values), ops._contig(scales)
        if values.shape[1] % 128 != 0:
            raise ValueError("the 8-bit cache needs head_dim 64")
        ops.check_cache(self.kv_bank, self.kv_scale, self.scale_rows, self.tokens_per_chapter, values.shape[1] // 128)
        return self

    def attend(self, q: torch.Tensor, chapter_indices: torch.Tensor, chapter_weights: torch.Tensor, num_heads: int,
               num_kv_heads: Optional[int] = None, counts: Optional[torch.Tensor] = None, scale: Optional[float] = None,
               return_lse: bool = False):
        """Attention of projected queries [B, n_q, H*64] bf16 over each sequence's listed chapters, one joint softmax over their rows
        scaled by the chapters' weights ([B, n] ids and weights: a router's joint list).  ``counts`` [B] int32: how many entries of
        each list count (what lies behind them is not read; none: zeros, lse -inf).  Returns [B, n_q, H*64] bf16, with
        ``return_lse`` also the natural log of the softmax's denominator [B, n_q, H] fp32.  A chapter id outside the cache raises the
        device status and is left out.  For generation: it has no gradients; a query or a cache that requires
        one is refused, and the chapters' weights are taken as numbers (a router's, whatever graph they hang on).

        Scores, softmax and sums are fp32 over either cache.  Over an 8-bit one, queries go into the products as
        fp16 numbers (exact but for elements below 2^-24 of their head's largest, which are off by 2^-32 of it at most) and probabilities as two
        (off by 2^-21 of their own, not below 2^-32 of the largest among 32 neighbouring rows, times those rows' scales)."""
        heads, kv_heads = int(num_heads), int(num_heads if num_kv_heads is None else num_kv_heads)
        L.require_cuda(q, chapter_indices, chapter_weights, counts)
        if any(map(_carries_gradient, (q, self.kv_bank, self.kv_scale))):
            raise RuntimeError("attention over the cache has no gradients: call it under torch.no_grad(), or on detached tensors")
        if q.dtype != torch.bfloat16 or q.dim() != 3:
            raise TypeError("attend takes bf16 queries [B, n_q, H * head_dim]")
        b, n_q, hd = q.shape
        if heads <= 0 or kv_heads <= 0 or heads % kv_heads != 0 or hd != heads * 64:
            raise ValueError(f"queries of width {hd} are not {heads} heads of 64 on {kv_heads} KV heads")
        if self.kv_bank.shape[1] != 2 * kv_heads * 64:
            raise ValueError(f"the cache holds {self.kv_bank.shape[1] // 128} KV heads, not {kv_heads}")
        if chapter_indices.dim() != 2 or chapter_indices.shape != chapter_weights.shape or chapter_indices.shape[0] != b:
            raise ValueError("chapter_indices and chapter_weights must both be [B, n]")
        if counts is not None and tuple(counts.shape) != (b,):
            raise ValueError("counts must be [B]")
        device = self.kv_bank.device
        if q.device != device or chapter_indices.device != device or chapter_weights.device != device or (
                counts is not None and counts.device != device):
            raise ValueError("all tensors must be on the device of the cache")
        if b == 0 or n_q == 0 or chapter_indices.shape[1] == 0:
            out, lse = torch.zeros_like(q), q.new_full((b, n_q, heads), float("-inf"), dtype=torch.float32)
            return (out, lse) if return_lse else out
        idx = _whole(chapter_indices)
        out, lse = ops.decode_attn_cache(ops._contig(q), self.kv_bank, self.kv_scale, self.scale_rows, idx,
                                         _as(chapter_weights, torch.float32), None if counts is None else _whole(counts),
                                         heads, kv_heads, self.tokens_per_chapter, 0.125 if scale is None else float(scale), return_lse)
        return (out, lse) if return_lse else out


def _carries_gradient(t: Optional[torch.Tensor]) -> bool:
    if t is None:
        return False
    return (t.requires_grad and torch.is_grad_enabled()) or (
        forward_ad._current_level >= 0 and forward_ad.unpack_dual(t).tangent is not None)


def _whole(t: torch.Tensor) -> torch.Tensor:
    """Ids or counts as int32; what does not fit stays out of range instead of wrapping into it."""
    return _as(t if t.dtype == torch.int32 else t.clamp(-(2 ** 31), 2 ** 31 - 1) if t.dtype == torch.int64 else t, torch.int32)


def _as(t: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    return ops._contig(t if t.dtype == dtype else t.to(dtype))


class RoutingWindow:
    """Routing state of one memory layer during cached generation (model.py:630-660).

    ``prefill(h)`` returns the states the router pools for the prompt and keeps the last ``window`` of them;
    ``step(h)`` appends the new states and returns the window to pool.  ``hybrid`` pools the whole prompt at
    prefill; ``rolling`` pools the window from the start.
    """

    def __init__(self, window_size: int = 128, strategy: str = "hybrid"):
        if strategy not in ("rolling", "hybrid"):
            raise ValueError("strategy must be 'rolling' or 'hybrid'")
        self.window_size = int(window_size)
        self.strategy = strategy
        self.cache: Optional[torch.Tensor] = None

    def reset(self) -> None:
        self.cache = None

    def prefill(self, hidden_states: torch.Tensor) -> torch.Tensor:
        if self.strategy == "rolling":
            return self.step(hidden_states)
        self.cache = hidden_states[:, -self.window_size:].detach()
        return hidden_states

    def step(self, hidden_states: torch.Tensor) -> torch.Tensor:
        if self.cache is not None and hidden_states.dim() == 3 and not (torch.is_grad_enabled() and hidden_states.requires_grad):
            rows = min(self.window_size, self.cache.shape[1] + hidden_states.shape[1])
            window = ops.roll_window(self.cache, hidden_states, rows)
            if window is not None:
                self.cache = window
                return window
        combined = hidden_states if self.cache is None else torch.cat([self.cache, hidden_states], dim=1)
        if combined.shape[1] > self.window_size:
            combined = combined[:, -self.window_size:]
        self.cache = combined.detach()
        return combined


class MemoryDecoder:
    """One memory layer in generation mode over a :class:`ProjectedBankCache`."""

    def __init__(self, cache: ProjectedBankCache, router_weight: torch.Tensor, router_bias: Optional[torch.Tensor],
                 wq: torch.Tensor, wo: torch.Tensor, *, num_heads: int, num_kv_heads: Optional[int] = None,
                 top_k: int, num_shared_chapters: int = 1, routed_scaling_factor: float = 2.5, router=None):
        """``router``: a ``ChapterRouter``; its weights, ``top_k`` and rules (scores, balance bias, groups) stand for ``router_weight``,
        ``router_bias`` and ``top_k`` then, which are not read.  One of the reference's rules is part of the native step."""
        self.cache = cache
        self.router = router
        self.router_weight, self.router_bias = router_weight, router_bias
        self.num_heads = int(num_heads)
        self.num_kv_heads = int(num_kv_heads or num_heads)
        self.top_k, self.num_shared = int(top_k), int(num_shared_chapters)
        self.routed_scale = float(routed_scaling_factor)
        cd = torch.bfloat16
        self.wq_c, self.wo_c = ops.cast(wq.contiguous(), cd), ops.cast(wo.contiguous(), cd)
        self.scale = (wq.shape[0] // self.num_heads) ** -0.5
        self._plans: dict = {}

    def step(self, hidden_states: torch.Tensor, routing_states: torch.Tensor) -> Tuple[torch.Tensor, dict]:
        """``hidden_states`` [B, n_q, d]: the tokens being decoded (input of the cross attention);
        ``routing_states`` [B, W, d]: the states the router mean-pools (a :class:`RoutingWindow` result).
        Returns (output [B, n_q, d] in the dtype of ``hidden_states``, routing info)."""
        weight, bias, top_k = self.router_weight, self.router_bias, self.top_k
        if self.router is not None:
            if self.router.by_logits:
                return self._step_by_router(hidden_states, routing_states)
            linear = self.router.router
            weight, bias, top_k = linear.weight.detach(), None if linear.bias is None else linear.bias.detach(), self.router.top_k
        out, idx, w, cidx, cw = ops.decode_step(
            hidden_states, routing_states, weight, bias, self.wq_c, self.wo_c, self.cache.kv_bank,
            num_heads=self.num_heads, num_kv_heads=self.num_kv_heads, tokens_per_chapter=self.cache.tokens_per_chapter,
            top_k=top_k, num_shared=self.num_shared, routed_scale=self.routed_scale, scale=self.scale,
            plans=self._plans, kv_scale=getattr(self.cache, "kv_scale", None), scale_rows=getattr(self.cache, "scale_rows", 0))
        return out, {"indices": idx, "weights": w, "combined_indices": cidx, "combined_weights": cw}

    @torch.no_grad()
    def _step_by_router(self, hidden_states: torch.Tensor, routing_states: torch.Tensor) -> Tuple[torch.Tensor, dict]:
        if hidden_states.dim() != 3 or hidden_states.shape[0] != routing_states.shape[0]:
            raise ValueError("hidden_states and routing_states must share the batch")
        idx, w, cidx, cw, _ = self.router.route_with_shared(routing_states, self.num_shared, self.routed_scale)
        b, n_q, d = hidden_states.shape
        x = hidden_states.reshape(b * n_q, d)
        q = ops.gemm(x if x.dtype == torch.bfloat16 else ops.cast(x, torch.bfloat16), self.wq_c, tag="q")
        o = self.cache.attend(q.view(b, n_q, -1), cidx, cw, self.num_heads, self.num_kv_heads, scale=self.scale)
        out = ops.gemm(o.view(b * n_q, -1), self.wo_c, out_dtype=hidden_states.dtype, tag="o").view(b, n_q, -1)
        return out, {"indices": idx, "weights": w, "combined_indices": cidx, "combined_weights": cw}
