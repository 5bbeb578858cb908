"""Pieces shared by the benchmark models.

* ``compute_dtype()`` reads the active autocast dtype: under bf16/fp16
  autocast on CUDA the models run on the native sm_100a kernels with fp32
  master parameters (the same numerics contract as autocast: fp32 params,
  low-precision GEMM operands, fp32 accumulation); otherwise they run the
  plain-PyTorch reference path.
* ``LowPrecisionShadows`` keeps a bf16/fp16 copy of every GEMM weight. A copy
  is refreshed only when its parameter changed through PyTorch (tracked by the
  tensor version counter); the fused optimizer writes the copies itself in the
  same pass that updates the parameters.
"""

from __future__ import annotations

import threading
from typing import Any, Dict, Iterable, List, Optional

import torch
import torch.nn as nn

from ..ops import functional as kf
from ..parallel.ddp import check_entry


def compute_dtype(device: torch.device) -> Optional[torch.dtype]:
    """Low-precision compute dtype for native kernels, or None for the reference path."""

    if device.type != "cuda":
        return None
    if not torch.is_autocast_enabled("cuda"):
        return None
    dt = torch.get_autocast_dtype("cuda")
    return dt if dt in (torch.bfloat16, torch.float16) else None


def shadow_of(param: torch.Tensor, dtype: torch.dtype) -> Optional[torch.Tensor]:
    sh = getattr(param, "_kb_shadow", None)
    if sh is None or sh.dtype != dtype or sh.device != param.device or sh.shape != param.shape:
        return None
    return sh


class LowPrecisionShadows:
    """bf16/fp16 copies of a fixed list of fp32 matrix parameters.

    ``fused_groups`` lists groups of matrices with equal column counts whose
    copies should be row blocks of one buffer (for example q, k and v): the
    forward pass then runs one GEMM on the stacked weight while every matrix
    stays its own parameter (Muon orthogonalises each separately).
    """

    def __init__(self, params: Iterable[nn.Parameter], fused_groups: Iterable[Iterable[nn.Parameter]] = ()) -> None:
        self.params: List[nn.Parameter] = list(params)
        self.fused_groups: List[List[nn.Parameter]] = [list(g) for g in fused_groups]
        known = {id(p) for p in self.params}
        for g in self.fused_groups:
            if any(id(p) not in known for p in g) or len({p.shape[1] for p in g}) != 1:
                raise ValueError("fused shadow groups must be listed parameters with equal column counts")
        self._fused: Dict[tuple, torch.Tensor] = {}

    def _ensure_fused(self, dtype: torch.dtype) -> None:
        for gi, g in enumerate(self.fused_groups):
            buf = self._fused.get((gi, dtype))
            if buf is not None and buf.device == g[0].device and all(
                    getattr(getattr(p, "_kb_shadow", None), "_base", None) is buf for p in g):
                continue
            rows = sum(p.shape[0] for p in g)
            buf = torch.empty((rows, g[0].shape[1]), device=g[0].device, dtype=dtype)
            r = 0
            for p in g:
                p._kb_shadow = buf[r:r + p.shape[0]]  # type: ignore[attr-defined]
                p._kb_shadow_version = -1  # type: ignore[attr-defined]
                r += p.shape[0]
            self._fused[(gi, dtype)] = buf

    def fused(self, index: int, dtype: torch.dtype) -> torch.Tensor:
        """The stacked copy of fused group ``index`` (valid after ``get(dtype)``)."""

        return self._fused[(index, dtype)]

    def refresh(self) -> None:
        """Bring every 16-bit copy handed out so far up to date with its parameter."""

        for dtype in list(getattr(self, "_dtypes_seen", ())):
            self.get(dtype)

    def get(self, dtype: torch.dtype) -> Dict[int, torch.Tensor]:
        seen = self.__dict__.setdefault("_dtypes_seen", set())
        seen.add(dtype)
        if self.fused_groups:
            self._ensure_fused(dtype)
        stale_src: List[torch.Tensor] = []
        stale_dst: List[torch.Tensor] = []
        out: Dict[int, torch.Tensor] = {}
        for p in self.params:
            sh = shadow_of(p, dtype)
            if sh is None:
                sh = torch.empty(p.shape, device=p.device, dtype=dtype)
                p._kb_shadow = sh  # type: ignore[attr-defined]
                p._kb_shadow_version = -1  # type: ignore[attr-defined]
            if getattr(p, "_kb_shadow_version", -1) != p._version:
                stale_src.append(p.detach())
                stale_dst.append(sh)
                p._kb_shadow_version = p._version  # type: ignore[attr-defined]
            out[id(p)] = sh
        if stale_src:
            kf.cast_multi(stale_src, stale_dst)
        return out


def mark_shadow_fresh(param: torch.Tensor) -> None:
    """Called by kernels that rewrote ``param`` and its shadow together."""

    if getattr(param, "_kb_shadow", None) is not None:
        param._kb_shadow_version = param._version  # type: ignore[attr-defined]


def to_lp(t: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    """fp32 -> bf16/fp16 cast on the native kernel (contiguous input)."""

    t = t.contiguous()
    out = torch.empty(t.shape, device=t.device, dtype=dtype)
    kf.cast_multi([t], [out])
    return out


def accumulation_target(*params: torch.Tensor) -> Optional[torch.Tensor]:
    """The existing fp32 gradient buffer of ``params`` that a backward may add into directly, or None.

    Under gradient accumulation the second and later micro-steps would
    otherwise produce a fresh weight gradient that autograd then adds into
    ``.grad`` (one more read and write of every gradient). A backward may
    instead accumulate into ``.grad`` itself (a GEMM with the old gradient as
    its D operand) and return None for that weight, when nothing could
    observe the difference: gradients are not being recorded, every
    parameter already has a contiguous fp32 gradient of its own shape, no
    hook is registered on the parameters (a hook expects to see the
    accumulation), and -- for several parameters -- their gradients lie back
    to back in one buffer (the layout autograd keeps when it adopted the
    split views of one fused gradient on the first micro-step). Returns a
    [sum of rows, cols] view over those gradients.
    """

    if torch.is_grad_enabled() or not params:
        return None
    grads = []
    for p in params:
        g = p.grad
        if (g is None or g.dtype != torch.float32 or not g.is_contiguous() or g.shape != p.shape
                or p._backward_hooks or getattr(p, "_post_accumulate_grad_hooks", None)):
            return None
        grads.append(g)
    first = grads[0]
    cols = first.numel() // first.shape[0]
    rows = 0
    for g in grads:
        if (g.numel() // g.shape[0] != cols or g.untyped_storage().data_ptr() != first.untyped_storage().data_ptr()
                or g.data_ptr() != first.data_ptr() + rows * cols * 4):
            return None
        rows += g.shape[0]
    return first.as_strided((rows, cols), (cols, 1))


class HeadLogits(torch.autograd.Function):
    """Final norm and LM head: ``[B, S, vocab]`` logits in the compute dtype (rows padded to 64 columns)."""

    @staticmethod
    def forward(ctx, x, norm_w, norm_b, head_w, head_w16, eps, rms):
        B, S, C = x.shape
        M, V = B * S, head_w.shape[0]
        cdt = head_w16.dtype
        x2 = x.reshape(M, C)
        h, mean, rstd = kf.norm_forward(x2, norm_w, norm_b, eps, rms=rms, out_dtype=cdt)
        vpad = (V + 63) // 64 * 64
        # A tensor of its own, not a view of a padded one: callers may mask it in place.
        logits = torch.empty_strided((B, S, V), (S * vpad, vpad, 1), device=x.device, dtype=cdt)
        kf.gemm(h, head_w16, out=logits.view(M, V))
        ctx.save_for_backward(x2, h, mean, rstd, norm_w, head_w16)
        ctx.meta = (B, S, C, V, rms)
        return logits

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dlogits):
        x2, h, mean, rstd, norm_w, head_w16 = ctx.saved_tensors
        B, S, C, V, rms = ctx.meta
        dlog = dlogits.to(h.dtype).reshape(B * S, V)
        # The GEMM's operands: rows of their own (a gradient may be one row, expanded) at 16-byte boundaries.
        if dlog.stride(1) != 1 or dlog.stride(0) < V or dlog.stride(0) % 8 or dlog.data_ptr() % 16:
            padded = torch.empty((B * S, (V + 63) // 64 * 64), device=h.device, dtype=h.dtype)[:, :V]
            dlog = padded.copy_(dlog)
        dh = kf.gemm(dlog, head_w16, b_mn_major=True)
        dw = kf.gemm(dlog, h, a_mn_major=True, b_mn_major=True, out_dtype=torch.float32)
        dx, dnorm_w, dnorm_b, dx_lp = kf.norm_backward(dh, x2, norm_w, mean, rstd, rms=rms, dx_dtype=torch.float32,
                                                       want_lp=True)
        dx = dx.view(B, S, C)
        dx._kb_lp = dx_lp  # the 16-bit copy the last layer's backward starts from
        return dx, dnorm_w, dnorm_b, dw, None, None, None


class TokenLosses:
    """Per-token losses of a language model over its vocabulary; mixed into models that have ``logits(idx)``.

    ``model(idx, method="distillation_loss", ...)`` is ``model.distillation_loss(idx, ...)`` by way of ``forward``, which
    data-parallel wrappers need: theirs starts the reduction of the gradients. ``DataParallel`` has the methods too.
    """

    _entered = threading.local()  # .model: the one whose forward hands a call on

    def _by_method(self, method: str, idx: torch.Tensor, targets, ignore_index: int, options: Dict[str, Any]):
        if method not in ("logits", "token_logprobs", "distillation_loss"):
            raise ValueError(f"method must be 'logits', 'token_logprobs' or 'distillation_loss', got {method!r}")
        if targets is not None:
            raise ValueError(f"targets do not go with method={method!r}")
        if method == "token_logprobs":
            options = {"ignore_index": ignore_index, **options}
        before = getattr(self._entered, "model", None)
        self._entered.model = self
        try:
            return getattr(self, method)(idx, **options)
        finally:
            self._entered.model = before

    def _check_entry(self, name: str) -> None:
        if getattr(self._entered, "model", None) is not self:
            check_entry(self, name)

    def token_logprobs(self, idx: torch.Tensor, tokens: Optional[torch.Tensor] = None, *, top_k: int = 0,
                       temperature: float = 1.0, ignore_index: int = -100) -> kf.TokenLogprobs:
        """``ops.functional.token_logprobs`` of the model's logits: scoring of given tokens, entropies, alternatives.

        ``token_logprobs(idx, top_k=k)`` of a teacher gives the ``top_ids`` and ``top_logprobs`` that a student's
        ``distillation_loss(..., tail=True)`` takes.
        """

        self._check_entry("token_logprobs")
        return kf.token_logprobs(self.logits(idx), tokens, top_k=top_k, temperature=temperature,
                                 ignore_index=ignore_index)

    def distillation_loss(self, idx: torch.Tensor, teacher_ids: torch.Tensor, teacher_logits: torch.Tensor, *,
                          weight: Optional[torch.Tensor] = None, temperature: float = 1.0,
                          tail: bool = False) -> torch.Tensor:
        """Mean of ``ops.functional.topk_distillation`` over the positions that have teacher slots, or the mean
        weighted by ``weight`` (``[B, S]``)."""

        self._check_entry("distillation_loss")
        logits = self.logits(idx)
        if weight is None:
            weight = ((teacher_ids >= 0) & (teacher_ids < logits.shape[-1])).any(-1)
        weight = weight.float()
        weight = weight / weight.sum().clamp_min(torch.finfo(torch.float32).tiny)
        return kf.topk_distillation(logits, teacher_ids, teacher_logits, temperature=temperature, tail=tail,
                                    weight=weight, reduction="sum")
