"""Thin, shape-checked wrappers over the native kernels, with PyTorch references.

Every ``*_ref`` function is the plain-PyTorch definition of the same op in
fp32; tests compare the native kernels against them. The native wrappers
allocate their outputs (and scratch) from PyTorch's caching allocator so that
out-of-memory surfaces as ``torch.OutOfMemoryError``.
"""

from __future__ import annotations

import math
from typing import NamedTuple, Optional, Sequence

import torch
import torch.nn.functional as F

from ._ext import native, use_native

ACT_NONE, ACT_GELU, ACT_GELU_BWD = 0, 1, 2

# Alternatives of token_logprobs, or teacher slots of topk_distillation, per row.
MAX_TOP_K = 128
MAX_LIST_VOCAB = 1 << 19


# ----------------------------------------------------------------- GEMM


def gemm(
    a: torch.Tensor,
    b: torch.Tensor,
    *,
    a_mn_major: bool = False,
    b_mn_major: bool = False,
    out: Optional[torch.Tensor] = None,
    out_dtype: Optional[torch.dtype] = None,
    d: Optional[torch.Tensor] = None,
    alpha: float = 1.0,
    beta: float = 0.0,
    bias: Optional[torch.Tensor] = None,
    aux: Optional[torch.Tensor] = None,
    act: int = ACT_NONE,
    block_n: int = 0,
    symmetric: bool = False,
) -> torch.Tensor:
    """``out = epilogue(alpha * A @ B^T)`` on tcgen05 tensor cores.

    ``a`` is ``[.., M, K]`` (K-major) or, with ``a_mn_major``, ``[.., K, M]``.
    ``b`` is ``[.., N, K]`` or, with ``b_mn_major``, ``[.., K, N]``.
    Epilogue: ``+ bias[n]``; ``act=GELU`` stores the pre-activation to ``aux``
    and applies tanh-GELU; ``act=GELU_BWD`` multiplies by GELU'(d);
    otherwise ``+ beta * d``.

    ``symmetric=True`` declares the result symmetric (``X X^T``, or ``A A``
    plus ``beta * D`` with ``A`` and ``D`` symmetric; 16-bit output, no bias
    or activation): only the tiles on or above the diagonal are computed and
    the epilogue mirrors them, about half the work for large square outputs.
    Elements next to the diagonal may be written from both sides; both
    values are the same product up to rounding.
    """

    M = a.shape[-1] if a_mn_major else a.shape[-2]
    N = b.shape[-1] if b_mn_major else b.shape[-2]
    if out is None:
        shape = (*a.shape[:-2], M, N)
        out = torch.empty(shape, device=a.device, dtype=out_dtype or a.dtype)
    native().gemm(a, a_mn_major, b, b_mn_major, out, d, float(alpha), float(beta), bias, aux, int(act), int(block_n),
                  1 if symmetric else 0)
    return out


def gemm_ref(a, b, *, a_mn_major=False, b_mn_major=False, d=None, alpha=1.0, beta=0.0, bias=None, act=ACT_NONE):
    A = a.float().transpose(-1, -2) if a_mn_major else a.float()
    B = b.float().transpose(-1, -2) if b_mn_major else b.float()
    y = alpha * (A @ B.transpose(-1, -2))
    if bias is not None:
        y = y + bias.float()
    if act == ACT_GELU:
        return F.gelu(y, approximate="tanh"), y
    if act == ACT_GELU_BWD:
        h = d.float().detach().requires_grad_(True)
        with torch.enable_grad():
            g = torch.autograd.grad(F.gelu(h, approximate="tanh").sum(), h)[0]
        return y * g
    if d is not None and beta != 0.0:
        y = y + beta * d.float()
    return y


# ----------------------------------------------------------------- norms


def norm_forward(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor], eps: float, *, rms: bool,
                 out_dtype: torch.dtype):
    rows = x.numel() // x.shape[-1]
    y = torch.empty(x.shape, device=x.device, dtype=out_dtype)
    rstd = torch.empty(rows, device=x.device, dtype=torch.float32)
    mean = None if rms else torch.empty(rows, device=x.device, dtype=torch.float32)
    native().norm_forward(x, weight, bias, y, mean, rstd, float(eps), bool(rms))
    return y, mean, rstd


def norm_backward(dy, x, weight, mean, rstd, *, rms: bool, dres: Optional[torch.Tensor] = None,
                  dx_dtype: Optional[torch.dtype] = None, need_bias_grad: bool = True, want_lp: bool = False):
    """Returns (dx, dweight, dbias[, dx in dy's dtype when ``want_lp``])."""

    C = x.shape[-1]
    rows = x.numel() // C
    dx = torch.empty(x.shape, device=x.device, dtype=dx_dtype or (dres.dtype if dres is not None else x.dtype))
    dw = torch.empty(C, device=x.device, dtype=torch.float32)
    db = None if (rms or not need_bias_grad) else torch.empty(C, device=x.device, dtype=torch.float32)
    ws = torch.empty(native().norm_backward_workspace_elems(rows, C, x.device.index or 0), device=x.device,
                     dtype=torch.float32)
    lp = torch.empty(x.shape, device=x.device, dtype=dy.dtype) if want_lp else None
    native().norm_backward(dy, x, weight, mean, rstd, dres, dx, dw, db, ws, bool(rms), False, lp)
    if want_lp:
        return dx, dw, db, lp
    return dx, dw, db


def layer_norm_ref(x, w, b, eps):
    return F.layer_norm(x.float(), (x.shape[-1],), w.float(), None if b is None else b.float(), eps)


def rms_norm_ref(x, w, eps):
    xf = x.float()
    return xf * torch.rsqrt(xf.pow(2).mean(-1, keepdim=True) + eps) * w.float()


# ----------------------------------------------------------------- attention


def flash_attention_forward(q, k, v, *, causal: bool, scale: Optional[float] = None, out=None):
    """q, k, v: [B, S, H, D] views (token stride free). Returns (o, lse[B, H, S])."""

    B, S, H, D = q.shape
    scale = (1.0 / math.sqrt(D)) if scale is None else scale
    if out is None:
        out = torch.empty((B, S, H, D), device=q.device, dtype=q.dtype)
    lse = torch.empty((B, H, S), device=q.device, dtype=torch.float32)
    native().flash_attention_forward(q, k, v, out, lse, float(scale), bool(causal))
    return out, lse


def flash_attention_backward(q, k, v, o, do, lse, *, causal: bool, scale: Optional[float] = None, dq=None, dk=None,
                             dv=None):
    B, S, H, D = q.shape
    scale = (1.0 / math.sqrt(D)) if scale is None else scale
    dq = torch.empty_like(q, memory_format=torch.contiguous_format) if dq is None else dq
    dk = torch.empty_like(k, memory_format=torch.contiguous_format) if dk is None else dk
    dv = torch.empty_like(v, memory_format=torch.contiguous_format) if dv is None else dv
    ws = torch.empty(B * S * H * D + B * H * S, device=q.device, dtype=torch.float32)
    native().flash_attention_backward(q, k, v, o, do, lse, dq, dk, dv, ws, float(scale), bool(causal))
    return dq, dk, dv


def attention_ref(q, k, v, *, causal: bool, scale: Optional[float] = None):
    """[B, S, H, D] inputs, fp32 math."""

    qf, kf, vf = (t.float().transpose(1, 2) for t in (q, k, v))
    o = F.scaled_dot_product_attention(qf, kf, vf, is_causal=causal, scale=scale)
    return o.transpose(1, 2)


# ----------------------------------------------------------------- misc


def embedding_forward(idx, wte, wpe, seq_len):
    out = torch.empty((*idx.shape, wte.shape[1]), device=idx.device, dtype=torch.float32)
    native().embedding_forward(idx.contiguous(), wte, wpe, out, int(seq_len))
    return out


def embedding_backward(idx, dout, vocab, wpe_rows, seq_len, want_wpe=True):
    C = dout.shape[-1]
    dwte = torch.zeros((vocab, C), device=dout.device, dtype=torch.float32)
    dwpe = torch.zeros((wpe_rows, C), device=dout.device, dtype=torch.float32) if want_wpe else None
    native().embedding_backward(idx.contiguous(), dout.contiguous(), dwte, dwpe, int(seq_len))
    return dwte, dwpe


def cross_entropy_forward(logits, target, vocab, ignore_index=-100):
    rows = target.numel()
    loss = torch.empty(rows, device=logits.device, dtype=torch.float32)
    lse = torch.empty(rows, device=logits.device, dtype=torch.float32)
    native().cross_entropy_forward(logits, target.reshape(-1).contiguous(), loss, lse, int(vocab), int(ignore_index))
    return loss, lse


def cross_entropy_backward_(logits, target, lse, gscale, vocab, ignore_index=-100):
    native().cross_entropy_backward(logits, target.reshape(-1).contiguous(), lse, gscale, int(vocab), int(ignore_index))
    return logits


# ------------------------------------------- per-token losses over a vocabulary


class TokenLogprobs(NamedTuple):
    """What ``token_logprobs`` returns; every tensor has the logits' leading shape.

    ``logprobs`` (None without tokens) and ``entropy`` carry gradients;
    ``top_logprobs`` and ``top_ids`` (both ``[..., top_k]``, None for
    ``top_k=0``) do not.
    """

    logprobs: Optional[torch.Tensor]
    entropy: torch.Tensor
    top_logprobs: Optional[torch.Tensor]
    top_ids: Optional[torch.Tensor]


def _vocab_rows(logits: torch.Tensor, name: str) -> torch.Tensor:
    """``logits`` as [rows, vocab] with unit inner stride (a view where the strides allow it)."""

    if logits.dim() < 1 or logits.shape[-1] < 1:
        raise ValueError(f"{name}: logits must be [..., vocab] with at least one column")
    if logits.shape[-1] > MAX_LIST_VOCAB:
        raise ValueError(f"{name}: vocabularies of more than {MAX_LIST_VOCAB} entries are not supported")
    if logits.dtype not in (torch.bfloat16, torch.float16, torch.float32):
        raise TypeError(f"{name}: logits must be bf16, fp16 or fp32, got {logits.dtype}")
    rows = logits.numel() // logits.shape[-1]
    z = logits.reshape(rows, logits.shape[-1])
    return z if z.stride(1) == 1 or z.shape[1] == 1 else z.contiguous()


def _check_temperature(temperature: float, name: str) -> None:
    if not 1e-4 <= temperature <= 1e4:
        raise ValueError(f"{name}: temperature must lie in [1e-4, 1e4], got {temperature}")


def _like_rows(z: torch.Tensor) -> torch.Tensor:
    """An uninitialised [rows, vocab] tensor whose rows start where ``z``'s do modulo 16 bytes, if z's rows do not
    overlap."""

    rows, vocab = z.shape
    ld = z.stride(0) if rows > 1 and vocab <= z.stride(0) <= vocab + 1024 else vocab
    return torch.empty((rows, ld), device=z.device, dtype=z.dtype)[:, :vocab]


def token_logprobs_forward(logits, tokens, *, top_k: int = 0, temperature: float = 1.0, ignore_index: int = -100):
    """Returns (logprobs, entropy, stats, top_logprobs, top_ids) of 2-D ``logits`` (unit inner stride).

    ``stats`` is what ``token_logprobs_backward`` needs; ``logprobs`` is None
    without ``tokens``, the last two for ``top_k=0``.
    """

    rows, vocab = logits.shape
    dev = logits.device
    entropy = torch.empty(rows, device=dev, dtype=torch.float32)
    stats = torch.empty((rows, native().TOKEN_LOGPROBS_STATS), device=dev, dtype=torch.float32)
    logprobs = torch.empty(rows, device=dev, dtype=torch.float32) if tokens is not None else None
    top_logprobs = torch.empty((rows, top_k), device=dev, dtype=torch.float32) if top_k else None
    top_ids = torch.empty((rows, top_k), device=dev, dtype=torch.int64) if top_k else None
    native().token_logprobs_forward(logits, tokens, logprobs, entropy, stats, top_logprobs, top_ids, int(vocab),
                                    float(temperature), int(ignore_index))
    return logprobs, entropy, stats, top_logprobs, top_ids


def token_logprobs_backward(logits, tokens, stats, entropy, dlogprobs, dentropy, *, temperature: float = 1.0,
                            ignore_index: int = -100, out: Optional[torch.Tensor] = None):
    """Gradient of the logits from those of ``logprobs`` and ``entropy`` (fp32 rows, or None).

    ``out=logits`` overwrites the logits with their gradient. Rows whose
    gradients both are zero, and ignored rows, get zeros without being read.
    """

    out = _like_rows(logits) if out is None else out
    native().token_logprobs_backward(logits, tokens, stats, entropy, dlogprobs, dentropy, out, int(logits.shape[1]),
                                     float(temperature), int(ignore_index))
    return out


def token_logprobs(logits: torch.Tensor, tokens: Optional[torch.Tensor] = None, *, top_k: int = 0,
                   temperature: float = 1.0, ignore_index: int = -100) -> TokenLogprobs:
    """Log probabilities of given tokens, entropies and the most likely alternatives, in one pass over the logits.

    ``logits`` is ``[..., vocab]`` in bf16, fp16 or fp32 (any row stride),
    ``tokens`` ``[...]`` (int64; None when only entropy and alternatives are
    wanted). With ``p = softmax(logits / temperature)``: ``logprobs`` is
    ``log p[token]``, ``entropy`` ``-sum p log p`` in nats, ``top_ids`` the
    ``top_k`` (at most 128) largest logits in descending order, equal logits
    by their index, and ``top_logprobs`` their log probabilities. All are fp32
    but the ids. The results of a row with ``tokens == ignore_index`` are
    zeros and ids of -1; a token outside the vocabulary has a NaN log
    probability, and a NaN gradient where the upstream one is not zero. Logits
    of -inf are never produced (they add nothing to the entropy); a row of -inf
    only, or with a NaN or +inf, gives NaN. NaN logits rank above all others.
    On CUDA, logits with a forward-mode tangent are refused.
    """

    if use_native(logits):
        return TokenLogprobs(*native().token_logprobs(logits, tokens, top_k, temperature, ignore_index))
    name = "token_logprobs"
    z = _vocab_rows(logits, name)
    lead, vocab = logits.shape[:-1], logits.shape[-1]
    _check_temperature(temperature, name)
    if not 0 <= top_k <= min(MAX_TOP_K, vocab):
        raise ValueError(f"{name}: top_k must lie in [0, {min(MAX_TOP_K, vocab)}], got {top_k}")
    if tokens is not None:
        if tokens.shape != lead or tokens.dtype != torch.int64 or tokens.device != logits.device:
            raise ValueError(f"{name}: tokens must be int64 of shape {tuple(lead)} on {logits.device}")
        tokens = tokens.reshape(-1)
    logprobs, entropy, top_logprobs, top_ids = token_logprobs_ref(z, tokens, top_k=top_k, temperature=temperature,
                                                                  ignore_index=ignore_index)
    return TokenLogprobs(None if logprobs is None else logprobs.view(lead), entropy.view(lead),
                         None if top_logprobs is None else top_logprobs.view(*lead, top_k),
                         None if top_ids is None else top_ids.view(*lead, top_k))


def token_logprobs_ref(logits, tokens, *, top_k: int = 0, temperature: float = 1.0, ignore_index: int = -100):
    """2-D logits, 1-D tokens; (logprobs, entropy, top_logprobs, top_ids) in fp32 (fp64 for fp64 logits)."""

    zf = logits if logits.dtype == torch.float64 else logits.float()
    counted = torch.ones(len(zf), dtype=torch.bool, device=zf.device) if tokens is None else tokens != ignore_index
    if not counted.all():  # rows left out have gradient zero, whatever they hold
        zf = torch.where(counted[:, None], zf, 0.0)
    logp = torch.log_softmax(zf / temperature, dim=-1)
    masked = torch.isneginf(zf) & torch.isfinite(logp.detach().amax(-1, keepdim=True))
    entropy = -torch.where(masked, 0.0, logp.exp() * logp.masked_fill(masked, 0.0)).sum(-1)
    logprobs = top_logprobs = top_ids = None
    if tokens is not None:
        inside = (tokens >= 0) & (tokens < logits.shape[1])
        got = logp.gather(1, torch.where(inside, tokens, 0)[:, None])[:, 0]
        if got.requires_grad:  # the gradient of a NaN is one, if any of it is asked for
            got.register_hook(lambda g: g if g is None else torch.where(inside | (g == 0), g, math.nan))
        logprobs = torch.where(counted, got + torch.where(inside, 0.0, math.nan), 0.0)
    if top_k:
        ids = zf.detach().sort(dim=-1, descending=True, stable=True).indices[:, :top_k]
        top_logprobs = torch.where(counted[:, None], logp.detach().gather(1, ids), 0.0)
        top_ids = torch.where(counted[:, None], ids, -1)
    return logprobs, torch.where(counted, entropy, 0.0), top_logprobs, top_ids


def topk_distillation_forward(logits, teacher_ids, teacher_logits, *, weight=None, temperature: float = 1.0,
                              tail: bool = False):
    """Returns (loss rows, stats for the backward pass) of 2-D ``logits`` and ``[rows, k]`` teachers.

    ``weight`` (fp32 rows) multiplies the losses; rows of weight zero are not read.
    """

    rows, vocab = logits.shape
    loss = torch.empty(rows, device=logits.device, dtype=torch.float32)
    stats = torch.empty((rows, native().TOPK_DISTILLATION_STATS), device=logits.device, dtype=torch.float32)
    native().topk_distillation_forward(logits, teacher_ids, teacher_logits, weight, loss, stats, None, int(vocab),
                                       float(temperature), bool(tail))
    return loss, stats


def topk_distillation_grad(logits, teacher_ids, teacher_logits, *, weight=None, temperature: float = 1.0,
                           tail: bool = False, out: Optional[torch.Tensor] = None):
    """Forward and backward in one kernel: (weighted loss rows, stats, gradient of their sum).

    The logits are read from memory once; ``out=logits`` overwrites them with
    their gradient.
    """

    rows, vocab = logits.shape
    loss = torch.empty(rows, device=logits.device, dtype=torch.float32)
    stats = torch.empty((rows, native().TOPK_DISTILLATION_STATS), device=logits.device, dtype=torch.float32)
    out = _like_rows(logits) if out is None else out
    native().topk_distillation_forward(logits, teacher_ids, teacher_logits, weight, loss, stats, out, int(vocab),
                                       float(temperature), bool(tail))
    return loss, stats, out


def topk_distillation_backward(logits, teacher_ids, teacher_logits, stats, *, row_scale=None, scale=None,
                               temperature: float = 1.0, tail: bool = False, out: Optional[torch.Tensor] = None):
    """Gradient of ``sum(row_scale * loss) * scale`` (fp32 rows and scalar on the device; None is one).

    ``out=logits`` overwrites the logits with their gradient. Rows of scale
    zero, and rows without slots, get zeros without being read.
    """

    out = _like_rows(logits) if out is None else out
    native().topk_distillation_backward(logits, teacher_ids, teacher_logits, stats, row_scale, scale, out,
                                        int(logits.shape[1]), float(temperature), bool(tail), False)
    return out


def topk_distillation(logits: torch.Tensor, teacher_ids: torch.Tensor, teacher_logits: torch.Tensor, *,
                      temperature: float = 1.0, tail: bool = False, weight: Optional[torch.Tensor] = None,
                      reduction: str = "none") -> torch.Tensor:
    """KL divergence of a student's distribution from a teacher known by its top logits.

    ``logits`` is ``[..., vocab]`` (bf16, fp16 or fp32, any row stride), the
    teacher's ``teacher_ids`` (int64) and ``teacher_logits`` (floating) are
    ``[..., k]`` with 1 to 128 slots. Ids outside the vocabulary are empty
    slots, so rows may hold fewer; ids of a row should differ (equal ones
    count as separate slots). With ``p = softmax(logits / temperature)``:

    * ``tail=False``: ``q = softmax(teacher_logits / temperature)`` over the
      row's slots; the loss is ``sum q (log q - log p[id])``.
    * ``tail=True``: ``teacher_logits`` are log probabilities at this
      temperature (``token_logprobs(...).top_logprobs``), ``q`` their
      exponentials, and the teacher's remaining mass ``1 - sum q`` is compared
      with the student's mass outside the listed tokens as one more slot.
      Where the student has none, the loss is infinite and that slot adds
      nothing to the gradient, but a rest below 2^-18, which rounding alone
      leaves of a teacher that lists everything, counts as none there.

    Rows without slots have loss and gradient zero. ``reduction="none"``
    returns fp32 losses ``[...]``; ``"sum"`` returns their sum weighted by
    ``weight`` (``[...]``, ones when None), where rows of weight zero are left
    out altogether. The gradient reaches the logits only; it is not scaled by
    the temperature's square. On CUDA, logits with a forward-mode tangent are
    refused.
    """

    name = "topk_distillation"
    if reduction not in ("none", "sum"):
        raise ValueError(f"{name}: reduction must be 'none' or 'sum', got {reduction!r}")
    if use_native(logits):
        return native().topk_distillation(logits, teacher_ids, teacher_logits, temperature, tail, weight,
                                          reduction == "sum")
    lead = logits.shape[:-1]
    z = _vocab_rows(logits, name)
    _check_temperature(temperature, name)
    if teacher_ids.dim() != logits.dim() or teacher_ids.shape[:-1] != lead or teacher_ids.dtype != torch.int64:
        raise ValueError(f"{name}: teacher_ids must be int64 of shape {(*lead, 'k')}")
    if teacher_logits.shape != teacher_ids.shape or not teacher_logits.is_floating_point():
        raise ValueError(f"{name}: teacher_logits must be floating, of teacher_ids' shape")
    if not 1 <= teacher_ids.shape[-1] <= MAX_TOP_K:
        raise ValueError(f"{name}: 1 to {MAX_TOP_K} teacher slots per row, got {teacher_ids.shape[-1]}")
    if weight is not None and (reduction != "sum" or weight.shape != lead):
        raise ValueError(f"{name}: weight goes with reduction='sum' and has shape {tuple(lead)}")
    for other in (teacher_ids, teacher_logits, weight):
        if other is not None and other.device != logits.device:
            raise ValueError(f"{name}: all tensors must be on {logits.device}")
    k = teacher_ids.shape[-1]
    ids = teacher_ids.reshape(-1, k)
    if weight is not None:
        weight = weight.detach().float().reshape(-1)
        ids = torch.where((weight != 0)[:, None], ids, -1)
    loss = topk_distillation_ref(z, ids, teacher_logits.detach().reshape(-1, k).float(), temperature=temperature,
                                 tail=tail)
    if reduction == "none":
        return loss.view(lead)
    return loss.sum() if weight is None else torch.where(weight == 0, 0.0, loss * weight).sum()


def topk_distillation_ref(logits, teacher_ids, teacher_logits, *, temperature: float = 1.0, tail: bool = False):
    """2-D logits and ``[rows, k]`` teachers; loss rows in fp32 (fp64 for fp64 logits)."""

    zf = logits if logits.dtype == torch.float64 else logits.float()
    valid = (teacher_ids >= 0) & (teacher_ids < logits.shape[1])
    some = valid.any(-1)
    if not some.all():  # rows without slots have gradient zero, whatever they hold
        zf = torch.where(some[:, None], zf, 0.0)
    x = zf / temperature
    logp = torch.log_softmax(x, dim=-1)
    at = torch.where(valid, teacher_ids, 0)
    t = torch.where(valid, teacher_logits.to(zf.dtype), -math.inf)
    if tail:
        q, logq = t.exp(), t
    else:
        t = t / temperature
        high = t.amax(-1, keepdim=True)
        e = (t - torch.where(high == -math.inf, 0.0, high)).exp()
        total = e.sum(-1, keepdim=True)
        q = torch.where(total == 0, 0.0, e / total)
        logq = q.log()
    loss = torch.where(q == 0, 0.0, q * (logq - logp.gather(1, at)).masked_fill(q == 0, 0.0)).sum(-1)
    if tail:
        listed = torch.zeros_like(logp.detach()).scatter_add_(1, at, valid.to(logp.dtype)) > 0
        rest = (1.0 - q.sum(-1)).clamp_min(0.0)
        # From the largest logit off the list, whose distance from the row's may have no digits below one.
        top = x.detach().amax(-1, keepdim=True)
        high = x.detach().masked_fill(listed, -math.inf).amax(-1, keepdim=True)
        none = high == -math.inf  # no student mass off the list: an infinite constant
        off = (x - torch.where(none, 0.0, high)).masked_fill(listed, -math.inf).masked_fill(none, 0.0)
        log_rest = torch.logsumexp(off, -1) + (high - top)[:, 0] - torch.logsumexp(x - top, -1)
        log_rest = torch.where(none[:, 0], -math.inf, log_rest)
        # What rounding leaves of a teacher that lists everything, where the student has no mass for it.
        rest = torch.where((rest <= 2.0**-18) & (log_rest.detach() < -126 * math.log(2.0)), 0.0, rest)
        loss = loss + torch.where(rest == 0, 0.0, rest * (rest.log() - log_rest).masked_fill(rest == 0, 0.0))
    return torch.where(some, loss, 0.0)


def bias_grad(g: torch.Tensor) -> torch.Tensor:
    """Column sums of ``g`` in fp32 (the bias gradient), deterministic (two passes, no atomics)."""

    out = torch.empty(g.shape[-1], device=g.device, dtype=torch.float32)
    native().bias_grad(g, out, False)
    return out


def cast_multi(src: Sequence[torch.Tensor], dst: Sequence[torch.Tensor]) -> None:
    native().cast_multi(list(src), list(dst))


def swiglu_forward(gu):
    F_ = gu.shape[-1] // 2
    h = torch.empty((*gu.shape[:-1], F_), device=gu.device, dtype=gu.dtype)
    native().swiglu_forward(gu, h)
    return h


def swiglu_backward(gu, dh):
    dgu = torch.empty_like(gu)
    native().swiglu_backward(gu, dh, dgu)
    return dgu


def swiglu_ref(gu):
    g, u = gu.float().chunk(2, dim=-1)
    return F.silu(g) * u


def patchify(images, patch: int, dtype: torch.dtype):
    """fp32 NCHW images -> [B * patches, C * patch * patch] rows in ``dtype`` (Conv2d weight column order)."""

    B, C, H, W = images.shape
    out = torch.empty((B * (H // patch) * (W // patch), C * patch * patch), device=images.device, dtype=dtype)
    native().patchify(images.contiguous(), out, int(patch))
    return out


def patchify_ref(images, patch: int):
    B, C, H, W = images.shape
    x = images.reshape(B, C, H // patch, patch, W // patch, patch)
    return x.permute(0, 2, 4, 1, 3, 5).reshape(B * (H // patch) * (W // patch), C * patch * patch)


def rope_apply_(x, cos, sin, inverse=False):
    B, S, H, D = x.shape
    native().rope_apply(x, cos, sin, S, H, D, bool(inverse))
    return x


def rope_ref(x, cos, sin):
    """x: [B, S, H, D]; cos/sin: [S, D/2]. Rotate-half convention."""

    xf = x.float()
    half = xf.shape[-1] // 2
    x1, x2 = xf[..., :half], xf[..., half:]
    c = cos[None, :, None, :]
    s = sin[None, :, None, :]
    return torch.cat([x1 * c - x2 * s, x2 * c + x1 * s], dim=-1)
