"""Fused softmax + sparse categorical cross-entropy.

``softmax_cross_entropy(logits, labels)`` returns the per-example loss vector
with no reduction, which is what the reference's ``loss`` helper returns
(reference centralized/client.py:11-13); ``reduction='sum'`` reproduces the
gradient the reference's ``tape.gradient`` of that vector computes
(client.py:16-19), ``'mean'`` is the usual default elsewhere.

``probs_clip_eps`` selects the reference's exact formulation, which applies the
loss to softmax *probabilities* clipped to ``[eps, 1 - eps]`` and renormalised
(what Keras does for ``from_logits=False``); it runs in plain torch since it is
a parity option for 10-class outputs, not a hot path.

``token_log_probs(logits, tokens, top=k)`` scores given tokens: their log
probabilities, the entropy of each row and its ``k`` best alternatives, in one
pass over the logits, with gradients (front end of ``csrc/kernels/token_logp.hip``).
"""
from __future__ import annotations

import ctypes
from typing import NamedTuple

import torch

from . import _lib


def _label_code(y: torch.Tensor) -> int:
    if y.dtype == torch.int32:
        return 0
    if y.dtype == torch.int64:
        return 1
    raise TypeError("labels must be int32 or int64")


def _row_padded(t: torch.Tensor) -> bool:
    """Rows that are read in place: contiguous, or padded to the next multiple of 16 bytes in a 16-byte aligned
    buffer (the layout ``ops.dense.linear`` gives logits whose width is not a multiple of 8). Any other view -- a
    column slice, rows of a much wider matrix -- is copied: backward allocates its gradient with the same row
    stride and needs the same alignment as the input."""
    if t.dim() != 2 or t.stride(1) != 1 or t.shape[0] <= 0:
        return False
    C, ld = t.shape[1], t.stride(0)
    if ld == C:
        return True
    per16 = 16 // t.element_size()
    return t.data_ptr() % 16 == 0 and ld == -(-C // per16) * per16


def _fwd(logits: torch.Tensor, labels: torch.Tensor, want_correct: bool):
    B, C = logits.shape
    if logits.is_cuda:
        # rows may be padded (stride(0) > C): the logits of a vocabulary whose size is not a multiple of 8 come in a
        # buffer with 16-byte aligned rows (ops.dense.linear), and are read in place
        x = logits if _row_padded(logits) else logits.contiguous()
        y = labels.contiguous()
        loss = torch.empty(B, dtype=torch.float32, device=x.device)
        lse = torch.empty(B, dtype=torch.float32, device=x.device)
        correct = torch.empty(B, dtype=torch.uint8, device=x.device) if want_correct else None
        rc = _lib.kernels().dtf_softmax_ce_fwd_ld(_lib.ptr(x), _lib.ptr(y), _lib.ptr(loss), _lib.ptr(lse),
                                                  _lib.ptr(correct), B, C, ctypes.c_longlong(x.stride(0)),
                                                  _lib.dtype_code(x.dtype), _label_code(y), _lib.stream_ptr(x.device))
        _lib.check(rc, "softmax_ce_fwd")
        return x, y, loss, lse, correct
    xf = logits.float()
    lse = torch.logsumexp(xf, dim=1)
    valid = (labels >= 0) & (labels < C)
    safe = labels.clamp(0, C - 1).long()
    loss = torch.where(valid, lse - xf.gather(1, safe[:, None])[:, 0], torch.zeros_like(lse))
    correct = (xf.argmax(1) == labels).to(torch.uint8) if want_correct else None
    return logits, labels, loss, lse, correct


class _SoftmaxCE(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, labels):
        x, y, loss, lse, _ = _fwd(logits, labels, False)
        ctx.save_for_backward(x, y, lse)
        return loss

    @staticmethod
    def backward(ctx, gout):
        x, y, lse = ctx.saved_tensors
        B, C = x.shape
        g = gout.contiguous().float()
        if x.is_cuda:
            ld = x.stride(0)
            # same row padding as the logits; the kernel zeroes the padding of the gradient
            dx = torch.empty((B, ld), dtype=x.dtype, device=x.device)[:, :C]
            rc = _lib.kernels().dtf_softmax_ce_bwd_ld(_lib.ptr(x), _lib.ptr(y), _lib.ptr(lse), _lib.ptr(g), _lib.ptr(dx),
                                                      B, C, ctypes.c_longlong(ld), _lib.dtype_code(x.dtype),
                                                      _label_code(y), _lib.stream_ptr(x.device))
            _lib.check(rc, "softmax_ce_bwd")
            return dx, None
        valid = ((y >= 0) & (y < C))
        p = torch.exp(x.float() - lse[:, None])
        p[torch.arange(B), y.clamp(0, C - 1).long()] -= 1.0
        dx = p * (g * valid)[:, None]
        return dx.to(x.dtype), None


def _clipped_probs_loss(logits, labels, eps):
    p = torch.softmax(logits.float(), dim=1).clamp(eps, 1.0 - eps)
    q = p / p.sum(dim=1, keepdim=True)
    return -torch.log(q.gather(1, labels.long()[:, None])[:, 0])


def softmax_cross_entropy(logits: torch.Tensor, labels: torch.Tensor, reduction: str = "none",
                          probs_clip_eps: float | None = None) -> torch.Tensor:
    """Loss of ``[B, C]`` logits against ``[B]`` integer labels (label < 0: ignored row)."""
    if logits.dim() != 2:
        logits = logits.reshape(-1, logits.shape[-1])
        labels = labels.reshape(-1)
    if probs_clip_eps is not None:
        loss = _clipped_probs_loss(logits, labels, probs_clip_eps)
    else:
        loss = _SoftmaxCE.apply(logits, labels)
    if reduction == "none":
        return loss
    if reduction == "sum":
        return loss.sum()
    if reduction == "mean":
        n = (labels >= 0).sum().clamp(min=1)
        return loss.sum() / n
    raise ValueError(f"unknown reduction {reduction!r}")


@torch.no_grad()
def softmax_ce_eval(logits: torch.Tensor, labels: torch.Tensor):
    """(per-example loss, correct flags) in one pass; used by evaluation loops
    (reference centralized/server.py:24-37 computes argmax accuracy separately)."""
    if logits.dim() != 2:
        logits = logits.reshape(-1, logits.shape[-1])
        labels = labels.reshape(-1)
    _, _, loss, _, correct = _fwd(logits, labels, True)
    return loss, correct


class TokenLogProbs(NamedTuple):
    logp: torch.Tensor       # log probability of the token
    entropy: torch.Tensor    # of the row's distribution, in nats
    top_logp: torch.Tensor   # [..., top], descending
    top_ids: torch.Tensor    # [..., top] int64


MAX_TOP = 32


def _token_logp(logits, tokens, top, keep):
    """(logits and tokens as the kernel reads them, statistics for the backward pass when ``keep``, the four results)."""
    x = logits if _row_padded(logits) else logits.contiguous()
    N, C = x.shape
    y, dev = tokens.contiguous(), x.device
    logp, entropy = (torch.empty(N, dtype=torch.float32, device=dev) for _ in range(2))
    stat = torch.empty(2, N, dtype=torch.float32, device=dev) if keep else None   # row maximum, log of the row's sum above it
    top_logp = torch.empty(N, top, dtype=torch.float32, device=dev)
    top_ids = torch.empty(N, top, dtype=torch.int64, device=dev)
    with _lib.on_device(x):
        rc = _lib.kernels().dtf_token_logp_fwd(_lib.ptr(x), _lib.ptr(y), _lib.ptr(logp), _lib.ptr(entropy), _lib.ptr(top_logp),
                                               _lib.ptr(top_ids), _lib.ptr(stat), N, C,
                                               ctypes.c_longlong(x.stride(0) if N > 1 else C), top, _lib.dtype_code(x.dtype),
                                               _label_code(y), _lib.stream_ptr(dev))
    _lib.check(rc, "token_logp_fwd")
    return x, y, stat, logp, entropy, top_logp, top_ids


class _TokenLogp(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, tokens, top):
        x, y, stat, logp, entropy, top_logp, top_ids = _token_logp(logits, tokens, top, True)
        ctx.save_for_backward(x, y, stat, entropy, top_ids)
        ctx.mark_non_differentiable(top_ids)
        ctx.set_materialize_grads(False)
        return logp, entropy, top_logp, top_ids

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g_logp, g_ent, g_top, _):
        x, y, stat, entropy, top_ids = ctx.saved_tensors
        if g_logp is None and g_ent is None and g_top is None:
            return None, None, None
        if not _row_padded(x):                     # (hooks on saved tensors may lay it out anew)
            x = x.contiguous()
        g_logp, g_ent, g_top = (None if g is None else g.float().contiguous() for g in (g_logp, g_ent, g_top))
        N, C = x.shape
        ld = x.stride(0) if N > 1 else C
        # the rows of dx as those of x, in stride and in alignment
        shift = x.data_ptr() % 16 // x.element_size()
        dx = torch.empty(N * ld + shift, dtype=x.dtype, device=x.device)[shift:].view(N, ld)[:, :C]
        k = 0 if g_top is None else top_ids.shape[1]
        with _lib.on_device(x):
            rc = _lib.kernels().dtf_token_logp_bwd(_lib.ptr(x), _lib.ptr(y), _lib.ptr(stat), _lib.ptr(entropy), _lib.ptr(top_ids),
                                                   _lib.ptr(g_logp), _lib.ptr(g_ent), _lib.ptr(g_top), _lib.ptr(dx), N, C,
                                                   ctypes.c_longlong(ld), k, _lib.dtype_code(x.dtype), _label_code(y),
                                                   _lib.stream_ptr(x.device))
        _lib.check(rc, "token_logp_bwd")
        return dx, None, None


def _token_logp_composed(logits, tokens, top):
    x = logits.float()
    ok = (tokens >= 0) & (tokens < x.shape[1])
    best = x.detach().amax(1, keepdim=True)
    none = best == -torch.inf                       # a row without a distribution: entropy 0, no gradient
    z = torch.where(none, x.detach(), x) - best.masked_fill(none, 0.0)
    total = z.exp().sum(1, keepdim=True)
    lp = z - total.masked_fill(none, 1.0).log()
    logp = torch.where(ok, lp.gather(1, tokens.clamp(0, x.shape[1] - 1).long()[:, None])[:, 0], 0.0)
    seen = lp != -torch.inf
    entropy = -(lp.exp() * torch.where(seen, lp, 0.0)).sum(1)
    top_ids = torch.sort(x.detach(), dim=1, descending=True, stable=True).indices[:, :top]
    return logp, entropy, lp.gather(1, top_ids), top_ids


def token_log_probs(logits: torch.Tensor, tokens: torch.Tensor, top: int = 0) -> TokenLogProbs:
    """Scores ``tokens[...]`` (int32 or int64) under ``logits[..., V]`` (float32 or bfloat16): ``logp``, ``entropy``,
    ``top_logp`` in float32 and ``top_ids``, all shaped like ``tokens`` (the last two with ``top`` more, at most 32).

    A token outside ``[0, V)`` (an ignored position) has ``logp`` 0 and no gradient through it. Alternatives of equal
    logits come lowest index first. Logits of -inf are words that cannot be; in a row of nothing else the log
    probabilities are -inf, the entropy 0 and the gradients 0. The three floating results have gradients; on a GPU
    forward-mode derivatives and traces are refused."""
    if logits.dim() < 1 or logits.shape[:-1] != tokens.shape:
        raise ValueError(f"logits [..., V] and tokens [...] do not fit: {tuple(logits.shape)}, {tuple(tokens.shape)}")
    if logits.device != tokens.device:
        raise ValueError(f"logits are on {logits.device}, tokens on {tokens.device}")
    _lib.dtype_code(logits.dtype)
    _label_code(tokens)
    V, shape = logits.shape[-1], tokens.shape
    if not 0 <= top <= min(MAX_TOP, V):
        raise ValueError(f"top {top}: need 0 to {MAX_TOP}, and no more than the {V} logits of a row")
    if V < 1 or V > 1 << 30 or tokens.numel() >= 1 << 22:
        raise ValueError(f"{tokens.numel()} rows of {V} logits: need at least 1 logit a row and fewer than {1 << 22} rows")
    flat = tokens.dim() == 1
    x, y = (logits, tokens) if flat else (logits.reshape(-1, V), tokens.reshape(-1))
    if not (x.is_cuda and y.numel()):
        r = _token_logp_composed(x, y, int(top))
    elif _lib.differentiated(x):
        r = _TokenLogp.apply(x, y, int(top))
    else:
        r = _token_logp(x, y, int(top), False)[3:]
    if flat:
        return TokenLogProbs(*r)
    return TokenLogProbs(r[0].view(shape), r[1].view(shape), r[2].view(*shape, top), r[3].view(*shape, top))
