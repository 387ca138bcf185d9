"""Multi-head attention.

:func:`attention` takes separate queries, keys and values of any lengths (causal, padded, grouped heads, relative position
bias; bf16 and fp32) and runs the fused kernels of ``csrc/kernels/attention.h``, forward and backward.

:func:`self_attention` without options is the encoder's path on the batched MFMA GEMM plus the fused softmax kernels, and
with options the general one on the same buffer. Its input is the fused QKV projection ``qkv[B, S, 3, nh, hd]`` (one GEMM output); the three products
``S = Q K^T``, ``O = P V`` and their four gradient products address Q, K and V *inside* that
buffer through leading dimensions and two-level batch strides (batch, head), so no head
split / transpose copies are made. The scale ``1/sqrt(hd)`` and the optional additive
key-padding bias are fused into the softmax kernel.

Two paths: head dimension 64 with ``S % 128 == 0`` (the BERT-base configuration) runs the fused
flash-style kernels of ``csrc/kernels/flash_attn.hip`` (scores never leave registers; backward
recomputes the probabilities from the stored log-sum-exp). Other shapes materialise the scores
(``[B, nh, S, S]`` bf16) and run the batched GEMM + fused softmax kernels. ``set_flash(False)`` or
``DTF_FLASH=0`` forces the second path.
"""
from __future__ import annotations

import ctypes
import math
import os

import torch

from . import _lib
from . import gemm as G
from . import relative_bias as _rel


_flash = os.environ.get("DTF_FLASH", "1") == "1"


def set_flash(on: bool) -> None:
    global _flash
    _flash = bool(on)


def _flash_ok(qkv: torch.Tensor) -> bool:
    B, S, three, nh, hd = qkv.shape
    return _flash and hd == 64 and S % 128 == 0 and S >= 128


class _FlashFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, qkv, bias):
        B, S, _, nh, hd = qkv.shape
        out = torch.empty(B, S, nh, hd, dtype=qkv.dtype, device=qkv.device)
        lse = torch.empty(B, nh, S, dtype=torch.float32, device=qkv.device)
        rc = _lib.kernels().dtf_flash_attn_fwd(_lib.ptr(qkv), _lib.ptr(bias), _lib.ptr(out), _lib.ptr(lse), B, S, nh, hd,
                                               ctypes.c_float(1.0 / math.sqrt(hd)), _lib.stream_ptr(qkv.device))
        _lib.check(rc, "flash_attn_fwd")
        ctx.save_for_backward(qkv, bias if bias is not None else lse, out, lse)
        ctx.has_bias = bias is not None
        return out

    @staticmethod
    def backward(ctx, dout):
        qkv, bias, out, lse = ctx.saved_tensors
        B, S, _, nh, hd = qkv.shape
        dout = dout.contiguous()
        dqkv = torch.empty_like(qkv)
        delta = torch.empty(B, nh, S, dtype=torch.float32, device=qkv.device)
        # the kernels also sum the columns of the dqkv they store (per wave, finished by one small kernel): the bias
        # gradient of the fused QKV projection, offered to that layer's backward under dqkv's address
        from . import layernorm as _ln
        parts = sums = None
        if _ln.hand_over_enabled():
            parts = torch.empty((B * (S // 32), 3 * nh * hd), dtype=torch.float32, device=qkv.device)
            sums = torch.empty(3 * nh * hd, dtype=torch.float32, device=qkv.device)
        rc = _lib.kernels().dtf_flash_attn_bwd_cs(_lib.ptr(qkv), _lib.ptr(bias if ctx.has_bias else None), _lib.ptr(out),
                                                  _lib.ptr(lse), _lib.ptr(dout), _lib.ptr(delta), _lib.ptr(dqkv), B, S,
                                                  nh, hd, ctypes.c_float(1.0 / math.sqrt(hd)), _lib.ptr(parts),
                                                  _lib.ptr(sums), _lib.stream_ptr(qkv.device))
        _lib.check(rc, "flash_attn_bwd")
        if sums is not None:
            _ln.offer_col_sum(dqkv, sums)
        return dqkv, None


def _fast(qkv: torch.Tensor) -> bool:
    B, S, three, nh, hd = qkv.shape
    return (qkv.is_cuda and qkv.dtype == torch.bfloat16 and qkv.is_contiguous() and hd % 8 == 0 and S % 8 == 0
            and S <= 4096 and three == 3)


def _softmax_fwd(scores, bias, rows_per_batch, scale):
    L = scores.shape[-1]
    rows = scores.numel() // L
    rc = _lib.kernels().dtf_softmax_fwd(_lib.ptr(scores), _lib.ptr(scores), _lib.ptr(bias), ctypes.c_longlong(rows), L,
                                        ctypes.c_longlong(rows_per_batch), ctypes.c_float(scale),
                                        _lib.stream_ptr(scores.device))
    _lib.check(rc, "softmax_fwd")
    return scores


def _softmax_bwd(p, dp, scale):
    L = p.shape[-1]
    rows = p.numel() // L
    rc = _lib.kernels().dtf_softmax_bwd(_lib.ptr(p), _lib.ptr(dp), _lib.ptr(dp), ctypes.c_longlong(rows), L,
                                        ctypes.c_float(scale), _lib.stream_ptr(p.device))
    _lib.check(rc, "softmax_bwd")
    return dp


class _AttnFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, qkv, bias):
        B, S, _, nh, hd = qkv.shape
        dev = qkv.device
        ld = 3 * nh * hd                      # row stride of a token inside qkv
        q, k, v = qkv[:, :, 0], qkv[:, :, 1], qkv[:, :, 2]   # views; only their data_ptr is used
        scores = torch.empty(B, nh, S, S, dtype=qkv.dtype, device=dev)
        sb = (S * ld, hd)                     # (batch, head) strides inside qkv
        sc = (nh * S * S, S * S)
        G.gemm_raw(G.NT, q, k, scores, S, S, hd, ld, ld, S, extra=G.batch_dims(B, nh, sb, sb, sc))
        p = _softmax_fwd(scores, bias, nh * S, 1.0 / math.sqrt(hd))
        out = torch.empty(B, S, nh, hd, dtype=qkv.dtype, device=dev)
        so = (S * nh * hd, hd)
        G.gemm_raw(G.NN, p, v, out, S, hd, S, S, ld, nh * hd, extra=G.batch_dims(B, nh, sc, sb, so))
        ctx.save_for_backward(qkv, p)
        return out

    @staticmethod
    def backward(ctx, dout):
        qkv, p = ctx.saved_tensors
        B, S, _, nh, hd = qkv.shape
        dev = qkv.device
        ld = 3 * nh * hd
        dout = dout.contiguous()
        q, k, v = qkv[:, :, 0], qkv[:, :, 1], qkv[:, :, 2]
        dqkv = torch.empty_like(qkv)
        dq, dk, dv = dqkv[:, :, 0], dqkv[:, :, 1], dqkv[:, :, 2]
        sb = (S * ld, hd)
        sc = (nh * S * S, S * S)
        so = (S * nh * hd, hd)
        lo = nh * hd
        # dV = P^T dO
        G.gemm_raw(G.TN, p, dout, dv, S, hd, S, S, lo, ld, extra=G.batch_dims(B, nh, sc, so, sb))
        # dP = dO V^T
        dp = torch.empty_like(p)
        G.gemm_raw(G.NT, dout, v, dp, S, S, hd, lo, ld, S, extra=G.batch_dims(B, nh, so, sb, sc))
        ds = _softmax_bwd(p, dp, 1.0 / math.sqrt(hd))
        # dQ = dS K ; dK = dS^T Q
        G.gemm_raw(G.NN, ds, k, dq, S, hd, S, S, ld, ld, extra=G.batch_dims(B, nh, sc, sb, sb))
        G.gemm_raw(G.TN, ds, q, dk, S, hd, S, S, ld, ld, extra=G.batch_dims(B, nh, sc, sb, sb))
        return dqkv, None

# ---------------------------------------------------------------------------------------- general attention
# csrc/kernels/attention.h: any lengths, causal, grouped key / value heads, padded batches, strided operands, relative
# position bias; bf16 and fp32. The words below are the enum of csrc/kernels/attention.hip.
def _strides(t: torch.Tensor) -> tuple[int, int, int]:
    """(batch, token, head) strides; those of axes of one element, which torch leaves arbitrary, as in a dense tensor."""
    (B, S, n, hd), (sb, ss, sh, _) = t.shape, t.stride()
    return (sb if B > 1 else 0), (ss if S > 1 else n * hd), (sh if n > 1 else 0)


def _usable(t: torch.Tensor) -> torch.Tensor:
    """``t``, or a dense copy of it when the kernels cannot address it in place: they read 16 bytes at a time along the
    head, rows must not overlap, and a tile's offsets are 32-bit."""
    per16 = 16 // t.element_size()
    sb, ss, sh = _strides(t)
    if (t.stride(3) == 1 or t.shape[3] == 1) and t.data_ptr() % 16 == 0 and not (sb % per16 or ss % per16 or sh % per16) \
            and t.shape[3] <= ss <= 1 << 22:
        return t
    return t.contiguous() if not t.is_contiguous() else t.clone(memory_format=torch.contiguous_format)


def _words(ptrs, B, Sq, Sk, nh, nkv, hd, opts, key_bias, lens, starts, table, stat, delta=0, parts=0, dtable=0):
    """``ptrs``: (pointer, strides) of q, k, v, out, dout, dq, dk, dv; ``None`` for those a pass has not."""
    causal, _, start0, max_distance, bidirectional = opts
    w = [0 if t is None else t[0] for t in ptrs]
    for t in ptrs:
        w += (0, 0, 0) if t is None else t[1]
    borders = ()
    if table is not None:
        borders = _rel.bucket_borders(table.shape[0], max_distance, bidirectional)
    w += (0 if key_bias is None else key_bias.data_ptr(), 0 if lens is None else lens.data_ptr(),
          0 if starts is None else starts.data_ptr(), start0, 0 if table is None else table.data_ptr(),
          int(table is not None and table.dtype == torch.bfloat16), 0 if table is None else table.shape[0], max_distance,
          int(bidirectional), stat.data_ptr(), delta, parts, dtable, B, Sq, Sk, nh, nkv, hd, int(causal))
    return w, borders


def _call(name, w, borders, bf16, scale, like):
    w = [*w, int(bf16), *borders]
    with _lib.on_device(like):
        rc = getattr(_lib.kernels(), name)((ctypes.c_longlong * len(w))(*w), len(w), ctypes.c_float(scale),
                                           _lib.stream_ptr(like.device))
    _lib.check(rc, name)


def _view(t: torch.Tensor, first: int, heads: int):
    """(pointer, strides) of ``heads`` heads of ``t`` from ``first`` on."""
    st = _strides(t)
    return t.data_ptr() + first * t.stride(2) * t.element_size(), st


class _GeneralFn(torch.autograd.Function):
    """``k is None``: ``q`` is the fused ``[B, S, nh + 2 nkv, hd]`` buffer, and so is its gradient."""

    @staticmethod
    def forward(ctx, q, k, v, table, key_bias, lens, starts, nkv, opts):
        packed = k is None
        q = _usable(q)
        if packed:
            B, Sq, n, hd = q.shape
            Sk, nh = Sq, n - 2 * nkv
            qkv = (_view(q, 0, nh), _view(q, nh, nkv), _view(q, nh + nkv, nkv))
        else:
            k, v = _usable(k), _usable(v)
            B, Sq, nh, hd = q.shape
            Sk = k.shape[1]
            qkv = tuple((t.data_ptr(), _strides(t)) for t in (q, k, v))
        out = torch.empty(B, Sq, nh, hd, dtype=q.dtype, device=q.device)
        stat = torch.empty(2, B, nh, Sq, dtype=torch.float32, device=q.device)
        ctx.meta = (B, Sq, Sk, nh, nkv, hd, packed, opts)
        ctx.table_like = None if table is None else (table.shape, table.dtype)
        table = None if table is None else table.contiguous()
        ctx.save_for_backward(q, k, v, table, key_bias, lens, starts, out, stat)
        if Sk == 0:
            return out.zero_()
        if out.numel():
            w, borders = _words((*qkv, (out.data_ptr(), _strides(out)), None, None, None, None), B, Sq, Sk, nh, nkv, hd,
                                opts, key_bias, lens, starts, table, stat)
            _call("dtf_attention_fwd", w, borders, q.dtype == torch.bfloat16, opts[1], q)
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout):
        q, k, v, table, key_bias, lens, starts, out, stat = ctx.saved_tensors
        B, Sq, Sk, nh, nkv, hd, packed, opts = ctx.meta
        dev = q.device
        if packed:
            dq, dk, dv = torch.empty(B, Sq, nh + 2 * nkv, hd, dtype=q.dtype, device=dev), None, None
            qkv = (_view(q, 0, nh), _view(q, nh, nkv), _view(q, nh + nkv, nkv))
            grads = (_view(dq, 0, nh), _view(dq, nh, nkv), _view(dq, nh + nkv, nkv))
        else:
            dq, dk, dv = (torch.empty(t.shape, dtype=t.dtype, device=dev) for t in (q, k, v))
            qkv = tuple((t.data_ptr(), _strides(t)) for t in (q, k, v))
            grads = tuple((t.data_ptr(), _strides(t)) for t in (dq, dk, dv))
        dtable = parts = None
        if table is not None and ctx.needs_input_grad[3]:
            shape, dt = ctx.table_like
            dtable = torch.empty(shape, dtype=dt, device=dev)
        if out.numel() == 0 or Sk == 0:
            return (dq.zero_(), None if packed else dk.zero_(), None if packed else dv.zero_(),
                    None if dtable is None else dtable.zero_(), None, None, None, None, None)
        if dtable is not None:
            parts = torch.empty(B * (-(-Sq // 128)) * dtable.numel(), dtype=torch.float32, device=dev)
        dout = _usable(dout)
        delta = torch.empty(B, nh, Sq, dtype=torch.float32, device=dev)
        w, borders = _words((*qkv, (out.data_ptr(), _strides(out)), (dout.data_ptr(), _strides(dout)), *grads), B, Sq, Sk,
                            nh, nkv, hd, opts, key_bias, lens, starts, table, stat, delta.data_ptr(),
                            0 if parts is None else parts.data_ptr(), 0 if dtable is None else dtable.data_ptr())
        _call("dtf_attention_bwd", w, borders, q.dtype == torch.bfloat16, opts[1], q)
        return dq, dk, dv, dtable, None, None, None, None, None


def _composed(q, k, v, table, key_bias, lens, starts, nkv, opts):
    """The same function in torch operations, for tensors that are not on a GPU."""
    causal, scale, start0, max_distance, bidirectional = opts
    if k is None:
        q, k, v = q.split((q.shape[2] - 2 * nkv, nkv, nkv), 2)
    B, Sq, nh, _ = q.shape
    Sk = k.shape[1]
    ok = torch.ones(B, Sk, dtype=torch.bool)
    if lens is not None:
        ok &= torch.arange(Sk) < lens[:, None]
    if key_bias is not None:
        ok &= key_bias != -math.inf
    k, v = (t.float().masked_fill(~ok[:, :, None, None], 0.0).transpose(1, 2).repeat_interleave(nh // nkv, 1) for t in (k, v))
    t = q.float().transpose(1, 2) @ k.transpose(2, 3) * scale
    first = torch.full((B,), start0) if starts is None else starts.long()
    dist = torch.arange(Sk) - (torch.arange(Sq)[:, None] + first[:, None, None])               # [B, Sq, Sk]
    if table is not None:
        bucket = _rel.relative_bucket(dist, table.shape[0], max_distance, bidirectional)
        t = t + table.float()[bucket].permute(0, 3, 1, 2)
    if key_bias is not None:
        t = t + key_bias[:, None, None, :]
    seen = ok[:, None, :] & (dist <= 0) if causal else ok[:, None, :].expand(B, Sq, Sk)
    t = t.masked_fill(~seen[:, None], -math.inf)
    top = t.detach().amax(-1, keepdim=True) if Sk else t.detach().sum(-1, keepdim=True)
    e = torch.exp(t - top.masked_fill(top == -math.inf, 0.0))
    total = e.sum(-1, keepdim=True)
    p = e / total.masked_fill(total == 0, 1.0)
    return (p @ v).transpose(1, 2).to(q.dtype).contiguous()


def _int_vector(t, name, B, device):
    if not isinstance(t, torch.Tensor) or t.shape != (B,) or t.dtype not in (torch.int32, torch.int64) or t.device != device:
        raise ValueError(f"{name} is an int32 or int64 tensor [{B}] on {device}")
    return t if t.dtype == torch.int32 and t.is_contiguous() else t.to(torch.int32).contiguous()


def _general(q, k, v, nkv, key_bias, causal, scale, key_lengths, q_start, rel_table, rel_max_distance, rel_bidirectional):
    B, Sq, n, hd = q.shape
    nh, Sk = (n - 2 * nkv, Sq) if k is None else (n, k.shape[1])
    _lib.dtype_code(q.dtype)
    if hd % 8 or not 8 <= hd <= 128:
        raise ValueError(f"head size {hd}: need a multiple of 8 up to 128")
    if nkv < 1 or nh < 1 or nh % nkv:
        raise ValueError(f"{nh} query heads do not divide over {nkv} key / value heads")
    if max(B, Sq, Sk) > 1 << 28 or nh > 1 << 16:
        raise ValueError(f"sizes {tuple(q.shape)} with {Sk} keys are out of range")
    scale = 1.0 / math.sqrt(hd) if scale is None else float(scale)
    if not 1e-30 < scale < 1e30:
        raise ValueError(f"scale {scale}: need a positive number between 1e-30 and 1e30")
    if key_bias is not None:
        if key_bias.shape != (B, Sk) or key_bias.device != q.device or not key_bias.is_floating_point():
            raise ValueError(f"key_bias is a floating tensor [{B}, {Sk}] on {q.device}, got {tuple(key_bias.shape)}")
        if key_bias.requires_grad:
            raise ValueError("key_bias has no gradient: pass it detached")
        key_bias = key_bias.float().contiguous()
    lens = None if key_lengths is None else _int_vector(key_lengths, "key_lengths", B, q.device)
    starts, start0 = None, Sk - Sq
    if isinstance(q_start, torch.Tensor):
        starts = _int_vector(q_start, "q_start", B, q.device)
    elif q_start is not None:
        start0 = int(q_start)
        if abs(start0) > 1 << 29:
            raise ValueError(f"q_start {start0} is out of range")
    bidirectional = (not causal) if rel_bidirectional is None else bool(rel_bidirectional)
    if rel_table is not None:
        _rel.check_buckets(rel_table, nh, rel_max_distance, bidirectional)
        if rel_table.device != q.device:
            raise ValueError(f"rel_table is on {rel_table.device}, the queries on {q.device}")
    opts = (bool(causal), scale, start0, int(rel_max_distance), bidirectional)
    run = _GeneralFn.apply if q.is_cuda else _composed
    return run(q, k, v, rel_table, key_bias, lens, starts, nkv, opts)


def attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, key_bias: torch.Tensor | None = None, *,
              causal: bool = False, scale: float | None = None, key_lengths: torch.Tensor | None = None,
              q_start: int | torch.Tensor | None = None, rel_table: torch.Tensor | None = None,
              rel_max_distance: int = 128, rel_bidirectional: bool | None = None) -> torch.Tensor:
    """``q[B, Sq, nh, hd]``, ``k, v[B, Sk, nkv, hd]`` -> context ``[B, Sq, nh, hd]``; float32 or bfloat16, with gradients
    for ``q``, ``k``, ``v`` and ``rel_table``.

    Strides are free (views into larger buffers are read in place when 16-byte aligned); ``nh`` is a multiple of
    ``nkv``, and query head ``h`` reads key head ``h // (nh // nkv)``; ``hd`` is a multiple of 8 up to 128.

    ``key_bias[B, Sk]`` is added to the scores of every query; a key with ``-inf`` takes no part, whatever ``k`` and
    ``v`` hold there. ``key_lengths[B]`` (int32, else converted; values are clamped to ``[0, Sk]``) ends each
    sequence's keys: what lies behind is never used. Query ``i`` stands at position ``q_start + i`` among the keys
    (default: the queries are the last ``Sq`` of ``Sk`` positions; a tensor ``[B]`` gives each sequence its own, as for
    new tokens over caches filled to different lengths). ``causal``: keys after the query's position take no part.
    ``rel_table[buckets, nh]`` adds the learned bias of ``ops/relative_bias.py`` for the distance to that position
    (``rel_bidirectional`` defaults to ``not causal``). A query that no key is left for gets zeros, and zero gradients.

    K and V of keys that only ``causal`` hides have to be finite."""
    if q.dim() != 4 or k.dim() != 4 or k.shape != v.shape or k.shape[0] != q.shape[0] or k.shape[3] != q.shape[3]:
        raise ValueError(f"q[B, Sq, nh, hd] and k, v[B, Sk, nkv, hd] do not fit: {tuple(q.shape)}, {tuple(k.shape)}, "
                         f"{tuple(v.shape)}")
    if not (q.dtype == k.dtype == v.dtype and q.device == k.device == v.device):
        raise ValueError("q, k and v are of one type and on one device")
    return _general(q, k, v, k.shape[2], key_bias, causal, scale, key_lengths, q_start, rel_table, rel_max_distance,
                    rel_bidirectional)


def self_attention(qkv: torch.Tensor, key_bias: torch.Tensor | None = None, *, kv_heads: int | None = None,
                   causal: bool = False, scale: float | None = None, key_lengths: torch.Tensor | None = None,
                   q_start: int | torch.Tensor | None = None, rel_table: torch.Tensor | None = None,
                   rel_max_distance: int = 128, rel_bidirectional: bool | None = None) -> torch.Tensor:
    """``qkv[B, S, 3, nh, hd]`` -> context ``[B, S, nh, hd]``. ``key_bias[B, S]`` (fp32) is added to
    the scores of every query of that batch element (0 for real tokens, -inf for padding).

    With ``kv_heads`` the buffer is ``[B, S, nh + 2 * kv_heads, hd]`` (query heads, then key heads, then value heads).
    It and the other options are those of :func:`attention`, whose kernels then run, on the buffer in place: the gradient
    comes back as one buffer too."""
    if kv_heads is not None or causal or scale is not None or key_lengths is not None or q_start is not None \
            or rel_table is not None:
        if kv_heads is None:
            if qkv.dim() != 5 or qkv.shape[2] != 3:
                raise ValueError(f"qkv is [B, S, 3, nh, hd], got {tuple(qkv.shape)}")
            kv_heads = qkv.shape[3]
            qkv = qkv.flatten(2, 3)
        if qkv.dim() != 4 or qkv.shape[2] <= 2 * kv_heads:
            raise ValueError(f"qkv is [B, S, nh + 2 * {kv_heads}, hd], got {tuple(qkv.shape)}")
        return _general(qkv, None, None, int(kv_heads), key_bias, causal, scale, key_lengths, q_start, rel_table,
                        rel_max_distance, rel_bidirectional)
    if _fast(qkv):
        if key_bias is not None:
            key_bias = key_bias.float().contiguous()
        if _flash_ok(qkv):
            return _FlashFn.apply(qkv, key_bias)
        return _AttnFn.apply(qkv, key_bias)
    B, S, _, nh, hd = qkv.shape
    q, k, v = (qkv[:, :, i].permute(0, 2, 1, 3).float() for i in range(3))
    s = q @ k.transpose(-1, -2) / math.sqrt(hd)
    if key_bias is not None:
        s = s + key_bias[:, None, None, :].float()
    o = torch.softmax(s, dim=-1) @ v
    return o.permute(0, 2, 1, 3).to(qkv.dtype).contiguous()
