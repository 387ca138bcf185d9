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
# position bias; bf16 and fp32. A call is an array of 64-bit words, the enum of csrc/kernels/attention.hip: four for each
# of q, k, v, out, dout, dq, dk, dv (pointer; batch, token and head stride), then the rest.
_NONE = (0, 0, 0, 0)
_entry: dict = {}


def _call(name: str, words, scale: float, like: torch.Tensor) -> None:
    fn = _entry.get(name)
    if fn is None:
        fn = getattr(_lib.kernels(), name)
        fn.argtypes = (ctypes.c_char_p, ctypes.c_int, ctypes.c_float, ctypes.c_void_p)
        _entry[name] = fn
    n = len(words)
    with _lib.on_device(like):
        rc = fn(_lib.pack_words(words), n, scale, _lib.stream_ptr(like.device))
    if rc:
        _lib.check(rc, name)


def _address(t: torch.Tensor):
    """The four words of ``t``, or ``None`` when the kernels cannot address it in place: they read 16 bytes at a time
    along the head, rows must not overlap, and a tile's offsets are 32-bit. The strides of axes of one element, which torch
    leaves arbitrary, are those of a dense tensor."""
    B, S, n, hd = t.shape
    sb, ss, sh, se = t.stride()
    if B == 1:
        sb = 0
    if S == 1:
        ss = n * hd
    if n == 1:
        sh = 0
    p = t.data_ptr()
    if se != 1 or not hd <= ss <= 1 << 22 or (p | (sb | ss | sh) * t.element_size()) & 15:
        return None
    return p, sb, ss, sh


def _usable(t: torch.Tensor):
    """(tensor, address): ``t`` itself or a dense copy."""
    w = _address(t)
    if w is None:
        t = t.contiguous() if not t.is_contiguous() else t.clone(memory_format=torch.contiguous_format)
        w = _address(t)
    return t, w


def _heads(t: torch.Tensor, w, nh: int, nkv: int):
    """The words of the query, key and value heads of a fused buffer."""
    p, sb, ss, sh = w
    step = t.stride(2) * t.element_size()
    return p, sb, ss, sh, p + nh * step, sb, ss, sh, p + (nh + nkv) * step, sb, ss, sh


def _dense(p, S, n, hd):
    return p, S * n * hd, n * hd, hd


def _inputs(q, k, v, nkv):
    """q, k, v as the kernels read them, and their twelve words."""
    q, w = _usable(q)
    if k is None:
        return q, k, v, _heads(q, w, q.shape[2] - 2 * nkv, nkv)
    (k, kw), (v, vw) = _usable(k), _usable(v)
    return q, k, v, (*w, *kw, *vw)


def _forward(q, k, v, table, key_bias, lens, starts, nkv, opts, stat, fine):
    """(out, q, k, v as the kernels read them, table, words of the call)."""
    causal, scale, start0, max_distance, bidirectional = opts
    q, k, v, ins = _inputs(q, k, v, nkv)
    B, Sq, nh, hd = q.shape
    if k is None:
        nh -= 2 * nkv
    Sk = Sq if k is None else k.shape[1]
    out = torch.empty(B, Sq, nh, hd, dtype=q.dtype, device=q.device)
    bf16, rel, borders = int(q.dtype == torch.bfloat16), (0, 0, 0), ()
    if table is not None:
        table = table.contiguous()
        rel = (table.data_ptr(), int(table.dtype == torch.bfloat16), table.shape[0])
        borders = _rel.bucket_borders(table.shape[0], max_distance, bidirectional)
    part, splits = 0, 1
    if B and Sq * nh <= 32 * nkv and Sk > 256:           # few queries: the keys may be split over workgroups
        splits = _lib.kernels().dtf_attention_splits(B, Sq, Sk, nh, nkv)
        if splits > 1:
            part = torch.empty(splits * B * nh * Sq * (-(-hd // 32) * 32 + 2), dtype=torch.float32, device=q.device)
    words = (*ins, *_dense(out.data_ptr(), Sq, nh, hd), *_NONE, *_NONE, *_NONE, *_NONE,
             0 if key_bias is None else key_bias.data_ptr(), 0 if lens is None else lens.data_ptr(),
             0 if starts is None else starts.data_ptr(), start0, *rel, max_distance, int(bidirectional),
             0 if stat is None else stat.data_ptr(), 0, 0, 0, B, Sq, Sk, nh, nkv, hd, int(causal), bf16,
             part.data_ptr() if splits > 1 else 0, 0 if fine is None else fine.data_ptr(), *borders)
    if Sk == 0:
        out.zero_()
    elif out.numel():
        _call("dtf_attention_fwd", words, scale, q)
    return out, q, k, v, table, words


class _GeneralFn(torch.autograd.Function):
    """``k is None``: ``q`` is the fused ``[B, S, nh + 2 nkv, hd]`` buffer, and so is its gradient."""

    @staticmethod
    def forward(ctx, q, k, v, table, key_bias, lens, starts, nkv, opts):
        B, Sq, n = q.shape[:3]
        stat = torch.empty(2, B, n - 2 * nkv if k is None else n, Sq, dtype=torch.float32, device=q.device)
        ctx.table_like = None if table is None else (table.shape, table.dtype)
        # the bits of the output that bfloat16 cuts off, for the backward pass's rowsum(dO * O)
        fine = None
        if q.dtype == torch.bfloat16:
            fine = torch.empty(B, Sq, n - 2 * nkv if k is None else n, q.shape[3], dtype=torch.uint8, device=q.device)
        out, q, k, v, table, ctx.words = _forward(q, k, v, table, key_bias, lens, starts, nkv, opts, stat, fine)
        ctx.scale = opts[1]
        ctx.save_for_backward(q, k, v, table, key_bias, lens, starts, stat, fine, out)
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout):
        # the words of the forward pass hold the sizes; what they point to may have moved (hooks on saved tensors put them
        # elsewhere, checkpointing computes them anew)
        q, k, v, table, key_bias, lens, starts, stat, fine, out = ctx.saved_tensors
        words = ctx.words
        B, Sq, Sk, nh, nkv, hd = words[45:51]
        q, k, v, ins = _inputs(q, k, v, nkv)
        dev, dt = q.device, q.dtype
        dq = torch.empty(q.shape, dtype=dt, device=dev)
        dk = dv = dtable = None
        if k is None:
            grads = _heads(dq, _dense(dq.data_ptr(), Sq, nh + 2 * nkv, hd), nh, nkv)
        else:
            dk, dv = torch.empty(k.shape, dtype=dt, device=dev), torch.empty(k.shape, dtype=dt, device=dev)
            grads = (*_dense(dq.data_ptr(), Sq, nh, hd), *_dense(dk.data_ptr(), Sk, nkv, hd),
                     *_dense(dv.data_ptr(), Sk, nkv, hd))
        if table is not None and ctx.needs_input_grad[3]:
            dtable = torch.empty(ctx.table_like[0], dtype=ctx.table_like[1], device=dev)
        if out.numel() == 0 or Sk == 0:
            for t in (dq, dk, dv, dtable):
                if t is not None:
                    t.zero_()
            return dq, dk, dv, dtable, None, None, None, None, None
        # statistics of the queries for the dK / dV kernel, then the partial sums of the table's gradient
        n = B * nh * -(-Sq // 128) * 512
        scratch = torch.empty(n + (0 if dtable is None else B * -(-Sq // 128) * dtable.numel()), dtype=torch.float32, device=dev)
        p = scratch.data_ptr()
        part, splits = 0, 1
        if nh > nkv:                               # grouped heads: dK and dV may be summed in splits of the group
            splits = _lib.kernels().dtf_attention_bwd_splits(B, Sk, nh, nkv)
            if splits > 1:
                part = torch.empty(splits * 2 * B * nkv * Sk * (-(-hd // 32) * 32), dtype=torch.float32, device=dev)
        dout, dw = _usable(dout)
        keys, lengths, first, bias, stats, low = (0 if t is None else t.data_ptr() for t in (key_bias, lens, starts, table, stat, fine))
        _call("dtf_attention_bwd", (*ins, *_dense(out.data_ptr(), Sq, nh, hd), *dw, *grads, keys, lengths, first, words[35], bias,
              *words[37:41], stats, p, *((0, 0) if dtable is None else (p + 4 * n, dtable.data_ptr())), *words[45:53],
              part.data_ptr() if splits > 1 else 0, low, *words[55:]), ctx.scale, q)
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
    first = torch.full((B,), start0) if starts is None else starts.long()
    if causal:
        ok &= torch.arange(Sk) < (first + Sq)[:, None]         # (nothing behind the last query is read)
    k, v = (t.float().masked_fill(~ok[:, :, None, None], 0.0).transpose(1, 2).repeat_interleave(nh // nkv, 1) for t in (k, v))
    t = q.float().transpose(1, 2) @ k.transpose(2, 3) * scale
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
    if t.dtype == torch.int64:                     # (values that 32 bits do not hold stay as far out as they are)
        t = t.clamp(-(1 << 30), 1 << 30).int()
    return t.contiguous()


def _general(q, k, v, nkv, key_bias, causal, scale, key_lengths, q_start, rel_table, rel_max_distance, rel_bidirectional):
    B, Sq, n, hd = q.shape
    nh, Sk = (n - 2 * nkv, Sq) if k is None else (n, k.shape[1])
    _lib.dtype_code(q.dtype)
    if hd % 8 or not 8 <= hd <= 128:
        raise ValueError(f"head size {hd}: need a multiple of 8 up to 128")
    if nkv < 1 or nh < 1 or nh % nkv:
        raise ValueError(f"{nh} query heads do not divide over {nkv} key / value heads")
    if max(B, Sq, Sk) > 1 << 28 or nh > 1 << 16 or n * hd > 1 << 22:
        raise ValueError(f"sizes {tuple(q.shape)} with {Sk} keys are out of range")
    scale = 1.0 / math.sqrt(hd) if scale is None else float(scale)
    if not 1e-30 < scale < 1e30:
        raise ValueError(f"scale {scale}: need a positive number between 1e-30 and 1e30")
    if key_bias is not None:
        if key_bias.shape != (B, Sk) or key_bias.device != q.device or not key_bias.is_floating_point():
            raise ValueError(f"key_bias is a floating tensor [{B}, {Sk}] on {q.device}, got {tuple(key_bias.shape)}")
        if key_bias.requires_grad:
            raise ValueError("key_bias has no gradient: pass it detached")
        if key_bias.dtype == torch.float64:        # (a finite bias that 32 bits do not hold is none of their infinities)
            top = torch.finfo(torch.float32).max
            key_bias = torch.where(key_bias.isinf(), key_bias, key_bias.clamp(-top, top))
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
    if not q.is_cuda:
        return _composed(q, k, v, rel_table, key_bias, lens, starts, nkv, opts)
    if _lib.differentiated(q, k, v, rel_table):
        return _GeneralFn.apply(q, k, v, rel_table, key_bias, lens, starts, nkv, opts)
    return _forward(q, k, v, rel_table, key_bias, lens, starts, nkv, opts, None, None)[0]


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
    (``rel_bidirectional`` defaults to ``not causal``); ``-inf`` in it masks a bucket's distances, other values count up to
    1.1e7 either way. A query that no key is left for gets zeros, and zero gradients.

    With ``causal`` what lies behind the last query's position is never used either (the unfilled end of a cache); K and V
    of the keys up to it have to be finite, though earlier queries do not see them all. On a GPU forward-mode derivatives
    and traces are refused."""
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
