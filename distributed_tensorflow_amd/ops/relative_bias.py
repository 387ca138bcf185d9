"""Learned relative position bias by buckets (front end of ``csrc/kernels/relative_bias.hip``).

A table of ``[buckets, heads]`` learned values is added to the attention scores: the score of query ``i`` and key ``j``
gets ``table[bucket(j - pos_i), head]`` with ``pos_i = q_start + i``. Distances up to ``exact - 1`` have a bucket each,
farther ones share buckets by the logarithm of the distance, and from ``max_distance`` on there is one bucket:

* ``bidirectional``: ``half = buckets / 2`` buckets for keys at or before the query, the other half for keys after it;
* one-sided: ``half = buckets``, and keys after the query count as distance 0;
* with ``a`` the distance and ``exact = half // 2``: bucket ``a`` when ``a < exact``, else
  ``exact + min(half - exact - 1, floor(log(a / exact) / log(max_distance / exact) * (half - exact)))``.

The borders between the buckets are computed in whole numbers (``a^(half - exact) * exact^t >= max_distance^t *
exact^(half - exact)``), so a distance that lies on a border is not decided by rounding.

:func:`relative_bias` writes the ``[heads, q_len, k_len]`` bias out, with the gradient of the table. The fused attention
(``ops/attention.py``, ``rel_table=``) adds the same bias without ever writing it.
"""
from __future__ import annotations

from functools import lru_cache

import torch

from . import _lib

MAX_BUCKETS, MAX_DISTANCE = 128, 2048


@lru_cache(maxsize=64)
def bucket_borders(buckets: int, max_distance: int, bidirectional: bool) -> tuple[int, ...]:
    """Smallest distance of each bucket after the first logarithmic one."""
    half = buckets // 2 if bidirectional else buckets
    exact = half // 2
    n = half - exact
    out, a = [], exact
    for t in range(1, n):
        need = max_distance ** t * exact ** (n - t)          # a^n >= max_distance^t exact^(n - t)
        while a ** n < need:
            a += 1
        out.append(a)
    return tuple(out)


def check_buckets(table: torch.Tensor, heads: int | None, max_distance: int, bidirectional: bool) -> None:
    if table.dim() != 2 or (heads is not None and table.shape[1] != heads):
        raise ValueError(f"the table is [buckets, heads], got {tuple(table.shape)} for {heads} heads")
    n = table.shape[0]
    _lib.dtype_code(table.dtype)
    half = n // 2 if bidirectional else n
    if n > MAX_BUCKETS or half < 2 or (bidirectional and n % 2) or table.shape[1] < 1:
        raise ValueError(f"{n} buckets: need 2 to {MAX_BUCKETS}, an even number of at least 4 when bidirectional")
    if not half // 2 < max_distance <= MAX_DISTANCE:
        raise ValueError(f"max_distance {max_distance}: need more than {half // 2} (a bucket each) and at most {MAX_DISTANCE}")


def relative_bucket(distance: torch.Tensor, buckets: int, max_distance: int = 128, bidirectional: bool = True) -> torch.Tensor:
    """Bucket (int64) of every signed distance key - query."""
    d = distance.long()
    half = buckets // 2 if bidirectional else buckets
    exact = half // 2
    a = d.abs() if bidirectional else (-d).clamp(min=0)
    far = torch.full_like(a, exact)
    for border in bucket_borders(buckets, max_distance, bidirectional):
        far += a >= border
    b = torch.where(a < exact, a, far)
    return b + half * (d > 0) if bidirectional else b


@lru_cache(maxsize=256)
def _words(q_len: int, k_len: int, heads: int, q_start: int, buckets: int, max_distance: int, bidirectional: bool):
    w = (q_len, k_len, heads, q_start, buckets, max_distance, int(bidirectional),
         *bucket_borders(buckets, max_distance, bidirectional))          # (the sizes of a call as its C entry reads them)
    return _lib.pack_words(w), len(w)


def _forward(table, q_len, k_len, q_start, max_distance, bidirectional):
    t = table.contiguous()
    out = torch.empty(t.shape[1], q_len, k_len, dtype=t.dtype, device=t.device)
    if out.numel():
        w = _words(q_len, k_len, t.shape[1], q_start, t.shape[0], max_distance, bidirectional)
        with _lib.on_device(t):
            rc = _lib.kernels().dtf_relative_bias_fwd(*w, _lib.ptr(t), _lib.ptr(out), _lib.dtype_code(t.dtype),
                                                      _lib.stream_ptr(t.device))
        _lib.check(rc, "relative_bias_fwd")
    return out


class _BiasFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, table, *args):
        ctx.meta = (*args, table.shape, table.dtype)
        return _forward(table, *args)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g):
        q_len, k_len, q_start, max_distance, bidirectional, shape, dt = ctx.meta
        if g.numel() == 0:
            return torch.zeros(shape, dtype=dt, device=g.device), None, None, None, None, None
        g = g.contiguous()
        d = torch.empty(shape, dtype=dt, device=g.device)
        lib = _lib.kernels()
        parts = torch.empty(lib.dtf_relative_bias_parts(q_len, k_len, shape[1]) * shape[0] * shape[1], dtype=torch.float32,
                            device=g.device)
        w = _words(q_len, k_len, shape[1], q_start, shape[0], max_distance, bidirectional)
        with _lib.on_device(g):
            rc = lib.dtf_relative_bias_bwd(*w, _lib.ptr(g), _lib.ptr(parts), _lib.ptr(d), _lib.dtype_code(dt),
                                           _lib.stream_ptr(g.device))
        _lib.check(rc, "relative_bias_bwd")
        return d, None, None, None, None, None


def relative_bias(table: torch.Tensor, q_len: int, k_len: int, *, max_distance: int = 128, bidirectional: bool = True,
                  q_start: int | None = None) -> torch.Tensor:
    """``[heads, q_len, k_len]`` bias, in the type of ``table`` (``[buckets, heads]``, float32 or bfloat16).

    ``q_start`` is the position of the first query counted from the first key; by default the queries are the last
    ``q_len`` of the ``k_len`` positions (0 for self-attention). On a GPU forward-mode derivatives and traces are refused."""
    check_buckets(table, None, max_distance, bidirectional)
    q_start = k_len - q_len if q_start is None else int(q_start)
    if q_len < 0 or k_len < 0 or max(q_len, k_len) > 1 << 28 or abs(q_start) > 1 << 29:
        raise ValueError(f"lengths {q_len} and {k_len} with the first query at {q_start} are out of range")
    if table.is_cuda:
        run = _BiasFn.apply if _lib.differentiated(table) else _forward
        return run(table, q_len, k_len, q_start, max_distance, bool(bidirectional))
    d = torch.arange(k_len)[None, :] - (torch.arange(q_len)[:, None] + q_start)
    return table.t()[:, relative_bucket(d, table.shape[0], max_distance, bidirectional)]
