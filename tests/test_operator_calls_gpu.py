"""Calls of general attention, relative position bias and token log probabilities that their documentation allows beyond the
ordinary ones, on the GPU against the 64-bit oracles (bounds: operator_oracles.py)."""
import math
import os
import sys

import pytest
import torch
from torch.autograd import forward_ad as fwAD

sys.path.insert(0, os.path.dirname(__file__))
import operator_oracles as O  # noqa: E402
from distributed_tensorflow_amd.engine.graph import collected  # noqa: E402
from test_operators_gpu import BF16, DEV, FP32, _compare, _compare_logp, _dev, _inputs, _logits  # noqa: E402

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------------------------------ tangents and traces
def _one_call_each():
    """(name, its differentiable inputs, call)"""
    from distributed_tensorflow_amd.ops.attention import attention, self_attention
    from distributed_tensorflow_amd.ops.relative_bias import relative_bias
    from distributed_tensorflow_amd.ops.softmax_ce import token_log_probs
    q, k, v, _, table = (t.to(DEV) for t in _inputs(2, 40, 50, 2, 1, 16, FP32, 8))
    few = q[:, :1].contiguous()
    bias = torch.zeros(2, 50, device=DEV)
    x, tok = torch.randn(6, 40, device=DEV), torch.arange(6, device=DEV)
    return [("attention", (q, k, v, bias, table), lambda q, k, v, b, t: attention(q, k, v, b, rel_table=t)),
            ("attention, few queries", (few, k, v, bias, table), lambda q, k, v, b, t: attention(q, k, v, b, rel_table=t)),
            ("self_attention", (k.repeat(1, 1, 4, 1), table), lambda x, t: self_attention(x, kv_heads=1, rel_table=t)),
            ("relative_bias", (table,), lambda t: relative_bias(t, 9, 12)),
            ("token_log_probs", (x,), lambda x: token_log_probs(x, tok, 3).logp)]


def test_a_tangent_is_refused_and_not_dropped():
    for name, ins, call in _one_call_each():
        want = call(*ins)
        for i in range(len(ins)):
            for grad in (True, False):
                with torch.set_grad_enabled(grad), fwAD.dual_level():
                    with pytest.raises(NotImplementedError):
                        call(*ins[:i], fwAD.make_dual(ins[i], torch.ones_like(ins[i])), *ins[i + 1:])
                    assert torch.equal(call(*ins), want), name             # (a level without a tangent changes nothing)
        assert torch.equal(call(*ins), want), name


def test_a_trace_is_refused_and_not_left_without_the_kernels():
    from torch.fx.experimental.proxy_tensor import make_fx
    for name, ins, call in _one_call_each():
        for trace in (lambda: torch.jit.trace(call, ins), lambda: make_fx(call)(*ins)):
            with pytest.raises(RuntimeError, match="trace"):
                trace()
        call(*ins)
        with pytest.raises(RuntimeError, match="trace"):
            torch.jit.trace(call, (ins[0].detach().clone().requires_grad_(), *ins[1:]))


# ------------------------------------------------------------------------------------------ inside a compiled function
def test_calls_inside_a_compiled_function():
    """torch.compile breaks its graph around the kernels: the same results and gradients as without it."""
    from distributed_tensorflow_amd.ops.attention import attention
    from distributed_tensorflow_amd.ops.relative_bias import relative_bias
    from distributed_tensorflow_amd.ops.softmax_ce import token_log_probs
    q, k, v, _, table = (t.to(DEV) for t in _inputs(2, 40, 50, 2, 1, 16, FP32, 8))
    tok = torch.arange(16, device=DEV)
    for call in (lambda q, k, v, t: attention(q * 1, k, v, causal=True, rel_table=t) + 1,
                 lambda q, k, v, t: attention(q[:, :1] * 1, k, v, rel_table=t) + 1,
                 lambda q, k, v, t: relative_bias(t * 2, 9, 12) + 1,
                 lambda q, k, v, t: token_log_probs(q.reshape(16, 160) * 1, tok, 2).logp + 1):
        torch._dynamo.reset()
        fast, runs = torch.compile(call, backend="eager"), []
        for f in (call, fast):
            leaves = [t.clone().requires_grad_() for t in (q, k, v, table)]
            out = f(*leaves)
            grads = torch.autograd.grad(out.sum(), leaves, allow_unused=True)
            with torch.no_grad():
                runs.append([out, f(*leaves), *(g for g in grads if g is not None)])
        assert len(runs[0]) == len(runs[1]) and all(torch.equal(a, b) for a, b in zip(*runs))


# ------------------------------------------------------------------------------------------ key biases at the ends of their type
@pytest.mark.parametrize("dt", [BF16, FP32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("Sq,Sk", [(70, 90), (3, 700)], ids=["rows", "few"])
@pytest.mark.parametrize("scale", [None, 0.3, 3.0, 1e-3])
@pytest.mark.parametrize("rel", [0, 8])
def test_attention_key_biases_of_any_finite_value(dt, Sq, Sk, scale, rel):
    """The largest value on one key and on several, large ones of both signs, and rows of lowest values of two types."""
    q, k, v, do, table = _inputs(5, Sq, Sk, 4, 2, 40, dt, rel, seed=2)
    kb = torch.zeros(5, Sk)
    kb[0, 17] = torch.finfo(FP32).max
    kb[1, 3:60:7] = torch.finfo(FP32).max
    kb[1, 5], kb[1, 9] = -math.inf, torch.finfo(FP32).min
    kb[2, ::2], kb[2, 1::2] = 1e37, 2e38
    kb[3], kb[3, 11:40:3] = torch.finfo(FP32).min, torch.finfo(BF16).min
    kb[4, :] = -1e38
    kb[4, Sk // 2:] = -3e38
    _compare(q, k, v, do, table, key_bias=kb, scale=scale, rel_max_distance=20)


@pytest.mark.parametrize("dt", [BF16, FP32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("Sq", [70, 3], ids=["rows", "few"])
def test_attention_key_biases_beside_the_smallest_scale(dt, Sq):
    """scale 2e-30: the biases alone decide, ordinary ones and those that 1 / scale would carry past the type."""
    q, k, v, do, _ = _inputs(3, Sq, 300, 2, 2, 16, dt, seed=6)
    kb = torch.randn(3, 300, generator=torch.Generator().manual_seed(1))
    kb[1, 40:50] = torch.arange(10.0) * 1e31
    kb[2] = -1e31
    kb[2, 7::2] = -2e31
    _compare(q, k, v, do, key_bias=kb, scale=2e-30)


# ------------------------------------------------------------------------------------------ key biases in 64 bits
@pytest.mark.parametrize("dt", [BF16, FP32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("Sq", [70, 3], ids=["rows", "few"])
def test_attention_key_bias_in_64_bits(dt, Sq):
    """float64's lowest value is finite: no mask, whatever 32 bits make of it."""
    q, k, v, do, _ = _inputs(2, Sq, 300, 2, 2, 16, dt, seed=7)
    kb = torch.zeros(2, 300, dtype=torch.float64)
    kb[0] = torch.finfo(torch.float64).min
    kb[1, 40:50] = torch.finfo(torch.float64).max
    kb[1, 60] = -math.inf
    _compare(q, k, v, do, key_bias=kb)


# ------------------------------------------------------------------------------------------ few queries
@pytest.mark.parametrize("dt", [BF16, FP32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("Sk", [200, 1700], ids=["one_piece", "split"])
@pytest.mark.parametrize("Sq,nh", [(1, 4), (5, 8), (16, 4)], ids=["2_rows", "20_rows", "32_rows"])
@pytest.mark.parametrize("rel", [0, 16])
@pytest.mark.parametrize("causal", [False, True], ids=["full", "causal"])
def test_few_queries_with_key_biases_and_garbage_behind_masks(dt, Sk, Sq, nh, rel, causal):
    """-inf keys with NaN and infinities behind them, alone, with lengths and with a table; rows that no key is left for."""
    B, nkv, hd = 5, 2, 64
    q, k, v, do, table = _inputs(B, Sq, Sk, nh, nkv, hd, dt, rel, seed=8)
    kb = torch.randn(B, Sk, generator=torch.Generator().manual_seed(2))
    kb[0, ::3] = -math.inf
    kb[1] = -math.inf
    kb[2, 1:] = -math.inf
    kb[3, :150] = -math.inf
    for b, value in ((0, math.nan), (1, math.inf), (2, -math.inf), (3, math.nan)):
        k[b, kb[b] == -math.inf], v[b, kb[b] == -math.inf] = value, value
    n = torch.tensor([Sk, Sk - 9, Sk, Sk - 40, 0], dtype=torch.int32)
    for b, m in enumerate(n.tolist()):
        k[b, m:], v[b, m:], kb[b, m:] = math.nan, math.inf, math.nan
    # (causal needs finite K and V where only it hides them: the queries are the last, or stand where every key that they do
    # not see is masked anyway)
    out, got = _compare(q, k, v, do, table, causal=causal, key_bias=kb, key_lengths=n, q_start=n - Sq if causal else None,
                        rel_max_distance=60)
    for b in (1, 4):
        assert not out[b].any() and not any(g[b].any() for g in got[:3])


@pytest.mark.parametrize("Sq,nh", [(1, 4), (5, 8), (16, 4), (33, 2)], ids=["2_rows", "20_rows", "32_rows", "66_rows"])
@pytest.mark.parametrize("dt", [BF16, FP32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("cfg", [(32, 128, True), (128, 2048, False), (4, 3, True)], ids=str)
def test_few_queries_with_a_table(dt, Sq, nh, cfg):
    q, k, v, do, table = _inputs(2, Sq, 1100, nh, 2 if nh > 2 else 1, 96, dt, cfg[0])
    _compare(q, k, v, do, table, causal=not cfg[2], rel_max_distance=cfg[1], rel_bidirectional=cfg[2],
             q_start=torch.tensor([1100 - Sq, 500]))


# ------------------------------------------------------------------------------------------ unfilled caches
@pytest.mark.parametrize("dt", [BF16, FP32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("Sq,Sk", [(1, 90), (1, 2000), (7, 700), (150, 300)], ids=str)
@pytest.mark.parametrize("extra", ["", "table", "key_bias", "lengths"])
def test_attention_over_the_filled_part_of_a_cache(dt, Sq, Sk, extra):
    """NaN and infinities behind the last query's position, without key_lengths: causal alone keeps them out, of the result
    and of the gradients."""
    B, nh, nkv, hd = 4, 4, 2, 64
    q, k, v, do, table = _inputs(B, Sq, Sk, nh, nkv, hd, dt, 16 if extra == "table" else 0, seed=11)
    filled = torch.tensor([Sk, Sq, Sk // 2 + 5 if Sq < 100 else 260, Sk - 1], dtype=torch.int32)
    kw = {}
    if extra == "key_bias":
        kw["key_bias"] = torch.randn(B, Sk, generator=torch.Generator().manual_seed(3))
    if extra == "lengths":
        kw["key_lengths"] = torch.tensor([Sk, Sk, Sk // 2, 1], dtype=torch.int32)
    clean = [t.clone() for t in (k, v)]
    for b, n in enumerate(filled.tolist()):
        k[b, n:], v[b, n:] = math.nan, math.inf
        for t in clean:
            t[b, n:] = 0
    from distributed_tensorflow_amd.ops.attention import attention
    kw.update(causal=True, q_start=filled - Sq)
    val, tol = O.attention(q, *clean, do, rel_table=table, **kw)
    leaves = [t.to(DEV).requires_grad_() for t in (q, k, v)] + ([] if table is None else [table.to(DEV).requires_grad_()])
    out = attention(*leaves[:3], rel_table=None if table is None else leaves[3], **{n: _dev(x) for n, x in kw.items()})
    O.check("out", out, val["out"], tol["out"])
    for n, g in zip(("dq", "dk", "dv", "dtable"), torch.autograd.grad(out, leaves, do.to(DEV))):
        O.check(n, g, val[n], tol[n])


# ------------------------------------------------------------------------------------------ distances masked by the table
@pytest.mark.parametrize("dt", [BF16, FP32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("mask", [-math.inf, torch.finfo(BF16).min], ids=["inf", "lowest"])
@pytest.mark.parametrize("Sq,Sk", [(200, 200), (2, 900)], ids=["rows", "few"])
@pytest.mark.parametrize("bias", [False, True], ids=["", "key_bias"])
def test_attention_with_distances_that_the_table_masks(dt, mask, Sq, Sk, bias):
    """-inf, or the type's lowest value, in some buckets, the far ones among them: the keys there take no part. (The oracle is
    given -1e31, which leaves them none either: every row has other keys.)"""
    q, k, v, do, table = _inputs(2, Sq, Sk, 4, 2, 64, dt, 16, seed=12)
    table[7], table[15], table[3, 1], table[11] = mask, mask, mask, mask
    low = table.clone()
    low[table.float() < -1e30] = -1e31
    kw = dict(rel_max_distance=30, rel_bidirectional=True)
    if bias:
        kw["key_bias"] = torch.randn(2, Sk, generator=torch.Generator().manual_seed(4))
        kw["key_bias"][0, ::5] = -math.inf
    from distributed_tensorflow_amd.ops.attention import attention
    val, tol = O.attention(q, k, v, do, rel_table=low, **kw)
    leaves = [t.to(DEV).requires_grad_() for t in (q, k, v, table)]
    out = attention(*leaves[:3], rel_table=leaves[3], **{n: _dev(x) for n, x in kw.items()})
    O.check("out", out, val["out"], tol["out"])
    for n, g in zip(("dq", "dk", "dv", "dtable"), torch.autograd.grad(out, leaves, do.to(DEV))):
        O.check(n, g, val[n], tol[n])
    if mask == -math.inf:                                    # a head whose every distance is masked
        with torch.no_grad():
            leaves[3][:, 2] = mask
        out = attention(*leaves[:3], rel_table=leaves[3], **{n: _dev(x) for n, x in kw.items()})
        gq, gk, gv, gt = torch.autograd.grad(out, leaves, do.to(DEV))
        assert not out[:, :, 2].any() and not gq[:, :, 2].any() and not gt[:, 2].any()
        assert all(torch.isfinite(t).all() for t in (out, gq, gk, gv, gt))


# ------------------------------------------------------------------------------------------ captured decoding
@pytest.mark.parametrize("ints", [torch.int32, torch.int64], ids=["int32", "int64"])
@pytest.mark.parametrize("table", [False, True], ids=["", "table"])
def test_new_tokens_over_a_growing_cache_in_a_graph(ints, table):
    """One captured call, replayed while the caches fill: lengths and starts are read anew from the caller's tensors."""
    from distributed_tensorflow_amd.ops.attention import attention
    B, nh, nkv, hd, Sk = 3, 8, 2, 64, 1500
    g = torch.Generator(DEV).manual_seed(5)
    k, v = (torch.full((B, Sk, nkv, hd), math.nan, dtype=BF16, device=DEV) for _ in range(2))
    q = torch.randn(B, 1, nh, hd, dtype=BF16, device=DEV, generator=g)
    t = torch.randn(16, nh, dtype=BF16, device=DEV, generator=g) if table else None
    n, at = (torch.zeros(B, dtype=ints, device=DEV) for _ in range(2))

    def call():
        return attention(q, k, v, causal=True, key_lengths=n, q_start=at, rel_table=t)

    def fill(step):
        for b, m in enumerate((1 + step, 700 * step, 1500 - step)):
            k[b, :m] = torch.randn(m, nkv, hd, dtype=BF16, device=DEV, generator=g)
            v[b, :m] = torch.randn(m, nkv, hd, dtype=BF16, device=DEV, generator=g)
            n[b], at[b] = m, m - 1

    fill(0)
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with collected(), torch.cuda.graph(graph):
        out = call()
    for step in range(3):
        fill(step)
        q.mul_(-1.5)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, call()) and torch.isfinite(out).all()
        assert bool(out[1].any()) == (step > 0)              # (an empty cache gives zeros)


# ------------------------------------------------------------------------------------------ large grids
def test_few_queries_over_more_keys_than_the_other_kernels_grids_hold():
    """One token of 32 heads over 2^25 keys of one head: 32 x 262145 tiles of 128 keys, which no kernel of this pass has as
    its grid. A few keys far apart hold nearly all the weight. Bound: P and the result are rounded to bf16 (u); a score of 8
    products 2 (8 + 8) u32 A; a lane adds at most 2^25 / (64 x 4 x 4) terms of P, a wave 2^25 / (64 x 4 x 32) products."""
    from distributed_tensorflow_amd.ops.attention import attention
    nh, hd, Sk = 32, 8, (1 << 25) + 77
    g = torch.Generator(DEV).manual_seed(4)
    q = torch.randn(1, 1, nh, hd, device=DEV, generator=g).to(BF16)
    k = (torch.randn(1, Sk, 1, hd, device=DEV, generator=g) * 0.1).to(BF16)
    v = torch.randn(1, Sk, 1, hd, device=DEV, generator=g).to(BF16)
    for i, at in enumerate((0, 5_000_000, (1 << 24) + 1, Sk - 78, Sk - 1)):
        k[0, at, 0] = 60 * q[0, 0, 6 * i].float() / q[0, 0, 6 * i].float().norm() ** 2
    out = attention(q, k, v)
    t = q[0, 0].double() @ k[0, :, 0].double().t() / math.sqrt(hd)
    A = q[0, 0].double().abs() @ k[0, :, 0].double().abs().t() / math.sqrt(hd)
    p = torch.softmax(t, 1)
    del t
    want, u = p @ v[0, :, 0].double(), O.half_step(BF16)
    terms = Sk // (64 * 4 * 4) + Sk // (64 * 4 * 32) + 512
    tol = (p * (u + O.U32 * (2 * (hd + 8) * A + terms + 16))) @ v[0, :, 0].double().abs() + u * want.abs()
    O.check("out", out[0, 0], want.cpu(), 1.01 * tol.cpu())


# ------------------------------------------------------------------------------------------ parts of the gradients
@pytest.mark.parametrize("dt", [BF16, FP32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("fused", [False, True], ids=["separate", "fused"])
def test_attention_gradients_of_some_inputs(dt, fused):
    """Any subset of q, k, v and the table may ask for its gradient: the same numbers as together."""
    from distributed_tensorflow_amd.ops.attention import attention, self_attention
    q, k, v, do, table = (t.to(DEV) for t in _inputs(2, 140, 140, 4, 2, 64, dt, 16))
    ins = [torch.cat((q, k, v), 2), table] if fused else [q, k, v, table]

    def grads(wanted):
        leaves = [t.clone().requires_grad_(i in wanted) for i, t in enumerate(ins)]
        out = self_attention(leaves[0], kv_heads=2, causal=True, rel_table=leaves[1]) if fused else \
            attention(*leaves[:3], causal=True, rel_table=leaves[3])
        return torch.autograd.grad(out, [leaves[i] for i in wanted], do)

    every = grads(range(len(ins)))
    for bits in range(1, 1 << len(ins)):
        wanted = [i for i in range(len(ins)) if bits >> i & 1]
        assert all(torch.equal(a, every[i]) for i, a in zip(wanted, grads(wanted))), wanted


# ------------------------------------------------------------------------------------------ the written bias
@pytest.mark.parametrize("dt", [BF16, FP32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("cfg", [(3001, 2999, 20, 32, 128, True, None), (4099, 1501, 24, 16, 50, False, -900),
                                 (1203, 5003, 17, 128, 2048, True, 1700), (60007, 33, 3, 8, 8, True, -20000)], ids=str)
def test_relative_bias_gradient_of_several_tiles_a_wave(dt, cfg):
    """heads x tiles (8 rows x 512 columns) beyond twice 8192, so that a wave walks several of them, at odd lengths and with a
    last wave whose share is short. The sums are made in 64 bits on the GPU, diagonal by diagonal; bound as the oracle's,
    with the terms that a wave adds up in a row: a register takes 64 elements of each tile, an LDS sum 15."""
    from distributed_tensorflow_amd.ops.relative_bias import relative_bias
    q_len, k_len, heads, buckets, far, bidir, start = cfg
    tiles = -(-q_len // 8) * -(-k_len // 512)
    per = tiles * heads // 8192
    assert per >= 2 and tiles % per
    g = torch.Generator(DEV).manual_seed(q_len)
    table = torch.randn(buckets, heads, device=DEV, generator=g).to(dt).requires_grad_()
    do = torch.randn(heads, q_len, k_len, device=DEV, generator=g).to(dt)
    first = k_len - q_len if start is None else start
    out = relative_bias(table, q_len, k_len, max_distance=far, bidirectional=bidir, q_start=start)
    got, = torch.autograd.grad(out, table, do)
    low = -(q_len - 1) - first
    of = O.buckets_between(low, k_len - 1 - first, buckets, far, bidir).to(DEV)
    assert torch.equal(out[0], table[:, 0][of].unfold(0, k_len, 1).flip(0))
    where = (torch.arange(k_len, device=DEV)[None] - torch.arange(q_len, device=DEV)[:, None] + (q_len - 1)).flatten()
    want, mag = (torch.zeros(buckets, heads, dtype=torch.float64, device=DEV) for _ in range(2))
    for h in range(heads):
        x = do[h].flatten().double()
        for w, y in ((want, x), (mag, x.abs())):
            diag = torch.zeros(q_len + k_len - 1, dtype=torch.float64, device=DEV).index_add_(0, where, y)
            w[:, h].index_add_(0, of, diag)
    tol = (64 * per + 4096) * O.U32 * mag + O.half_step(dt) * want.abs()
    O.check("dtable", got, want.cpu(), 1.01 * tol.cpu() + 1e-30)
    again, = torch.autograd.grad(relative_bias(table, q_len, k_len, max_distance=far, bidirectional=bidir, q_start=start), table, do)
    assert torch.equal(got, again)


@pytest.mark.parametrize("dt", [BF16, FP32], ids=["bf16", "fp32"])
def test_relative_bias_of_more_rows_than_a_grid(dt):
    from distributed_tensorflow_amd.ops.relative_bias import relative_bias
    q_len, k_len, heads, buckets = 140001, 37, 2, 32
    table = torch.randn(buckets, heads, generator=torch.Generator().manual_seed(1)).to(dt).to(DEV).requires_grad_()
    out = relative_bias(table, q_len, k_len, q_start=-70000)
    of = O.buckets_between(-(q_len - 1) + 70000, k_len - 1 + 70000, buckets, 128, True).to(DEV)
    for h in range(heads):
        assert torch.equal(out[h], table[:, h][of].unfold(0, k_len, 1).flip(0)), h
    # (a gradient of ones counts a bucket's elements: whole numbers below 2^24, summed exactly, rounded once)
    count = torch.bincount(of, torch.minimum(torch.minimum(torch.arange(1, q_len + k_len, device=DEV), torch.tensor(k_len, device=DEV)),
                                             torch.arange(q_len + k_len - 1, 0, -1, device=DEV)).double(), minlength=buckets)
    got, = torch.autograd.grad(out, table, torch.ones_like(out))
    assert torch.equal(got, count[:, None].expand(-1, heads).to(dt))


# ------------------------------------------------------------------------------------------ token log probabilities
@pytest.mark.parametrize("dt", [BF16, FP32], ids=["bf16", "fp32"])
def test_token_log_probs_of_subnormal_logits(dt):
    """Logits below the smallest normal number, of both signs: their order is that of the values all the same."""
    x, tok, g = _logits(6, 5003, dt)
    tiny = torch.finfo(dt).tiny
    x[0] = (torch.randn(5003, generator=g) * tiny / 8).to(dt)
    x[1] = -(torch.rand(5003, generator=g) * tiny / 8).to(dt)
    x[2, 100:] = -tiny / 4
    x[2, :100] = -tiny / 2
    gs = (torch.randn(6, generator=g), torch.randn(6, generator=g), torch.randn(6, 9, generator=g))
    _compare_logp(x, tok, 9, gs)


# ------------------------------------------------------------------------------------------ logits far from zero
@pytest.mark.parametrize("dt", [BF16, FP32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("N,V", [(9, 353), (9, 5003), (9, 30522), (600, 6001)])
def test_token_log_probs_of_logits_far_from_zero(dt, N, V):
    """What all logits of a row have in common leaves no trace: rows of nothing but the type's lowest value or its largest, rows
    far from zero either way, and rows masked to few by the lowest value."""
    x, tok, g = _logits(N, V, dt)
    x[0] = torch.finfo(dt).min
    x[1] = torch.finfo(dt).max
    for i, off in ((2, 3e4), (3, -3e4), (4, 1e6), (5, -1e20)):
        x[i] = (x[i].float() + off).to(dt)
    x[6] = torch.finfo(dt).min
    x[6, V // 2:V // 2 + 3] = x[2, :3]
    x[7] = torch.finfo(dt).min
    x[7, 5::7] = 1.0
    tok[6] = V // 2 + 1
    gs = (torch.randn(N, generator=g), torch.randn(N, generator=g), torch.randn(N, 9, generator=g))
    _compare_logp(x, tok, 9, gs)


# ------------------------------------------------------------------------------------------ offsets beyond 32 bits
def test_token_log_probs_beyond_32_bits():
    """70001 x 32000 logits: the last rows are those of a call on them alone."""
    from distributed_tensorflow_amd.ops.softmax_ce import token_log_probs
    N, V, n = 70001, 32000, 777
    x = torch.randn(N, V, dtype=BF16, device=DEV, generator=torch.Generator(DEV).manual_seed(1))
    tok = torch.randint(0, V, (N,), device=DEV)

    def run(x, tok):
        x = x.detach().requires_grad_()
        r = token_log_probs(x, tok, 3)
        d, = torch.autograd.grad((r.logp.sum(), r.entropy.sum(), r.top_logp.sum()), x)
        return [*r, d]

    assert all(torch.equal(a[-n:], b) for a, b in zip(run(x, tok), run(x[-n:].clone(), tok[-n:])))


def test_relative_bias_beyond_32_bits():
    from distributed_tensorflow_amd.ops.relative_bias import relative_bias
    q_len, k_len, heads, buckets = 12001, 11987, 16, 32
    table = torch.randn(buckets, heads, dtype=BF16, device=DEV, generator=torch.Generator(DEV).manual_seed(2)).requires_grad_()
    out = relative_bias(table, q_len, k_len)
    low = -(q_len - 1) - (k_len - q_len)
    of = O.buckets_between(low, q_len - 1, buckets, 128, True).to(DEV)
    assert torch.equal(out[-1], table[:, -1][of].unfold(0, k_len, 1).flip(0))
    # the gradient where only the last head's last rows count: those rows' elements, whole numbers, added exactly
    g = torch.zeros_like(out)
    g[-1, -5:] = 1
    got, = torch.autograd.grad(out, table, g)
    want = torch.zeros(buckets, heads, device=DEV)
    for i in range(q_len - 5, q_len):
        want[:, -1] += torch.bincount(of[q_len - 1 - i:q_len - 1 - i + k_len], minlength=buckets)
    assert torch.equal(got, want.to(BF16))


@pytest.mark.parametrize("fused", [False, True], ids=["separate", "fused"])
def test_attention_beyond_32_bits(fused):
    """41 x 8192 x 64 heads of 128, few keys: the last sequences are those of a call on them alone (the same kernel variants
    in the same order of sums)."""
    from distributed_tensorflow_amd.ops.attention import attention, self_attention
    B, S, nh, hd, n = (41, 8192, 64, 128, 6) if not fused else (700, 200, 64, 128, 90)
    g = torch.Generator(DEV).manual_seed(3)
    if fused:
        ins = [torch.randn(B, S, 3 * nh, hd, dtype=BF16, device=DEV, generator=g)]
    else:
        ins = [torch.randn(B, s, nh, hd, dtype=BF16, device=DEV, generator=g) for s in (S, 100, 100)]
    do = torch.randn(B, S, nh, hd, dtype=BF16, device=DEV, generator=g)
    lens = torch.randint(1, 100, (B,), device=DEV, dtype=torch.int32)
    assert ins[0].numel() > 1 << 31

    def run(ins, do, lens):
        ins = [t.detach().requires_grad_() for t in ins]
        out = self_attention(*ins, kv_heads=nh, key_lengths=lens) if fused else attention(*ins, key_lengths=lens)
        return [out, *torch.autograd.grad(out, ins, do)]

    whole = run(ins, do, lens)
    part = run([t[-n:].clone() for t in ins], do[-n:].clone(), lens[-n:].clone())
    assert all(torch.equal(a[-n:], b) for a, b in zip(whole, part))
