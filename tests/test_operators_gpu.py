"""General attention, relative position bias and token log probabilities on the GPU against the 64-bit oracles, whose
bounds are derived in operator_oracles.py."""
import math
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.dirname(__file__))
import operator_oracles as O  # noqa: E402
from distributed_tensorflow_amd.engine.graph import collected  # noqa: E402

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16, FP32 = torch.bfloat16, torch.float32


def _inputs(B, Sq, Sk, nh, nkv, hd, dt, buckets=0, seed=0):
    g = torch.Generator().manual_seed(seed + 7919 * Sq + 31 * Sk + hd)
    q, k, v, do = (torch.randn(B, s, n, hd, generator=g).to(dt) for s, n in ((Sq, nh), (Sk, nkv), (Sk, nkv), (Sq, nh)))
    table = torch.randn(buckets, nh, generator=g).to(dt) if buckets else None
    return q, k, v, do, table


def _dev(x):
    return x.to(DEV) if isinstance(x, torch.Tensor) else x


def _compare(q, k, v, do, table=None, **kw):
    from distributed_tensorflow_amd.ops.attention import attention
    val, tol = O.attention(q, k, v, do, rel_table=table, **kw)
    leaves = [t.to(DEV).requires_grad_() for t in (q, k, v)]
    tab = None if table is None else table.to(DEV).requires_grad_()
    out = attention(*leaves, rel_table=tab, **{n: _dev(x) for n, x in kw.items()})
    got = torch.autograd.grad(out, leaves + ([tab] if tab is not None else []), do.to(DEV))
    O.check("out", out, val["out"], tol["out"])
    for n, t in zip(("dq", "dk", "dv", "dtable"), got):
        O.check(n, t, val[n], tol[n])
    return out, got


SHAPES = [  # B, Sq, Sk, nh, nkv, hd
    (1, 1, 1, 1, 1, 8), (2, 1, 37, 4, 2, 64), (1, 33, 1, 2, 2, 40), (2, 31, 65, 2, 1, 16), (1, 64, 64, 2, 2, 32),
    (2, 65, 63, 3, 3, 72), (1, 127, 129, 4, 1, 64), (1, 130, 257, 2, 2, 128), (1, 200, 140, 6, 2, 96), (3, 128, 128, 1, 1, 64),
    (1, 5, 300, 8, 2, 128), (1, 300, 5, 2, 2, 80),
]


@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("dt", [BF16, FP32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("causal", [False, True], ids=["full", "causal"])
def test_attention_shapes(shape, dt, causal):
    q, k, v, do, _ = _inputs(*shape, dt)
    _compare(q, k, v, do, causal=causal)


@pytest.mark.parametrize("dt", [BF16, FP32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("causal", [False, True], ids=["full", "causal"])
@pytest.mark.parametrize("mask", ["lengths", "bias", "both"])
def test_attention_masks_with_empty_rows_and_garbage_behind_them(dt, causal, mask):
    B, S, nh, nkv, hd = 4, 150, 4, 2, 64
    q, k, v, do, _ = _inputs(B, S, S, nh, nkv, hd, dt, seed=3)
    kw = {}
    if mask != "bias":
        kw["key_lengths"] = torch.tensor([0, 1, 150, 77], dtype=torch.int32)
        for b, n in enumerate(kw["key_lengths"].tolist()):
            k[b, n:] = math.nan
            v[b, n:] = math.inf
    if mask != "lengths":
        kb = torch.randn(B, S)
        kb[1, 40:] = -math.inf
        kb[2, ::3] = -math.inf
        kb[3] = -math.inf
        kw["key_bias"] = kb
        k[2, ::3] = math.nan
        v[2, ::3] = math.nan
    out, got = _compare(q, k, v, do, causal=causal, **kw)
    if mask != "bias":
        assert not out[0].any() and not got[0][0].any() and not got[1][0].any()


@pytest.mark.parametrize("dt", [BF16, FP32], ids=["bf16", "fp32"])
def test_attention_lowest_value_masks(dt):
    """A bias of the type's lowest value masks a key next to others, and cancels out where every key has it."""
    B, S, nh, hd = 2, 70, 2, 64
    q, k, v, do, _ = _inputs(B, S, S, nh, nh, hd, dt, seed=4)
    kb = torch.zeros(B, S)
    kb[0, 30:] = torch.finfo(FP32).min
    kb[1] = torch.finfo(FP32).min
    # (rows of equal huge biases: the scores are absorbed, the probabilities uniform, and so are they in the oracle)
    _compare(q, k, v, do, key_bias=kb)


@pytest.mark.parametrize("dt", [BF16, FP32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("cfg", [(32, 128, None), (8, 5, True), (16, 300, False), (128, 2048, True), (2, 3, False)], ids=str)
@pytest.mark.parametrize("shape", [(2, 150, 150, 3, 3, 64), (1, 40, 333, 4, 2, 32), (1, 330, 90, 2, 1, 128), (3, 1, 200, 2, 2, 64)], ids=str)
@pytest.mark.parametrize("causal", [False, True], ids=["full", "causal"])
def test_attention_relative_bias(dt, cfg, shape, causal):
    buckets, far, bidir = cfg
    if bidir is None:
        bidir = not causal
    q, k, v, do, table = _inputs(*shape, dt, buckets)
    _compare(q, k, v, do, table, causal=causal, rel_max_distance=far, rel_bidirectional=bidir)


def test_attention_relative_bias_with_masks_and_per_sequence_starts():
    B, Sq, Sk, nh, nkv, hd = 3, 70, 210, 4, 2, 64
    q, k, v, do, table = _inputs(B, Sq, Sk, nh, nkv, hd, BF16, 32)
    kb = torch.randn(B, Sk)
    kb[:, 100:103] = -math.inf
    _compare(q, k, v, do, table, causal=True, key_bias=kb, key_lengths=torch.tensor([210, 130, 5]),
             q_start=torch.tensor([140, 60, -65]))


@pytest.mark.parametrize("dt", [BF16, FP32], ids=["bf16", "fp32"])
def test_attention_few_queries_over_a_long_cache(dt):
    B, Sq, Sk, nh, nkv, hd = 3, 2, 5003, 8, 2, 128
    q, k, v, do, table = _inputs(B, Sq, Sk, nh, nkv, hd, dt, 32)
    n = torch.tensor([5003, 2, 1700], dtype=torch.int32)
    _compare(q, k, v, do, table, causal=True, key_lengths=n, q_start=n - Sq)
    _compare(q[:, :1], k, v, do[:, :1], causal=True, key_lengths=n, q_start=n - 1)


def test_attention_reads_views_in_place_and_copies_what_it_cannot():
    from distributed_tensorflow_amd.ops.attention import attention, self_attention
    B, S, nh, nkv, hd = 2, 75, 4, 2, 64
    g = torch.Generator().manual_seed(1)
    qkv = torch.randn(B, S, nh + 2 * nkv, hd, generator=g).to(BF16).to(DEV)
    do = torch.randn(B, S, nh, hd, generator=g).to(BF16).to(DEV)
    q, k, v = qkv.split((nh, nkv, nkv), 2)
    want = attention(q.contiguous(), k.contiguous(), v.contiguous(), causal=True)
    assert torch.equal(attention(q, k, v, causal=True), want)
    assert torch.equal(self_attention(qkv, kv_heads=nkv, causal=True), want)
    odd = torch.empty(B * S * nh * hd + 1, dtype=BF16, device=DEV)[1:].view(B, S, nh, hd).copy_(q)   # 2-byte aligned
    assert torch.equal(attention(odd, k, v, causal=True), want)
    heads_first = q.transpose(1, 2).contiguous().transpose(1, 2)
    assert torch.equal(attention(heads_first, k, v, causal=True), want)
    one = k[:1, :, :1].expand(B, S, nkv, hd)                         # stride 0 over the batch and the heads
    assert torch.equal(attention(q, one, v, causal=True), attention(q, one.contiguous(), v, causal=True))
    same = k[:, :1].expand(B, S, nkv, hd)                            # stride 0 over the tokens: copied
    assert torch.equal(attention(q, same, v), attention(q, same.contiguous(), v))
    wide = torch.zeros(B, S, nh, 2 * hd, dtype=BF16, device=DEV)
    wide[..., ::2] = q                                               # no unit stride
    assert torch.equal(attention(wide[..., ::2], k, v, causal=True), want)
    # gradients through the views arrive where they belong
    x = qkv.clone().requires_grad_()
    gx, = torch.autograd.grad(self_attention(x, kv_heads=nkv, causal=True), x, do)
    leaves = [t.contiguous().requires_grad_() for t in (q, k, v)]
    gs = torch.autograd.grad(attention(*leaves, causal=True), leaves, do.transpose(1, 2).contiguous().transpose(1, 2))
    assert torch.equal(gx, torch.cat(gs, 2))
    y = qkv[:, :, : 3 * nkv].reshape(B, S, 3, nkv, hd)
    a = self_attention(y, causal=True)
    assert torch.equal(a, attention(y[:, :, 0], y[:, :, 1], y[:, :, 2], causal=True))


def test_attention_without_keys_or_queries():
    from distributed_tensorflow_amd.ops.attention import attention
    for Sq, Sk in ((0, 5), (5, 0), (0, 0)):
        q, k, v = (torch.randn(2, s, 2, 64, device=DEV, dtype=BF16).requires_grad_() for s in (Sq, Sk, Sk))
        t = torch.randn(8, 2, device=DEV, dtype=BF16).requires_grad_()
        out = attention(q, k, v, rel_table=t)
        assert out.shape == q.shape and not out.any()
        for x in torch.autograd.grad(out, (q, k, v, t), torch.randn_like(out)):
            assert not x.any()


def test_attention_is_the_same_every_time():
    q, k, v, do, table = (t.to(DEV) for t in _inputs(2, 700, 700, 4, 2, 64, BF16, 32))
    from distributed_tensorflow_amd.ops.attention import attention
    runs = []
    for _ in range(3):
        leaves = [t.clone().requires_grad_() for t in (q, k, v, table)]
        out = attention(*leaves[:3], rel_table=leaves[3])
        runs.append([out, *torch.autograd.grad(out, leaves, do)])
    for r in runs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(r, runs[0]))


def test_attention_gradient_agrees_with_differences():
    """(f(x + h d) - f(x - h d)) / 2h of the fp32 kernels against their gradient, f = sum(out * w). What the quotient is
    off by for h itself is taken from the oracle in 64 bits; the kernels' own error adds bound(f) / h."""
    from distributed_tensorflow_amd.ops.attention import attention
    q, k, v, w, table = _inputs(1, 40, 60, 2, 1, 32, FP32, 16)
    ins, h = (q, k, v, table), 2.0 ** -7
    leaves = [t.to(DEV).requires_grad_() for t in ins]
    out = attention(*leaves[:3], rel_table=leaves[3], causal=True)
    grads = torch.autograd.grad(out, leaves, w.to(DEV))
    for n, (t, g) in enumerate(zip(ins, grads)):
        d = torch.randn(t.shape, generator=torch.Generator().manual_seed(n))
        f, exact, err = [], [], 0.0
        for s in (1, -1):
            moved = [x + s * h * d if i == n else x for i, x in enumerate(ins)]
            o = attention(*(x.to(DEV) for x in moved[:3]), rel_table=moved[3].to(DEV), causal=True)
            val, tol = O.attention(*moved[:3], rel_table=moved[3], causal=True)
            f.append(float((o.double().cpu() * w).sum()))
            exact.append(float((val["out"] * w).sum()))
            err += float((tol["out"] * w.abs()).sum())
        val, tol = O.attention(q, k, v, w, rel_table=table, causal=True)
        name = ("dq", "dk", "dv", "dtable")[n]
        slope = float((val[name] * d).sum())
        off = abs((exact[0] - exact[1]) / (2 * h) - slope)
        got = float((g.double().cpu() * d).sum())
        assert abs((f[0] - f[1]) / (2 * h) - got) <= off + err / (2 * h) + float((tol[name] * d.abs()).sum())


def test_attention_on_another_stream_and_in_a_graph():
    from distributed_tensorflow_amd.ops.attention import attention
    q, k, v, do, table = (t.to(DEV) for t in _inputs(2, 140, 140, 2, 2, 64, BF16, 32))

    def run(leaves):
        out = attention(*leaves[:3], rel_table=leaves[3], causal=True)
        return [out, *torch.autograd.grad(out, leaves, do)]

    want = run([t.clone().requires_grad_() for t in (q, k, v, table)])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    leaves = [t.clone().requires_grad_() for t in (q, k, v, table)]
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            got = run(leaves)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    del got
    g = torch.cuda.CUDAGraph()
    with collected(), torch.cuda.graph(g):
        outs = run(leaves)
    for i in range(4):
        with torch.no_grad():
            leaves[0].copy_(q * (i + 1) * 0.5)
        g.replay()
        torch.cuda.synchronize()
        new = run([leaves[0].detach().clone().requires_grad_(), *[t.clone().requires_grad_() for t in (k, v, table)]])
        assert all(torch.equal(a, b) for a, b in zip(outs, new)), i


@pytest.mark.parametrize("Sq,masked", [(40, False), (40, True), (7, False)], ids=["rows", "key_bias", "few"])
def test_table_gradient_of_bf16_attention_is_finer_than_bf16(Sq, masked):
    """An fp32 table beside bf16 q, k, v. Nothing that a row's dT = P (dP - D) is made of may be rounded to 8 bits: P enters
    O in two parts of 8 bits and D reads O to 16. Bound: D off by 2^-17 of sum P |dP| and of sum |dO O| each, doubled; P and
    dP by fp32 roundings, 64 + 64 terms of 2^-24 and an exponent of up to 16, below 2^-17."""
    from distributed_tensorflow_amd.ops.attention import attention
    Sk, nh, hd, buckets = 90, 3, 64, 8
    q, k, v, do, table = _inputs(1, Sq, Sk, nh, nh, hd, BF16, buckets)
    table = 0.5 * table.float()
    bias = torch.where(torch.arange(Sk) % 9 == 0, -1.0, 0.0)[None] if masked else None
    d = torch.arange(Sk)[None, :] - (torch.arange(Sq)[:, None] + Sk - Sq)
    of = O.buckets_between(int(d.min()), int(d.max()), buckets, 30, True)[d - int(d.min())]
    want, tol = torch.zeros(buckets, nh, dtype=torch.float64), torch.zeros(buckets, nh, dtype=torch.float64)
    for h in range(nh):
        qq, kk, vv, dd = (t[0, :, h].double() for t in (q, k, v, do))
        t = qq @ kk.t() / math.sqrt(hd) + table[:, h].double()[of] + (bias.double() if masked else 0.0)
        p = torch.softmax(t, 1)
        dp, o = dd @ vv.t(), p @ vv
        D = (dd * o).sum(1, keepdim=True)
        off = 2.0 ** -16 * ((p * dp.abs()).sum(1, keepdim=True) + (dd * o).abs().sum(1, keepdim=True))
        mag = dd.abs() @ vv.abs().t() + D.abs()
        for u in range(buckets):
            want[u, h] = (p * (dp - D))[of == u].sum()
            tol[u, h] = (p * (off + 2.0 ** -17 * mag))[of == u].sum() + 1e-30       # (0 in a bucket with no distance)
    leaf = table.to(DEV).requires_grad_()
    out = attention(q.to(DEV), k.to(DEV), v.to(DEV), _dev(bias), rel_table=leaf, rel_max_distance=30)
    got, = torch.autograd.grad(out, leaf, do.to(DEV))
    O.check("dtable", got, want, tol)


@pytest.mark.parametrize("dt", [BF16, FP32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("hd", [24, 64, 88, 128])
@pytest.mark.parametrize("mode", ["plain", "causal_table", "key_bias"])
def test_attention_of_more_workgroups_than_cus(dt, hd, mode):
    """Grids beyond which a workgroup's waves walk the tiles together, over more than four tiles."""
    B, Sq, Sk, nh, nkv = 8, 270, 390, 12, 12
    q, k, v, do, table = _inputs(B, Sq, Sk, nh, nkv, hd, dt, 16)
    if mode == "plain":
        _compare(q, k, v, do, key_lengths=torch.tensor([390, 0, 389, 257, 64, 1, 300, 128]))
    elif mode == "causal_table":
        _compare(q, k, v, do, table, causal=True, rel_max_distance=40)
    else:
        bias = torch.randn(B, Sk, generator=torch.Generator().manual_seed(1))
        bias[1], bias[2, 200:], bias[3, ::3] = -math.inf, -math.inf, -math.inf
        _compare(q, k, v, do, table, key_bias=bias, rel_max_distance=300)


def test_attention_over_a_cache_that_passes_32_bits():
    """Rows 2^22 elements apart (the widest that are read in place): the last ones lie 5 GB behind the first."""
    from distributed_tensorflow_amd.ops.attention import attention
    Sk, row = 650, 1 << 22
    buf = torch.empty(Sk * row, dtype=BF16, device=DEV)
    kv = buf.as_strided((1, Sk, 4, 64), (Sk * row, row, 64, 1))
    kv.copy_(torch.randn(1, Sk, 4, 64, generator=torch.Generator().manual_seed(3)).to(BF16))
    for Sq in (1, 70):
        q, _, _, do, _ = (None if t is None else t.to(DEV) for t in _inputs(1, Sq, Sk, 4, 2, 64, BF16))

        def run(kv):
            leaves = [t.requires_grad_() for t in (q.clone(), kv[:, :, :2].detach(), kv[:, :, 2:].detach())]
            out = attention(*leaves, causal=True)
            return [out, *torch.autograd.grad(out, leaves, do)]

        assert all(torch.equal(a, b) for a, b in zip(run(kv), run(kv.contiguous())))


@pytest.mark.parametrize("how", ["offload", "checkpoint"])
def test_gradients_with_saved_tensors_moved(how):
    """Hooks put what the backward pass needs elsewhere (the forward's own copies are freed), or it is computed anew."""
    from torch.utils.checkpoint import checkpoint
    from distributed_tensorflow_amd.ops.attention import attention, self_attention
    from distributed_tensorflow_amd.ops.relative_bias import relative_bias
    from distributed_tensorflow_amd.ops.softmax_ce import token_log_probs
    q, k, v, do, table = (t.to(DEV) for t in _inputs(2, 130, 130, 4, 2, 64, BF16, 32))
    bias = torch.zeros(2, 130, device=DEV)
    bias[0, 100:] = -math.inf
    lens = torch.tensor([130, 90], device=DEV)
    tok = torch.arange(260, device=DEV)

    def step(q, k, v, table):
        wide = torch.cat((q, k, v), 2) * 1.5                       # (only the graph holds these)
        a = attention(q * 2, k * 2, v * 2, bias * 1, rel_table=table * 2, causal=True)
        b = self_attention(wide, kv_heads=2, key_lengths=lens + 0, rel_table=table * 3)
        r = token_log_probs((a + b).reshape(260, 256)[:, :250] * 1, tok, 3)
        w = relative_bias(table * 2, 130, 130)
        return (a * do).float().sum() + (b * do).float().sum() + r.logp.sum() + r.top_logp.sum() + r.entropy.sum() + w.float().sum()

    def grads(run):
        leaves = [t.clone().requires_grad_() for t in (q, k, v, table)]
        loss = run(leaves)
        junk = [torch.full((1 << n,), math.nan, device=DEV) for n in range(8, 22)]       # over whatever was freed
        return torch.autograd.grad(loss, leaves), junk

    def moved(leaves):
        if how == "checkpoint":
            return checkpoint(step, *leaves, use_reentrant=False)
        with torch.autograd.graph.save_on_cpu():
            return step(*leaves)

    want, got = grads(lambda leaves: step(*leaves))[0], grads(moved)[0]
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_attention_of_no_sequences_and_of_lengths_beyond_32_bits():
    from distributed_tensorflow_amd.ops.attention import attention
    for B, Sq in ((0, 1), (0, 200), (2, 0)):
        q, k, v, do, _ = (None if t is None else t.to(DEV) for t in _inputs(B, Sq, 400, 4, 2, 64, BF16))
        leaves = [t.requires_grad_() for t in (q, k, v)]
        out = attention(*leaves, causal=True)
        assert out.shape == (B, Sq, 4, 64)
        assert all(float(g.abs().sum()) == 0 for g in torch.autograd.grad(out, leaves, do))
        assert attention(q.detach(), k.detach(), v.detach()).shape == out.shape
    q, k, v, _, _ = (None if t is None else t.to(DEV) for t in _inputs(3, 70, 90, 2, 2, 64, FP32))
    far = torch.tensor([1 << 40, -(1 << 33), (1 << 32) + 5], device=DEV)
    assert torch.equal(attention(q, k, v, key_lengths=far), attention(q, k, v, key_lengths=far.clamp(0, 90).int()))
    assert torch.equal(attention(q, k, v, q_start=far, causal=True), attention(q, k, v, q_start=far.clamp(-200, 200), causal=True))


# ------------------------------------------------------------------------------------------------ relative bias
@pytest.mark.parametrize("dt", [BF16, FP32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("cfg", [(1, 1, 3, 32, 128, True), (70, 70, 2, 32, 128, True), (129, 300, 3, 16, 50, False),
                                 (300, 129, 1, 8, 8, True), (1, 1000, 4, 32, 128, False), (515, 517, 2, 128, 2048, True),
                                 (33, 65, 2, 2, 3, False), (64, 2500, 1, 64, 200, True)], ids=str)
@pytest.mark.parametrize("q_start", [None, 0, 400, -700])
def test_relative_bias(dt, cfg, q_start):
    from distributed_tensorflow_amd.ops.relative_bias import relative_bias
    q_len, k_len, heads, buckets, far, bidir = cfg
    g = torch.Generator().manual_seed(q_len + buckets)
    table, do = torch.randn(buckets, heads, generator=g).to(dt), torch.randn(heads, q_len, k_len, generator=g).to(dt)
    start = k_len - q_len if q_start is None else q_start
    bias, d, tol = O.relative_bias(table, q_len, k_len, far, bidir, start, do)
    t = table.to(DEV).requires_grad_()
    out = relative_bias(t, q_len, k_len, max_distance=far, bidirectional=bidir, q_start=q_start)
    assert torch.equal(out.cpu(), bias)
    got, = torch.autograd.grad(out, t, do.to(DEV))
    O.check("dtable", got, d, tol)
    again, = torch.autograd.grad(relative_bias(t, q_len, k_len, max_distance=far, bidirectional=bidir, q_start=q_start), t,
                                 do.to(DEV).transpose(1, 2).contiguous().transpose(1, 2))
    assert torch.equal(got, again)


@pytest.mark.parametrize("dt", [BF16, FP32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("q_len,k_len", [(4003, 5001), (2999, 7003)])
def test_relative_bias_larger_than_the_caches(dt, q_len, k_len):
    """Every row at another alignment, most of it beyond the band: the values of the table at the oracle's buckets."""
    from distributed_tensorflow_amd.ops.relative_bias import relative_bias
    heads, buckets = 11, 32
    table = torch.randn(buckets, heads, generator=torch.Generator().manual_seed(5)).to(dt).to(DEV)
    bias = relative_bias(table, q_len, k_len, q_start=700)
    low = -(q_len - 1) - 700
    of = O.buckets_between(low, k_len - 1 - 700, buckets, 128, True).to(DEV)
    for h in range(heads):
        assert torch.equal(bias[h], table[:, h][of].unfold(0, k_len, 1).flip(0)), h


def test_attention_adds_the_bias_that_relative_bias_writes():
    """Both entry points read a table the same way: key biases made of its rows for one query."""
    from distributed_tensorflow_amd.ops.attention import attention
    from distributed_tensorflow_amd.ops.relative_bias import relative_bias
    q, k, v, _, table = (t.to(DEV) for t in _inputs(1, 1, 300, 1, 1, 64, FP32, 32))
    bias = relative_bias(table, 1, 300, q_start=120)
    a = attention(q, k, v, rel_table=table, q_start=120)
    b = attention(q, k, v, key_bias=bias[0])
    # the two add the same numbers in another order: one rounding of the score more
    assert float((a - b).abs().max()) <= 64 * O.U32 * float(v.abs().max())


# ------------------------------------------------------------------------------------------------ token log probabilities
def _logits(N, V, dt, seed=0):
    g = torch.Generator().manual_seed(seed + N + V)
    x = (2 * torch.randn(N, V, generator=g)).to(dt)
    tok = torch.randint(0, V, (N,), generator=g)
    return x, tok, g


def _compare_logp(x, tok, top, gs=None, device_x=None):
    from distributed_tensorflow_amd.ops.softmax_ce import token_log_probs
    val, tol, ids = O.token_log_probs(x, tok, top, gs)
    leaf = x.to(DEV) if device_x is None else device_x
    leaf = leaf.requires_grad_()
    r = token_log_probs(leaf, tok.to(DEV), top)
    assert torch.equal(r.top_ids.cpu(), ids)
    for n in ("logp", "entropy", "top_logp"):
        O.check(n, getattr(r, n), val[n], tol[n])
    if gs is not None:
        n = 3 if top else 2
        d, = torch.autograd.grad((r.logp, r.entropy, r.top_logp)[:n], leaf, [t.to(DEV) for t in gs[:n]])
        O.check("dlogits", d, val["dlogits"], tol["dlogits"])
        return d


@pytest.mark.parametrize("dt", [BF16, FP32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("N,V,top", [(1, 1, 1), (3, 2, 0), (5, 33, 32), (7, 64, 20), (4, 1000, 5), (9, 4099, 32), (3, 8192, 10),
                                     (2, 8193, 10), (5, 30522, 10), (2, 40001, 32), (2, 131072, 20), (3, 100003, 1)])
def test_token_log_probs(dt, N, V, top):
    x, tok, g = _logits(N, V, dt)
    if N > 2:
        tok[1], tok[2] = -1, V
    gs = (torch.randn(N, generator=g), torch.randn(N, generator=g), torch.randn(N, top, generator=g))
    _compare_logp(x, tok, top, gs)
    _compare_logp(x, tok.int(), top)


@pytest.mark.parametrize("dt", [BF16, FP32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("V", [50, 30522, 70001])
def test_token_log_probs_of_degenerate_rows(dt, V):
    """Equal logits, sorted ones either way, one finite logit, none, sure rows, +-0, and all but a few masked: the number
    of candidates for the top is anything from none to the whole row."""
    x = torch.zeros(9, V)
    x[1] = torch.arange(V) / V
    x[2] = -torch.arange(V) / V
    x[3, :-1] = -math.inf
    x[4] = -math.inf
    x[5, V // 2] = 60.0
    x[6, ::2] = -0.0
    x[7] = -math.inf
    x[7, 5::7] = 1.0
    x[8, V // 3:V // 3 + 40] = torch.arange(40.0)[: min(40, V - V // 3)]
    tok = torch.tensor([0, V - 1, 0, V - 1, 3, V // 2, 1, 0, V // 3])
    gs = tuple(torch.ones(s) for s in ((9,), (9,), (9, 20)))
    _compare_logp(x.to(dt), tok, 20, gs)


@pytest.mark.parametrize("dt", [BF16, FP32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("N,V,top", [(600, 4097, 5), (513, 9001, 32), (2000, 1000, 20), (700, 300, 32)])
def test_token_log_probs_of_many_rows(dt, N, V, top):
    """As many rows as give each fewer threads; every seventh row is constant, every eleventh sorted, some masked to few."""
    x, tok, g = _logits(N, V, dt)
    x[::7] = 1.5
    x[3::11] = (torch.arange(V) / V - 0.5).to(dt)
    x[5::13, 40:] = -math.inf
    x[6::13, : V - 9] = torch.finfo(dt).min
    tok[9] = -1
    tok[5::13] = 3
    tok[6::13] = V - 1
    gs = (torch.randn(N, generator=g), torch.randn(N, generator=g), torch.randn(N, top, generator=g))
    _compare_logp(x, tok, top, gs)


def test_token_log_probs_with_nan_and_infinity():
    from distributed_tensorflow_amd.ops.softmax_ce import token_log_probs
    x = torch.randn(3, 30000)
    x[0, 17], x[0, 29000], x[1, 5] = math.nan, math.nan, math.inf
    r = token_log_probs(x.to(DEV), torch.tensor([1, 2, 3], device=DEV), 3)
    assert torch.isnan(r.logp[:2]).all() and torch.isnan(r.entropy[:2]).all() and torch.isfinite(r.logp[2])
    assert r.top_ids[0, :2].tolist() == [17, 29000] and int(r.top_ids[1, 0]) == 5       # NaN counts as the largest
    assert r.top_ids[2].tolist() == torch.sort(x[2], descending=True, stable=True).indices[:3].tolist()


@pytest.mark.parametrize("dt", [BF16, FP32], ids=["bf16", "fp32"])
def test_token_log_probs_of_padded_and_misaligned_rows(dt):
    x, tok, g = _logits(6, 1003, dt)
    gs = (torch.randn(6, generator=g), torch.randn(6, generator=g), torch.randn(6, 4, generator=g))
    want = _compare_logp(x, tok, 4, gs)
    ld = 1008
    wide = torch.full((6, ld), 7.0, dtype=dt, device=DEV)
    wide[:, :1003] = x.to(DEV)
    assert torch.equal(_compare_logp(x, tok, 4, gs, wide[:, :1003].detach()), want)
    flat = torch.empty(6 * 1003 + 1, dtype=dt, device=DEV)
    moved = flat[1:].view(6, 1003)
    moved.copy_(x)
    _compare_logp(x, tok, 4, gs, moved.detach())
    _compare_logp(x, tok, 4, gs, x.to(DEV).t().contiguous().t().detach())


def test_token_log_probs_keeps_leading_axes_and_single_gradients():
    from distributed_tensorflow_amd.ops.softmax_ce import softmax_cross_entropy, token_log_probs
    x, tok, _ = _logits(24, 999, FP32)
    leaf = x.to(DEV).view(2, 3, 4, 999).requires_grad_()
    r = token_log_probs(leaf, tok.to(DEV).view(2, 3, 4), 2)
    assert r.logp.shape == (2, 3, 4) and r.top_ids.shape == (2, 3, 4, 2)
    # -logp is the loss that trains: same gradient as softmax_cross_entropy's, to the two kernels' roundings
    a, = torch.autograd.grad(-r.logp.sum(), leaf, retain_graph=True)
    other = leaf.detach().view(24, 999).requires_grad_()
    b, = torch.autograd.grad(softmax_cross_entropy(other, tok.to(DEV), "sum"), other)
    assert float((a.view(24, 999) - b).abs().max()) <= 2.0 ** -19
    c, = torch.autograd.grad(r.entropy.sum(), leaf, retain_graph=True)
    assert float(c.sum(-1).abs().max()) <= 1e-4          # moving every logit alike moves no probability
    d, = torch.autograd.grad(r.top_logp[..., 0].sum(), leaf)
    assert float(d.sum(-1).abs().max()) <= 1e-4
    empty = token_log_probs(torch.empty(0, 10, device=DEV), torch.empty(0, dtype=torch.long, device=DEV), 3)
    assert empty.logp.shape == (0,) and empty.top_ids.shape == (0, 3)


def test_token_log_probs_in_a_graph():
    from distributed_tensorflow_amd.ops.softmax_ce import token_log_probs
    x, tok, _ = _logits(40, 30522, BF16)
    leaf, t = x.to(DEV).requires_grad_(), tok.to(DEV)

    def run(v):
        r = token_log_probs(v, t, 5)
        return [*r, torch.autograd.grad((r.logp.sum(), r.entropy.sum()), v)[0]]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run(leaf)
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with collected(), torch.cuda.graph(g):
        outs = run(leaf)
    for i in range(4):
        with torch.no_grad():
            leaf.copy_(torch.roll(x, i, 1))
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, run(leaf.detach().clone().requires_grad_()))), i


# ------------------------------------------------------------------------------------------------ large grids, head splits
@pytest.mark.parametrize("dt", [BF16, FP32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("cfg", [(40, 260, 260, 32, 32, 8, False), (66, 300, 129, 16, 4, 16, True), (260, 33, 300, 8, 8, 24, False)], ids=str)
@pytest.mark.parametrize("rel", [0, 16])
def test_attention_with_a_grid_that_fills_the_chip(dt, cfg, rel):
    """Small grids run workgroups of two halves; these run the single ones over several tiles. Two distinct sequences,
    repeated: every copy is bitwise the same (the table's gradient aside, which sums them), and right."""
    from distributed_tensorflow_amd.ops.attention import attention
    B, Sq, Sk, nh, nkv, hd, causal = cfg
    q, k, v, do, table = _inputs(2, Sq, Sk, nh, nkv, hd, dt, rel, seed=9)
    val, tol = O.attention(q, k, v, do, causal=causal, rel_table=table, rel_max_distance=40)
    big = [t.to(DEV).repeat(B // 2, 1, 1, 1).requires_grad_() for t in (q, k, v)]
    tab = None if table is None else table.to(DEV).requires_grad_()
    out = attention(*big, causal=causal, rel_table=tab, rel_max_distance=40)
    got = torch.autograd.grad(out, big + ([tab] if rel else []), do.to(DEV).repeat(B // 2, 1, 1, 1))
    for n, t in zip(("out", "dq", "dk", "dv"), (out, *got)):
        assert torch.equal(t, t[:2].repeat(B // 2, 1, 1, 1)), n
        O.check(n, t[:2], val[n], tol[n])
    if rel:                                   # (B / 2 times the sums; the bound's own rounding is already one of the result)
        O.check("dtable", got[3], val["dtable"] * (B // 2), tol["dtable"] * (B // 2))


@pytest.mark.parametrize("shape", [(1, 300, 300, 8, 1, 64), (1, 200, 333, 12, 2, 128), (2, 140, 140, 6, 2, 32)], ids=str)
@pytest.mark.parametrize("causal", [False, True], ids=["full", "causal"])
def test_attention_sums_shared_heads_over_splits(shape, causal):
    """Many query heads to a key head and few key heads: dK and dV are summed in parts and joined."""
    q, k, v, do, table = _inputs(*shape, BF16, 16, seed=5)
    _compare(q, k, v, do, table, causal=causal, rel_max_distance=60)


# ------------------------------------------------------------------------------------------------ together, in the model
def _tiny(device, dtype, seed=0):
    from distributed_tensorflow_amd.models.bert import bert_tiny
    torch.manual_seed(seed)
    return bert_tiny(seq_len=77, vocab=1000, rel_buckets=16, rel_max_distance=50).to(device=device, dtype=dtype)


def test_bert_with_relative_positions_matches_the_cpu_model():
    """The fp32 model on the GPU (general attention with the relative bias and padded batches, scoring) against the same
    weights on the CPU in fp32: two layers of sums of at most 1024 terms, both sides off by at most some 1024 * 2^-24 of
    the largest magnitude each."""
    from distributed_tensorflow_amd.models.bert import synthetic_mlm_batch
    x, y = synthetic_mlm_batch(3, 77, 1000, "cpu", n_pred=9)
    n = torch.tensor([77, 40, 1], dtype=torch.int32)
    res = []
    for dev in ("cpu", DEV):
        m = _tiny("cpu", FP32).to(dev)
        logits = m(x.to(dev), logits=True, key_lengths=n.to(dev))
        (logits.float().logsumexp(1).sum() - logits[torch.arange(27), y].sum()).backward()
        s = m.score(x.to(dev), y.to(dev), 5, key_lengths=n.to(dev))
        res.append((logits, m.rel.grad, m.layers[0].qkv.weight.grad, m.word.grad, s.logp, s.entropy, s.top_logp))
    for a, b in zip(*res):
        a, b = a.detach(), b.detach().cpu()
        assert float((a - b).abs().max()) <= 2 * 1024 * O.U32 * 8 * float(a.abs().max())


def test_bert_with_relative_positions_trains_in_bf16_and_in_a_graph():
    """Training steps of the strategy, eager and captured: the same losses and weights to the bit, finite, and the table
    moves."""
    from distributed_tensorflow_amd.comm.backend import Comm
    from distributed_tensorflow_amd.engine.optimizer import Adam
    from distributed_tensorflow_amd.engine.replica import TrainConfig
    from distributed_tensorflow_amd.models.bert import synthetic_mlm_batch
    from distributed_tensorflow_amd.parallel.mirrored import MirroredStrategy
    x, y = synthetic_mlm_batch(6, 77, 1000, DEV, n_pred=9)
    runs = []
    for graph in (False, True):
        cfg = TrainConfig(loss="mlm", param_dtype=BF16, grad_dtype=BF16, graph=graph)
        st = MirroredStrategy(_tiny("cpu", FP32), Comm(0, 1, torch.device(DEV)), cfg, optimizer=Adam(1e-3))
        before = st.replica.model.rel.detach().clone()
        step = st.step_callable() if graph else st.train_step
        losses = [float(step(x, y)) for _ in range(10)]
        assert all(math.isfinite(v) for v in losses) and not torch.equal(before, st.replica.model.rel)
        runs.append((losses, st.flat.master.clone()))
    assert runs[0][0] == pytest.approx(runs[1][0], rel=1e-6)
    assert torch.equal(runs[0][1], runs[1][1])


def test_operators_in_two_graphs_and_on_two_streams_at_once():
    """Two captured passes that are replayed in turn and two streams at a time: no call shares a workspace with another."""
    from distributed_tensorflow_amd.ops.attention import attention
    from distributed_tensorflow_amd.ops.relative_bias import relative_bias
    from distributed_tensorflow_amd.ops.softmax_ce import token_log_probs

    def make(seed):
        q, k, v, do, table = (t.to(DEV) for t in _inputs(2, 200, 200, 4, 2, 64, BF16, 32, seed=seed))
        x = torch.randn(60, 5000, device=DEV, generator=torch.Generator(DEV).manual_seed(seed)).to(BF16)
        tok = torch.randint(0, 5000, (60,), device=DEV)
        cache = [torch.randn(2, n, h, 64, device=DEV).to(BF16) for n, h in ((1, 8), (3000, 2), (3000, 2))]

        def run():
            leaves = [t.detach().requires_grad_() for t in (q, k, v, table)]
            out = attention(*leaves[:3], rel_table=leaves[3], causal=True)
            grads = torch.autograd.grad(out, leaves, do)
            t = table.detach().requires_grad_()
            bias = relative_bias(t, 200, 200)
            dt, = torch.autograd.grad(bias, t, bias.detach())
            lx = x.detach().requires_grad_()
            r = token_log_probs(lx, tok, 4)
            dx, = torch.autograd.grad(r.logp.sum(), lx)
            return [out.detach(), *grads, bias.detach(), dt, *[z.detach() for z in r], dx, attention(*cache)]
        return run

    runs = [make(1), make(2)]
    want = [[t.clone() for t in r()] for r in runs]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = [None, None]
    for _ in range(3):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i] = runs[i]()
    torch.cuda.synchronize()
    for g, w in zip(got, want):
        assert all(torch.equal(a, b) for a, b in zip(g, w))
    del got
    graphs, outs = [], []
    for r in runs:
        g = torch.cuda.CUDAGraph()
        with collected(), torch.cuda.graph(g):
            outs.append(r())
        graphs.append(g)
    for _ in range(3):
        for g in graphs:
            g.replay()
        runs[0]()
    torch.cuda.synchronize()
    for g, w in zip(outs, want):
        assert all(torch.equal(a, b) for a, b in zip(g, w))
