"""General attention, relative position bias and token log probabilities: what they refuse, their torch form against the
64-bit oracles, and the oracles' gradients against differences. No GPU."""
import math
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.dirname(__file__))
import operator_oracles as O  # noqa: E402
from distributed_tensorflow_amd.ops.attention import attention, self_attention  # noqa: E402
from distributed_tensorflow_amd.ops.relative_bias import bucket_borders, relative_bias, relative_bucket  # noqa: E402
from distributed_tensorflow_amd.ops.softmax_ce import token_log_probs  # noqa: E402


def _t(*shape, dt=torch.float32):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(sum(shape))).to(dt)


@pytest.mark.parametrize("kw,err", [
    (dict(q=_t(2, 5, 4)), ValueError), (dict(k=_t(2, 7, 2, 24)), ValueError), (dict(k=_t(3, 7, 2, 16)), ValueError),
    (dict(v=_t(2, 8, 2, 16)), ValueError), (dict(q=_t(2, 5, 3, 16)), ValueError),
    (dict(q=_t(2, 5, 4, 12), k=_t(2, 7, 2, 12), v=_t(2, 7, 2, 12)), ValueError),
    (dict(q=_t(2, 5, 4, 136), k=_t(2, 7, 2, 136), v=_t(2, 7, 2, 136)), ValueError),
    (dict(q=_t(2, 5, 4, 16, dt=torch.bfloat16)), ValueError),
    (dict(q=_t(2, 5, 4, 16).half(), k=_t(2, 7, 2, 16).half(), v=_t(2, 7, 2, 16).half()), TypeError),
    (dict(scale=0.0), ValueError), (dict(scale=-1.0), ValueError), (dict(scale=math.inf), ValueError),
    (dict(scale=math.nan), ValueError),
    (dict(key_bias=_t(2, 6)), ValueError), (dict(key_bias=_t(2, 7).requires_grad_()), ValueError),
    (dict(key_bias=torch.zeros(2, 7, dtype=torch.int32)), ValueError),
    (dict(key_lengths=torch.tensor([1.0, 2.0])), ValueError), (dict(key_lengths=torch.tensor([1])), ValueError),
    (dict(key_lengths=[1, 2]), ValueError),
    (dict(q_start=torch.tensor([1.0, 2.0])), ValueError), (dict(q_start=1 << 30), ValueError),
    (dict(rel_table=_t(8, 3)), ValueError), (dict(rel_table=_t(8, 4, 1)), ValueError), (dict(rel_table=_t(7, 4)), ValueError),
    (dict(rel_table=_t(130, 4)), ValueError), (dict(rel_table=_t(2, 4)), ValueError),
    (dict(rel_table=_t(8, 4), rel_max_distance=2), ValueError), (dict(rel_table=_t(8, 4), rel_max_distance=2049), ValueError),
    (dict(rel_table=_t(8, 4).half()), TypeError),
])
def test_attention_refuses(kw, err):
    args = dict(q=_t(2, 5, 4, 16), k=_t(2, 7, 2, 16), v=_t(2, 7, 2, 16))
    args.update(kw)
    with pytest.raises(err):
        attention(args.pop("q"), args.pop("k"), args.pop("v"), **args)


def test_attention_refuses_rows_wider_than_its_offsets():
    x = torch.empty(1, 1, 65536, 72)
    with pytest.raises(ValueError):
        attention(x, x, x)
    with pytest.raises(ValueError):
        self_attention(x, kv_heads=16384)


def test_splits_of_an_empty_batch():
    from distributed_tensorflow_amd.ops import _lib
    lib = _lib.kernels()
    assert lib.dtf_attention_splits(0, 1, 4001, 16, 4) == 1 and lib.dtf_attention_splits(8, 1, 4001, 16, 4) > 1
    assert lib.dtf_attention_bwd_splits(0, 4001, 16, 4) >= 1


def test_self_attention_refuses():
    for x, kw in ((_t(2, 5, 8, 16), dict(kv_heads=4)), (_t(2, 5, 8, 16), dict(kv_heads=0)), (_t(2, 5, 7, 16), dict(kv_heads=2)),
                  (_t(2, 5, 2, 4, 16), dict(causal=True)), (_t(2, 5, 3, 4, 16), dict(kv_heads=4)), (_t(2, 5, 8, 16), dict(causal=True))):
        with pytest.raises(ValueError):
            self_attention(x, **kw)


def test_relative_bias_refuses():
    for t, kw in ((_t(8), {}), (_t(3, 2), dict(bidirectional=True)), (_t(1, 2), dict(bidirectional=False)), (_t(8, 0), {}),
                  (_t(8, 2), dict(max_distance=2)), (_t(8, 2), dict(q_start=1 << 30))):
        with pytest.raises(ValueError):
            relative_bias(t, 4, 4, **kw)
    with pytest.raises(ValueError):
        relative_bias(_t(8, 2), -1, 4)
    with pytest.raises(TypeError):
        relative_bias(_t(8, 2).half(), 4, 4)


def test_token_log_probs_refuses():
    x, t = _t(4, 10), torch.zeros(4, dtype=torch.long)
    for a, b, top in ((x, t[:3], 0), (x, t, 11), (x, t, -1), (_t(4, 100), t, 33), (torch.empty(4, 0), t, 0), (x, t[:, None], 0)):
        with pytest.raises(ValueError):
            token_log_probs(a, b, top)
    for a, b in ((x.half(), t), (x, t.float())):
        with pytest.raises(TypeError):
            token_log_probs(a, b)


@pytest.mark.parametrize("buckets,far,bidir", [(32, 128, True), (32, 128, False), (8, 8, True), (2, 3, False), (128, 2048, True),
                                               (64, 200, False), (4, 2, True)])
def test_buckets_are_those_of_whole_numbers(buckets, far, bidir):
    d = torch.arange(-far - 70, far + 71)
    want = torch.tensor([O.bucket(int(x), buckets, far, bidir) for x in d])
    assert torch.equal(relative_bucket(d, buckets, far, bidir), want)
    half = buckets // 2 if bidir else buckets
    assert len(bucket_borders(buckets, far, bidir)) == half - half // 2 - 1
    assert int(relative_bucket(torch.tensor(-far), buckets, far, bidir)) == half - 1


@pytest.mark.parametrize("shape", [(2, 5, 9, 4, 2, 16), (1, 9, 5, 2, 2, 8), (1, 1, 1, 1, 1, 8)])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
def test_attention_torch_form(shape, causal, dt):
    B, Sq, Sk, nh, nkv, hd = shape
    q, k, v, do, table = _t(B, Sq, nh, hd, dt=dt), _t(B, Sk, nkv, hd, dt=dt), _t(B, Sk, nkv, hd, dt=dt) * 2, _t(B, Sq, nh, hd, dt=dt), _t(8, nh, dt=dt)
    kb = torch.zeros(B, Sk)
    kb[:, Sk // 2] = -math.inf
    kw = dict(key_bias=kb, key_lengths=torch.tensor([Sk, 3][:B]), causal=causal, rel_max_distance=9)
    val, tol = O.attention(q, k, v, do, rel_table=table, **kw)
    leaves = [t.clone().requires_grad_() for t in (q, k, v, table)]
    with torch.no_grad():
        leaves[1][:, Sk // 2], leaves[2][:, Sk // 2] = math.nan, math.inf       # what a masked key holds is not read
    out = attention(*leaves[:3], rel_table=leaves[3], **kw)
    O.check("out", out, val["out"], tol["out"])
    for n, g in zip(("dq", "dk", "dv", "dtable"), torch.autograd.grad(out, leaves, do)):
        O.check(n, g, val[n], tol[n])


def test_oracle_gradients_agree_with_differences():
    q, k, v, w, table = _t(1, 6, 4, 8).double(), _t(1, 9, 2, 8).double(), _t(1, 9, 2, 8).double() * 2, _t(1, 6, 4, 8).double(), _t(8, 4).double()
    kw = dict(causal=True, rel_max_distance=6, key_bias=torch.randn(1, 9).double())
    ins = [q, k, v, table]
    val, _ = O.attention(q, k, v, w, rel_table=table, **kw)
    f = lambda t: float((O.attention(*t[:3], rel_table=t[3], **kw)[0]["out"] * w).sum())  # noqa: E731
    for n, name in enumerate(("dq", "dk", "dv", "dtable")):
        d, h = torch.randn(ins[n].shape, dtype=torch.float64), 1e-5
        up, down = ([x + s * h * d if i == n else x for i, x in enumerate(ins)] for s in (1, -1))
        # truncation h^2 f''' / 6 and rounding eps f / h are both far below 1e-7 here
        assert abs((f(up) - f(down)) / (2 * h) - float((val[name] * d).sum())) < 1e-7
    x, tok = _t(3, 20).double(), torch.tensor([4, -1, 19])
    gs = (_t(3).double(), _t(3, 1)[:, 0].double(), _t(3, 5).double())
    top = O.token_log_probs(x, tok, 5, gs)
    def loss(z):
        val, _, _ = O.token_log_probs(z, tok, 5)
        return float(sum((val[n] * g).sum() for n, g in zip(("logp", "entropy", "top_logp"), gs)))
    d = torch.randn(3, 20, dtype=torch.float64)
    assert abs((loss(x + 1e-5 * d) - loss(x - 1e-5 * d)) / 2e-5 - float((top[0]["dlogits"] * d).sum())) < 1e-7


def test_token_log_probs_torch_form():
    x, tok = _t(6, 40), torch.tensor([0, 39, -1, 40, 7, 5])
    x[4] = -math.inf
    x[5, 3:] = -math.inf
    gs = tuple(_t(*s) for s in ((6,), (6, 1), (6, 4)))
    gs = (gs[0], gs[1][:, 0], gs[2])
    val, tol, ids = O.token_log_probs(x, tok, 4, gs)
    leaf = x.clone().requires_grad_()
    r = token_log_probs(leaf, tok, 4)
    assert torch.equal(r.top_ids, ids)
    for n in ("logp", "entropy", "top_logp"):
        O.check(n, getattr(r, n), val[n], tol[n])
    rows = torch.tensor([0, 1, 2, 3])                     # (rows with infinities: the kernels' business)
    d, = torch.autograd.grad((r.logp[rows], r.entropy[rows], r.top_logp[rows]), leaf, [g[rows] for g in gs])
    O.check("dlogits", d[rows], val["dlogits"][rows], tol["dlogits"][rows])


def test_no_garbage_is_collected_while_a_graph_is_captured():
    import gc
    import weakref
    from distributed_tensorflow_amd.engine.graph import collected

    class Node:
        pass

    def cycle():
        a = Node()
        a.me = a
        return weakref.ref(a)

    old = cycle()
    with collected():
        assert old() is None and not gc.isenabled()
        new = cycle()
        kept = [[] for _ in range(20000)]                # (more than one generation's worth of containers)
        assert new() is not None and kept
    assert gc.isenabled()
