"""Attention, relative position bias and token log probabilities in 64 bits, with bounds of what the kernels may be off by.

The bounds follow the kernels' roundings. With ``u`` half a step of the operands' type (``torch.finfo(t).eps / 2``) and
``e`` the relative error of a probability in 32 bits:

* ``e``: a score sums ``hd`` products, so it is off by at most ``hd u32 A`` with ``A = scale sum |q||k| + |bias|``; the
  maximum that is taken off and the exponential's argument add a few ``u32 (|t| + |m|)``, the exponential itself a few
  ``u32``, the row's sum of ``Sk`` terms ``Sk u32``: ``e = u32 (2 (hd + 8) A + Sk + 16)``;
* out: P is rounded to the operands' type (``u``), the result too: ``(u + e + Sk u32) P|v| + u |out|``;
* D = rowsum(dO * O) takes the stored O: ``eD = |dO| . err(out) + hd u32 |dO| . |O|``;
* dT = P (dP - D): ``eT = P (2 e |dP - D| + eD + hd u32 |dO||v|)``; it is rounded to the operands' type (``u |dT|``)
  where it enters a product, and not where it enters the table's gradient;
* dQ, dK, dV, dTable: those, summed over absolute values, ``n u32`` more for a sum of n terms, and the result's rounding.
"""
import math

import torch

U32 = 2.0 ** -24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def bucket(d, buckets, max_distance, bidirectional):
    """Bucket of one signed distance, in whole numbers."""
    half = buckets // 2 if bidirectional else buckets
    exact, a = half // 2, (abs(d) if bidirectional else max(-d, 0))
    n = half - exact
    b = a
    if a >= exact:
        t = 0
        while t < n - 1 and a ** n * exact ** (t + 1) >= max_distance ** (t + 1) * exact ** n:
            t += 1
        b = exact + t
    return b + (half if bidirectional and d > 0 else 0)


def buckets_between(low, high, buckets, max_distance, bidirectional):
    return torch.tensor([bucket(d, buckets, max_distance, bidirectional) for d in range(low, high + 1)])


def attention(q, k, v, dout=None, key_bias=None, causal=False, scale=None, key_lengths=None, q_start=None, rel_table=None,
              rel_max_distance=128, rel_bidirectional=None):
    """Values and bounds: two dicts with out and, when ``dout`` is given, dq, dk, dv, dtable. Inputs on the CPU."""
    dt = q.dtype
    u = half_step(dt)
    B, Sq, nh, hd = q.shape
    Sk, nkv = k.shape[1:3]
    group = nh // nkv
    scale = 1 / math.sqrt(hd) if scale is None else scale
    bidir = (not causal) if rel_bidirectional is None else rel_bidirectional
    starts = torch.full((B,), Sk - Sq) if q_start is None else torch.as_tensor(q_start).expand(B)
    val = {n: torch.zeros(s, dtype=torch.float64) for n, s in
           dict(out=q.shape, dq=q.shape, dk=k.shape, dv=v.shape).items()}
    tol = {n: t.clone() for n, t in val.items()}
    if rel_table is not None:
        val["dtable"], tol["dtable"] = (torch.zeros(rel_table.shape, dtype=torch.float64) for _ in range(2))
    for b in range(B):
        d = torch.arange(Sk)[None, :] - (torch.arange(Sq)[:, None] + int(starts[b]))
        seen = torch.ones(Sq, Sk, dtype=torch.bool)
        if key_lengths is not None:
            seen &= (torch.arange(Sk) < int(key_lengths[b]))[None]
        if key_bias is not None:
            seen &= (key_bias[b] != -math.inf)[None]
        alive = seen.any(0)
        if causal:
            seen &= d <= 0
        if rel_table is not None and Sk:
            low = int(d.min())
            of = buckets_between(low, int(d.max()), rel_table.shape[0], rel_max_distance, bidir)[d - low]
        for h in range(nh):
            qq = q[b, :, h].double()
            kk, vv = (x[b, :, h // group].double().masked_fill(~alive[:, None], 0.0) for x in (k, v))
            t, A = qq @ kk.t() * scale, qq.abs() @ kk.abs().t() * scale
            bias = torch.zeros(Sq, Sk, dtype=torch.float64)
            if rel_table is not None:
                bias = bias + rel_table[:, h].double()[of]
            if key_bias is not None:
                bias = bias + key_bias[b].double().masked_fill(~alive, 0.0)
            big = bias.abs() > 1e30                          # lowest-value masks: absorbed alike in 32 bits
            t = torch.where(big, bias, t + bias).masked_fill(~seen, -math.inf)
            A = (A + torch.where(big, 0.0, bias.abs()))
            top = t.amax(1, keepdim=True)
            p = torch.exp(t - top.masked_fill(top == -math.inf, 0.0))
            total = p.sum(1, keepdim=True)
            p = p / total.masked_fill(total == 0, 1.0)
            e = U32 * (2 * (hd + 8) * A + Sk + 16)
            o = p @ vv
            eo = (p * (e + u + Sk * U32)) @ vv.abs() + u * o.abs()
            val["out"][b, :, h], tol["out"][b, :, h] = o, eo
            if dout is None:
                continue
            do = dout[b, :, h].double()
            dp, adp = do @ vv.t(), do.abs() @ vv.abs().t()
            D = (do * o).sum(1, keepdim=True)
            eD = (do.abs() * (eo + hd * U32 * o.abs())).sum(1, keepdim=True)
            ds = p * (dp - D)
            es = p * (2 * e * (dp - D).abs() + eD + 2 * hd * U32 * adp)
            er = es + u * ds.abs()
            kvh = h // group
            val["dq"][b, :, h] = scale * ds @ kk
            tol["dq"][b, :, h] = scale * (er + Sk * U32 * ds.abs()) @ kk.abs()
            val["dk"][b, :, kvh] += scale * ds.t() @ qq
            tol["dk"][b, :, kvh] += scale * (er + group * Sq * U32 * ds.abs()).t() @ qq.abs()
            val["dv"][b, :, kvh] += p.t() @ do
            tol["dv"][b, :, kvh] += (p * (e + u + group * Sq * U32)).t() @ do.abs()
            if rel_table is not None:
                n = B * Sq * Sk
                for w, x in ((val, ds), (tol, es + min(n, 4096) * U32 * ds.abs())):
                    w["dtable"][:, h].index_add_(0, of.flatten(), x.flatten())
    names = ["out"] if dout is None else ["out", "dq", "dk", "dv"] + (["dtable"] if rel_table is not None else [])
    for n in names:
        if n != "out":                                       # (out's own rounding is in already: D sees it)
            tol[n] += half_step(rel_table.dtype if n == "dtable" else dt) * val[n].abs()
        tol[n] = 1.01 * tol[n] + 1e-30
    return {n: val[n] for n in names}, {n: tol[n] for n in names}


def relative_bias(table, q_len, k_len, max_distance, bidirectional, q_start, g):
    """(bias, dtable, bound of dtable)."""
    d = torch.arange(k_len)[None, :] - (torch.arange(q_len)[:, None] + q_start)
    low = int(d.min())
    of = buckets_between(low, int(d.max()), table.shape[0], max_distance, bidirectional)[d - low]
    bias = table.t()[:, of]
    dt, mag = (torch.zeros(table.shape, dtype=torch.float64) for _ in range(2))
    for h in range(table.shape[1]):
        dt[:, h].index_add_(0, of.flatten(), g[h].double().flatten())
        mag[:, h].index_add_(0, of.flatten(), g[h].double().abs().flatten())
    # sums of up to 4096 terms in a row in 32 bits, of partial sums after that
    return bias, dt, 1.01 * (min(q_len * k_len, 4096) * U32 * mag + half_step(table.dtype) * dt.abs()) + 1e-30


def token_log_probs(x, tokens, top, g=None):
    """Values and bounds of logp, entropy, top_logp (and dlogits for ``g = (g_logp, g_entropy, g_top)``), and top_ids."""
    xd, (N, V) = x.double(), x.shape
    ok = (tokens >= 0) & (tokens < V)
    best = xd.amax(1, keepdim=True)
    none = best == -math.inf
    z = xd - best.masked_fill(none, 0.0)
    total = z.exp().sum(1, keepdim=True)
    lp = z - total.masked_fill(none, 1.0).log()
    p = lp.exp()
    fin = torch.where(lp == -math.inf, 0.0, lp)
    H = -(p * fin).sum(1, keepdim=True)
    pick = lp.gather(1, tokens.clamp(0, V - 1).long()[:, None])[:, 0]
    ids = torch.sort(x.float(), dim=1, descending=True, stable=True).indices[:, :top]
    val = dict(logp=torch.where(ok, pick, 0.0), entropy=H[:, 0], top_logp=lp.gather(1, ids))
    # x - m: one rounding; e^z: its argument's, u32 |z| log2 e, and its own; sums of V terms: the threads hold V / 256 of
    # them in a row and add tree-wise, 64 in a row at most here
    sums = U32 * (64 + V / 256)
    es = U32 * ((p * (3 * fin.abs() + 8)).sum(1, keepdim=True)) + sums
    tol = dict(logp=torch.where(ok, (es[:, 0] + 3 * U32 * (pick.abs().nan_to_num(posinf=0.0) + 1)), 0.0),
               entropy=(2 * es * (1 + H) + U32 * (p * (3 * fin.abs() + 8) * fin.abs()).sum(1, keepdim=True))[:, 0] + 4 * U32,
               top_logp=es + 3 * U32 * (val["top_logp"].abs().nan_to_num(posinf=0.0) + 1))
    if g is not None:
        ga, gh, gt = (t.double() for t in g)
        ga = torch.where(ok, ga, 0.0)
        one = torch.zeros_like(xd)
        one[torch.arange(N), tokens.clamp(0, V - 1).long()] += ga
        one.scatter_add_(1, ids, gt)
        all_ = one.sum(1, keepdim=True)
        inner = all_ + gh[:, None] * (fin + H)
        mag = ga.abs()[:, None] + gt.abs().sum(1, keepdim=True) + gh.abs()[:, None] * (fin.abs() + H)
        d = torch.where(none, 0.0, one - p * inner)
        val["dlogits"] = d
        ep = es + U32 * (4 * fin.abs() + 16)
        tol["dlogits"] = torch.where(none, 0.0, p * (ep * inner.abs() + 40 * U32 * mag + gh.abs()[:, None] * tol["entropy"][:, None])
                                     + 4 * U32 * one.abs() + half_step(x.dtype) * d.abs())
    return val, {n: 1.01 * t + 1e-30 for n, t in tol.items()}, ids


def check(name, got, want, tol):
    got = got.detach().double().cpu()
    assert got.shape == want.shape, (name, got.shape, want.shape)
    nan, inf = torch.isnan(want), torch.isinf(want)
    assert torch.equal(torch.isnan(got), nan) and torch.equal(got[inf], want[inf]), f"{name}: other NaN or infinities"
    fine = ~(nan | inf)
    over = ((got - want).abs() / tol)[fine]
    if over.numel():
        assert float(over.max()) <= 1.0, f"{name}: {float(over.max()):.3g} times the bound, at {int(over.argmax())} of {over.numel()}"
