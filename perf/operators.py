"""Cases of the transformer operators: attention with its backward pass (general shapes and masks), the learned relative
position bias by buckets with its gradient, and the log probabilities of given tokens with entropy and top alternatives.

With ``own`` false, ``run`` computes an operator from its definition with elementary torch operations in 32 bits; with
``own`` true it calls the framework's operator. ``exact`` is the definition in 64 bits.
"""
import math

import torch

own = False

DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


# ------------------------------------------------------------------------------------------------------------- cases
def _attention(name, B, Sq, Sk, nh, nkv, hd, dtype="bf16", causal=False, buckets=0, max_distance=128, mask="none",
               grad=True, packed=False, cache=False):
    c = dict(op="attention", B=B, Sq=Sq, Sk=Sk, nh=nh, nkv=nkv, hd=hd, dtype=dtype, causal=causal, buckets=buckets,
             max_distance=max_distance, mask=mask, grad=grad, packed=packed, cache=cache)
    return dict(c, name=name) if name else c


def _bias(name, Sq, Sk, nh, dtype="bf16", buckets=32, max_distance=128, bidirectional=True):
    c = dict(op="bias", Sq=Sq, Sk=Sk, nh=nh, dtype=dtype, buckets=buckets, max_distance=max_distance,
             bidirectional=bidirectional)
    return dict(c, name=name) if name else c


def _logp(name, N, V, top, dtype="bf16", grad=False, masked=0):
    c = dict(op="logp", N=N, V=V, top=top, dtype=dtype, grad=grad, masked=masked)
    return dict(c, name=name) if name else c


def listed():
    return [
        # one encoder layer of BERT-base's sizes in training, relative positions instead of position embeddings
        _attention("encoder_512_relative", 64, 512, 512, 12, 12, 64, buckets=32, packed=True),
        # the same heads on sequences of an odd length, the batch padded to its longest member
        _attention("encoder_197_padded", 96, 197, 197, 12, 12, 64, mask="lengths", packed=True),
        # the launcher's default type, the small BERT's heads, an additive key mask
        _attention("encoder_fp32_key_bias", 64, 128, 128, 2, 2, 64, dtype="fp32", mask="bias"),
        # a decoder layer in training: causal, four query heads to a key head, head size 128
        _attention("decoder_2048_grouped", 4, 2048, 2048, 16, 4, 128, causal=True),
        # one long document: causal, relative positions, far distances in one bucket
        _attention("decoder_8192_relative", 1, 8192, 8192, 8, 8, 64, causal=True, buckets=32),
        # queries of one sequence on the tokens of another, of unequal odd lengths, head size 80
        _attention("cross_333_on_1000", 8, 333, 1000, 10, 10, 80, mask="bias"),
        # one new token of each of eight sequences over a cache of keys and values filled to different lengths
        _attention("one_token_on_4001", 8, 1, 4001, 16, 4, 128, causal=True, mask="lengths", grad=False, cache=True),
        # the bias of BERT-base's heads written out for a short and a long sequence, with the table's gradient
        _bias("bias_512", 512, 512, 12),
        _bias("bias_4099", 4099, 4099, 16),
        # scores of the 80 masked positions of 64 sequences over BERT's vocabulary, trained through
        _logp("mlm_scores_trained", 5120, 30522, 5, grad=True),
        # the same scores of one position, where only latency counts, in the launcher's default type
        _logp("one_position", 1, 30522, 10, dtype="fp32"),
        # scoring a batch of documents over a vocabulary padded to a round size
        _logp("documents_131072", 2048, 131072, 20, masked=71),
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["attention", "attention", "attention", "bias", "logp", "logp"])
    if op == "bias":
        buckets = rng.choice([8, 16, 32, 64])
        return _bias("", _spread(rng, 1, 4000), _spread(rng, 1, 4000), rng.randint(1, 16), rng.choice(["bf16", "fp32"]),
                     buckets, rng.choice([buckets, 100, 128, 200]), rng.random() < 0.5)
    if op == "logp":
        V = _spread(rng, 32, 131072)
        N = _spread(rng, 1, min(20000, 200_000_000 // V))
        return _logp("", N, V, rng.choice([0, 1, 5, 20, 32]), rng.choice(["bf16", "bf16", "fp32"]), rng.random() < 0.5,
                     rng.choice([0, 0, min(17, V // 3)]))
    hd = rng.choice([16, 32, 40, 64, 64, 80, 96, 128])
    nkv = rng.choice([1, 2, 3, 4, 8])
    nh = nkv * rng.choice([1, 1, 2, 3])
    dtype = rng.choice(["bf16", "bf16", "bf16", "fp32"])
    buckets, max_distance = rng.choice([(0, 128), (0, 128), (32, 128), (16, 77), (32, 300)])
    if rng.random() < 0.25:                      # a few new tokens over a cache
        B, Sq, Sk = _spread(rng, 1, 64), rng.choice([1, 1, 2, 5]), _spread(rng, 5, 20000)
        return _attention("", B, Sq, Sk, nh, nkv, hd, dtype, True, buckets, max_distance, "lengths", False, False, True)
    Sq = _spread(rng, 1, 3000)
    self_attention = rng.random() < 0.6
    Sk = Sq if self_attention else _spread(rng, 1, 3000)
    B = _spread(rng, 1, max(1, min(32, 100_000_000 // (Sq * Sk * nh))))
    return _attention("", B, Sq, Sk, nh, nkv, hd, dtype, rng.random() < 0.5, buckets, max_distance,
                      rng.choice(["none", "lengths", "bias"]), rng.random() < 0.7 and Sk >= 8,   # with one key, dq is 0
                      self_attention and rng.random() < 0.6)


# ------------------------------------------------------------------------------------------------------------ inputs
def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    dt = TYPES[case["dtype"]]

    def normal(*shape, std=1.0):
        return (torch.randn(*shape, generator=g, device=DEV) * std).to(dt)

    def uniform(*shape):
        return torch.rand(*shape, generator=g, device=DEV)

    s = {"case": case}
    if case["op"] == "bias":
        s["table"] = normal(case["buckets"], case["nh"], std=0.5).requires_grad_()
        s["grad"] = normal(case["nh"], case["Sq"], case["Sk"])
        return s
    if case["op"] == "logp":
        N, V = case["N"], case["V"]
        x = normal(N, V, std=2.0)
        if case["masked"]:                       # words that the vocabulary was padded with
            x[:, V - case["masked"]:] = -math.inf
        s["tokens"] = torch.randint(0, V - case["masked"], (N,), generator=g, device=DEV)
        if N > 8:                                # padding of the batch: no token there
            s["tokens"][N // 3] = -1
        # a language model is often sure of the token
        x[torch.arange(N, device=DEV), s["tokens"].clamp(min=0)] += (8.0 * uniform(N)).to(dt)
        s["logits"] = x.requires_grad_(case["grad"])
        s["g"] = (uniform(N) - 0.5, 0.1 * (uniform(N) - 0.5), 0.1 * (uniform(N, case["top"]) - 0.5))
        return s
    B, Sq, Sk, nh, nkv, hd, train = (case[n] for n in ("B", "Sq", "Sk", "nh", "nkv", "hd", "grad"))
    if case["packed"]:
        s["qkv"] = normal(B, Sq, nh + 2 * nkv, hd).requires_grad_(train)
    else:
        s["q"] = normal(B, Sq, nh, hd, std=1.5).requires_grad_(train)
        s["k"] = normal(B, Sk, nkv, hd).requires_grad_(train)
        s["v"] = normal(B, Sk, nkv, hd).requires_grad_(train)
    s["table"] = normal(case["buckets"], nh).requires_grad_(train) if case["buckets"] else None
    s["lengths"] = s["key_bias"] = s["q_start"] = None
    if case["mask"] == "lengths":
        s["lengths"] = (Sk - (uniform(B) * (Sk // 2 + 1)).long()).clamp(min=min(Sq, Sk) if case["cache"] else 0).int()
    elif case["mask"] == "bias":                 # padded keys, and some that are merely unlikely
        kb = torch.where(uniform(B, Sk) < 0.1, -2.0, 0.0)
        n = Sk - (uniform(B) * (Sk // 2 + 1)).long()
        s["key_bias"] = kb.masked_fill(torch.arange(Sk, device=DEV) >= n[:, None], -math.inf)
    if case["cache"]:                            # the new tokens are the last ones of their sequences
        s["q_start"] = s["lengths"] - min(Sq, Sk)
    if train:
        s["dout"] = normal(B, Sq, nh, hd)
    return s


# ------------------------------------------------------------------------------------- the framework's operators' calls
def _run_own(s):
    c = s["case"]
    if c["op"] == "bias":
        from distributed_tensorflow_amd.ops.relative_bias import relative_bias
        bias = relative_bias(s["table"], c["Sq"], c["Sk"], max_distance=c["max_distance"],
                             bidirectional=c["bidirectional"])
        return {"bias": bias, "dtable": torch.autograd.grad(bias, s["table"], s["grad"])[0]}
    if c["op"] == "logp":
        from distributed_tensorflow_amd.ops.softmax_ce import token_log_probs
        r = token_log_probs(s["logits"], s["tokens"], top=c["top"])
        out = {"logp": r.logp, "entropy": r.entropy, "top_logp": r.top_logp, "top_ids": r.top_ids}
        if c["grad"]:
            n = 3 if c["top"] else 2
            out["dlogits"] = torch.autograd.grad((r.logp, r.entropy, r.top_logp)[:n], s["logits"], s["g"][:n])[0]
        return out
    from distributed_tensorflow_amd.ops.attention import attention, self_attention
    more = dict(causal=c["causal"], key_lengths=s["lengths"], q_start=s["q_start"], rel_table=s["table"],
                rel_max_distance=c["max_distance"])
    if c["packed"]:
        out = self_attention(s["qkv"], s["key_bias"], kv_heads=c["nkv"], **more)
        wrt = {"dqkv": s["qkv"]}
    else:
        out = attention(s["q"], s["k"], s["v"], s["key_bias"], **more)
        wrt = {"dq": s["q"], "dk": s["k"], "dv": s["v"]}
    if not c["grad"]:
        return {"out": out}
    if s["table"] is not None:
        wrt["dtable"] = s["table"]
    return {"out": out, **dict(zip(wrt, torch.autograd.grad(out, list(wrt.values()), s["dout"])))}


# -------------------------------------------------------------------------------------------------- the plain forms
def _buckets(delta, buckets, max_distance, bidirectional):
    """The bucket of each signed distance key - query: near ones alone, far ones together by the distance's logarithm."""
    half = buckets // 2 if bidirectional else buckets
    far = delta.abs() if bidirectional else (-delta).clamp(min=0)
    exact = half // 2
    log = torch.log(far.clamp(min=1).double() / exact) / math.log(max_distance / exact) * (half - exact)
    step = (exact + torch.floor(log + 1e-9)).clamp(max=half - 1).long()
    b = torch.where(far < exact, far, step)
    return b + half * (delta > 0) if bidirectional else b


def _diagonal_sums(t):
    """[..., Sq, Sk] -> [..., Sq + Sk - 1]: the sum over each key - query = Sk - 1 ... 1 - Sq, ascending."""
    Sq, Sk = t.shape[-2:]
    w = torch.nn.functional.pad(t.flip(-2), (0, Sq)).flatten(-2)[..., :Sq * (Sq + Sk - 1)]
    return w.unflatten(-1, (Sq, Sq + Sk - 1)).sum(-2, dtype=torch.float64)


def _plain_bias(s, c):
    dt, Sq, Sk = s["table"].dtype, c["Sq"], c["Sk"]
    start = Sk - Sq
    d = torch.arange(-(Sq - 1) - start, Sk - start, device=DEV)
    of = _buckets(d, c["buckets"], c["max_distance"], c["bidirectional"])
    with torch.no_grad():
        bias = s["table"].t()[:, of].unfold(1, Sk, 1).flip(1)
        sums = _diagonal_sums(s["grad"].float())
        dtable = torch.zeros(c["buckets"], c["nh"], dtype=torch.float64, device=DEV).index_add_(0, of, sums.t())
    return {"bias": bias, "dtable": dtable.to(dt)}


def _plain_logp(s, c):
    with torch.no_grad():
        x, tok = s["logits"].float(), s["tokens"]
        ok = tok >= 0
        rows = torch.arange(len(tok), device=DEV)
        z = x - x.amax(1, keepdim=True)
        e = torch.exp(z)
        total = e.sum(1, keepdim=True)
        p, lp = e / total, z - torch.log(total)
        plp = torch.where(p > 0, p * lp, 0.0)
        logp = torch.where(ok, lp[rows, tok.clamp(min=0)], 0.0)
        entropy = -plp.sum(1)
        ids = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :c["top"]]
        top = lp.gather(1, ids)
        out = {"logp": logp, "entropy": entropy, "top_logp": top, "top_ids": ids}
        if c["grad"]:
            ga, gh, gt = s["g"]
            ga = torch.where(ok, ga, 0.0)
            d = p * -(ga + gt.sum(1))[:, None] - gh[:, None] * (plp + p * entropy[:, None])
            d[rows, tok.clamp(min=0)] += ga
            d.scatter_add_(1, ids, gt)
            out["dlogits"] = d.to(s["logits"].dtype)
        return out


def _plain_attention(s, c):
    B, Sq, Sk, nh, nkv, hd = (c[n] for n in ("B", "Sq", "Sk", "nh", "nkv", "hd"))
    group, scale = nh // nkv, 1.0 / math.sqrt(hd)
    with torch.no_grad():
        q, k, v = s["qkv"].split((nh, nkv, nkv), 2) if c["packed"] else (s["q"], s["k"], s["v"])
        dt = q.dtype
        q, k, v = (t.float().transpose(1, 2) for t in (q, k, v))
        k, v = (t.repeat_interleave(group, 1) for t in (k, v))
        start = s["q_start"][:, None, None] if c["cache"] else Sk - Sq
        delta = torch.arange(Sk, device=DEV) - torch.arange(Sq, device=DEV)[:, None] - start    # [(B,) Sq, Sk]
        t = (q @ k.transpose(2, 3)) * scale
        if c["buckets"] and c["cache"]:
            of = _buckets(delta, c["buckets"], c["max_distance"], not c["causal"])
            t += s["table"].float()[of].permute(0, 3, 1, 2)
        elif c["buckets"]:                       # the rows of the bias are windows into one row of all distances
            d = torch.arange(-(Sq - 1) - start, Sk - start, device=DEV)
            of = _buckets(d, c["buckets"], c["max_distance"], not c["causal"])
            t += s["table"].float().t()[:, of].unfold(1, Sk, 1).flip(1)
        if s["key_bias"] is not None:
            t += s["key_bias"][:, None, None, :]
        if c["causal"]:
            t.masked_fill_((delta > 0)[:, None] if c["cache"] else delta > 0, -math.inf)
        if s["lengths"] is not None:
            t.masked_fill_((torch.arange(Sk, device=DEV) >= s["lengths"][:, None])[:, None, None, :], -math.inf)
        t -= t.amax(-1, keepdim=True).clamp(min=torch.finfo(torch.float32).min)
        p = torch.exp(t)
        del t
        p /= p.sum(-1, keepdim=True).clamp(min=torch.finfo(torch.float32).tiny)
        out = p @ v
        res = {"out": out.transpose(1, 2).to(dt).contiguous()}
        if not c["grad"]:
            return res
        do = s["dout"].float().transpose(1, 2)
        dv = p.transpose(2, 3) @ do
        dp = do @ v.transpose(2, 3)
        dp -= (do * out).sum(-1, keepdim=True)
        dp *= p
        del p
        dq = (dp @ k) * scale
        dk = (dp.transpose(2, 3) @ q) * scale
        dk, dv = (t.unflatten(1, (nkv, group)).sum(2) for t in (dk, dv))
        dq, dk, dv = (t.transpose(1, 2).to(dt) for t in (dq, dk, dv))
        if c["packed"]:
            res["dqkv"] = torch.cat((dq, dk, dv), 2)
        else:
            res.update(dq=dq.contiguous(), dk=dk.contiguous(), dv=dv.contiguous())
        if c["buckets"]:
            sums = _diagonal_sums(dp.sum(0))
            dtable = torch.zeros(c["buckets"], nh, dtype=torch.float64, device=DEV).index_add_(0, of, sums.t())
            res["dtable"] = dtable.to(dt)
        return res


def run(state):
    if own:
        return _run_own(state)
    c = state["case"]
    return {"attention": _plain_attention, "bias": _plain_bias, "logp": _plain_logp}[c["op"]](state, c)


# ---------------------------------------------------------------------------------------------------------- 64 bits
def _exact_bucket_list(low, high, buckets, max_distance, bidirectional):
    """Buckets of the distances low .. high, in whole numbers: (a / exact)^(half - exact) >= (max / exact)^t."""
    half = buckets // 2 if bidirectional else buckets
    exact = half // 2
    n = half - exact
    got = []
    for d in range(low, high + 1):
        a = min(abs(d) if bidirectional else max(-d, 0), max_distance)
        b = a
        if a >= exact:
            t = 0
            while t < n - 1 and a ** n * exact ** (t + 1) >= max_distance ** (t + 1) * exact ** n:
                t += 1
            b = exact + t
        got.append(b + (half if bidirectional and d > 0 else 0))
    return torch.tensor(got, device=DEV)


def _exact_attention(case, s):
    B, Sq, Sk, nh, nkv, hd = (case[n] for n in ("B", "Sq", "Sk", "nh", "nkv", "hd"))
    if case["packed"]:
        x = s["qkv"].detach()
        q, k, v = x[:, :, :nh], x[:, :, nh:nh + nkv], x[:, :, nh + nkv:]
    else:
        q, k, v = s["q"].detach(), s["k"].detach(), s["v"].detach()
    f8 = dict(dtype=torch.float64, device=DEV)
    out, dq = torch.zeros(B, Sq, nh, hd, **f8), torch.zeros(B, Sq, nh, hd, **f8)
    dk, dv = torch.zeros(B, Sk, nkv, hd, **f8), torch.zeros(B, Sk, nkv, hd, **f8)
    dtable = torch.zeros(max(case["buckets"], 1), nh, **f8)
    starts = s["q_start"].tolist() if case["cache"] else [Sk - Sq] * B
    lengths = s["lengths"].tolist() if s["lengths"] is not None else [Sk] * B
    j, i = torch.arange(Sk, device=DEV), torch.arange(Sq, device=DEV)
    of, start_of = None, None
    for b in range(B):
        off = j[None, :] - (i[:, None] + starts[b])
        if case["buckets"] and start_of != starts[b]:
            start_of = starts[b]
            low = -(Sq - 1) - start_of
            of = _exact_bucket_list(low, Sk - 1 - start_of, case["buckets"], case["max_distance"], not case["causal"])
            of = of[off - low]
        gone = (j >= lengths[b])[None, :].expand(Sq, Sk)
        if case["causal"]:
            gone = gone | (off > 0)
        if s["key_bias"] is not None:
            gone = gone | (s["key_bias"][b] == -math.inf)[None, :]
        some = (~gone).any(1)
        for h in range(nh):
            kh = h // (nh // nkv)
            qq, kk, vv = q[b, :, h].double(), k[b, :, kh].double(), v[b, :, kh].double()
            t = qq @ kk.t() / math.sqrt(hd)
            if case["buckets"]:
                t = t + s["table"].detach().double()[:, h][of]
            if s["key_bias"] is not None:
                t = t + s["key_bias"][b].double()
            t = t.masked_fill(gone, -math.inf)
            p = torch.softmax(t[some], 1)
            o = p @ vv
            out[b, some, h] = o
            if not case["grad"]:
                continue
            do = s["dout"][b, some, h].double()
            dt = p * (do @ vv.t() - (do * o).sum(1, keepdim=True))
            dq[b, some, h] = dt @ kk / math.sqrt(hd)
            dk[b, :, kh] += dt.t() @ qq[some] / math.sqrt(hd)
            dv[b, :, kh] += p.t() @ do
            if case["buckets"]:
                of_some = of[some]
                dtable[:, h] += torch.stack([(dt * (of_some == u)).sum() for u in range(case["buckets"])])
    res = {"out": out}
    if case["grad"]:
        res.update({"dqkv": torch.cat((dq, dk, dv), 2)} if case["packed"] else {"dq": dq, "dk": dk, "dv": dv})
        if case["buckets"]:
            res["dtable"] = dtable
    return res


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "attention":
        return _exact_attention(case, s)
    if case["op"] == "bias":
        Sq, Sk = case["Sq"], case["Sk"]
        of = _exact_bucket_list(1 - Sk, Sq - 1, case["buckets"], case["max_distance"], case["bidirectional"])
        table, bias, dtable = s["table"].detach().double(), [], []
        place = torch.arange(Sk, device=DEV)[None, :] + torch.arange(Sq - 1, -1, -1, device=DEV)[:, None]
        of = of[place].flatten()
        for h in range(case["nh"]):
            bias.append(table[:, h][of].view(Sq, Sk).to(TYPES[case["dtype"]]))
            t = s["grad"][h].double().flatten()
            dtable.append(torch.stack([(t * (of == u)).sum() for u in range(case["buckets"])]))
        return {"bias": torch.stack(bias), "dtable": torch.stack(dtable, 1)}
    res = {"logp": [], "entropy": [], "top_logp": [], "dlogits": []}
    for rows in torch.arange(case["N"], device=DEV).split(max(1, 100_000_000 // case["V"])):
        x, tok = s["logits"].detach()[rows].double(), s["tokens"][rows]
        lp = torch.log_softmax(x, 1)
        p = lp.exp()
        h = torch.special.entr(p).sum(1)
        res["logp"].append(lp.gather(1, tok.clamp(min=0)[:, None])[:, 0] * (tok >= 0))
        res["entropy"].append(h)
        res["top_logp"].append(lp.topk(case["top"], 1).values)
        if case["grad"]:
            ga, gh, gt = (t[rows].double() for t in s["g"])
            ga = ga * (tok >= 0)
            top = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :case["top"]]
            one = torch.zeros_like(x).scatter_(1, tok.clamp(min=0)[:, None], ga[:, None]).scatter_add_(1, top, gt)
            d = one - p * one.sum(1, keepdim=True)
            res["dlogits"].append(d + gh[:, None] * (torch.special.entr(p) - p * h[:, None]))
    res = {n: torch.cat(t) if t else None for n, t in res.items()}
    res["top_ids"] = None
    if not case["grad"]:
        del res["dlogits"]
    return res


# ------------------------------------------------------------------------------------------------------------- work
def work(case):
    size = 2 if case["dtype"] == "bf16" else 4
    if case["op"] == "bias":
        return {"bytes": 2 * size * case["nh"] * case["Sq"] * case["Sk"], "flops": case["nh"] * case["Sq"] * case["Sk"]}
    if case["op"] == "logp":
        n = case["N"] * case["V"]
        return {"bytes": size * n * (2 if case["grad"] else 1), "flops": n * (8 if case["grad"] else 4)}
    B, Sq, Sk, nh, nkv, hd = (case[n] for n in ("B", "Sq", "Sk", "nh", "nkv", "hd"))
    full = 0.75 if case["mask"] != "none" else 1.0        # the mean share of keys that are no padding
    pairs = Sq * Sk
    if case["causal"] and not case["cache"]:
        pairs = sum(min(max(i + Sk - Sq + 1, 0), Sk) for i in range(Sq))
    queries, keys = B * Sq * nh * hd, B * Sk * nkv * hd
    if case["grad"]:
        return {"bytes": size * (4 * queries + 4 * keys), "flops": 14 * hd * B * nh * pairs * full}
    return {"bytes": size * (2 * queries + 2 * keys * full), "flops": 4 * hd * B * nh * pairs * full}
