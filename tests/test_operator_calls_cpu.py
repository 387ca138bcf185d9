"""Calls of general attention, relative position bias and token log probabilities that their documentation allows beyond the
ordinary ones: what can be told without a GPU."""
import pytest
import torch
from torch.autograd import forward_ad as fwAD

from distributed_tensorflow_amd.ops import _lib


def test_calls_that_need_their_autograd_function():
    x, y = torch.randn(3), torch.randn(3, requires_grad=True)
    assert not _lib.differentiated(x, None) and _lib.differentiated(x, None, y)
    with torch.no_grad():
        assert not _lib.differentiated(x, y)
        with fwAD.dual_level():                              # a tangent does not ask for requires_grad, nor for grad mode
            assert _lib.differentiated(fwAD.make_dual(x, torch.ones(3)))
    assert not _lib.differentiated(x)


def test_traces_are_refused():
    from torch.fx.experimental.proxy_tensor import make_fx

    def call(t):
        _lib.differentiated(t)
        return t * 2

    x = torch.randn(3)
    for trace in (lambda: torch.jit.trace(call, x), lambda: make_fx(call)(x), lambda: make_fx(call, tracing_mode="fake")(x)):
        with pytest.raises(RuntimeError, match="trace"):
            trace()
    call(x)


def test_attention_key_bias_in_64_bits():
    """A finite bias that 32 bits do not hold masks nothing: its keys share the row where no other is left."""
    from distributed_tensorflow_amd.ops.attention import attention
    q, k, v = (torch.randn(2, n, 2, 16, generator=torch.Generator().manual_seed(n)) for n in (3, 9, 9))
    bias = torch.zeros(2, 9, dtype=torch.float64)
    bias[0] = torch.finfo(torch.float64).min
    bias[0, 4], bias[1, 2] = -torch.inf, torch.finfo(torch.float64).max
    out = attention(q, k, v, bias)
    alone = bias[0] != -torch.inf
    # a mean of 8 numbers: 8 roundings of 2^-24 of their magnitudes, and the softmax's few
    assert float((out[0] - v[0, alone].mean(0)).abs().max()) <= 32 * 2.0 ** -24 * float(v.abs().max())
    assert torch.equal(out[1], v[1, 2].expand(3, 2, 16))


@pytest.mark.parametrize("table", [False, True])
def test_a_call_with_other_words_is_refused(table):
    """A word too few or too many (another order of them, that is) is an error code, before anything is launched. The right
    number comes past that check, to the one of the operands, which are none here."""
    import ctypes
    import struct
    from distributed_tensorflow_amd.ops.relative_bias import bucket_borders
    words = [0] * 55
    words[45:51] = (1, 1, 1, 1, 1, 8)                        # B, Sq, Sk, nh, nkv, hd
    if table:
        words[36:41] = (64, 0, 32, 128, 1)
        words += bucket_borders(32, 128, True)
    lib = _lib.kernels()
    for name in ("dtf_attention_fwd", "dtf_attention_bwd"):
        fn = getattr(lib, name)
        for more in (-1, 1):
            w = (words + [0])[: len(words) + more]
            assert fn(struct.pack(f"{len(w)}q", *w), len(w), ctypes.c_float(1.0), None) == -1
        assert fn(struct.pack(f"{len(words)}q", *words), len(words), ctypes.c_float(1.0), None) == -2


@pytest.mark.parametrize("Sq,Sk", [(1, 9), (4, 11)])
def test_attention_over_the_filled_part_of_a_cache(Sq, Sk):
    """NaN and infinities behind the last query's position, without key_lengths: causal alone keeps them out, of the result
    and of the gradients."""
    from distributed_tensorflow_amd.ops.attention import attention
    filled = torch.tensor([Sk, Sq, Sk - 3], dtype=torch.int32)
    q, k, v = (torch.randn(3, n, 2, 16, generator=torch.Generator().manual_seed(n)) for n in (Sq, Sk, Sk))
    runs = []
    for fill in (0.0, torch.nan):
        kk, vv = k.clone(), v.clone()
        for b, n in enumerate(filled.tolist()):
            kk[b, n:], vv[b, n:] = fill, fill
        leaves = [t.clone().requires_grad_() for t in (q, kk, vv)]
        out = attention(*leaves, causal=True, q_start=filled - Sq)
        runs.append([out, *torch.autograd.grad(out.sum(), leaves)])
    assert all(torch.equal(a, b) for a, b in zip(*runs)) and torch.isfinite(runs[0][0]).all()
