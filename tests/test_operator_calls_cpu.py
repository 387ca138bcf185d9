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
