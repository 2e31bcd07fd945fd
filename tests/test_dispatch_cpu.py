"""CPU: when the operators on a paged cache and rotary positions go through the dispatcher."""
import pytest
import torch
from torch.utils._python_dispatch import TorchDispatchMode

from splitd_flash_attn.rotary import _traced


class Passing(TorchDispatchMode):
    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        return func(*args, **(kwargs or {}))


def test_plain_calls_go_past_the_dispatcher():
    x = torch.ones(2)
    assert not _traced(x, None)
    with torch.no_grad():
        assert not _traced(x)
    with torch.inference_mode():
        assert not _traced(x)
    with torch.autocast("cpu", dtype=torch.bfloat16):
        assert not _traced(x)
    with torch.autograd.set_detect_anomaly(True):
        assert not _traced(x)


def test_whatever_watches_operators_sees_them():
    from torch.fx.experimental.proxy_tensor import make_fx

    seen = []

    def fn(x):
        seen.append(_traced(x))
        return x + 1

    x = torch.ones(2)
    with Passing():
        fn(x)
    make_fx(fn)(x)
    make_fx(fn, pre_dispatch=True)(x)
    torch.jit.trace(fn, x, check_trace=False)
    torch.vmap(fn)(x)
    torch.func.grad(lambda y: fn(y).sum())(x)
    torch.func.functionalize(fn)(x)
    fn(torch.nn.Parameter(x))
    assert seen == [True] * len(seen) and len(seen) >= 8
    assert not _traced(x)  # and nothing stays behind
