"""Calls of the operators around a decoder layer's products that autograd must not pass over, without a GPU."""

import pytest
import torch
from test_layer_cpu import BF, E4, cache, i32, z

import torch_xdna
from torch_xdna import XdnaError, XdnaUnavailable, generate

FORMATS = [torch.int8, E4]


def floats(c):
    """The places of a cache's tensors that can require grad."""
    return [i for i, t in enumerate(c) if t.is_floating_point()]


@pytest.fixture
def binding(monkeypatch):
    """The binding, with what its calls returned."""
    with pytest.raises(XdnaError):
        torch_xdna.rotary(torch.zeros(3), i32(3), torch.zeros(1))    # loads it
    native, seen = generate._native, []

    class Spy:
        def __getattr__(self, name):
            def call(*args):
                seen.append(getattr(native, name)(*args))
                return seen[-1]

            return call

    monkeypatch.setattr(generate, "_native", Spy())
    return seen


@pytest.mark.parametrize("fmt", FORMATS)
def test_attention_hands_caches_that_require_grad_back(binding, fmt):
    """As an input that requires grad, a scale or a code (of a floating type) makes the custom op make the call, whose result
    raises in backward, where one without history would leave its gradient out without a word."""
    for i in floats(cache(dtype=fmt)):
        c = list(cache(dtype=fmt))
        c[i].requires_grad_()
        with pytest.raises(XdnaUnavailable):                         # raised by the op's call, which is not recorded
            torch_xdna.paged_attention(z(3, 4, 64), *c, i32(3, 2), i32(3))
        assert binding == [None], i
        binding.clear()
        with torch.no_grad(), pytest.raises(XdnaUnavailable):
            torch_xdna.paged_attention(z(3, 4, 64), *c, i32(3, 2), i32(3))
        assert not binding, i                                        # raised by the direct call


def test_attention_over_scales_that_require_grad_raises_in_backward(monkeypatch):
    from test_layer_cpu import _Fake

    monkeypatch.setattr(generate, "_native", _Fake())
    for i in (2, 3):
        c = list(cache())
        c[i].requires_grad_()
        for ns in (torch_xdna, torch.ops.xdna):
            y = ns.paged_attention(z(3, 4, 64, dtype=BF), *c, i32(3, 2), i32(3))
            assert y.requires_grad
            with pytest.raises(RuntimeError, match="autograd"):
                y.sum().backward()


@pytest.mark.parametrize("fmt", FORMATS)
def test_a_cache_that_requires_grad_is_not_written(binding, fmt):
    """What a call writes in place has no history: refused where autograd would want one, as keys that require grad are."""
    for i in floats(cache(dtype=fmt)):
        c = list(cache(dtype=fmt))
        c[i].requires_grad_()
        for more in ({}, dict(q=z(3, 4, 64).requires_grad_())):
            with pytest.raises(XdnaError, match="no gradients"):
                torch_xdna.cache_append(z(3, 2, 64), z(3, 2, 64), *c, i32(3, 2), i32(3), **more)
        with torch.no_grad(), pytest.raises(XdnaUnavailable):
            torch_xdna.cache_append(z(3, 2, 64), z(3, 2, 64), *c, i32(3, 2), i32(3))
