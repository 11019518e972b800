"""The generation operators at the edges of their contracts, without a GPU."""

import pytest
import torch

import torch_xdna
from torch_xdna import XdnaError, kernels


def test_scales_whose_products_overflow_are_refused():
    """The kernels work in powers of two: a scale times log2(e) has to stay finite too."""
    q, k, c = torch.zeros(5, 4, 64).bfloat16(), torch.zeros(5, 2, 64).bfloat16(), torch.zeros(5, 3, 2, 64).bfloat16()
    n = torch.zeros(5, dtype=torch.int32)
    for scale in (2.4e38, 3.0e38, 1e300):
        with pytest.raises(XdnaError, match="scale"):
            torch_xdna.packed_attention(q, k, k, n, scale)
        with pytest.raises(XdnaError, match="scale"):
            torch_xdna.shared_prefix_attention(q, k, k, c, c, n, scale)
    entry = kernels.lib().xdna_packed_attention
    assert entry(None, 8, 8, None, 8, 8, None, 8, 8, None, 1, 5, 4, 2, 64, kernels.BF16, 2.4e38, None, None, 0, None) == -1
    assert b"scale" in kernels.lib().xdna_last_error()


class _Fake:
    """The binding's calls: None where autograd would record them, else zeros of the right shape without history."""

    def launches(self):
        return 1

    def __getattr__(self, name):
        def call(*args):
            if torch.is_grad_enabled() and any(isinstance(a, torch.Tensor) and a.requires_grad for a in args):
                return None
            shape = (*args[0].shape[:-1], len(args[1])) if name == "linear_w4" else args[0].shape
            return torch.zeros(shape, dtype=args[0].dtype)

        return call


def _calls():
    def f(*shape):
        return torch.zeros(*shape, dtype=torch.bfloat16, requires_grad=True)

    n = torch.zeros(5, dtype=torch.int32)
    codes = torch.zeros(9, 128, dtype=torch.uint8)
    one = torch.zeros(3, requires_grad=True)
    tokens = torch.zeros(3, 2, dtype=torch.int32)
    plain = torch.zeros(3, 100)
    q, c = torch.zeros(5, 4, 64).bfloat16(), torch.zeros(5, 3, 2, 64).bfloat16()
    return [lambda ns: ns.packed_attention(f(5, 4, 64), f(5, 2, 64), f(5, 2, 64), n),
            lambda ns: ns.packed_attention(q, q, f(5, 4, 64), n),
            lambda ns: ns.shared_prefix_attention(f(5, 4, 64), f(7, 2, 64), f(7, 2, 64), c, c, n),
            lambda ns: ns.shared_prefix_attention(q, f(7, 2, 64), f(7, 2, 64), f(5, 3, 2, 64), c, n),
            lambda ns: ns.linear_w4(f(2, 200), codes, torch.zeros(9, 4).bfloat16(), 64),
            lambda ns: ns.linear_w4(torch.zeros(2, 200), codes, f(9, 4), 64),
            lambda ns: ns.linear_w4(torch.zeros(2, 200), codes, torch.zeros(9, 4).bfloat16(), 64, f(9)),
            lambda ns: ns.process_logits(f(3, 100)),
            lambda ns: ns.process_logits(plain, tokens, repetition=one),
            lambda ns: ns.process_logits(plain, bias=torch.zeros(100, requires_grad=True))]


def test_gradients_do_not_vanish_in_silence(monkeypatch):
    """The operators have no backward pass. Where an input requires grad, the direct call's result does too and says so
    in backward, as the custom op's; without grad mode both are as ever."""
    from torch_xdna import generate

    monkeypatch.setattr(generate, "_native", _Fake())
    for call in _calls():
        for ns in (torch_xdna, torch.ops.xdna):
            y = call(ns)
            assert y.requires_grad
            with pytest.raises(RuntimeError, match="autograd"):
                y.sum().backward()
            with torch.no_grad():
                assert not call(ns).requires_grad
            with torch.inference_mode():
                call(ns)


def test_the_binding_hands_recorded_calls_back():
    """Each input that may require grad, through the binding's own check (before it looks for a GPU)."""
    from torch_xdna import generate

    seen = []

    class Spy:
        def __getattr__(self, name):
            def call(*args):
                seen.append(getattr(binding, name)(*args))
                return seen[-1]

            return call

    with pytest.raises(XdnaError):
        torch_xdna.process_logits(torch.zeros(3))            # loads the binding
    binding = generate._native
    generate._native = Spy()
    try:
        for call in _calls():
            with pytest.raises(torch_xdna.XdnaUnavailable):  # raised by the op's call, which is not recorded
                call(torch_xdna)
            assert seen == [None]
            seen.clear()
    finally:
        generate._native = binding
