"""The operators around a decoder layer's products without a GPU: refusals of bad arguments, the shape functions, the C
entries' checks, recorded calls, and the frequencies of rotary positions."""

import math

import pytest
import torch

import torch_xdna
from torch_xdna import XdnaError, XdnaUnavailable, kernels

BF, E4 = torch.bfloat16, torch.float8_e4m3fn


def z(*shape, dtype=BF):
    return torch.zeros(*shape, dtype=dtype)


def i32(*shape):
    return torch.zeros(*shape, dtype=torch.int32)


def f32(*shape):
    return torch.zeros(*shape)


def refuse(fn, *args, match, **kw):
    with pytest.raises(XdnaError, match=match):
        fn(*args, **kw)


def cache(pages=4, heads=2, page=16, dim=64, dtype=torch.int8):
    return torch_xdna.paged_cache(pages, heads, dim, page, dtype, device="cpu")


def test_rotary_refusals():
    f, x, pos, freq = torch_xdna.rotary, z(5, 4, 64), i32(5), f32(32)
    refuse(f, z(5, 64), pos, freq, match="T, H, D")
    refuse(f, x.double(), pos, freq, match="f32, bf16 or f16")
    for d in (4, 12, 264):
        refuse(f, z(5, 4, d), pos, f32(2), match="head dimension")
    for bad in (i32(4), i32(5, 1), f32(5), i32(10)[::2]):
        refuse(f, x, bad, freq, match="positions")
    for bad in (f32(33), freq.double(), f32(8, 4), f32(64)[::2]):
        refuse(f, x, pos, bad, match="inv_freq")
    for bad in (f32(32), f32(3, 64), i32(64), f32(1, 4, 64)):
        refuse(f, x, pos, freq, norm=bad, match="norm")
    for bad in (-1.0, float("nan"), float("inf")):
        refuse(f, x, pos, freq, eps=bad, match="eps")
    for bad in (float("nan"), float("inf")):
        refuse(f, x, pos, freq, factor=bad, match="factor")
    refuse(f, [1], pos, freq, match="not a tensor")
    with pytest.raises(XdnaUnavailable):
        f(x, pos, freq)


def test_add_norm_refusals():
    f, x, w = torch_xdna.add_norm, z(3, 100), f32(100)
    refuse(f, x, z(3, 99), w, match="one shape")
    refuse(f, x, z(100), w, match="one shape")
    refuse(f, x, x.double(), w, match="one shape")
    refuse(f, torch.tensor(1.0), torch.tensor(1.0), w, match="one shape")
    refuse(f, z(3, 0), z(3, 0), f32(0), match="entries")
    refuse(f, z(1, 16385), z(1, 16385), f32(16385), match="entries")
    for bad in (f32(99), f32(1, 100), i32(100)):
        refuse(f, x, x, bad, match="weight")
        refuse(f, x, x, w, post=bad, match="post")
    for bad in (f32(99), f32(3, 1), f32(2, 100), i32(100), f32(1, 3, 100)):
        refuse(f, x, x, w, gate=bad, match="gate")
    refuse(f, x, x, w, scale=float("inf"), match="scale")
    refuse(f, x, x, w, eps=-1e-6, match="eps")
    with pytest.raises(XdnaUnavailable):
        f(x, x, w, w, w)


def test_weights_of_no_dimension():
    one, c, t, n = torch.tensor(1.0), cache(), z(3, 2, dtype=torch.int32), i32(3)
    refuse(torch_xdna.rotary, z(5, 4, 64), i32(5), f32(32), norm=one, match="norm")
    refuse(torch_xdna.rotary, z(5, 4, 64), i32(5), one, match="inv_freq")
    refuse(torch_xdna.add_norm, z(3, 100), z(3, 100), one, match="weight")
    refuse(torch_xdna.add_norm, z(3, 100), z(3, 100), f32(100), post=one, match="post")
    refuse(torch_xdna.add_norm, z(3, 100), z(3, 100), f32(100), gate=one, match="gate")
    refuse(torch_xdna.cache_append, z(3, 2, 64), z(3, 2, 64), *c, t, n, k_norm=one, match="k_norm")
    refuse(torch_xdna.cache_append, z(3, 2, 64), z(3, 2, 64), *c, t, n, q=z(3, 4, 64), q_norm=one, match="q_norm")


def test_paged_cache():
    for dtype in (torch.int8, E4):
        c = cache(3, 5, 32, 128, dtype)
        assert c.k.shape == c.v.shape == (3, 5, 32, 128) and c.k.dtype == c.v.dtype == dtype
        assert c.k_scales.shape == c.v_scales.shape == (3, 5) and c.k_scales.dtype == torch.float32
        assert all(t.is_contiguous() for t in c) and all(not t.float().any() for t in c)
    for args in ((-1, 2, 64), (3, 0, 64), (3, 2, 80), (3, 2, 64, 48)):
        refuse(torch_xdna.paged_cache, *args, device="cpu", match="pages")
    refuse(torch_xdna.paged_cache, 3, 2, 64, dtype=torch.uint8, device="cpu", match="codes")


def test_append_refusals():
    f, k, t, s = torch_xdna.cache_append, z(3, 2, 64), i32(3, 2), i32(3)
    c = cache()
    refuse(f, k, z(4, 2, 64), *c, t, s, match="need")
    refuse(f, z(3, 3, 64), z(3, 3, 64), *c, t, s, match="need")
    refuse(f, z(3, 2, 128), z(3, 2, 128), *c, t, s, match="need")
    refuse(f, k.float(), k.float(), *c, t, s, match="need")
    refuse(f, k, k.half(), *c, t, s, match="need")
    refuse(f, k, k, c.k, c.v[:3], *c[2:], t, s, match="caches")
    refuse(f, k, k, c.k.view(E4), c.v, *c[2:], t, s, match="caches")
    refuse(f, k, k, c.k.view(torch.uint8), c.v.view(torch.uint8), *c[2:], t, s, match="caches")
    for page in (8, 48, 256):
        bad = torch.zeros(4, 2, page, 64, dtype=torch.int8)
        refuse(f, k, k, bad, bad, *c[2:], t, s, match="pages of")
    bad = torch.zeros(4, 2, 16, 96, dtype=torch.int8)
    refuse(f, z(3, 2, 96), z(3, 2, 96), bad, bad, *c[2:], t, s, match="head dimension")
    swapped = torch.zeros(4, 16, 2, 64, dtype=torch.int8).transpose(1, 2)
    refuse(f, k, k, swapped, c.v, *c[2:], t, s, match="contiguous")
    refuse(f, k, k, c.k, c.v, c.k_scales[:3], c.v_scales, t, s, match="scales")
    refuse(f, k, k, c.k, c.v, c.k_scales.half(), c.v_scales, t, s, match="scales")
    for bad in (i32(2, 2), i32(3), i32(3, 2).long(), i32(2, 3).t()):
        refuse(f, k, k, *c, bad, s, match="table")
    for bad in (i32(2), s.long(), i32(3, 1), i32(6)[::2]):
        refuse(f, k, k, *c, t, bad, match="starts")
    refuse(f, k, k, *c, t, s, i32(3), match="table")             # two sequences
    refuse(f, k, k, *c, t, s, i32(0), match="cu_seqlens")
    refuse(f, k, k, *c, t, s, i32(4).long(), match="cu_seqlens")
    refuse(f, k, k, *c, t, s, inv_freq=f32(33), match="inv_freq")
    refuse(f, k, k, *c, t, s, k_norm=f32(3, 64), match="k_norm")
    refuse(f, k, k, *c, t, s, q_norm=f32(64), match="q_norm without q")
    for bad in (z(4, 4, 64), z(3, 0, 64), z(3, 4, 128), z(3, 4, 64, dtype=torch.float16), z(3, 64)):
        refuse(f, k, k, *c, t, s, q=bad, match="q:")
    refuse(f, k, k, *c, t, s, q=z(3, 4, 64), q_norm=f32(2, 64), match="q_norm")
    with pytest.raises(XdnaUnavailable):
        f(k, k, *c, t, s, i32(4), f32(32), 1.0, True, f32(64), z(3, 4, 64), f32(4, 64))


def test_paged_refusals():
    f, q, t, n = torch_xdna.paged_attention, z(3, 4, 64), i32(3, 2), i32(3)
    c = cache()
    refuse(f, z(3, 64), *c, t, n, match="need")
    refuse(f, z(3, 4, 128), *c, t, n, match="need")
    refuse(f, q.float(), *c, t, n, match="bf16 or f16")
    refuse(f, z(3, 3, 64), *c, t, n, match="share")
    refuse(f, z(3, 258, 64), *c, t, n, match="share")
    refuse(f, z(3, 0, 64), *c, t, n, match="share")
    refuse(f, q, c.k, c.v, c.k_scales, c.v_scales[:, :1], t, n, match="scales")
    for bad in (i32(2, 2), i32(3), t.long()):
        refuse(f, q, *c, bad, n, match="table")
    for bad in (i32(2), n.long()):
        refuse(f, q, *c, t, bad, match="lens")
    for s in (0.0, -1.0, float("nan"), 2.4e38):
        refuse(f, q, *c, t, n, scale=s, match="scale")
    with pytest.raises(XdnaUnavailable):
        f(z(3, 2, 4, 64), *c, t, n)


def test_shape_functions():
    from torch._subclasses.fake_tensor import FakeTensorMode

    ops = torch.ops.xdna
    with FakeTensorMode():
        x = z(5, 9, 64)[:, 2:6]
        assert ops.rotary(x, i32(5), f32(32)).shape == (5, 4, 64)
        a, b = ops.add_norm(f32(2, 3, 8), z(2, 3, 8), f32(8))
        assert a.shape == b.shape == (2, 3, 8) and a.dtype == torch.float32 and b.dtype == BF
        c = [torch.zeros(4, 2, 16, 64, dtype=torch.int8) for _ in range(2)] + [f32(4, 2) for _ in range(2)]
        assert ops.cache_append(z(5, 2, 64), z(5, 2, 64), *c, i32(5, 3), i32(5)).shape == (0,)
        assert ops.cache_append(z(5, 2, 64), z(5, 2, 64), *c, i32(5, 3), i32(5), q=x).shape == (5, 4, 64)
        assert ops.paged_attention(z(5, 3, 4, 64), *c, i32(5, 3), i32(5)).shape == (5, 3, 4, 64)


def test_c_entries_refuse_before_the_device():
    """The C entries' own checks of sizes and types come before any device call."""
    L = kernels.lib()
    assert L.xdna_rotary(None, kernels.I32, 1, 1, 64, 8, 8, None, 4, None, 32, 1.0, 0, None, 0, 0, 1e-6, None, None) == -1
    assert L.xdna_rotary(None, kernels.F32, 1, 1, 60, 8, 8, None, 4, None, 8, 1.0, 0, None, 0, 0, 1e-6, None, None) == -2
    assert L.xdna_rotary(None, kernels.F32, 1, 1, 64, 8, 8, None, 4, None, 33, 1.0, 0, None, 0, 0, 1e-6, None, None) == -1
    assert L.xdna_rotary(None, kernels.F32, 1, 1, 64, 8, 8, None, 2, None, 32, 1.0, 0, None, 0, 0, 1e-6, None, None) == -1
    assert L.xdna_add_norm(None, 0, 8, None, 0, 8, 1, 16385, None, 0, None, 0, None, 0, 0, 1.0, 1e-6, None, None, None) == -2
    assert L.xdna_add_norm(None, kernels.I8, 8, None, 0, 8, 1, 8, None, 0, None, 0, None, 0, 0, 1.0, 1e-6, None, None, None) == -1
    append = [None, 8, 8, None, 8, 8, kernels.BF16, 1, 2, 64, None, 0, None, 0, kernels.I8, None, 0, None, 0, 4, 16, None, 0,
              2, None, None, 1, None, 0, 1.0, 0, None, 0, 0, 1e-6, None, 8, 8, 0, None, 0, 0, None, None]
    assert L.xdna_cache_append.argtypes is not None and len(append) == len(L.xdna_cache_append.argtypes)
    for at, bad, code in ((6, kernels.F32, -1), (9, 96, -2), (20, 24, -2), (14, kernels.BF16, -1), (26, 2, -1), (28, 33, -1),
                          (19, -1, -1), (23, 2 ** 30, -1), (8, 0, -1)):
        args = list(append)
        args[at] = bad
        assert L.xdna_cache_append(*args) == code, (at, bad)
    paged = [None, 8, 8, 8, kernels.BF16, 1, 1, 4, 2, 64, None, 0, None, 0, kernels.E4M3, None, 0, None, 0, 4, 16, None, 0, 2,
             None, 1.0, None, None, 0, None]
    assert len(paged) == len(L.xdna_paged_attention.argtypes)
    for at, bad, code in ((4, kernels.F32, -1), (7, 5, -1), (9, 80, -2), (14, kernels.U8, -1), (20, 8, -2), (25, 0.0, -1),
                          (25, 2.4e38, -1), (5, -1, -1), (6, 1 << 30, -1)):
        args = list(paged)
        args[at] = bad
        assert L.xdna_paged_attention(*args) == code, (at, bad)
    assert b"paged_attention" in L.xdna_last_error()


class _Fake:
    """The binding's calls: None where autograd would record them, else results of the right shape without history."""

    def launches(self):
        return 1

    def __getattr__(self, name):
        def call(*args):
            at = [a for i, a in enumerate(args) if not (name == "cache_append" and i in (0, 1, 12))]
            if torch.is_grad_enabled() and any(isinstance(a, torch.Tensor) and a.requires_grad for a in at):
                return None
            if name == "add_norm":
                return torch.zeros_like(args[0]), torch.zeros_like(args[1])
            if name == "cache_append":
                return False if args[13] is None else torch.zeros(args[13].shape)
            return torch.zeros(args[0].shape)

        return call


def _grad(*shape, dtype=BF):
    return torch.zeros(*shape, dtype=dtype, requires_grad=True)


def _calls():
    x, c, t, n = z(3, 4, 64), cache(), i32(3, 2), i32(3)
    return [lambda ns: ns.rotary(_grad(3, 4, 64), n, f32(32)),
            lambda ns: ns.rotary(x, n, f32(32), norm=_grad(64)),
            lambda ns: ns.rotary(x, n, _grad(32, dtype=torch.float32)),
            lambda ns: ns.add_norm(_grad(3, 8), z(3, 8), f32(8))[0],
            lambda ns: ns.add_norm(z(3, 8), _grad(3, 8), f32(8))[1],
            lambda ns: ns.add_norm(z(3, 8), z(3, 8), _grad(8), f32(8))[1],
            lambda ns: ns.add_norm(z(3, 8), z(3, 8), f32(8), _grad(8), None)[0],
            lambda ns: ns.add_norm(z(3, 8), z(3, 8), f32(8), None, _grad(3, 8))[0],
            lambda ns: ns.cache_append(z(3, 2, 64), z(3, 2, 64), *c, t, n, q=_grad(3, 4, 64)),
            lambda ns: ns.cache_append(z(3, 2, 64), z(3, 2, 64), *c, t, n, q=x, q_norm=_grad(64)),
            lambda ns: ns.paged_attention(_grad(3, 4, 64), *c, t, n)]


def test_gradients_do_not_vanish_in_silence(monkeypatch):
    """No operator has a backward pass. Where an input requires grad the direct call's result does too, and says so in
    backward, as the custom op's; without grad mode both are as ever."""
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
    from torch_xdna import generate

    seen = []

    class Spy:
        def __getattr__(self, name):
            def call(*args):
                seen.append(getattr(binding, name)(*args))
                return seen[-1]

            return call

    with pytest.raises(XdnaError):
        torch_xdna.rotary(torch.zeros(3), i32(3), f32(1))        # loads the binding
    binding = generate._native
    generate._native = Spy()
    try:
        for call in _calls():
            with pytest.raises(XdnaUnavailable):                 # raised by the op's call, which is not recorded
                call(torch_xdna)
            assert seen == [None]
            seen.clear()
    finally:
        generate._native = binding


def test_a_cache_keeps_no_gradients():
    f, c, t, n = torch_xdna.cache_append, cache(), i32(3, 2), i32(3)
    refuse(f, _grad(3, 2, 64), z(3, 2, 64), *c, t, n, match="no gradients")
    refuse(f, z(3, 2, 64), _grad(3, 2, 64), *c, t, n, match="no gradients")
    refuse(f, z(3, 2, 64), z(3, 2, 64), *c, t, n, k_norm=_grad(64), match="no gradients")
    with torch.no_grad(), pytest.raises(XdnaUnavailable):
        f(_grad(3, 2, 64), z(3, 2, 64), *c, t, n)


def test_frequencies():
    """Against the formulas, entry by entry; yarn and llama3 leave fast entries and divide slow ones."""
    def near(a, b):
        assert a.dtype == torch.float32 and torch.allclose(a.double(), torch.tensor(b, dtype=torch.float64), rtol=1e-7, atol=0)

    f = torch_xdna.rotary_frequencies
    plain = [1e6 ** (-2 * i / 64) for i in range(32)]
    freq, factor = f(64, 1e6, device="cpu")
    near(freq, plain)
    assert factor == 1.0
    near(f(64, 1e6, "linear", 4.0, device="cpu")[0], [x / 4 for x in plain])
    freq = f(64, 1e6, "ntk", 4.0, device="cpu")[0]
    near(freq, [(1e6 * 4 ** (64 / 62)) ** (-2 * i / 64) for i in range(32)])
    assert abs(float(freq[-1]) / (plain[-1] / 4) - 1) < 1e-6     # the slowest entry is divided by the factor
    turns = [4096 * x / (2 * math.pi) for x in plain]
    freq, factor = f(64, 1e6, "llama3", 8.0, original=4096, device="cpu")
    assert factor == 1.0
    for x, y, n in zip(plain, freq.tolist(), turns):
        want = x if n >= 4 else x / 8 if n <= 1 else x / 8 + (x - x / 8) * (n - 1) / 3
        assert abs(y / want - 1) < 1e-6
    freq, factor = f(64, 1e6, "yarn", 8.0, original=4096, device="cpu")
    assert factor == 1 + 0.1 * math.log(8)
    ratio = [y / x for x, y in zip(plain, freq.tolist())]
    assert all(abs(r - 1) < 1e-6 for r, n in zip(ratio, turns) if n > 50)
    assert all(abs(r - 0.125) < 1e-6 for r, n in zip(ratio, turns) if n < 0.5)
    assert all(a >= b - 1e-6 for a, b in zip(ratio, ratio[1:]))
    for bad in (dict(dim=63), dict(dim=0), dict(dim=64, base=1.0), dict(dim=64, factor=0.5), dict(dim=64, scaling="yarn"),
                dict(dim=64, scaling="what"), dict(dim=64, scaling="llama3", original=4096, low=4.0, high=1.0),
                dict(dim=2, scaling="ntk"), dict(dim=64, factor=float("nan"))):
        refuse(f, **bad, device="cpu", match="rotary_frequencies")
