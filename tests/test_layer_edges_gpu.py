"""The operators around a decoder layer's products on the B200 where they are most easily wrong, against their definitions."""

import math

import pytest
import torch
from test_layer_gpu import (E, FORMATS, _clean, check_attention, close, filled, freqs,  # noqa: F401
                            i32, power, randn, rounding, step, table_of, values)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("b,keys", [(1, 60000), (2, 1000), (460, 1000)])
def test_paged_a_peak_without_a_value(cuda, fmt, b, keys):
    """One key that has nearly all of the weight and nothing to say, and many that share the rest: their weights, 2^-21 of
    the peak's, count in full. Work shared out among blocks of threads, in clusters and among warps (460 sequences over one
    set of pages). All small weights are alike, so that a rounding of them is not lost among the signs of others. Tolerance:
    half a step of the weights in f16 (2^-11), four times the scores' 12 sums of 15 at 2^-23 each, 2^-20 for exponentials and
    sums, and the output's rounding; nothing that grows with the number of keys."""
    import torch_xdna

    d, page = 64, 64
    pages = -(-keys // page)
    g = torch.Generator(device="cuda").manual_seed(keys)
    k = torch.zeros(pages, 1, page, d, device="cuda")
    v = torch.randint(8, 15, k.shape, generator=g, device="cuda").float()    # exact in both formats
    q = torch.zeros(b, 1, d, dtype=torch.float16, device="cuda")
    q[..., 0] = 1.0
    one = torch.ones(pages, 1, device="cuda")
    for at in (0, keys // 2, keys - 1):
        kc, vc = k.clone(), v.clone()
        kc[at // page, 0, at % page, 0] = 120.0                              # a score of 15 beside zeros
        vc[at // page, 0, at % page] = 0.0
        c = (kc.to(fmt), vc.to(fmt), one, one)
        table = torch.arange(pages, dtype=torch.int32, device="cuda").expand(b, pages)
        got = torch_xdna.paged_attention(q, *c, table, i32(*[keys] * b), 0.125)
        p = torch.softmax(torch.where(torch.arange(keys, device="cuda") == at, 15.0, 0.0).double(), 0)
        want = (p @ vc[:, 0].reshape(-1, d)[:keys].double()).expand(b, 1, d)
        close(got, want, want * (2.0 ** -11 + 4 * 12 * 15 * 2.0 ** -23 + 2.0 ** -20) + rounding(want, torch.float16))


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("b,keys,t", [(2, 700, 1), (3, 5000, 2), (230, 260, 1)])
def test_paged_scales_that_are_no_powers_of_two(cuda, fmt, b, keys, t):
    """Of a cache that something else has filled: keys and values are code * scale whatever the scale."""
    page, hkv, d = 16, 2, 64
    lens = [(keys * (i + 1)) // b for i in range(b)]
    counts = [-(-n // page) for n in lens]
    c = filled(sum(counts) + 1, hkv, page, d, fmt, seed=b)
    g = torch.Generator(device="cuda").manual_seed(b)
    for s in c[2:]:
        s.mul_(1 + torch.rand(s.shape, generator=g, device="cuda"))
    check_attention(randn(b, t, 4, d, seed=2, dtype=torch.float16), c, table_of(counts, sum(counts) + 1), lens)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("packed", [False, True])
def test_append_behind_scales_that_are_no_powers_of_two(cuda, fmt, packed):
    """Older tokens of a block whose scale is no power of two keep their values, to half a step of the block's new scale: the
    least power of two that holds it and the new tokens. (The product of a code and a factor is itself rounded, to 2^-24.)"""
    import torch_xdna

    page, hkv, d, lo = 32, 3, 64, 9
    for factor, size in ((1.0, 1e-3), (1.37, 1e-3), (1.999, 1e-3), (1.37, 30.0), (1.5, 2000.0)):
        c = filled(2, hkv, page, d, fmt, seed=3)
        c.k_scales.mul_(factor), c.v_scales.mul_(factor)
        old = [x.clone() for x in c]
        n = 4 if packed else 1
        k, v = randn(n, hkv, d, seed=4, scale=size), randn(n, hkv, d, seed=5, scale=size)
        torch_xdna.cache_append(k, v, *c, i32(1).view(1, 1), i32(lo), i32(0, n) if packed else None)
        for i, x in ((0, k), (1, v)):
            new, was = x.double().transpose(0, 1), values(old[i][1], old[2 + i][1])[:, :lo]
            mantissa, e = torch.frexp(old[2 + i][1].double())            # mantissas from 1/2 on
            held = torch.ldexp(torch.ones_like(mantissa), e - (mantissa == 0.5).int())
            scale = torch.maximum(power(new.abs().amax((1, 2)), fmt), held)
            assert torch.equal(c[2 + i][1].double(), scale)
            got, s = values(c[i][1], c[2 + i][1]), scale[:, None, None]
            assert ((got[:, lo:lo + n] - new).abs() <= step(new, s, fmt)).all()
            assert ((got[:, :lo] - was).abs() <= step(was, s, fmt) + was.abs() * E).all()


def test_append_says_that_it_wrote(cuda):
    """A tensor of the cache that autograd saved before an append is noticed in backward, as with the custom op; caches of
    inference mode, which count nothing, are written outside of it too."""
    import torch_xdna

    for ns in (torch_xdna, torch.ops.xdna):
        c, k, table = filled(2, 2, 16, 64, torch.float8_e4m3fn), randn(1, 2, 64), i32(1).view(1, 1)
        for t in c:
            w = torch.ones((), device="cuda", requires_grad=True)
            with torch.enable_grad():
                y = (t.float() if t is c.k or t is c.v else t) * w       # saves scales themselves
                versions = [x._version for x in c]
                ns.cache_append(k, k, *c, table, i32(3))
                assert all(x._version > n for x, n in zip(c, versions))
                if t is c.k_scales or t is c.v_scales:
                    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
                        y.sum().backward()
    with torch.inference_mode():
        c = filled(2, 2, 16, 64, torch.int8)
    before = c.k.clone()
    torch_xdna.cache_append(k, k, *c, table, i32(3))
    assert c.k.is_inference() and not torch.equal(c.k, before)


def test_rotary_angles_far_out(cuda):
    """Positions beyond 32 bits against angles in exact arithmetic: the angle is good to the position times 2^-64 turns, at 2^40
    2^-21.3, 6.5 units of 2^-24; cos and sin as ever 7; within the tolerance of near ones."""
    from fractions import Fraction

    import torch_xdna

    two_pi = 2 * Fraction(314159265358979323846264338327950288419716939937510582097494459, 10 ** 62)
    pos = [2 ** 31 - 1, 2 ** 33 + 12345, 2 ** 37 - 1, -(2 ** 37) + 99, 2 ** 40, 2 ** 40 - 7]
    for base in (1e4, 1e6):
        f = freqs(64, base)
        x = torch.zeros(len(pos), 1, 128, device="cuda")
        x[..., :64] = 1.0                                            # (1, 0) turns to (cos, sin)
        angle = torch.empty(len(pos), 64, dtype=torch.float64)
        for i, n in enumerate(pos):
            for j, y in enumerate(f.tolist()):
                turns = n * Fraction(y) / two_pi
                angle[i, j] = float((turns - (turns.numerator // turns.denominator)) * two_pi)
        want = torch.cat((angle.cos(), angle.sin()), 1)[:, None].cuda()
        for interleaved in (False, True):
            y = x.clone()
            if interleaved:
                y.zero_()[..., ::2] = 1.0
            got = torch_xdna.rotary(y, torch.tensor(pos, device="cuda"), f, interleaved=interleaved)
            if interleaved:
                got = torch.cat((got[..., ::2], got[..., 1::2]), -1)
            close(got, want, torch.full_like(want, 32 * E))


@pytest.mark.parametrize("d", [8, 64, 72, 80, 96, 112, 128, 200, 256])
@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary_norm_of_non_finite_heads(cuda, d, interleaved):
    """Heads with an infinity or a NaN leave the others of their token, which share a warp and its sums, as they were without."""
    import torch_xdna

    t, h = 5, 13
    f, pos, w = freqs(d // 2), torch.arange(t, device="cuda"), randn(h, d, seed=2, dtype=torch.float32)
    for dtype in (torch.float32, torch.bfloat16):
        x = randn(t, h, d, seed=d, dtype=dtype)
        want = torch_xdna.rotary(x, pos, f, 1.0, interleaved, w)
        bad = torch.zeros(t, h, dtype=torch.bool, device="cuda")
        for i, (a, b, e, y) in enumerate(((0, 0, 0, math.inf), (1, 5, d - 1, math.nan), (1, 6, 3, -math.inf), (2, 12, d // 2, math.nan),
                                          (4, 1, 5, math.inf))):
            x[a, b, e], bad[a, b] = y, True
        got = torch_xdna.rotary(x, pos, f, 1.0, interleaved, w)
        assert torch.equal(torch.isfinite(got).all(-1), ~bad)
        assert torch.equal(got[~bad], want[~bad])
