"""The operators around a decoder layer's products on the B200 against their definitions in 64 bits.

Tolerances, per element, from the arithmetic (u = 2^-8 for bf16, 2^-11 for f16, 2^-24 = e for f32):
  rotary    the root of the mean square: at most 24 sums (half of their error), a division, eps and rsqrtf (2 ulp): 20 e;
            two products with it: 22 e. cos and sin: the angle to 1.6 e, sincospif to 2 ulp, the factor: 7 e at most;
            the turn: 2 e. Together 32 e of factor * (|a| + |b|) for a pair (a, b), and the output's rounding.
  add_norm  a row's sum of squares in at most 42 sums (21 e of its root), rsqrtf 4 e, products: 36 e of z, 2 e of x'; h
            has 36 e of itself, what x' is off by, and as much again by its norm; then the output's rounding.
  append    the values as for rotary without the output's rounding; codes within half a step of them.
  attention the scores' sums of D exact products in steps of 16 (2^-23 each, at most D / 8 + 4 of them); twice that for a
            weight and for their sum; 2^-20 for exponentials and f32 sums; weights rounded to f16 (2^-11), at most 2^-25 of
            the row's largest p * V scale lost per key where they underflow; the output's rounding.
"""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu
E = 2.0 ** -24
U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: E}
HALF = [torch.bfloat16, torch.float16]
FORMATS = [torch.int8, torch.float8_e4m3fn]
TOP = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}


@pytest.fixture(autouse=True)
def _clean(cuda):
    """Each test leaves the device error word clear."""
    from torch_xdna import kernels

    kernels.take_device_error()
    with torch.no_grad():
        yield
    assert kernels.take_device_error() == (0, 0), "a kernel recorded a device-side error"


def randn(*shape, seed=0, dtype=torch.bfloat16, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)


def i32(*x):
    return torch.tensor(list(x), dtype=torch.int32).cuda()


def close(got, want, tol):
    got = got.double()
    assert got.shape == want.shape
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    same = (got == want) | torch.isnan(want)       # infinities too
    off = torch.where(same, 0.0, (got - want).abs() - tol)
    assert float(off.max() if off.numel() else 0.0) <= 0, (
        f"{int((off > 0).sum())} of {off.numel()} values, worst |d| {float((got - want).abs().nan_to_num(posinf=0).max()):.3g}")


def rounding(want, dtype):
    return U[dtype] * want.abs() * 1.001 + (2.0 ** -25 if dtype == torch.float16 else 1e-38)


# ------------------------------------------------------------------ rotary positions
def turned(x, pos, freq, factor=1.0, interleaved=False, norm=None, eps=1e-6):
    """(values, tolerance before rounding) in 64 bits of x [T, H, D]."""
    u = x.double()
    if norm is not None:
        u = u / (u.square().mean(-1, keepdim=True) + eps).sqrt() * norm.double()
    n = 0 if freq is None else len(freq)
    out, tol = u.clone(), 22 * E * u.abs()
    if n:
        angle = pos.double()[:, None] * freq.double()
        c, s = (angle.cos() * factor)[:, None], (angle.sin() * factor)[:, None]
        at = torch.arange(n, device=x.device)
        i, j = (2 * at, 2 * at + 1) if interleaved else (at, at + n)
        a, b = u[..., i], u[..., j]
        out[..., i], out[..., j] = a * c - b * s, b * c + a * s
        tol[..., i] = tol[..., j] = 32 * E * abs(factor) * (a.abs() + b.abs())
    return out, tol + 1e-37


def freqs(n, base=1e4):
    return torch.tensor([base ** (-i / max(n, 1)) for i in range(n)]).cuda()


@pytest.mark.parametrize("dtype", [torch.float32, *HALF])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("d,n", [(64, 32), (128, 64), (128, 16), (128, 5), (80, 16), (96, 12), (256, 32), (8, 4), (8, 1),
                                 (200, 100), (72, 36), (128, 63), (256, 127), (16, 0)])
def test_rotary(cuda, dtype, interleaved, d, n):
    import torch_xdna

    for t, h, far in ((1, 1, 0), (1, 24, 4000), (5, 3, 100000), (67, 9, 131072)):
        x, f = randn(t, h, d, seed=d + t, dtype=dtype, scale=1.5), freqs(n)
        pos = torch.arange(far, far + t, device="cuda", dtype=torch.int32 if t == 5 else torch.int64)
        norm = [None, randn(d, seed=1, dtype=torch.float32), randn(h, d, seed=2, dtype=dtype)][(t + h) % 3]
        got = torch_xdna.rotary(x, pos, f, 1.25, interleaved, norm)
        assert got.dtype == dtype and got.is_contiguous()
        want, tol = turned(x, pos, f, 1.25, interleaved, norm)
        close(got, want, tol + rounding(want, dtype))


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("d,n", [(48, 24), (64, 8), (80, 40), (96, 48), (112, 56)])
def test_rotary_heads_of_a_few_lanes(cuda, d, n, interleaved):
    """Rounds of as many heads as their lanes let into a warp, the last one part full, one warp per token and several."""
    import torch_xdna

    for t, h in ((2, 7), (5, 13), (4801, 11), (4801, 31)):
        x, f, pos = randn(t, h, d, seed=d + h), freqs(n), torch.arange(t, device="cuda")
        norm = randn(h, d, seed=2, dtype=torch.float32) if h != 13 else None
        want, tol = turned(x, pos, f, 1.0, interleaved, norm)
        close(torch_xdna.rotary(x, pos, f, 1.0, interleaved, norm), want, tol + rounding(want, x.dtype))


def test_rotary_far_and_negative_positions(cuda):
    """Angles far out are those of the exact product, for either type of positions."""
    import torch_xdna

    pos = torch.tensor([0, 1, -1, 999999, 2 ** 31 - 1, -2 ** 31, 123456789], device="cuda")
    x, f = randn(len(pos), 3, 128, dtype=torch.float32), freqs(64, 1e6)
    want, tol = turned(x, pos, f)
    close(torch_xdna.rotary(x, pos, f), want, tol + rounding(want, x.dtype))
    assert torch.equal(torch_xdna.rotary(x, pos, f), torch_xdna.rotary(x, pos.int(), f))


def test_rotary_strides_and_many(cuda):
    import torch_xdna

    qkv = randn(4099, 30, 128, seed=3)
    pos, f, w = torch.arange(4099, device="cuda"), freqs(64), randn(24, 128, seed=4, dtype=torch.float32)
    odd = randn(33, 5, 131, seed=5)[..., 1:129]                      # rows off their alignment: copied
    for x, norm in ((qkv[:, :24], w), (qkv[:, 3:27], w), (qkv[:, ::2][:, :12], None), (randn(24, 33, 128, seed=6).transpose(0, 1), w),
                    (odd, None), (qkv[::7, :1], None)):
        p = pos[:len(x)]
        want, tol = turned(x, p, f, norm=None if norm is None else norm[:x.shape[1]])
        close(torch_xdna.rotary(x, p, f, norm=None if norm is None else norm[:x.shape[1]]), want, tol + rounding(want, x.dtype))
    for shape in ((0, 4, 64), (4, 0, 64)):
        assert torch_xdna.rotary(torch.zeros(shape, device="cuda"), pos[:shape[0]], f[:32]).shape == shape


def test_rotary_non_finite(cuda):
    """What is not finite stays within its pair, or within its head where there is a norm."""
    import torch_xdna

    x = randn(3, 4, 64, dtype=torch.float32)
    x[0, 1, 5], x[1, 2, 40], x[2, 3, 63] = math.inf, math.nan, -math.inf
    pos, f = i32(3, 4, 5), freqs(8)                                  # entries from 16 on stay
    got = torch_xdna.rotary(x, pos, f)
    bad = torch.zeros_like(x, dtype=torch.bool)
    bad[0, 1, 5] = bad[0, 1, 13] = bad[1, 2, 40] = bad[2, 3, 63] = True
    assert torch.equal(~torch.isfinite(got), bad) and got[2, 3, 63] == -math.inf
    got = torch_xdna.rotary(x, pos, f, norm=torch.ones(64, device="cuda"))
    assert torch.equal(torch.isfinite(got).all(-1), ~bad.any(-1)) or not torch.isfinite(got[bad]).any()


# ------------------------------------------------------------------ norms around a block
def normed(x, y, w, post=None, gate=None, scale=1.0, eps=1e-6):
    """(x', tol, h, tol) in 64 bits, tolerances with the roundings."""
    z = y.double()
    if post is not None:
        z = z / (z.square().mean(-1, keepdim=True) + eps).sqrt() * post.double()
    z = scale * z if gate is None else scale * z * gate.double()
    new = x.double() + z
    d_new = 38 * E * z.abs() + 2 * E * new.abs() + 1e-37
    inv = 1 / (new.square().mean(-1, keepdim=True) + eps).sqrt()
    h = new * inv * w.double()
    off = d_new.square().sum(-1, keepdim=True).sqrt() / new.square().sum(-1, keepdim=True).sqrt().clamp_min(1e-30)
    d_h = h.abs() * (38 * E + off) + w.double().abs() * inv * d_new
    return new, d_new + rounding(new, x.dtype), h, d_h + rounding(h, y.dtype)


@pytest.mark.parametrize("tx", [torch.float32, *HALF])
@pytest.mark.parametrize("ty", [torch.float32, *HALF])
@pytest.mark.parametrize("t,d", [(1, 1024), (3, 64), (2, 1), (5, 7), (9, 1001), (4, 4093), (1, 16384), (2, 16383), (300, 512),
                                 (301, 1999), (7, 8200), (600, 40)])
def test_add_norm(cuda, tx, ty, t, d):
    import torch_xdna

    x, y = randn(t, d, seed=1, dtype=tx, scale=2.0), randn(t, d, seed=2, dtype=ty)
    w, post = randn(d, seed=3, dtype=torch.float32), randn(d, seed=4, dtype=ty)
    for post, gate, scale in ((None, None, 1.0), (post, None, 0.5), (None, randn(d, seed=5, dtype=tx), -1.5),
                              (post, randn(t, d, seed=6, dtype=ty), 0.7), (None, randn(t, d, seed=7, dtype=torch.float32), 1.0)):
        new, h = torch_xdna.add_norm(x, y, w, post, gate, scale)
        assert new.dtype == tx and h.dtype == ty
        a, da, b, db = normed(x, y, w, post, gate, scale)
        close(new, a, da)
        close(h, b, db)


def test_add_norm_shapes_and_strides(cuda):
    import torch_xdna

    w = randn(96, seed=1, dtype=torch.bfloat16)
    big = randn(2, 5, 4, 200, seed=2)
    cases = [(big[..., :96], big[..., 100:196]), (big[:, :, 1, 3:99], big[:, :, 2, :96]), (big[0, :, 0, :192:2], big[1, :, 3, :192:2]),
             (big[0, 0, 0, :96], big[0, 0, 1, :96]), (randn(3, 97, seed=3)[:, :96], randn(3, 96, seed=4)),
             (randn(3, 96, seed=5).t().contiguous().t(), randn(3, 96, seed=6)), (randn(1, 96, seed=7).expand(4, 96), randn(4, 96, seed=8))]
    for x, y in cases:
        for gate in (None, w, y * 0.5):
            new, h = torch_xdna.add_norm(x, y, w, gate=gate)
            assert new.shape == h.shape == x.shape
            a, da, b, db = normed(x, y, w, gate=gate)
            close(new, a, da)
            close(h, b, db)
    v = randn(97, seed=9, dtype=torch.float32)
    for at in (0, 1):                                                # weights off their alignment
        a, da, b, db = normed(cases[0][0], cases[0][1], v[at:at + 96], v[at:at + 96])
        new, h = torch_xdna.add_norm(cases[0][0], cases[0][1], v[at:at + 96], v[at:at + 96])
        close(new, a, da)
        close(h, b, db)
    for shape in ((0, 96), (2, 0, 96)):
        assert torch_xdna.add_norm(torch.zeros(shape, device="cuda"), torch.zeros(shape, device="cuda"), w)[1].shape == shape


def test_add_norm_non_finite_rows_stay_apart(cuda):
    import torch_xdna

    for d in (64, 77):
        x, y, w = randn(5, d, seed=1, dtype=torch.float32), randn(5, d, seed=2), torch.ones(d, device="cuda")
        y[1, 3], x[3, d - 1] = math.inf, math.nan
        new, h = torch_xdna.add_norm(x, y, w, torch.ones(d, device="cuda"))
        assert torch.isfinite(h[[0, 2, 4]]).all() and torch.isnan(h[[1, 3]]).any(1).all() and torch.isfinite(new[[0, 2, 4]]).all()


# ------------------------------------------------------------------ the paged cache: a model of it
def power(top, fmt):
    """The least power of two that holds the largest values in a format's top."""
    e = (top / TOP[fmt]).log2().round()
    return torch.exp2(torch.where(TOP[fmt] * torch.exp2(e) < top, e + 1, e).clamp_min(-126))


def step(x, scale, fmt):
    """How far a code's value may be from x: half of the distance between codes there."""
    return 0.5 * scale if fmt == torch.int8 else torch.maximum(x.abs() * 2.0 ** -4, scale * 2.0 ** -10)


def values(codes, scales):
    return codes.double() * scales.double()[..., None, None]


class Blocks:
    """What appends do to one tensor of codes: kept values with what they may be off by, before and after."""

    def __init__(self, codes, scales, fmt):
        self.fmt, self.codes, self.scales = fmt, codes.clone(), scales.clone()
        self.touched = torch.zeros(codes.shape[:3], dtype=torch.bool, device=codes.device)

    def check(self, codes, scales, runs, exact=False):
        """runs: (page, first slot, values [n, Hkv, D], tolerance) of this append, a page at most once."""
        seen = torch.zeros(codes.shape[:3], dtype=torch.bool, device=codes.device)
        pages = torch.zeros(len(codes), dtype=torch.bool, device=codes.device)
        for page, lo, x, tol in runs:
            n = len(x)
            x, tol = x.transpose(0, 1), tol.transpose(0, 1)              # [Hkv, n, D]
            low, high = (power((x.abs() - s * tol).amax((1, 2)).clamp_min(0), self.fmt) for s in (1, -1))
            old = self.scales[page].double()
            if lo > 0:
                low, high = torch.maximum(low, old), torch.maximum(high, old)
            new = scales[page].double()
            assert ((new == high) if exact else ((new >= low) & (new <= high))).all(), (page, new, low, high)
            got, s = values(codes[page], scales[page]), new[:, None, None]
            assert ((got[:, lo:lo + n] - x).abs() <= step(x, s, self.fmt) + tol).all(), page
            if lo > 0:
                was = values(self.codes[page], self.scales[page])[:, :lo]
                grown = new > old
                assert torch.equal(codes[page][~grown, :lo].float(), self.codes[page][~grown, :lo].float())
                assert ((got[:, :lo] - was).abs() <= step(was, s, self.fmt))[grown].all()
            seen[page, :, :lo + n] = True
            pages[page] = True
        raw, was = codes.view(torch.uint8), self.codes.view(torch.uint8)
        assert torch.equal(raw[~seen], was[~seen]), "slots behind a sequence, or other pages, were written"
        assert torch.equal(scales[~pages], self.scales[~pages])


def filled(pages, hkv, page, d, fmt, seed=0):
    """A cache full of codes, its scales of several sizes."""
    import torch_xdna

    c = torch_xdna.paged_cache(pages, hkv, d, page, fmt)
    for i, codes in enumerate((c.k, c.v)):
        x = randn(pages, hkv, page, d, seed=seed + i, dtype=torch.float32, scale=TOP[fmt] / 4).clamp(-TOP[fmt], TOP[fmt])
        codes.copy_(x.round() if fmt == torch.int8 else x)
    for i, s in enumerate((c.k_scales, c.v_scales)):
        e = torch.randint(-9, -3, s.shape, generator=torch.Generator(device="cuda").manual_seed(seed + 7 + i), device="cuda")
        s.copy_(torch.exp2(e.float()))
    return c


def table_of(counts, pages, seed=0):
    g = torch.Generator().manual_seed(seed)
    order = torch.randperm(pages, generator=g).int()
    width, at = max([1, *counts]), 0
    t = torch.full((len(counts), width), -1, dtype=torch.int32)
    for i, n in enumerate(counts):
        t[i, :n] = order[at:at + n]
        at += n
    return t.cuda()


def runs_of(x, tol, first, start, n, row, page):
    """The page runs of a sequence's new tokens: rows first .. first + n - 1 of x at positions from start on."""
    out, pos = [], start
    while pos < start + n:
        j, end = pos // page, min(start + n, (pos // page + 1) * page)
        if j < len(row) and 0 <= row[j]:
            at = first + pos - start
            out.append((row[j], pos % page, x[at:at + end - pos], tol[at:at + end - pos]))
        pos = end
    return out


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("hq,hkv,d,n,interleaved", [(16, 8, 128, 64, False), (3, 3, 64, 32, True), (14, 2, 64, 10, False),
                                                    (8, 1, 128, 13, False), (5, 5, 128, 16, True), (9, 3, 64, 0, False)])
@pytest.mark.parametrize("page", [16, 32, 64, 128])
def test_append_tokens(cuda, fmt, dtype, hq, hkv, d, n, interleaved, page):
    """One token of each sequence: at a page's first slot, inside, at its last one; rows that are not stored."""
    import torch_xdna

    starts = [0, 1, page - 1, page, 2 * page + 5, -1, 3 * page, 7, -2 ** 31]   # row 6: past the table
    pages = 20
    table = table_of([3, 1, 1, 2, 3, 3, 3, 1, 0], pages)
    table[7, 0] = pages                                             # no page
    c = filled(pages, hkv, page, d, fmt)
    before = [Blocks(c.k, c.k_scales, fmt), Blocks(c.v, c.v_scales, fmt)]
    qkv = randn(len(starts), hq + 2 * hkv, d, seed=9, dtype=dtype, scale=2.0)
    q, k, v = qkv.split((hq, hkv, hkv), 1)
    f = freqs(n)
    k_norm, q_norm = (None, None) if n == 16 else (randn(d, seed=3, dtype=torch.float32), randn(hq, d, seed=4, dtype=dtype))
    got = torch_xdna.cache_append(k, v, *c, table, i32(*starts), inv_freq=f if n else None, factor=1.1, interleaved=interleaved,
                                  k_norm=k_norm, q=q, q_norm=q_norm)
    pos = torch.tensor(starts, device="cuda")
    want, tol = turned(q, pos, f, 1.1, interleaved, q_norm)
    want[pos < 0] = 0
    close(got, want, tol + rounding(want, dtype))
    (kw, kt), vw = turned(k, pos, f, 1.1, interleaved, k_norm), v.double()
    if not n and k_norm is None:
        kt = torch.zeros_like(kt)
    rows = [[int(p) if 0 <= p < pages else -1 for p in r] for r in table.tolist()]
    for b, codes, scales, x, t in ((before[0], c.k, c.k_scales, kw, kt), (before[1], c.v, c.v_scales, vw, torch.zeros_like(vw))):
        runs = [r for i, s in enumerate(starts) if s >= 0 for r in runs_of(x, t, i, s, 1, rows[i], page)]
        assert len(runs) == 5
        b.check(codes, scales, runs, exact=codes is c.v)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("hq,hkv,d,n,interleaved", [(16, 8, 128, 64, False), (0, 3, 64, 32, True), (14, 2, 64, 10, False),
                                                    (0, 1, 128, 13, False), (4, 34, 64, 32, False), (0, 2, 128, 0, False)])
@pytest.mark.parametrize("page", [16, 32, 64, 128])
def test_append_packed(cuda, fmt, dtype, hq, hkv, d, n, interleaved, page):
    """Packed sequences: empty ones, ones that begin inside a page, that go past the table, that are not stored, and
    tokens of none before and behind them."""
    import torch_xdna

    lens, starts = [5, 0, 1, 2 * page + 3, page, 40, 0, page - 1, 150], [0, 3, page - 1, 7, page, -1, -1, 1, page // 2]
    counts = [-(-max(s + m, 0) // page) for s, m in zip(starts, lens)]
    counts[8] -= 1                                                   # the last tokens have no room
    pages = sum(counts) + 2
    table = table_of(counts, pages)
    table[3, 1] = -7                                                 # a page in the middle is none
    first, total = 2, sum(lens) + 2 + 3
    cu = torch.tensor([first] + lens).cumsum(0).int().cuda()
    c = filled(pages, hkv, page, d, fmt, seed=5)
    before = [Blocks(c.k, c.k_scales, fmt), Blocks(c.v, c.v_scales, fmt)]
    qkv = randn(total, hq + 2 * hkv, d, seed=8, dtype=dtype, scale=1.5)
    q, k, v = qkv.split((hq, hkv, hkv), 1)
    f, norm = freqs(n), None if n == 0 else randn(hkv, d, seed=3, dtype=torch.float32)
    got = torch_xdna.cache_append(k, v, *c, table, i32(*starts), cu, f if n else None, interleaved=interleaved, k_norm=norm,
                                  q=q if hq else None)
    pos = torch.full((total,), -1, dtype=torch.long)
    at = first
    for s, m in zip(starts, lens):
        if s >= 0:
            pos[at:at + m] = torch.arange(s, s + m)
        at += m
    pos = pos.cuda()
    if hq:
        want, tol = turned(q, pos, f, 1.0, interleaved)
        want[pos < 0] = 0
        close(got, want, tol + rounding(want, dtype))
    else:
        assert got is None
    kw, kt = turned(k, pos, f, 1.0, interleaved, norm)
    if n == 0:
        kt = torch.zeros_like(kt)
    rows = table.tolist()
    for b, codes, scales, x, t in ((before[0], c.k, c.k_scales, kw, kt), (before[1], c.v, c.v_scales, v.double(), torch.zeros_like(kt))):
        runs, at = [], first
        for i, (s, m) in enumerate(zip(starts, lens)):
            if s >= 0:
                runs += runs_of(x, t, at, s, m, rows[i][:counts[i]], page)
            at += m
        b.check(codes, scales, runs, exact=codes is c.v or n == 0)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("packed", [False, True])
def test_append_scales_exactly(cuda, fmt, packed):
    """Largest values at, just above and just below top * 2^e, zeros, tiny and huge ones, and what is not finite."""
    import torch_xdna

    top, page = TOP[fmt], 16
    tops = [top * 2.0 ** -4, top * 2.0 ** -4 * (1 + 2 ** -7), top * 2.0 ** -4 * (1 - 2 ** -7), 0.0, 1e-38, 2.0 ** -133, 3e38, 1.0, 2.0]
    x = torch.zeros(len(tops) + 2, 2, 64).bfloat16()
    for i, t in enumerate(tops):
        x[i, 0, 5], x[i, 0, 9], x[i, 1, 63] = t, -t / 3, -t
    x[len(tops), 0, 3], x[len(tops) + 1, 1, 4] = math.nan, -math.inf
    x[len(tops):, :, 7] = 1.0
    x = x.cuda()
    n = len(x)
    c = torch_xdna.paged_cache(n, 2, 64, page, fmt)
    table = torch.arange(n, dtype=torch.int32, device="cuda").view(-1, 1)
    cu = torch.arange(n + 1, dtype=torch.int32, device="cuda") if packed else None
    torch_xdna.cache_append(x, x, *c, table, torch.zeros(n, dtype=torch.int32, device="cuda"), cu)
    for codes, scales in ((c.k, c.k_scales), (c.v, c.v_scales)):
        want = power(x.double().abs().amax(2), fmt)
        odd = torch.isnan(x).any(2) | torch.isinf(x).any(2)
        assert torch.isnan(scales[odd]).all() and int(odd.sum()) == 2
        assert torch.equal(scales[~odd].double(), want[~odd])
        got = values(codes, scales)[:, :, 0]
        ok = (got - x.double()).abs() <= step(x.double(), want[..., None], fmt)
        assert ok[~odd].all() and torch.isnan(got[odd]).all()
        assert not codes[odd].float().any()
    # the block stays as it is until its page starts anew
    one = torch.ones_like(x)
    torch_xdna.cache_append(one, one, *c, table, torch.ones(n, dtype=torch.int32, device="cuda"), cu)
    assert torch.equal(torch.isnan(c.k_scales), odd)
    torch_xdna.cache_append(one, one, *c, table, torch.zeros(n, dtype=torch.int32, device="cuda"), cu)
    assert torch.equal(c.k_scales.double(), power(torch.ones(n, 2, dtype=torch.float64, device="cuda"), fmt))


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("page", [16, 64])
def test_append_growing_values(cuda, fmt, page):
    """A page whose every token is larger than the one before: int8 codes stay within a step of the final scale, however
    often they were rounded; e4m3 ones within half a step and what lies below its lowest value."""
    import torch_xdna

    hkv, d = 3, 128
    x = randn(page, hkv, d, dtype=torch.float32) * torch.exp2(torch.arange(page, device="cuda") * 0.7)[:, None, None]
    x = x.bfloat16()
    c, table = torch_xdna.paged_cache(2, hkv, d, page, fmt), i32(1).view(1, 1)
    for t in range(page):
        torch_xdna.cache_append(x[t:t + 1], x[t:t + 1], *c, table, i32(t))
    want, scale = x.double().transpose(0, 1), c.k_scales[1].double()[:, None, None]
    assert torch.equal(scale.flatten(), power(x.double().abs().amax((0, 2)), fmt))
    off = (values(c.k[1], c.k_scales[1]) - want).abs()
    assert (off <= (scale if fmt == torch.int8 else want.abs() * 2.0 ** -4 + scale * 2.0 ** -9)).all()
    whole = torch_xdna.paged_cache(2, hkv, d, page, fmt)            # the same tokens in one call
    torch_xdna.cache_append(x, x, *whole, table, i32(0), i32(0, page))
    assert torch.equal(whole.k_scales, c.k_scales)
    assert ((values(whole.k[1], whole.k_scales[1]) - want).abs() <= step(want, scale, fmt)).all()


def test_append_strides(cuda):
    """Keys and values of one allocation, page by page, rows that have to be copied, and tables with a pitch."""
    import torch_xdna

    kv = torch.zeros(6, 2, 4, 32, 64, dtype=torch.int8, device="cuda")
    scales = torch.zeros(6, 2, 4, device="cuda")
    c = (kv[:, 0], kv[:, 1], scales[:, 0], scales[:, 1])
    same = torch_xdna.paged_cache(6, 4, 64, 32)
    x = randn(70, 9, 131, seed=4)
    k, v = x[:, 1:5, 2:66], x[:, 5:9, 3:67]
    table = i32(3, 5, 1, 9, 0, 2, 4, 9).view(2, 4)[:, :3]
    for cache in (c, same):
        a = k if cache is c else k.contiguous()
        torch_xdna.cache_append(a, v, *cache, table, i32(0, 31), i32(0, 60, 70), freqs(32))
        torch_xdna.cache_append(a[:2], v[:2], *cache, table, i32(60, 41), inv_freq=freqs(32))
    for a, b in zip(c, same):
        assert torch.equal(a, b)
    assert torch_xdna.cache_append(k[:0], v[:0], *c, table[:0], i32()) is None
    assert torch_xdna.cache_append(k, v, *c, table[:0], i32(), i32(0), q=k).eq(0).all()   # no sequence: zeros


# ------------------------------------------------------------------ attention over it
def attended(q, c, table, lens, scale=None):
    """(o, tol) in 64 bits; q [B, T, Hq, D]."""
    b, t, hq, d = q.shape
    pages, hkv, page = c[0].shape[:3]
    scale = d ** -0.5 if scale is None else scale
    o = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    tol = torch.zeros_like(o)
    rep, top = hq // hkv, TOP[c[0].dtype]
    for i, n in enumerate(lens):
        n = min(max(n, 0), table.shape[1] * page)
        if n == 0:
            continue
        ids = table[i, :-(-n // page)].long()
        good = ((ids >= 0) & (ids < pages)).repeat_interleave(page)[:n]
        ids = ids.clamp(0, max(pages - 1, 0))
        s = c[3][ids].double().repeat_interleave(page, 0)[:n]                              # [n, Hkv]
        k, v = (values(x[ids], y[ids]).transpose(1, 2).reshape(-1, hkv, d)[:n] for x, y in ((c[0], c[2]), (c[1], c[3])))
        for j in range(t):
            see = n - t + j + 1
            if see <= 0 or not good[:see].any():
                continue
            at = good[:see].nonzero()[:, 0]
            for h in range(hkv):
                qr = q[i, j, h * rep:(h + 1) * rep].double()
                z = qr @ k[at, h].t() * scale
                size = (qr.abs() @ k[at, h].abs().t() * scale).amax(1, keepdim=True)
                p = torch.softmax(z, 1)
                o[i, j, h * rep:(h + 1) * rep] = p @ v[at, h]
                a = p @ v[at, h].abs()
                lost = (len(at) + 1) * 2.0 ** -25 * top * (p * s[at, h]).amax(1, keepdim=True)
                e_s = (d / 8 + 4) * 2.0 ** -23 * size
                tol[i, j, h * rep:(h + 1) * rep] = a * (2.0 ** -11 + 4 * e_s + 2.0 ** -20) + lost + rounding(o[i, j, h * rep:(h + 1) * rep].abs() + a, q.dtype)
    return o, tol


def check_attention(q, c, table, lens, scale=None):
    import torch_xdna

    got = torch_xdna.paged_attention(q, *c, table, i32(*lens), scale)
    assert got.shape == q.shape and got.dtype == q.dtype and got.is_contiguous()
    q4 = q if q.dim() == 4 else q[:, None]
    want, tol = attended(q4, c, table, lens, scale)
    close(got.view(want.shape), want, tol)
    return got


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("hq,hkv,d", [(16, 8, 128), (8, 8, 64), (14, 2, 64), (6, 1, 128), (20, 1, 64), (128, 1, 128), (24, 3, 128)])
@pytest.mark.parametrize("page", [16, 32, 64, 128])
def test_paged(cuda, fmt, dtype, hq, hkv, d, page):
    lens = [1, 15, 16, 17, 0, 31, 33, 64, 127, 128, 129, 300, 0, 513]
    counts = [-(-n // page) for n in lens]
    c = filled(sum(counts) + 3, hkv, page, d, fmt, seed=hq)
    check_attention(randn(len(lens), hq, d, seed=1, dtype=dtype), c, table_of(counts, sum(counts) + 3), lens)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("hq,hkv,d,t", [(16, 8, 128, 2), (16, 8, 128, 4), (16, 8, 128, 5), (14, 2, 64, 3), (8, 8, 64, 33),
                                        (7, 1, 128, 9), (12, 4, 64, 6)])
def test_paged_several_tokens(cuda, fmt, hq, hkv, d, t):
    """The last T tokens of each sequence, also of ones that are shorter than T."""
    lens, page = [t, t + 1, 1, t - 1, 0, 40, 130, 257], 16 if d == 64 else 32
    counts = [-(-n // page) for n in lens]
    c = filled(sum(counts) + 1, hkv, page, d, fmt, seed=t)
    check_attention(randn(len(lens), t, hq, d, seed=2), c, table_of(counts, sum(counts) + 1), lens)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("d,page", [(128, 64), (64, 16)])
def test_paged_many_short(cuda, fmt, d, page):
    """Enough sequences for shares of warps: lengths from none to a few tiles, whole runs without any."""
    g = torch.Generator().manual_seed(3)
    lens = torch.randint(0, 260, (230,), generator=g).tolist()
    lens[40:80] = [0] * 40
    lens[-1] = 0
    counts = [-(-n // page) for n in lens]
    c = filled(sum(counts) + 3, 4, page, d, fmt)
    table = table_of(counts, sum(counts) + 3)
    check_attention(randn(len(lens), 8, d, seed=5), c, table, lens)
    check_attention(randn(len(lens), 3, 8, d, seed=6), c, table, lens)
    check_attention(randn(len(lens), 5, 8, d, seed=7), c, table, lens)
    check_attention(randn(len(lens), 8, d, seed=5), c, table, [0] * len(lens))


@pytest.mark.parametrize("fmt", FORMATS)
def test_paged_long(cuda, fmt):
    """Lengths far apart, so that shares begin and end anywhere."""
    lens, page, hkv, d = [20011, 1, 7000, 64, 0, 3333], 64, 2, 128
    counts = [-(-n // page) for n in lens]
    c = filled(sum(counts) + 1, hkv, page, d, fmt)
    table = table_of(counts, sum(counts) + 1)
    check_attention(randn(len(lens), 4, d, seed=3), c, table, lens)
    check_attention(randn(len(lens), 2, 4, d, seed=4, dtype=torch.float16), c, table, lens, scale=0.3)
    small = [40, 1, 70, 64, 0, 33]                                   # few keys in a table with much room
    check_attention(randn(len(lens), 4, d, seed=3), c, table, small)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("hq,hkv,d,t", [(16, 8, 128, 1), (14, 2, 64, 4), (4, 4, 64, 1), (12, 1, 128, 1)])
def test_paged_at_the_borders_of_its_manners(cuda, fmt, hq, hkv, d, t):
    """Tables as wide as those from which on the work is shared out in another manner, one page less and one more, with
    sequences that fill them, that hardly begin, and none."""
    page = 32
    for b, keys in ((1, 2560), (1, 2592), (2, 160), (5, 1024), (5, 1056), (60, 1024), (60, 1056), (60, 128)):
        lens = [keys, 1, 0, keys // 2, 33][:b] + [(7 * i) % 60 for i in range(b - 5)]
        counts = [-(-n // page) for n in lens]
        c = filled(sum(counts) + 1, hkv, page, d, fmt, seed=b)
        table = table_of(counts, sum(counts) + 1)
        assert table.shape[1] * page == keys
        check_attention(randn(b, t, hq, d, seed=keys) if t > 1 else randn(b, hq, d, seed=keys), c, table, lens)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("hq,t,d", [(2, 1, 128), (10, 2, 64)])
@pytest.mark.parametrize("b,keys", [(370, 1024), (443, 256), (190, 896), (125, 960), (90, 1024), (77, 640), (60, 2048), (50, 2048), (40, 1920)])
def test_paged_as_many_sequences_as_the_multiprocessors_hold(cuda, fmt, hq, t, d, b, keys):
    """One to eight blocks of threads for each sequence, with lengths from none to the table's and parts without a key."""
    g = torch.Generator().manual_seed(b)
    lens = [keys, 0, 1, keys - 1] + torch.randint(0, keys, (b - 4,), generator=g).tolist()
    counts = [-(-n // 64) for n in lens]
    c = filled(sum(counts) + 1, 1, 64, d, fmt, seed=b)
    table = table_of(counts, sum(counts) + 1)
    check_attention(randn(b, t, hq, d, seed=keys), c, table, lens)


def test_paged_lengths_and_pages_that_are_none(cuda):
    """Lengths below zero and beyond the table; entries of the table that are no page, inside a tile and for whole ones;
    no pages, no table and no rows at all."""
    import torch_xdna

    page, hkv, d = 16, 2, 64
    c = filled(12, hkv, page, d, torch.int8)
    table = i32(3, -1, 5, 12, 7, 1, 2 ** 31 - 1, -2 ** 31, -1, -1, 0, 2).view(3, 4)
    for lens in ([64, 64, 64], [33, 20, 40], [1000, -5, 2 ** 31 - 1], [16, 17, 32]):
        check_attention(randn(3, 4, d, seed=1), c, table, lens)
        check_attention(randn(3, 3, 4, d, seed=2), c, table, lens)
    q = randn(3, 4, d)
    assert not torch_xdna.paged_attention(q, *c, table[:, :0], i32(5, 6, 7)).any()
    none = torch_xdna.paged_cache(0, hkv, d, page)
    assert not torch_xdna.paged_attention(q, *none, table, i32(5, 6, 7)).any()
    assert torch_xdna.paged_attention(q[:0], *c, table[:0], i32()).shape == (0, 4, d)
    assert torch_xdna.paged_attention(q[:, None][:, :0], *c, table, i32(1, 2, 3)).shape == (3, 0, 4, d)
    torch_xdna.cache_append(q[:, :2], q[:, :2], *none, table, i32(0, 1, 2))


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("page", [16, 64])
def test_paged_what_is_not_read(cuda, fmt, page):
    """Codes behind the last token, in whatever bits, and scales of other blocks do not matter; a scale of NaN makes the
    rows that see its block NaN, and no others."""
    import torch_xdna

    hkv, d, lens = 2, 128, [page + 3, 5, 3 * page]
    counts = [2, 1, 3]
    c = filled(8, hkv, page, d, fmt)
    table = table_of(counts, 8)
    q = randn(3, 2, 4, d, seed=1)
    want = check_attention(q, c, table, lens)
    for i, n in enumerate(lens):
        last = int(table[i, counts[i] - 1])
        if n % page:
            for x in (c.k, c.v):
                x.view(torch.uint8)[last, :, n % page:] = 0x7f
    for p in set(range(8)) - set(table.flatten().tolist()):
        for s in c[2:]:
            s[p] = math.nan
        for x in c[:2]:
            x.view(torch.uint8)[p] = 0xff
    assert torch.equal(torch_xdna.paged_attention(q, *c, table, i32(*lens)), want)
    c.v_scales[int(table[0, 1]), 1] = math.nan                      # seen by both rows of head 1 of sequence 0
    c.k_scales[int(table[2, 2]), 0] = math.nan
    got = torch_xdna.paged_attention(q, *c, table, i32(*lens))
    bad = torch.zeros_like(q, dtype=torch.bool)
    bad[0, :, 2:], bad[2, :, :2] = True, True
    assert torch.equal(torch.isnan(got), bad) and torch.equal(got[~bad], want[~bad])
    # the row before the block's first token does not see it
    lens[0] = page + 1
    want = torch_xdna.paged_attention(q, *c, table, i32(*lens))
    assert torch.isfinite(want[0, 0]).all() and torch.isnan(want[0, 1, 2:]).all()


@pytest.mark.parametrize("fmt", FORMATS)
def test_paged_scales_far_apart(cuda, fmt):
    """Blocks whose scales differ by thirty orders of two, for keys and for values: the weights that meet V are full where
    they count, and blocks without keys to speak of do not overflow."""
    page, hkv, d, lens = 16, 1, 64, [400]
    for spread_k, spread_v in ((0, 30), (30, 0), (12, 100), (0, 126)):
        c = filled(25, hkv, page, d, fmt, seed=spread_v)
        e = torch.arange(25, device="cuda").float() / 24
        c.k_scales[:, 0], c.v_scales[:, 0] = torch.exp2((-9 - spread_k * e).round()), torch.exp2((-spread_v * e.flip(0)).round())
        for order in (torch.arange(25), torch.arange(24, -1, -1)):
            check_attention(randn(1, 4, d, seed=1, dtype=torch.float16), c, order.int().cuda().view(1, -1), lens)
    c.v_scales.fill_(0.0)                                            # blocks of zeros
    c.v.zero_()
    assert not check_attention(randn(1, 4, d, seed=1), c, torch.arange(25).int().cuda().view(1, -1), lens).any()


def test_paged_queries_of_any_size(cuda):
    """Queries far above and below one, and peaked scores."""
    import torch_xdna

    page, hkv, d, lens = 32, 2, 64, [200, 77]
    c = filled(12, hkv, page, d, torch.int8)
    table = table_of([7, 3], 12)
    q = randn(2, 4, d, seed=1)
    for factor, scale in ((1e30, 1e-31), (1e-30, 1e29), (3e37, 1e-38), (1e-38, 1e36), (100.0, None)):
        check_attention((q.float() * factor).bfloat16(), c, table, lens, scale)
    check_attention((q.float() * 300).half(), c, table, lens)
    q[0, 1] = 0
    q[1, 2, 7], q[1, 0, 3] = math.nan, math.inf
    got = torch_xdna.paged_attention(q, *c, table, i32(*lens))
    assert torch.isfinite(got[0]).all() and torch.isfinite(got[1, [1, 3]]).all() and torch.isnan(got[1, 2]).all()


def test_paged_strides(cuda):
    import torch_xdna

    kv = filled(10, 4, 32, 64, torch.float8_e4m3fn)
    both = torch.stack((kv.k.view(torch.uint8), kv.v.view(torch.uint8)), 1)
    scales = torch.stack((kv.k_scales, kv.v_scales), 1)
    c = (both[:, 0].view(torch.float8_e4m3fn), both[:, 1].view(torch.float8_e4m3fn), scales[:, 0], scales[:, 1])
    qkv, wide = randn(4, 16, 70, seed=2), torch.zeros(4, 9, dtype=torch.int32, device="cuda")
    wide[:, :3] = i32(1, 2, 3, 9, 8, 7, 0, 4, 5, 6, 3, 1).view(4, 3)
    lens = [70, 96, 5, 33]
    want = torch_xdna.paged_attention(qkv[:, :8, 3:67].contiguous(), *kv, wide[:, :3].contiguous(), i32(*lens))
    for q in (qkv[:, :8, 3:67], qkv[:, :8, 3:67].contiguous()):
        assert torch.equal(torch_xdna.paged_attention(q, *c, wide[:, :3], i32(*lens)), want)
    check_attention(qkv[:, :8, 3:67], c, wide[:, :3], lens)
    t = randn(4, 8, 3, 64, seed=4).transpose(1, 2)                   # [B, T, Hq, D] by another order
    check_attention(t, c, wide[:, :3], lens)


def test_offsets_past_32_bits(cuda):
    """Pages more than 2^32 bytes from the first: written, read, and the table at its far end."""
    import torch_xdna

    hkv, page, d, pages = 8, 128, 128, 40000                         # 131072 bytes a page, 5.2 GB each
    if torch.cuda.mem_get_info()[0] < 14 << 30:
        pytest.skip("needs 14 GB")
    codes = [torch.empty(pages, hkv, page, d, dtype=torch.int8, device="cuda") for _ in range(2)]
    scales = [torch.zeros(pages, hkv, device="cuda") for _ in range(2)]
    c, near = (*codes, *scales), torch_xdna.paged_cache(4, hkv, d, page)
    far, low = i32(pages - 1, 33000, 39998, 1).view(2, 2), i32(3, 2, 1, 0).view(2, 2)
    k, v = randn(300, hkv, d, seed=1), randn(300, hkv, d, seed=2)
    for cache, table in ((c, far), (near, low)):
        torch_xdna.cache_append(k, v, *cache, table, i32(0, 0), i32(0, 200, 300), freqs(64))
        torch_xdna.cache_append(k[:2], v[:2], *cache, table, i32(200, 100), inv_freq=freqs(64))
    for a, b in zip(c, near):
        assert torch.equal(a[far.flatten().long()], b[low.flatten().long()])
    q = randn(2, 16, d, seed=3)
    assert torch.equal(torch_xdna.paged_attention(q, *c, far, i32(201, 101)), torch_xdna.paged_attention(q, *near, low, i32(201, 101)))


# ------------------------------------------------------------------ all of them as they are used
def test_results_do_not_depend_on_the_run(cuda):
    import torch_xdna

    page, hkv, d = 64, 2, 128
    lens = [5000, 33, 900, 0, 64, 7]
    counts = [-(-n // page) for n in lens]
    c = filled(sum(counts), hkv, page, d, torch.float8_e4m3fn)
    table, q = table_of(counts, sum(counts)), randn(len(lens), 8, d)
    want = torch_xdna.paged_attention(q, *c, table, i32(*lens))
    for _ in range(5):
        assert torch.equal(torch_xdna.paged_attention(q, *c, table, i32(*lens)), want)


def test_streams_and_graphs(cuda):
    """A decode step captured once and replayed with other lengths, tokens and tables, on another stream than the one that
    made the tensors; two graphs in turn."""
    import torch_xdna

    b, hq, hkv, d, page = 3, 8, 4, 64, 16
    f, w = freqs(32), torch.ones(hq * d, device="cuda")
    make = lambda: filled(30, hkv, page, d, torch.int8, seed=1)  # noqa: E731
    table = table_of([8, 8, 8], 30)
    state = dict(qkv=randn(b, hq + 2 * hkv, d, seed=1), starts=i32(0, 20, 100), x=randn(b, hq * d, seed=2, dtype=torch.float32))

    def layer(s, c):
        q, k, v = s["qkv"].split((hq, hkv, hkv), 1)
        q = torch_xdna.cache_append(k, v, *c, table, s["starts"], inv_freq=f, q=q)
        o = torch_xdna.paged_attention(q, *c, table, s["starts"] + 1)
        return torch_xdna.add_norm(s["x"], torch_xdna.rotary(o, s["starts"], f).flatten(1), w)

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graphs = []
    with torch.cuda.stream(stream):
        for _ in range(2):
            c = make()
            layer(state, c)
            torch.cuda.synchronize()
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=stream):
                out = layer(state, c)
            graphs.append((g, c, out))
    torch.cuda.synchronize()
    plain = make()
    for _, c, _ in graphs:
        for x, y in zip(c, plain):
            x.copy_(y)
    for step in range(6):
        state["qkv"].copy_(randn(b, hq + 2 * hkv, d, seed=10 + step))
        torch.cuda.synchronize()
        want = layer(state, plain)
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            for g, c, out in graphs:
                g.replay()
        torch.cuda.synchronize()
        for g, c, out in graphs:
            assert all(torch.equal(x, y) for x, y in zip(out, want))
            assert all(torch.equal(x, y) for x, y in zip(c, plain))
        state["starts"] += 1


def test_two_streams_at_once(cuda):
    import torch_xdna

    page, hkv, d = 64, 4, 128
    lens = [700, 64, 1, 2000]
    counts = [-(-n // page) for n in lens]
    c = filled(sum(counts), hkv, page, d, torch.int8)
    table, n = table_of(counts, sum(counts)), i32(*lens)
    qs = [randn(4, 8, d, seed=s) for s in range(2)]
    want = [torch_xdna.paged_attention(q, *c, table, n) for q in qs]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in qs], [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(torch_xdna.paged_attention(qs[i], *c, table, n))
    torch.cuda.synchronize()
    assert all(torch.equal(x, want[i]) for i in range(2) for x in got[i])


def test_custom_ops(cuda):
    """The same calls as torch.ops.xdna.*, also through torch.compile's functionalisation of the append."""
    import torch_xdna

    ops, f = torch.ops.xdna, freqs(32)
    x, pos = randn(5, 4, 64), torch.arange(5, device="cuda")
    assert torch.equal(ops.rotary(x, pos, f), torch_xdna.rotary(x, pos, f))
    w = torch.ones(64, device="cuda")
    for a, b in zip(ops.add_norm(x, x, w, None, None, 0.5), torch_xdna.add_norm(x, x, w, scale=0.5)):
        assert torch.equal(a, b)
    table, starts = table_of([1] * 5, 6), i32(0, 1, 2, 3, 4)

    def both(x, c):
        q = ops.cache_append(x[:, :2], x[:, 2:], *c, table, starts, None, f, q=x)
        return ops.paged_attention(q, *c, table, starts + 1)

    def direct(x, c):
        q = torch_xdna.cache_append(x[:, :2], x[:, 2:], *c, table, starts, inv_freq=f, q=x)
        return torch_xdna.paged_attention(q, *c, table, starts + 1)

    caches = [filled(6, 2, 16, 64, torch.int8) for _ in range(3)]
    want = direct(x, caches[0])
    assert torch.equal(both(x, caches[1]), want)
    assert torch.equal(torch.compile(both, backend="aot_eager")(x, caches[2]), want)
    for c in caches[1:]:
        assert all(torch.equal(a, b) for a, b in zip(c, caches[0]))
    before = torch_xdna.stats.launches
    torch_xdna.paged_attention(x, *caches[0], table, starts)
    assert torch_xdna.stats.launches == before + 1      # a cluster per sequence and key head: no second kernel


@pytest.mark.parametrize("fmt", FORMATS)
def test_prompts_then_tokens(cuda, fmt):
    """Prompts appended packed, then tokens one by one and three at once: every step's attention is that over the keys and
    values themselves, to what 8 bits leave of them."""
    import torch_xdna

    hq, hkv, d, page = 8, 4, 64, 32
    lens = [37, 1, 90]
    table, f = table_of([5, 3, 6], 16), freqs(32)
    c = torch_xdna.paged_cache(16, hkv, d, page, fmt)
    kept = [[], [], []]
    total = sum(lens)
    k, v = randn(total, hkv, d, seed=1), randn(total, hkv, d, seed=2)
    cu = torch.tensor([0] + lens).cumsum(0).int().cuda()
    torch_xdna.cache_append(k, v, *c, table, i32(0, 0, 0), cu, f)
    at = 0
    for i, n in enumerate(lens):
        pos = torch.arange(n, device="cuda")
        kept[i] = [turned(k[at:at + n], pos, f)[0], v[at:at + n].double()]
        at += n
    have = list(lens)
    for step in range(8):
        t = 3 if step % 4 == 3 else 1
        qkv = randn(3 * t, hq + 2 * hkv, d, seed=20 + step)
        q, k, v = qkv.split((hq, hkv, hkv), 1)
        cu = torch.arange(0, 3 * t + 1, t, dtype=torch.int32, device="cuda") if t > 1 else None
        q = torch_xdna.cache_append(k, v, *c, table, i32(*have), cu, f, q=q)
        for i in range(3):
            pos = torch.arange(have[i], have[i] + t, device="cuda")
            kept[i][0] = torch.cat((kept[i][0], turned(k[i * t:(i + 1) * t], pos, f)[0]))
            kept[i][1] = torch.cat((kept[i][1], v[i * t:(i + 1) * t].double()))
            have[i] += t
        got = check_attention(q.view(3, t, hq, d), c, table, have)
        for i in range(3):
            for h in range(hq):
                z = q.view(3, t, hq, d)[i, t - 1, h].double() @ kept[i][0][:, h // 2].t() * d ** -0.5
                want = torch.softmax(z, 0) @ kept[i][1][:, h // 2]
                off = float((got[i, t - 1, h].double() - want).norm() / kept[i][1][:, h // 2].norm(dim=1).mean())
                assert off < 0.05, (step, i, h, off)                # 8-bit codes: 1 to 3 % of a value each


@pytest.mark.parametrize("fmt", FORMATS)
def test_example_generates(cuda, fmt):
    """The example's model over its paged cache: whole prompts, then tokens, twice the same."""
    import importlib.util
    from pathlib import Path

    at = Path(__file__).resolve().parent.parent / "examples" / "generate_paged.py"
    spec = importlib.util.spec_from_file_location("generate_paged_example", at)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    gen = torch.Generator().manual_seed(5)
    vocab = 704
    prompts = [torch.randint(0, vocab, (n,), generator=gen).cuda() for n in (70, 1, 64)]
    model = example.Model(2, vocab, torch.device("cuda"))
    runs = []
    for some in (prompts, prompts):
        session = example.PagedSession(model, some, 6, fmt)
        for _ in range(6):
            assert torch.isfinite(session.logits.float()).all()
            session.step(session.choose())
        assert session.lens.tolist() == [76, 7, 70]
        runs.append(session.tokens.clone())
    assert torch.equal(*runs)
    for i, n in enumerate((70, 1, 64)):
        new = runs[0][i, n:n + 6]
        assert ((new >= 0) & (new < vocab)).all() and torch.equal(runs[0][i, :n], prompts[i].int())
