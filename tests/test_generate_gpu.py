"""The generation operators on the B200 against their definitions in 64 bits.

Tolerances, per element, from the arithmetic (u = 2^-8 for bf16, 2^-11 for f16, 2^-24 for f32):
  attention  the weights enter the second product rounded to the operands' type (u of A = sum p |v|), the output is
             rounded once (u |o| <= u A); everything else is f32, with at most 2^-13 A for the scores and exponentials
             of the magnitudes used here; f16 weights below 2^-14 are rounded to 2^-25 at worst.
  linear_w4  the products are exact in f32 (an f32 x is split exactly); at most K / 16 + 16 chopped sums of 2^-23 each;
             the output is rounded once.
  logits     at most six f32 operations on terms of the size of their sum, the output rounded once; -inf exactly.
"""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu
U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
HALF = [torch.bfloat16, torch.float16]


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


def close(got, want, tol):
    got = got.double()
    assert got.shape == want.shape
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    same = (got == want) | torch.isnan(want)       # infinities too
    off = torch.where(same, 0.0, (got - want).abs() - tol)
    assert float(off.max() if off.numel() else 0.0) <= 0, (
        f"{int((off > 0).sum())} of {off.numel()} values, worst |d| {float((got - want).abs().nan_to_num(posinf=0).max()):.3g}")


# ------------------------------------------------------------------ attention
def attend(q, k, v, scale, causal_from=None):
    """(o, tol) in 64 bits of one head: q [n, D], k, v [m, D]; row i sees keys 0 .. causal_from + i."""
    z = q.double() @ k.double().t() * scale
    if causal_from is not None:
        i, j = torch.meshgrid(torch.arange(z.shape[0]), torch.arange(z.shape[1]), indexing="ij")
        z = z.masked_fill((j > i + causal_from).to(z.device), -math.inf)
    p = torch.softmax(z, 1)
    o, a = p @ v.double(), p @ v.double().abs()
    u = U[q.dtype]
    tol = 2 * u * a * (1 + u) + 2.0 ** -13 * a + 1e-30
    if q.dtype == torch.float16:
        tol = tol + (k.shape[0] + 1) * 2.0 ** -25 * float(v.double().abs().max()) + 2.0 ** -25
    return o, tol


def packed_want(q, k, v, bounds, scale=None):
    rep, d = q.shape[1] // k.shape[1], q.shape[2]
    o = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    tol = torch.zeros_like(o)
    for a, b in bounds:
        for h in range(q.shape[1]):
            if b > a:
                o[a:b, h], tol[a:b, h] = attend(q[a:b, h], k[a:b, h // rep], v[a:b, h // rep],
                                                d ** -0.5 if scale is None else scale, 0)
    return o, tol


def cu_of(lens):
    return torch.tensor([0] + list(lens)).cumsum(0).to(torch.int32).cuda()


def bounds_of(lens):
    at = [0]
    for n in lens:
        at.append(at[-1] + n)
    return list(zip(at, at[1:]))


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("hq,hkv,d", [(16, 8, 128), (4, 4, 128), (12, 12, 64), (14, 2, 64), (6, 2, 128), (8, 1, 128),
                                      (20, 1, 64)])
@pytest.mark.parametrize("lens", [(1,), (2,), (127,), (128, 1), (129, 64, 63, 65), (0, 5, 0, 0, 300, 1, 0), (511, 257)])
def test_packed(cuda, dtype, hq, hkv, d, lens):
    import torch_xdna

    t = sum(lens)
    q, k, v = randn(t, hq, d, seed=1, dtype=dtype), randn(t, hkv, d, seed=2, dtype=dtype), randn(t, hkv, d, seed=3, dtype=dtype)
    got = torch_xdna.packed_attention(q, k, v, cu_of(lens))
    close(got, *packed_want(q, k, v, bounds_of(lens)))


def test_packed_long_and_many(cuda):
    import torch_xdna

    for lens, (hq, hkv, d) in (((4099, 1, 777), (4, 2, 128)), ([1 + i % 7 for i in range(700)], (4, 2, 64)),
                               ([33] * 90, (16, 8, 128))):
        t = sum(lens)
        q, k, v = randn(t, hq, d, seed=4), randn(t, hkv, d, seed=5), randn(t, hkv, d, seed=6)
        close(torch_xdna.packed_attention(q, k, v, cu_of(lens)), *packed_want(q, k, v, bounds_of(lens)))


def test_packed_peaked_scores(cuda):
    """Scores that rise by hundreds along a row and between rows: the running maximum moves all the time."""
    import torch_xdna

    lens, hq, hkv, d = (700, 300), 4, 2, 128
    t = sum(lens)
    ramp = torch.linspace(0.2, 3.0, t, device="cuda")[:, None, None]
    for sign in (1.0, -1.0):
        q = (randn(t, hq, d, seed=1, dtype=torch.float32).abs() * ramp).bfloat16()
        k = (randn(t, hkv, d, seed=2, dtype=torch.float32).abs() * ramp * sign).bfloat16()
        v = randn(t, hkv, d, seed=3)
        o, tol = packed_want(q, k, v, bounds_of(lens))
        close(torch_xdna.packed_attention(q, k, v, cu_of(lens)), o, tol * 2)  # scores of 10^3: f32 steps of 2^-14


def test_packed_strides_scale_and_views(cuda):
    import torch_xdna

    lens, hq, hkv, d = (37, 200, 91), 6, 3, 64
    t = sum(lens)
    cu = cu_of(lens)
    qkv = randn(t, hq + 2 * hkv, d, seed=7)
    q, k, v = qkv[:, :hq], qkv[:, hq:hq + hkv], qkv[:, hq + hkv:]
    want = packed_want(q, k, v, bounds_of(lens), 0.3)
    close(torch_xdna.packed_attention(q, k, v, cu, scale=0.3), *want)
    head_first = [x.transpose(0, 1).contiguous().transpose(0, 1) for x in (q, k, v)]
    close(torch_xdna.packed_attention(*head_first, cu, scale=0.3), *want)
    # layouts that are copied: columns apart, odd token strides, unaligned bases
    apart = [torch.stack((x, x), -1)[..., 0] for x in (q, k, v)]
    close(torch_xdna.packed_attention(*apart, cu, scale=0.3), *want)
    odd = [torch.cat((x.flatten(1), x.flatten(1)[:, :3]), 1)[:, :x[0].numel()].unflatten(1, (-1, d)) for x in (q, k, v)]
    close(torch_xdna.packed_attention(*odd, cu, scale=0.3), *want)
    shifted = [torch.cat((x.flatten()[:1], x.flatten()))[1:].view(x.shape) for x in (q, k, v)]
    close(torch_xdna.packed_attention(*shifted, cu, scale=0.3), *want)
    one = randn(t, 1, d, seed=8).expand(t, hkv, d)          # a broadcast head
    close(torch_xdna.packed_attention(q, one, one, cu), *packed_want(q, one, one, bounds_of(lens)))


def test_packed_offsets_past_32_bits(cuda):
    import torch_xdna

    base = torch.empty(2 * 2 ** 30 + 4096, dtype=torch.bfloat16, device="cuda")
    x = base.as_strided((3, 4, 64), (2 ** 30, 64, 1))
    x.copy_(randn(3, 4, 64, seed=9))
    small = x.clone()
    close(torch_xdna.packed_attention(x, x, x, cu_of((3,))), *packed_want(small, small, small, [(0, 3)]))


def test_packed_tokens_of_no_sequence(cuda):
    import torch_xdna

    q, k, v = randn(300, 4, 128, seed=1), randn(300, 2, 128, seed=2), randn(300, 2, 128, seed=3)
    k[250:], v[250:], q[250:] = float("nan"), float("inf"), float("nan")   # padding may hold anything
    got = torch_xdna.packed_attention(q, k, v, torch.tensor([20, 90, 250], dtype=torch.int32, device="cuda"))
    close(got, *packed_want(q, k, v, [(20, 90), (90, 250)]))
    assert not got[:20].any() and not got[250:].any()
    none = torch_xdna.packed_attention(q, k, v, torch.zeros(1, dtype=torch.int32, device="cuda"))
    assert none.shape == q.shape and not none.any()
    # words out of range or out of order are clamped: no access outside, the well-formed sequences right
    bad = torch.tensor([-5, 90, 90, 2 ** 31 - 1, 7, -2 ** 31], dtype=torch.int32, device="cuda")
    got = torch_xdna.packed_attention(q[:250], k[:250], v[:250], bad)
    close(got[:90], *(x[:90] for x in packed_want(q[:250], k[:250], v[:250], [(0, 90)])))
    assert torch_xdna.packed_attention(q[:0], k[:0], v[:0], torch.zeros(3, dtype=torch.int32, device="cuda")).shape == (0, 4, 128)


def test_packed_neighbours_do_not_leak(cuda):
    """NaN and infinity in one sequence stay in it, also where the sequences share tiles."""
    import torch_xdna

    lens = (50, 60, 70)
    q, k, v = randn(180, 4, 128, seed=1), randn(180, 2, 128, seed=2), randn(180, 2, 128, seed=3)
    k[60:110], v[50:110] = float("nan"), float("inf")
    got = torch_xdna.packed_attention(q, k, v, cu_of(lens))
    want, tol = packed_want(q, k, v, [(0, 50), (110, 180)])
    keep = torch.ones(180, dtype=torch.bool, device="cuda")
    keep[50:110] = False
    close(got[keep], want[keep], tol[keep])
    # a key after the query's place does not reach it either
    v[0:50], k[0:50] = randn(50, 2, 128, seed=4), randn(50, 2, 128, seed=5)
    k[40], v[40] = float("nan"), float("inf")
    got = torch_xdna.packed_attention(q, k, v, cu_of(lens))
    want, tol = packed_want(q, k, v, [(0, 40)])
    close(got[:40], want[:40], tol[:40])


def test_packed_is_repeatable(cuda):
    import torch_xdna

    lens = (333, 1, 900, 64)
    q, k, v = randn(1298, 16, 128, seed=1), randn(1298, 8, 128, seed=2), randn(1298, 8, 128, seed=3)
    first = torch_xdna.packed_attention(q, k, v, cu_of(lens))
    for _ in range(3):
        assert torch.equal(first, torch_xdna.packed_attention(q, k, v, cu_of(lens)))


def prefix_want(q, pk, pv, ck, cv, lens, scale=None):
    rep, d = q.shape[1] // pk.shape[1], q.shape[2]
    o = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    tol = torch.zeros_like(o)
    for b, n in enumerate(lens):
        n = min(max(n, 0), ck.shape[1])
        for h in range(q.shape[1]):
            k = torch.cat((pk[:, h // rep], ck[b, :n, h // rep]))
            v = torch.cat((pv[:, h // rep], cv[b, :n, h // rep]))
            if len(k):
                o[b, h], tol[b, h] = (x[0] for x in attend(q[b, h][None], k, v, d ** -0.5 if scale is None else scale))
    return o, tol


def prefix_inputs(b, p, s, hq, hkv, d, dtype=torch.bfloat16):
    return (randn(b, hq, d, seed=1, dtype=dtype), randn(p, hkv, d, seed=2, dtype=dtype), randn(p, hkv, d, seed=3, dtype=dtype),
            randn(b, s, hkv, d, seed=4, dtype=dtype), randn(b, s, hkv, d, seed=5, dtype=dtype))


def int32(xs):
    return torch.tensor(xs, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("hq,hkv,d", [(16, 8, 128), (4, 4, 128), (14, 2, 64), (6, 2, 128), (20, 1, 64)])
@pytest.mark.parametrize("b,p,s", [(1, 1, 1), (3, 0, 40), (2, 130, 0), (5, 127, 17), (9, 300, 129), (70, 257, 33)])
def test_prefix(cuda, dtype, hq, hkv, d, b, p, s):
    import torch_xdna

    x = prefix_inputs(b, p, s, hq, hkv, d, dtype)
    lens = [(7 * i * i + 3 * i) % (s + 1) for i in range(b)]     # from none to all of the cache
    close(torch_xdna.shared_prefix_attention(*x, int32(lens)), *prefix_want(*x, lens))


@pytest.mark.parametrize("b,p,s,hq,hkv,d", [(1, 9001, 3, 4, 2, 128), (1, 3, 5003, 4, 2, 128), (200, 1500, 70, 4, 2, 64),
                                            (2, 1, 2500, 16, 8, 128), (130, 40, 300, 8, 8, 128)])
def test_prefix_long_and_wide(cuda, b, p, s, hq, hkv, d):
    import torch_xdna

    x = prefix_inputs(b, p, s, hq, hkv, d)
    lens = [s - (i * 37) % (s + 1) for i in range(b)]
    close(torch_xdna.shared_prefix_attention(*x, int32(lens)), *prefix_want(*x, lens))


@pytest.mark.parametrize("b,p,s,hq,hkv,d", [(20, 1500, 300, 8, 4, 128), (12, 2100, 500, 14, 2, 64), (40, 333, 700, 16, 8, 128),
                                            (9, 1025, 129, 4, 4, 64), (50, 1100, 300, 14, 2, 64), (60, 513, 129, 4, 4, 64)])
def test_prefix_beside_split_caches(cuda, b, p, s, hq, hkv, d):
    """The prefix's kernel and the own keys' run side by side and are joined; calls in a row use the same memory."""
    import torch_xdna

    x = prefix_inputs(b, p, s, hq, hkv, d)
    y = [x[0].flip(0).contiguous(), x[2], x[1], x[4], x[3]]
    lens = [(i * i * 31 + 5) % (s + 1) if i % 4 else 0 for i in range(b)]
    a, z = int32(lens), int32(lens[::-1])
    first = torch_xdna.shared_prefix_attention(*x, a)
    close(first, *prefix_want(*x, lens))
    other = torch_xdna.shared_prefix_attention(*y, z)
    close(other, *prefix_want(*y, lens[::-1]))
    for _ in range(50):
        got, got2 = torch_xdna.shared_prefix_attention(*x, a), torch_xdna.shared_prefix_attention(*y, z)
        assert torch.equal(got, first) and torch.equal(got2, other)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("b,p,s,hq,hkv,d", [(130, 1001, 9, 3, 1, 64), (50, 1025, 1, 4, 2, 64), (65, 255, 33, 12, 4, 128),
                                            (33, 1537, 0, 8, 1, 128), (129, 513, 270, 10, 2, 128), (3, 33000, 17, 4, 1, 64)])
def test_prefix_through_the_tiles(cuda, dtype, b, p, s, hq, hkv, d):
    """Prefixes too long for the sequences to read each by itself, odd ends, groups that do not divide 128."""
    import torch_xdna

    x = prefix_inputs(b, p, s, hq, hkv, d, dtype)
    lens = [(5 * i * i + i) % (s + 1) for i in range(b)]
    close(torch_xdna.shared_prefix_attention(*x, int32(lens)), *prefix_want(*x, lens))


def test_prefix_empty_rows_and_clamped_lengths(cuda):
    import torch_xdna

    x = prefix_inputs(6, 0, 50, 4, 2, 128)
    lens = [0, 3, -4, 50, 51, 2 ** 31 - 1]
    got = torch_xdna.shared_prefix_attention(*x, int32(lens))
    close(got, *prefix_want(*x, lens))
    assert not got[0].any() and not got[2].any()
    x = prefix_inputs(3, 0, 0, 4, 2, 64)
    assert not torch_xdna.shared_prefix_attention(*x, int32([0, 1, 2])).any()
    x = prefix_inputs(0, 7, 5, 4, 2, 64)
    assert torch_xdna.shared_prefix_attention(*x, int32([])).shape == (0, 4, 64)


def test_prefix_unused_cache_may_hold_anything(cuda):
    import torch_xdna

    q, pk, pv, ck, cv = prefix_inputs(5, 200, 100, 4, 2, 128)
    lens = [0, 1, 31, 64, 99]
    for i, n in enumerate(lens):
        ck[i, n:], cv[i, n:] = float("nan"), float("inf")
    close(torch_xdna.shared_prefix_attention(q, pk, pv, ck, cv, int32(lens)), *prefix_want(q, pk, pv, ck, cv, lens))


def test_prefix_peaked_scores(cuda):
    """One side of the join far above the other, in both directions, and a prefix whose scores rise along it."""
    import torch_xdna

    q, pk, pv, ck, cv = prefix_inputs(4, 1000, 80, 4, 2, 128)
    q = q.abs()
    lens = [80, 5, 1, 0]
    for a, b in ((0.1, 4.0), (4.0, 0.1), (-3.0, 3.0)):
        kp = (pk.abs().float() * torch.linspace(0, a, 1000, device="cuda")[:, None, None]).bfloat16()
        kc = (ck.abs().float() * b).bfloat16()
        o, tol = prefix_want(q, kp, pv, kc, cv, lens)
        close(torch_xdna.shared_prefix_attention(q, kp, pv, kc, cv, int32(lens)), o, tol * 2)


def test_prefix_strides(cuda):
    import torch_xdna

    b, p, s, hq, hkv, d = 3, 140, 20, 4, 2, 64
    x = prefix_inputs(b, p, s, hq, hkv, d)
    lens = [20, 0, 11]
    want = prefix_want(*x, lens, scale=0.2)
    heads_first = [t.transpose(-3, -2).contiguous().transpose(-3, -2) for t in x]
    close(torch_xdna.shared_prefix_attention(*heads_first, int32(lens), scale=0.2), *want)
    apart = [torch.stack((t, t), -1)[..., 1] for t in x]
    close(torch_xdna.shared_prefix_attention(*apart, int32(lens), scale=0.2), *want)
    # keys and values of one cache [2, B, S, H, D] with room for more tokens than are passed
    big = torch.full((2, b, s + 13, hkv, d), float("nan"), dtype=x[3].dtype, device="cuda")
    big[0, :, :s], big[1, :, :s] = x[3], x[4]
    close(torch_xdna.shared_prefix_attention(*x[:3], big[0, :, :s], big[1, :, :s], int32(lens), scale=0.2), *want)


def test_prefix_offsets_past_32_bits(cuda):
    import torch_xdna

    base = torch.empty(2 ** 31 + 2 ** 20, dtype=torch.bfloat16, device="cuda")
    q, pk, pv, ck, cv = prefix_inputs(2, 33, 9, 4, 2, 64)
    far_c = base.as_strided((2, 9, 2, 64), (2 ** 31, 128, 64, 1))
    far_c.copy_(ck)
    close(torch_xdna.shared_prefix_attention(q, pk, pv, far_c, far_c, int32([9, 8])), *prefix_want(q, pk, pv, ck, ck, [9, 8]))
    far_p = base.as_strided((33, 2, 64), (2 ** 26, 64, 1))
    far_p.copy_(pk)
    close(torch_xdna.shared_prefix_attention(q, far_p, far_p, ck, cv, int32([9, 8])), *prefix_want(q, pk, pk, ck, cv, [9, 8]))


# ------------------------------------------------------------------ 4-bit linear
def unpack(codes, k):
    """The stored codes as [N, K] in 0..15, word by word."""
    words = codes.cpu().numpy().view("<u4")
    out = torch.empty(codes.shape[0], codes.shape[1] * 2, dtype=torch.int64)
    order = (0, 2, 4, 6, 1, 3, 5, 7)
    for i in range(words.shape[1]):
        block, t, w = i // 16, i % 16 // 4, i % 4
        for place, c in enumerate(order):
            out[:, block * 128 + 32 * w + 8 * t + c] = torch.from_numpy(((words[:, i] >> (4 * place)) & 15).astype("int64"))
    return out[:, :k]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n,k,group", [(1, 1, 32), (3, 130, 64), (16, 128, 128), (40, 1000, 32), (5, 257, 128)])
def test_w4_pack(cuda, dtype, n, k, group):
    import torch_xdna

    w = randn(n, k, seed=1, dtype=dtype, scale=0.05)
    w[0, :min(k, group)] = 0                                # a group of zeros
    codes, scales = torch_xdna.w4_pack(w, group)
    assert scales.dtype == (torch.float16 if dtype == torch.float32 else dtype)
    groups = -(-k // group)
    x = torch.nn.functional.pad(w.float().cpu(), (0, groups * group - k)).view(n, groups, group)
    want = (x.abs().amax(2) / 7).to(scales.dtype)
    assert torch.equal(scales.cpu(), want)
    s = want.float()[..., None]
    r = torch.where(s > 0, torch.round(x / torch.where(s > 0, s, 1.0)).clamp(-8, 7), 0.0)
    assert torch.equal(unpack(codes, k), (r + 8).long().view(n, -1)[:, :k])
    whole = unpack(codes, codes.shape[1] * 2)
    assert bool((whole[:, k:] == 8).all())


def w4_inputs(n, k, group, sdt=torch.bfloat16, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    codes = torch.randint(0, 256, (n, -(-k // 128) * 64), generator=g, device="cuda", dtype=torch.uint8)
    scales = (torch.rand(n, -(-k // group), generator=g, device="cuda") * 0.02 - 0.005).to(sdt)
    return codes, scales


def w4_want(x, codes, scales, group, bias):
    k = x.shape[1]
    w = (unpack(codes, k).cuda().double() - 8) * scales.double().repeat_interleave(group, 1)[:, :k]
    y, a = x.double() @ w.t(), x.double().abs() @ w.abs().t()
    if bias is not None:
        y, a = y + bias.double(), a + bias.double().abs()
    return y, U[x.dtype] * y.abs() + (k / 16 + 16) * 2.0 ** -23 * a + (2.0 ** -25 if x.dtype == torch.float16 else 0)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("m,n,k", [(1, 1, 1), (1, 16, 128), (1, 1024, 2048), (2, 17, 129), (3, 100, 1000), (5, 333, 31),
                                   (8, 64, 4000), (9, 65, 512), (16, 130, 300), (17, 48, 1024), (33, 31, 640)])
def test_linear_w4(cuda, dtype, group, m, n, k):
    import torch_xdna

    codes, scales = w4_inputs(n, k, group, torch.float16 if dtype == torch.float16 else torch.bfloat16)
    x = randn(m, k, seed=2, dtype=dtype)
    bias = randn(n, seed=3, dtype=torch.float32) if m % 2 else None
    close(torch_xdna.linear_w4(x, codes, scales, group, bias), *w4_want(x, codes, scales, group, bias))


@pytest.mark.parametrize("m,n,k", [(1, 20011, 512), (6, 20000, 1024), (70, 500, 700), (300, 257, 129), (2, 64, 30000),
                                   (12, 40, 20000)])
def test_linear_w4_large(cuda, m, n, k):
    import torch_xdna

    for dtype in (torch.bfloat16, torch.float32):
        codes, scales = w4_inputs(n, k, 64)
        x = randn(m, k, seed=2, dtype=dtype)
        bias = randn(n, seed=3)
        close(torch_xdna.linear_w4(x, codes, scales, 64, bias), *w4_want(x, codes, scales, 64, bias))


@pytest.mark.parametrize("m,n,k", [(32, 20000, 2500), (31, 21000, 2240), (33, 5000, 4300), (11, 3000, 5001)])
def test_linear_w4_x_in_runs(cuda, m, n, k):
    """x does not fit in shared memory: it is copied run by run, for each round of tiles again."""
    import torch_xdna

    for dtype, group in ((torch.float16, 32), (torch.bfloat16, 128), (torch.float32, 64)):
        codes, scales = w4_inputs(n, k, group)
        x = randn(m, k, seed=4, dtype=dtype)
        close(torch_xdna.linear_w4(x, codes, scales, group), *w4_want(x, codes, scales, group, None))


def test_linear_w4_strides_shapes_and_specials(cuda):
    import torch_xdna

    codes, scales = w4_inputs(70, 300, 32)
    x = randn(2, 3, 300, seed=2)
    want, tol = w4_want(x.view(6, 300), codes, scales, 32, None)
    close(torch_xdna.linear_w4(x, codes, scales, 32).view(6, 70), want, tol)
    wide = torch.full((6, 317), float("nan"), dtype=x.dtype, device="cuda")
    wide[:, 5:305] = x.view(6, 300)
    close(torch_xdna.linear_w4(wide[:, 5:305], codes, scales, 32), want, tol)       # odd pitch, unaligned base
    close(torch_xdna.linear_w4(x.view(6, 300).t().contiguous().t(), codes, scales, 32), want, tol)
    close(torch_xdna.linear_w4(x.view(6, 300)[2], codes, scales, 32), want[2], tol[2])
    close(torch_xdna.linear_w4(x.view(6, 300)[:1].expand(4, 300), codes, scales, 32), want[:1].expand(4, 70), tol[:1].expand(4, 70))
    assert torch_xdna.linear_w4(x[:0], codes, scales, 32).shape == (0, 3, 70)
    assert torch_xdna.linear_w4(x, codes[:0], scales[:0], 32).shape == (2, 3, 0)
    # a row with a NaN or an infinity does not reach its neighbours
    for dtype in (torch.bfloat16, torch.float32):
        y = x.view(6, 300).to(dtype).clone()
        y[1, 7], y[4, 299] = float("nan"), float("inf")
        got = torch_xdna.linear_w4(y, codes, scales, 32)
        keep = [0, 2, 3, 5]
        want2, tol2 = w4_want(y[keep], codes, scales, 32, None)
        close(got[keep], want2, tol2)
        assert bool(torch.isnan(got[1]).all())
        assert not bool(torch.isfinite(got[4][(unpack(codes, 300)[:, 299] != 8).cuda()]).any())


def test_linear_w4_range_of_f32(cuda):
    """f32 activations of very different sizes in one row keep their 24 bits."""
    import torch_xdna

    codes, scales = w4_inputs(64, 512, 128, torch.float16)
    x = randn(3, 512, seed=5, dtype=torch.float32) * torch.logspace(-20, 20, 512, device="cuda")
    close(torch_xdna.linear_w4(x, codes, scales, 128), *w4_want(x, codes, scales, 128, None))


def test_w4_pack_then_linear(cuda):
    """The whole way: the 4-bit linear of a packed weight is the product with the weight it stands for."""
    import torch_xdna

    w = randn(200, 777, seed=1, scale=0.05)
    x = randn(4, 777, seed=2)
    for group in (32, 64, 128):
        codes, scales = torch_xdna.w4_pack(w, group)
        stands = (unpack(codes, 777).cuda().double() - 8) * scales.double().repeat_interleave(group, 1)[:, :777]
        step = scales.double().repeat_interleave(group, 1)[:, :777]
        assert bool(((stands - w.double()).abs() <= step * (0.5 + 7 * 2.0 ** -8)).all())
        close(torch_xdna.linear_w4(x, codes, scales, group), *w4_want(x, codes, scales, group, None))


# ------------------------------------------------------------------ logits
def logits_want(logits, tokens=None, lens=None, prompt_lens=None, repetition=None, presence=None, frequency=None,
                bias=None, mask=None):
    y = logits.double().cpu()
    size = y.abs()
    B, V = y.shape
    for b in range(B):
        if tokens is None:
            continue
        n = tokens.shape[1] if lens is None else min(max(int(lens[b]), 0), tokens.shape[1])
        first = 0 if prompt_lens is None else int(prompt_lens[b])
        ids = [int(t) for t in tokens[b, :n]]
        for v in set(i for i in ids if 0 <= i < V):
            if repetition is not None:
                r = float(repetition[b])
                y[b, v] = y[b, v] / r if y[b, v] > 0 else y[b, v] * r
            c = sum(1 for at, i in enumerate(ids) if i == v and at >= first)
            size[b, v] = y[b, v].abs()
            if c:
                f = 0.0 if frequency is None else float(frequency[b])
                p = 0.0 if presence is None else float(presence[b])
                y[b, v] -= f * c + p
                size[b, v] += abs(f * c) + abs(p)
    if bias is not None:
        y, size = y + bias.double().cpu(), size + bias.double().cpu().abs()
    if mask is not None:
        at = torch.arange(V)
        ok = (mask.cpu().long()[:, at // 32] >> (at % 32)) & 1
        y = torch.where(ok.bool(), y, -math.inf)
    y = torch.where(y.abs() > torch.finfo(logits.dtype).max, y.sign() * math.inf, y)  # past the type's range
    size = torch.where(torch.isfinite(size), size, 0.0)
    tol = 6 * 2.0 ** -24 * size + U[logits.dtype] * torch.where(torch.isfinite(y), y.abs(), 0.0) * 1.01
    return y.cuda(), (tol + (2.0 ** -25 if logits.dtype == torch.float16 else 0)).cuda()


def some_params(b, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    u = torch.rand(3, b, generator=g, device="cuda")
    return dict(repetition=u[0] * 0.5 + 0.9, presence=u[1], frequency=u[2] * 0.3 - 0.05)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("b,v,t", [(1, 1, 1), (2, 31, 5), (3, 33, 0), (1, 4096, 300), (4, 4097, 64), (3, 8191, 1000),
                                   (2, 30011, 50)])
def test_logits(cuda, dtype, b, v, t):
    import torch_xdna

    g = torch.Generator(device="cuda").manual_seed(v)
    x = randn(b, v, seed=1, dtype=dtype, scale=3.0)
    tokens = torch.randint(0, max(1, v // 3), (b, t), generator=g, device="cuda", dtype=torch.int32)
    lens = int32([(t * (i + 1)) // b for i in range(b)])
    prompts = int32([int(n) // 2 for n in lens])
    mask = torch.randint(-2 ** 31, 2 ** 31, (b, -(-v // 32)), generator=g, device="cuda").to(torch.int32)
    shared = randn(v, seed=2, dtype=torch.float32)
    rows = randn(b, v, seed=3, dtype=torch.float32)
    for kw in (dict(tokens=tokens, lens=lens, prompt_lens=prompts, bias=shared, mask=mask, **some_params(b)),
               dict(tokens=tokens.long(), **some_params(b)), dict(bias=rows), dict(mask=mask[:1]), dict(),
               dict(tokens=tokens, lens=lens, bias=rows, mask=mask, presence=some_params(b)["presence"])):
        close(torch_xdna.process_logits(x, **kw), *logits_want(x, **kw))


def test_logits_masks_and_specials(cuda):
    import torch_xdna

    v = 5000
    x = randn(5, v, seed=1, dtype=torch.float32)
    x[0, 3], x[0, 4], x[0, 5] = float("nan"), float("inf"), -float("inf")
    x[1] = torch.finfo(torch.float32).min
    mask = torch.full((5, -(-v // 32)), -1, dtype=torch.int32, device="cuda")
    mask[0, 0] = ~0b111000                 # the special values stand in masked places
    mask[2] = 0                            # nothing is allowed
    tokens = int32([[3, 4, 5, 5, -1], [0, v - 1, v, v + 7, 2 ** 31 - 1], [1, 2, 3, 4, -2 ** 31], [7] * 5, [9, 9, 9, 8, 8]])
    kw = dict(tokens=tokens, mask=mask, **some_params(5))
    got = torch_xdna.process_logits(x, **kw)
    close(got, *logits_want(x, **kw))
    assert bool((got[2] == -math.inf).all()) and bool((got[0, 3:6] == -math.inf).all())
    kw.pop("mask")
    x[0, 3] = 1.0
    got = torch_xdna.process_logits(x, **kw)   # infinities that are allowed stay
    assert float(got[0, 4]) == math.inf and float(got[0, 5]) == -math.inf
    x[0, 3:6] = 0.0
    kw["tokens"] = torch.tensor([[2 ** 32 + 3, -2 ** 40, 5, 5, 5]] * 5, device="cuda")   # 64-bit ids are not cut
    close(torch_xdna.process_logits(x, **kw), *logits_want(x, **kw))


def test_logits_lengths_are_clamped(cuda):
    import torch_xdna

    x = randn(4, 700, seed=1, dtype=torch.bfloat16)
    tokens = torch.randint(0, 700, (4, 20), device="cuda", dtype=torch.int32)
    kw = dict(tokens=tokens, lens=int32([-3, 2 ** 31 - 1, 20, 1]), prompt_lens=int32([5, -1, 2 ** 31 - 1, -2 ** 31]),
              **some_params(4))
    close(torch_xdna.process_logits(x, **kw), *logits_want(x, **kw))


def test_logits_strides(cuda):
    import torch_xdna

    wide = randn(3, 4111, seed=1)
    big = torch.randint(0, 4000, (3, 90), device="cuda", dtype=torch.int32)
    kw = dict(tokens=big[:, 7:60], bias=randn(3, 4050, seed=2, dtype=torch.float32)[:, 3:4040],
              mask=torch.randint(-2 ** 31, 2 ** 31, (3, 200), device="cuda").to(torch.int32)[:, 5:132], **some_params(3))
    x = wide[:, 11:4048]                       # 4037 columns at an odd base and pitch
    close(torch_xdna.process_logits(x, **kw), *logits_want(x, **kw))
    t = x.t().contiguous().t()
    close(torch_xdna.process_logits(t, **dict(kw, tokens=kw["tokens"].t().contiguous().t())), *logits_want(x, **kw))
    base = torch.empty(2 ** 31 + 8192, dtype=torch.bfloat16, device="cuda")
    far = base.as_strided((2, 4037), (2 ** 31 + 1, 1))
    far.copy_(x[:2])
    small = {k: v[:2] for k, v in kw.items()}
    close(torch_xdna.process_logits(far, **small), *logits_want(x[:2], **small))


# ------------------------------------------------------------------ how they are called
def _calls():
    import torch_xdna

    q, k, v = randn(333, 16, 128, seed=1), randn(333, 8, 128, seed=2), randn(333, 8, 128, seed=3)
    cu = cu_of((200, 133))
    px = prefix_inputs(9, 700, 40, 16, 8, 128)
    lens = int32([40, 0, 3, 17, 22, 1, 39, 40, 8])
    codes, scales = w4_inputs(512, 1024, 128)
    x = randn(9, 1024, seed=4)
    logits = randn(9, 10000, seed=5)
    tokens = torch.randint(0, 10000, (9, 64), device="cuda", dtype=torch.int32)
    rep = torch.full((9,), 1.2, device="cuda")
    return [lambda ns: ns.packed_attention(q, k, v, cu),
            lambda ns: ns.shared_prefix_attention(*px, lens),
            lambda ns: ns.linear_w4(x, codes, scales, 128),
            lambda ns: ns.process_logits(logits, tokens, repetition=rep)], torch_xdna


def test_ops_streams_and_graphs(cuda):
    """The custom ops, a side stream and a captured graph give the direct call's bits; so does a repeat."""
    calls, pkg = _calls()
    direct = [c(pkg) for c in calls]
    torch.cuda.synchronize()
    for c, want in zip(calls, direct):
        assert torch.equal(c(torch.ops.xdna), want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        there = [c(pkg) for c in calls]
    torch.cuda.current_stream().wait_stream(side)
    for got, want in zip(there, direct):
        assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = [c(pkg) for c in calls]
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    for got, want in zip(captured, direct):
        assert torch.equal(got, want)


def test_report_counts_the_calls(cuda):
    calls, pkg = _calls()
    pkg.stats.reset()
    for c in calls:
        c(pkg)
    assert pkg.stats.calls["gpu"] == 4 and pkg.stats.launches >= 4


def test_launches_are_counted(cuda):
    """One kernel each where one is enough; the plan of many sequences, the prefix's tiles and the join are more."""
    import torch_xdna

    def launches(f):
        before = torch_xdna.stats.launches
        f()
        return torch_xdna.stats.launches - before

    q, k = randn(100, 4, 64), randn(100, 2, 64)
    assert launches(lambda: torch_xdna.packed_attention(q, k, k, cu_of((60, 40)))) == 1
    assert launches(lambda: torch_xdna.packed_attention(q, k, k, cu_of([2] * 50))) == 2
    x = prefix_inputs(3, 50, 20, 4, 2, 64)
    assert launches(lambda: torch_xdna.shared_prefix_attention(*x, int32([1, 2, 3]))) == 1
    x = prefix_inputs(70, 257, 20, 4, 2, 64)
    assert launches(lambda: torch_xdna.shared_prefix_attention(*x, int32([5] * 70))) == 2
    codes, scales = w4_inputs(64, 128, 32)
    assert launches(lambda: torch_xdna.linear_w4(randn(1, 128), codes, scales, 32)) == 1
    assert launches(lambda: torch_xdna.w4_pack(randn(4, 128))) == 1
    assert launches(lambda: torch_xdna.process_logits(randn(2, 100))) == 1


# ------------------------------------------------------------------ values at the ends of the types, both paths
@pytest.mark.parametrize("d", [64, 128])
def test_packed_large_and_special_values(cuda, d):
    import torch_xdna

    lens = (130, 170)
    q, k, v = randn(300, 4, d, seed=1), randn(300, 2, d, seed=2), randn(300, 2, d, seed=3)
    clean = packed_want(q, k, v, [(0, 130)])
    v[130:] = 3e38                                       # finite, of another sequence
    got = torch_xdna.packed_attention(q, k, v, cu_of(lens))
    close(got[:130], *(x[:130] for x in clean))
    # a NaN key reaches every later token of its sequence and no earlier one
    v[130:] = 1.0
    k[40, 0] = float("nan")
    got = torch_xdna.packed_attention(q, k, v, cu_of(lens))
    assert bool(torch.isnan(got[40:130, :2]).all()) and not bool(torch.isnan(got[:40]).any())
    assert not bool(torch.isnan(got[130:]).any()) and not bool(torch.isnan(got[:, 2:]).any())
    # a NaN value: only its own dimension
    k[40, 0] = 0.0
    v[41, 0, 3] = float("nan")
    got = torch_xdna.packed_attention(q, k, v, cu_of(lens))
    assert bool(torch.isnan(got[41:130, :2, 3]).all()) and not bool(torch.isnan(got[41:130, :2, 4:]).any())
    assert not bool(torch.isnan(got[:41]).any())


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("b", [3, 90])
def test_prefix_peaked_special_and_far(cuda, b, d):
    """b = 3: few sequences read the prefix themselves; 90: it goes through the tiles."""
    import torch_xdna

    p, s = 1000, 40
    q, pk, pv, ck, cv = prefix_inputs(b, p, s, 4, 2, d)
    q = q.abs()
    lens = [(11 * i) % (s + 1) for i in range(b)]
    for x, y in ((0.1, 4.0), (4.0, 0.1), (-3.0, 3.0), (3.0, -3.0)):
        kp = (pk.abs().float() * torch.linspace(0, x, p, device="cuda")[:, None, None]).bfloat16()
        kc = (ck.abs().float() * y).bfloat16()
        o, tol = prefix_want(q, kp, pv, kc, cv, lens)
        close(torch_xdna.shared_prefix_attention(q, kp, pv, kc, cv, int32(lens)), o, tol * 2)
    bad = pk.clone()
    bad[77, 1] = float("nan")
    got = torch_xdna.shared_prefix_attention(q, bad, pv, ck, cv, int32(lens))
    assert bool(torch.isnan(got[:, 2:]).all()) and not bool(torch.isnan(got[:, :2]).any())
    heads_first = [t.transpose(-3, -2).contiguous().transpose(-3, -2) for t in (q, pk, pv, ck, cv)]
    close(torch_xdna.shared_prefix_attention(*heads_first, int32(lens)), *prefix_want(q, pk, pv, ck, cv, lens))
    base = torch.empty(2 ** 31 + 2 ** 20, dtype=torch.bfloat16, device="cuda")
    far = base.as_strided((p, 2, d), (2 ** 21, d, 1))
    far.copy_(pk)
    close(torch_xdna.shared_prefix_attention(q, far, far, ck, cv, int32(lens)), *prefix_want(q, pk, pk, ck, cv, lens))


def test_linear_w4_scales_at_odd_places(cuda):
    """Views of larger weights: scales that start on two bytes, rows of an odd number of them, the array's last one."""
    import torch_xdna

    for k, group in ((300, 128), (1100, 128), (1500, 64), (900, 32)):
        codes, scales = w4_inputs(41, k, group)
        x = randn(3, k, seed=2)
        for i in (0, 1, 40):
            close(torch_xdna.linear_w4(x, codes[i:], scales[i:], group), *w4_want(x, codes[i:], scales[i:], group, None))


# ------------------------------------------------------------------ the operators together
def test_example_decode_agrees_with_prefill(cuda):
    """The example's decode (4-bit linears, caches, shared prefix) against its own packed prefill of the same tokens with
    the weights those bits stand for: the logits after the last step, within the 5e-2 (relative norm) that the package
    allows its bf16 linears, and tokens that obey the mask."""
    import importlib.util

    from conftest import ROOT

    spec = importlib.util.spec_from_file_location("generate_example", ROOT / "examples" / "generate.py")
    ex = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(ex)
    gen = torch.Generator().manual_seed(3)
    vocab, shared, steps = 1000, 140, 5
    system = torch.randint(0, vocab, (shared,), generator=gen)
    prompts = [torch.cat((system, torch.randint(0, vocab, (n,), generator=gen))).cuda() for n in (1, 30, 77)]
    model = ex.Model(2, vocab, torch.device("cuda"))
    session = ex.Session(model, prompts, shared, steps)
    mask = torch.full((1, -(-vocab // 32)), -1, dtype=torch.int32, device="cuda")
    mask[0, :16] = 0                                                     # only tokens from 512 on
    for _ in range(steps):
        token = session.choose(mask=mask)
        assert bool((token >= 512).all())
        session.step(token)
    whole = [session.tokens[j, :int(session.prompt_lens[j]) + steps].long() for j in range(3)]
    logits, _, cu = model.prefill(whole)
    want = logits[cu[1:].long() - 1].float()
    got = session.logits.float()
    assert float((got - want).norm() / want.norm()) < 5e-2
