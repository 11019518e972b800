"""The generation operators at the edges of their contracts: infinities and NaN in places that a row sees and in
places that it does not, long prompts, many rows. Definitions and tolerances are those of test_generate_gpu.py."""

import math

import pytest
import torch
from test_generate_gpu import (U, _clean, close, cu_of, int32, prefix_inputs, prefix_want, randn, unpack,  # noqa: F401
                               w4_inputs, w4_want)  # (_clean: autouse)

pytestmark = pytest.mark.gpu
HALF = [torch.bfloat16, torch.float16]


def row_want(q, k, v):
    """(o, tol) in 64 bits of one row q [D] over exactly the keys k, v [n, D]. Zero where no key weighs anything. The
    tolerance is that of the module named above, over the finite values (others have to be met exactly)."""
    z = k.double() @ q.double() * q.shape[0] ** -0.5
    if bool((z == -math.inf).all()):
        return torch.zeros_like(q, dtype=torch.float64), torch.zeros_like(q, dtype=torch.float64)
    p, x, u = torch.softmax(z, 0), v.double(), U[q.dtype]
    size = torch.where(torch.isfinite(x), x.abs(), 0.0)
    a = p.nan_to_num(nan=0.0) @ size
    tol = 2 * u * a * (1 + u) + 2.0 ** -13 * a + 1e-30
    if q.dtype == torch.float16:
        tol = tol + (len(z) + 1) * 2.0 ** -25 * float(size.max()) + 2.0 ** -25
    return (p[:, None] * x).sum(0), tol


def packed_rows(q, k, v, lens, rows=None):
    """row_want of the rows (tokens) `rows` of packed sequences, all heads: two tensors [rows, Hq, D]."""
    start = [0]
    for n in lens:
        start.append(start[-1] + n)
    rep = q.shape[1] // k.shape[1]
    out = []
    for t in range(start[-1]) if rows is None else rows:
        s = max(x for x in start if x <= t)
        out.append([row_want(q[t, h], k[s:t + 1, h // rep], v[s:t + 1, h // rep]) for h in range(q.shape[1])])
    return tuple(torch.stack([torch.stack([x[i] for x in heads]) for heads in out]) for i in range(2))


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("d", [64, 128])
def test_packed_infinite_key_at_the_start(cuda, dtype, d):
    """Scores of -inf at a sequence's first keys, with an infinity in V behind the mask of the rows that follow them:
    these keys weigh nothing and the rows stay finite. A row of which every score is -inf has no weights: zero."""
    import torch_xdna

    lens, first = (150, 60), 3
    q, k, v = (randn(210, h, d, seed=i, dtype=dtype) for i, h in enumerate((4, 2, 2)))
    q[..., 0] = -q[..., 0].abs() - 0.5
    k[:first, 0, 0] = math.inf                       # heads 0 and 1: -inf against every query
    v[40, 0, 5], v[100, 0, d - 1], v[170, 1] = math.inf, math.nan, math.inf
    got = torch_xdna.packed_attention(q, k, v, cu_of(lens))
    want, tol = packed_rows(q, k, v, lens)
    assert bool(torch.isfinite(want[:40]).all()) and not want[:first, :2].any()
    close(got, want, tol)


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("d", [64, 128])
def test_packed_non_finite_values_everywhere(cuda, dtype, d):
    """Infinities and NaN all over V, of keys that rows see and of keys that they do not, under weights from large to
    far below what 16 bits hold: each row is that of exactly its own keys."""
    import torch_xdna

    lens = (300, 1, 129, 260)
    q = randn(690, 4, d, seed=1, dtype=dtype, scale=6.0)
    k, v = randn(690, 2, d, seed=2, dtype=dtype), randn(690, 2, d, seed=3, dtype=dtype)
    g = torch.Generator(device="cuda").manual_seed(4)
    kind = torch.randint(0, 3, v.shape, generator=g, device="cuda")
    special = torch.tensor([math.inf, -math.inf, math.nan], device="cuda")[kind].to(dtype)
    v = torch.where(torch.rand(v.shape, generator=g, device="cuda") < 0.002, special, v)
    close(torch_xdna.packed_attention(q, k, v, cu_of(lens)), *packed_rows(q, k, v, lens))


@pytest.mark.parametrize("dtype", HALF)
def test_packed_non_finite_values_of_a_long_prompt(cuda, dtype):
    """One NaN and two infinities in the values of a prompt of 200000 tokens: the rows that see them, the rows that only
    share a tile with them, and all else, which keeps its bits."""
    import torch_xdna

    t, d = 200_000, 64
    q, k, v = (randn(t, h, d, seed=i, dtype=dtype) for i, h in enumerate((4, 2, 2)))
    k[7, 0] *= 24                                        # weights of the first infinity from large to nothing
    clean = torch_xdna.packed_attention(q, k, v, cu_of((t,)))
    v[7, 0, 1], v[100_003, 0, 2], v[9, 0, 3] = math.inf, -math.inf, math.nan
    got = torch_xdna.packed_attention(q, k, v, cu_of((t,)))
    assert torch.equal(got[:, 2:], clean[:, 2:]) and torch.equal(got[:, :2, 4:], clean[:, :2, 4:])
    for dim, first, value in ((1, 7, math.inf), (2, 100_003, -math.inf)):
        assert bool((got[first:, :2, dim] == value).all())
    assert bool(torch.isnan(got[9:, :2, 3]).all())
    rows = [0, 6, 7, 8, 9, 10, 63, 64, 127, 128, 99_999, 100_002, 100_003, 100_004, 100_095, 100_096, t - 1]
    close(got[rows], *packed_rows(q, k, v, (t,), rows))


def test_packed_non_finite_value_costs_little(cuda):
    """A NaN or an infinity in the values of each head is looked into once per tile, not once per row and key."""
    import torch_xdna

    def ms(fn):
        fn()
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        a.record()
        fn()
        b.record()
        b.synchronize()
        return a.elapsed_time(b)

    for dtype in HALF:
        q, k, v = (randn(8191, h, 128, seed=i, dtype=dtype) for i, h in enumerate((16, 8, 8)))
        cu = cu_of((8191,))
        clean = ms(lambda: torch_xdna.packed_attention(q, k, v, cu))
        for value in (math.nan, math.inf):
            v[50, :, 9] = value
            assert ms(lambda: torch_xdna.packed_attention(q, k, v, cu)) < 20 * clean + 1.0


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("group", [32, 64, 128])
def test_w4_pack_shows_non_finite_weights(cuda, dtype, group):
    """A group with a NaN or an infinity among its weights has a scale of NaN and codes of zero, and so its row's results
    are NaN; every other group is what it is without."""
    import torch_xdna

    n, k = 6, 300
    w = randn(n, k, seed=1, dtype=dtype, scale=0.05)
    clean_codes, clean_scales = torch_xdna.w4_pack(w, group)
    for row, col, value in ((0, 5, math.nan), (1, 200, math.inf), (2, 299, -math.inf), (3, 0, math.nan), (3, 1, math.inf)):
        w[row, col] = value
    codes, scales = torch_xdna.w4_pack(w, group)
    bad = torch.zeros(n, -(-k // group), dtype=torch.bool, device="cuda")
    bad[[0, 1, 2, 3], [5 // group, 200 // group, 299 // group, 0]] = True
    assert torch.equal(torch.isnan(scales), bad) and torch.equal(scales[~bad], clean_scales[~bad])
    hit = bad.repeat_interleave(group, 1)[:, :k].cpu()
    assert torch.equal(unpack(codes, k), torch.where(hit, 8, unpack(clean_codes, k)))
    x = randn(3, k, seed=2, dtype=dtype)
    y, clean = torch_xdna.linear_w4(x, codes, scales, group), torch_xdna.linear_w4(x, clean_codes, clean_scales, group)
    assert bool(torch.isnan(y[:, :4]).all()) and torch.equal(y[:, 4:], clean[:, 4:])


def test_w4_pack_past_the_range_of_f16_scales(cuda):
    """f32 weights that an f16 scale cannot hold: too large ones show in the result, bf16 scales hold them."""
    import torch_xdna

    w = randn(4, 128, seed=1, dtype=torch.float32)
    w[1] *= 1e6
    x = randn(2, 128, seed=2, dtype=torch.float32)
    y = torch_xdna.linear_w4(x, *torch_xdna.w4_pack(w, 64), 64)
    assert not bool(torch.isfinite(y[:, 1]).any()) and bool(torch.isfinite(y[:, [0, 2, 3]]).all())
    assert bool(torch.isfinite(torch_xdna.linear_w4(x, *torch_xdna.w4_pack(w, 64, torch.bfloat16), 64)).all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m,n,k", [(65_536, 40, 130), (70_001, 17, 64), (2 ** 19 + 5, 5, 33)])
def test_linear_w4_of_very_many_rows(cuda, dtype, m, n, k):
    import torch_xdna

    codes, scales = w4_inputs(n, k, 32, torch.float16 if dtype == torch.float16 else torch.bfloat16)
    x, bias = randn(m, k, seed=2, dtype=dtype), randn(n, seed=3, dtype=torch.float32)
    close(torch_xdna.linear_w4(x, codes, scales, 32, bias), *w4_want(x, codes, scales, 32, bias))


def test_inputs_that_require_grad(cuda):
    """The values are those without grad mode; backward raises."""
    import torch_xdna

    q, k, v = (randn(70, h, 64, seed=i) for i, h in enumerate((4, 2, 2)))
    codes, scales = w4_inputs(33, 200, 64)
    x, logits = randn(3, 200, seed=4), randn(3, 500, seed=5)
    calls = [(q, lambda y: torch_xdna.packed_attention(y, k, v, cu_of((30, 40)))),
             (q, lambda y: torch_xdna.shared_prefix_attention(y, k, v, k[:, None], v[:, None], cu_of([0] * 70)[:70])),
             (x, lambda y: torch_xdna.linear_w4(y, codes, scales, 64)),
             (scales, lambda y: torch_xdna.linear_w4(x, codes, y, 64)),
             (logits, torch_xdna.process_logits),
             (logits[0].float(), lambda y: torch_xdna.process_logits(logits, bias=y)),
             (logits[:, 0].float(), lambda y: torch_xdna.process_logits(logits, cu_of([1] * 8).view(3, 3), repetition=y + 1))]
    for value, call in calls:
        want = call(value)
        with torch.enable_grad():
            got = call(value.clone().requires_grad_())
            assert got.requires_grad and torch.equal(got, want)
            with pytest.raises(RuntimeError, match="autograd"):
                got.float().sum().backward()


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("d", [64, 128])
def test_results_at_the_end_of_the_type(cuda, dtype, d):
    """All values are the type's largest, and all weights but one round up: a mean of equal values is that value, to the
    tolerance of two roundings, and not infinite."""
    import torch_xdna

    top = torch.finfo(dtype).max
    size = top if dtype == torch.float16 else 2.0 ** 100   # bf16: sums over the keys have to stay within f32
    x = torch.arange(0.25, 3.0, 2.0 ** -7, device="cuda").to(dtype).double()
    p = torch.exp(-x)
    x = float(x[((p.to(dtype).double() - p) / p).argmax()])
    n, s = 600, 40
    q = torch.zeros(n, 2, d, dtype=dtype, device="cuda")
    q[..., 0] = 1
    k = torch.zeros(n, 1, d, dtype=dtype, device="cuda")
    k[1:, 0, 0] = -x
    v = torch.full_like(k, size)

    def right(y, value=size):
        return bool(torch.isfinite(y).all()) and bool(((y.double() - value).abs() <= 2 * U[dtype] * value).all())

    assert right(torch_xdna.packed_attention(q, k, v, cu_of((n,)), 1.0))
    if dtype == torch.bfloat16:                            # here the sums are summed again where they do not
        assert right(torch_xdna.packed_attention(q, k, torch.full_like(k, top), cu_of((n,)), 1.0), top)
    for b in (1, 3, 190):
        ck, cv = k[1:s + 1].expand(b, s, 1, d).contiguous(), v[:s].expand(b, s, 1, d).contiguous()
        lens = torch.full((b,), s, dtype=torch.int32, device="cuda")
        wide = q[:1].expand(b, 2, d).contiguous()
        for pk in (k, k[:0], torch.cat([k] * 12)):
            assert right(torch_xdna.shared_prefix_attention(wide, pk, torch.full_like(pk, size), ck, cv, lens, 1.0))



# ------------------------------------------------------------------ how a prefix call is split
@pytest.mark.parametrize("b,p,s,hq,hkv,d", [(190, 2500, 260, 8, 8, 64), (200, 3000, 300, 16, 8, 64), (180, 2000, 256, 6, 6, 128),
                                            (20, 1500, 300, 8, 4, 128), (50, 1100, 300, 14, 2, 64)])
def test_prefix_tiles_beside_split_caches_and_their_join(cuda, b, p, s, hq, hkv, d):
    """Three launches (the prefix's tiles, the caches in pieces beside them, the join), among them batches of which many
    caches wait for a place behind the tiles. Calls in a row use the same memory."""
    import torch_xdna

    x = prefix_inputs(b, p, s, hq, hkv, d)
    y = [x[0].flip(0).contiguous(), x[2], x[1], x[4], x[3]]
    lens = [(i * i * 31 + 5) % (s + 1) if i % 4 else 0 for i in range(b)]
    a, z = int32(lens), int32(lens[::-1])
    before = torch_xdna.stats.launches
    first = torch_xdna.shared_prefix_attention(*x, a)
    assert torch_xdna.stats.launches - before == 3
    close(first, *prefix_want(*x, lens))
    other = torch_xdna.shared_prefix_attention(*y, z)
    close(other, *prefix_want(*y, lens[::-1]))
    for _ in range(30):
        got, got2 = torch_xdna.shared_prefix_attention(*x, a), torch_xdna.shared_prefix_attention(*y, z)
        assert torch.equal(got, first) and torch.equal(got2, other)


@pytest.mark.parametrize("b,p,s,hq,hkv,d", [(1, 700, 9000, 16, 8, 128), (3, 100, 20000, 4, 2, 64), (33, 3000, 9000, 4, 2, 64),
                                            (64, 2100, 2000, 14, 2, 64), (130, 1500, 3000, 8, 4, 128)])
def test_prefix_caches_with_room_to_spare(cuda, b, p, s, hq, hkv, d):
    """Caches far longer than any sequence: most pieces of a cache are empty, and what lies past a length is not used."""
    import torch_xdna

    x = prefix_inputs(b, p, s, hq, hkv, d)
    lens = [(i * 37) % 90 for i in range(b)]
    for i, n in enumerate(lens):
        x[3][i, n:], x[4][i, n:] = math.nan, math.inf
    close(torch_xdna.shared_prefix_attention(*x, int32(lens)), *prefix_want(*x, lens))


@pytest.mark.parametrize("b,p", [(1, 300), (3, 50), (90, 1000), (20, 1500)])
def test_prefix_scores_of_minus_infinity_alone(cuda, b, p):
    """They weigh nothing: a sequence that has no other keys is zero, and one that has is as without them."""
    import torch_xdna

    q, pk, pv, ck, cv = prefix_inputs(b, p, 40, 4, 2, 128)
    q[..., 0] = -q[..., 0].abs() - 0.5
    pk[..., 0] = math.inf
    lens = [(i * 7) % 41 if i % 2 else 0 for i in range(b)]
    want = prefix_want(q, pk[:0], pv[:0], ck, cv, lens)
    got = torch_xdna.shared_prefix_attention(q, pk, pv, ck, cv, int32(lens))
    close(got, *want)
    assert not got[::2].any()


@pytest.mark.parametrize("lens", [[i % 3 for i in range(2500)], [0] * 1100 + [700, 1, 0, 129] + [5] * 1030,
                                  [1] * 1023 + [300], [1] * 1024 + [300], [2] * 1025])
def test_packed_many_sequences(cuda, lens):
    """The plan's block takes 1024 sequences at a time: fewer, just as many, more, empty ones among them."""
    import torch_xdna

    t = sum(lens)
    q, k, v = (randn(t, h, 64, seed=i) for i, h in enumerate((4, 2, 2)))
    got = torch_xdna.packed_attention(q, k, v, cu_of(lens))
    start = torch.tensor([0] + lens).cumsum(0)[:-1].tolist()
    rows = sorted({r for s, n in zip(start, lens) for r in (s, s + n // 2, s + n - 1) if n and s <= r < s + n})
    rows = rows[::max(1, len(rows) // 400)] + [t - 1]
    close(got[rows], *packed_rows(q, k, v, lens, rows))
