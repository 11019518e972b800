"""The generation operators at the edges of their contracts: infinities and NaN in places that a row sees and in
places that it does not, long prompts, many rows. Definitions and tolerances are those of test_generate_gpu.py."""

import math

import pytest
import torch
from test_generate_gpu import U, _clean, close, cu_of, randn  # noqa: F401 (_clean: autouse)

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
