"""The operators around a decoder layer's products on the B200 where they are most easily wrong, against their definitions."""

import pytest
import torch
from test_layer_gpu import (FORMATS, _clean, check_attention, close, filled, i32, randn,  # noqa: F401
                            rounding, step, table_of, values)

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
