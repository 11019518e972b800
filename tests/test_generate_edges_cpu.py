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
