"""The generation operators without a GPU: refusals of bad arguments, the shape functions, the C entries' checks."""

import pytest
import torch

import torch_xdna
from torch_xdna import XdnaError, XdnaUnavailable, kernels

BF = torch.bfloat16


def z(*shape, dtype=BF):
    return torch.zeros(*shape, dtype=dtype)


def i32(*shape):
    return torch.zeros(*shape, dtype=torch.int32)


def refuse(fn, *args, match, **kw):
    with pytest.raises(XdnaError, match=match):
        fn(*args, **kw)


def test_packed_refusals():
    f, cu = torch_xdna.packed_attention, i32(3)
    q, k = z(5, 4, 64), z(5, 2, 64)
    refuse(f, z(5, 256), k, k, cu, match="need")
    refuse(f, q, z(6, 2, 64), z(6, 2, 64), cu, match="need")
    refuse(f, q, k, z(5, 2, 128), cu, match="need")
    refuse(f, q, k, k.half(), cu, match="float16")
    refuse(f, q.float(), k.float(), k.float(), cu, match="bf16 or f16")
    refuse(f, q, z(5, 3, 64), z(5, 3, 64), cu, match="share")
    refuse(f, z(5, 129, 64), z(5, 1, 64), z(5, 1, 64), cu, match="share")
    refuse(f, z(5, 0, 64), z(5, 0, 64), z(5, 0, 64), cu, match="share")
    refuse(f, z(5, 4, 80), z(5, 2, 80), z(5, 2, 80), cu, match="head dimension")
    for bad in (cu.long(), i32(0), i32(3, 1), i32(6)[::2]):
        refuse(f, q, k, k, bad, match="cu_seqlens")
    for s in (0.0, -1.0, float("inf"), float("nan")):
        refuse(f, q, k, k, cu, scale=s, match="scale")
    with pytest.raises(XdnaUnavailable):
        f(q, k, k, cu)


def test_prefix_refusals():
    f, lens = torch_xdna.shared_prefix_attention, i32(3)
    q, p, c = z(3, 4, 64), z(7, 2, 64), z(3, 5, 2, 64)
    refuse(f, q, p, z(8, 2, 64), c, c, lens, match="need")
    refuse(f, q, p, p, c, z(3, 6, 2, 64), lens, match="need")
    refuse(f, q, p, p, z(2, 5, 2, 64), z(2, 5, 2, 64), lens, match="need")
    refuse(f, q, z(7, 4, 64), z(7, 4, 64), c, c, lens, match="need")
    refuse(f, q, z(7, 2, 128), z(7, 2, 128), z(3, 5, 2, 128), z(3, 5, 2, 128), lens, match="need")
    refuse(f, q, p.half(), p, c, c, lens, match="types")
    refuse(f, z(3, 5, 64), p, p, c, c, lens, match="share")
    refuse(f, q, p, p, c, c, i32(2), match="cache_lens")
    refuse(f, q, p, p, c, c, lens.long(), match="cache_lens")
    refuse(f, q, p, p, c, c, lens, scale=-2.0, match="scale")
    with pytest.raises(XdnaUnavailable):
        f(q, p, p, c, c, lens)


def test_w4_refusals():
    f = torch_xdna.w4_pack
    refuse(f, z(3), match="weight")
    refuse(f, z(3, 0), match="weight")
    refuse(f, z(3, 4, dtype=torch.float64), match="weight")
    refuse(f, z(3, 4), 16, match="group")
    refuse(f, z(3, 4), 32, torch.float32, match="scales")
    with pytest.raises(XdnaUnavailable):
        f(z(3, 4))
    f = torch_xdna.linear_w4
    x, codes, scales = z(2, 200), z(9, 128, dtype=torch.uint8), z(9, 4)
    refuse(f, x, codes, scales, 63, match="group")
    refuse(f, z(2, 200, dtype=torch.float64), codes, scales, 64, match="f32, bf16 or f16")
    refuse(f, z(2, 300), codes, scales, 64, match="codes")
    refuse(f, z(2, 0), z(9, 0, dtype=torch.uint8), z(9, 0), 64, match="codes")
    refuse(f, x, codes.to(torch.int8), scales, 64, match="codes")
    refuse(f, x, z(9, 256, dtype=torch.uint8)[:, ::2], scales, 64, match="codes")
    refuse(f, x, codes, z(9, 3), 64, match="scales")
    refuse(f, x, codes, scales.float(), 64, match="scales")
    refuse(f, x, codes, scales, 64, z(8), match="bias")
    with pytest.raises(XdnaUnavailable):
        f(x, codes, scales, 64)


def test_logits_refusals():
    f, x, t = torch_xdna.process_logits, z(3, 100), i32(3, 7)
    refuse(f, z(100), match="logits")
    refuse(f, x.double(), match="logits")
    refuse(f, x, i32(2, 7), match="tokens")
    refuse(f, x, t.float(), match="tokens")
    refuse(f, x, lens=i32(3), match="without tokens")
    refuse(f, x, presence=z(3, dtype=torch.float32), match="without tokens")
    refuse(f, x, t, lens=i32(2), match="lens")
    refuse(f, x, t, prompt_lens=i32(3).long(), match="prompt_lens")
    refuse(f, x, t, repetition=z(3), match="repetition")
    refuse(f, x, t, frequency=z(3, 1, dtype=torch.float32), match="frequency")
    refuse(f, x, bias=z(100), match="bias")
    refuse(f, x, bias=z(2, 100, dtype=torch.float32), match="bias")
    refuse(f, x, mask=i32(3, 3), match="mask")
    refuse(f, x, mask=i32(2, 4), match="mask")
    with pytest.raises(XdnaUnavailable):
        f(x)


def test_shape_functions():
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode():
        q, k = z(5, 4, 64)[:, :2], z(5, 2, 64)
        assert torch.ops.xdna.packed_attention(q, k, k, i32(2)).shape == (5, 2, 64)
        c = z(5, 9, 2, 64)
        assert torch.ops.xdna.shared_prefix_attention(q, k, k, c, c, i32(5)).shape == (5, 2, 64)
        y = torch.ops.xdna.linear_w4(z(2, 3, 200), z(9, 128, dtype=torch.uint8), z(9, 4), 64)
        assert y.shape == (2, 3, 9) and y.dtype == BF
        assert torch.ops.xdna.process_logits(z(3, 100)).shape == (3, 100)


def test_c_entries_refuse_before_the_device():
    """The C entries' own checks of sizes and types come before any device call."""
    L = kernels.lib()
    assert L.xdna_packed_attention(None, 8, 8, None, 8, 8, None, 8, 8, None, 1, 5, 4, 3, 64, kernels.BF16, 1.0, None,
                                   None, 0, None) == -1
    assert L.xdna_packed_attention(None, 8, 8, None, 8, 8, None, 8, 8, None, 1, 5, 4, 2, 96, kernels.BF16, 1.0, None,
                                   None, 0, None) == -2
    assert L.xdna_packed_attention(None, 8, 8, None, 8, 8, None, 8, 8, None, 1, 2 ** 30, 4, 2, 64, kernels.BF16, 1.0,
                                   None, None, 0, None) == -1
    assert L.xdna_prefix_attention(None, 8, 8, None, 8, 8, None, 8, 8, None, 8, 8, 8, None, 8, 8, 8, None, -1, 5, 5, 4,
                                   2, 64, kernels.F16, 1.0, None, None, 0, None) == -1
    assert L.xdna_linear_w4(None, kernels.I32, 1, 5, 5, None, None, kernels.F16, 32, 7, None, 0, None, 7, None) == -1
    assert L.xdna_linear_w4(None, kernels.F32, 1, 5, 5, None, None, kernels.F32, 32, 7, None, 0, None, 7, None) == -1
    assert L.xdna_w4_pack(None, kernels.F32, 3, 0, 5, 32, None, None, kernels.F16, None) == -1
    assert L.xdna_process_logits(None, kernels.F32, 70000, 5, 5, None, 4, 0, 0, None, None, None, None, None, None, 0,
                                 None, 0, None, 5, None) == -1
    assert b"process_logits" in L.xdna_last_error()
