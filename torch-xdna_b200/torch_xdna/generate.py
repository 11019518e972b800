"""Generation on the B200: from packed prompts to the next token.

  packed_attention         causal attention over prompts of different lengths, packed into one [T, H, D]
  shared_prefix_attention  a decode step's attention for a batch that shares a prefix
  w4_pack, linear_w4       linears with 4-bit weights and group scales for the few rows of a decode step
  process_logits           penalties, bias and grammar mask on the next token's logits

The reference answers with the logits of whole sequences and has no counterpart of these. Each call
enqueues kernels of libxdna_b200.so on the current stream and neither synchronises nor reads device
values on the host; a bad argument raises XdnaError, CPU tensors and a missing GPU XdnaUnavailable.
Inference only: there is no backward pass, and where an input requires grad, backward through the result
raises. The same calls are the ops torch.ops.xdna.* of these names (without w4_pack).
"""

import importlib.machinery
import importlib.util
import time
from pathlib import Path

import torch

from . import kernels
from .runtime import DEVICE, stats

ERR_INVALID = -1
W4_BLOCK = 128          # columns per block of the stored codes
BINDING_PATH = Path(__file__).resolve().parent / "lib" / "_xdna_generate.so"


class _NotLoaded:
    """Stands for the binding (csrc/binding.cpp: argument checks, allocation and the C calls) until its first use."""

    def __getattr__(self, name):
        global _native
        kernels.lib()
        if not BINDING_PATH.exists():
            raise kernels.XdnaUnavailable(
                f"{BINDING_PATH} is not built (run __graft_entry__.build() or make -C torch-xdna_b200/csrc)")
        loader = importlib.machinery.ExtensionFileLoader("_xdna_generate", str(BINDING_PATH))
        module = importlib.util.module_from_spec(importlib.util.spec_from_loader(loader.name, loader))
        loader.exec_module(module)
        module.init(kernels.XdnaError, kernels.XdnaUnavailable)
        _native = module
        return getattr(module, name)


_native = _NotLoaded()


def _ready(x):
    """Raises XdnaUnavailable where the kernels cannot run; CPU tensors are left to the binding, after its checks."""
    if not kernels._state["ok"] and getattr(x, "is_cuda", False):
        kernels.require()
    return time.perf_counter()


def _account(t0, launches=None):
    stats.calls[DEVICE] += 1
    stats.launches += _native.launches() if launches is None else launches
    stats.seconds[DEVICE] += time.perf_counter() - t0


def packed_attention(q, k, v, cu_seqlens, scale=None):
    """Causal attention over packed sequences: softmax(scale q k^T) v per sequence and head, each token over the
    tokens of its sequence up to itself.

    q [T, Hq, D], k and v [T, Hkv, D] (bf16 or f16, D 64 or 128, Hq a multiple of Hkv; any strides, copied where the
    kernels cannot read them); cu_seqlens [N + 1] int32 on the GPU: sequence i is tokens cu_seqlens[i] ..
    cu_seqlens[i + 1] - 1. Tokens of no sequence (padding past the last one) give zeros. scale: 1 / sqrt(D) unless
    given. Returns [T, Hq, D]."""
    t0 = _ready(q)
    out = _native.packed_attention(q, k, v, cu_seqlens, scale)
    if out is None:  # autograd records this call
        return torch.ops.xdna.packed_attention(q, k, v, cu_seqlens, scale)
    _account(t0)
    return out


def shared_prefix_attention(q, prefix_k, prefix_v, k_cache, v_cache, cache_lens, scale=None):
    """One decode step's attention for B sequences that share a prefix, read once for all of them.

    q [B, Hq, D]; prefix_k, prefix_v [P, Hkv, D]; k_cache, v_cache [B, S, Hkv, D], of which row b's first
    cache_lens[b] (int32 on the GPU, clamped to 0..S) are its own keys (bf16 or f16, D 64 or 128, Hq a multiple of
    Hkv; any strides, copied where the kernels cannot read them). Row b attends to the prefix and its own keys; with
    neither it is zero. scale: 1 / sqrt(D) unless given. Returns [B, Hq, D]. The lengths stay on the GPU, and the work
    is split by S: pass long caches cut to about the longest sequence (k_cache[:, :n], no copy)."""
    t0 = _ready(q)
    out = _native.shared_prefix_attention(q, prefix_k, prefix_v, k_cache, v_cache, cache_lens, scale)
    if out is None:  # autograd records this call
        return torch.ops.xdna.shared_prefix_attention(q, prefix_k, prefix_v, k_cache, v_cache, cache_lens, scale)
    _account(t0)
    return out


def w4_pack(w, group=128, scale_dtype=None):
    """A weight [N, K] (f32, bf16 or f16) in 4 bits: (codes uint8 [N, K' / 2], scales [N, ceil(K / group)]), K' = K
    rounded up to 128, w ~= (code - 8) * scale with scale = max |w| of the group / 7. group: 32, 64 or 128;
    scale_dtype: bf16 or f16, by default w's where it is one of them, else f16 (groups of max |w| from 2e-7 to 4.5e5). A
    group that is not finite has the scale NaN. The layout of the codes is described in include/xdna_b200.h."""
    t0 = _ready(w)
    bad = None
    if w.dim() != 2 or w.shape[1] < 1 or w.dtype not in (torch.float32, torch.bfloat16, torch.float16):
        bad = f"a [N, K] weight in f32, bf16 or f16, not {tuple(w.shape)} {w.dtype}"
    elif group not in (32, 64, 128):
        bad = f"group {group} (32, 64 or 128)"
    if scale_dtype is None:
        scale_dtype = torch.bfloat16 if w.dtype == torch.bfloat16 else torch.float16
    if scale_dtype not in (torch.bfloat16, torch.float16):
        bad = bad or f"scales in {scale_dtype} (bf16 or f16)"
    if bad:
        raise kernels.XdnaError("w4_pack", ERR_INVALID, bad)
    kernels._cuda(w)
    w = w.detach()
    if w.stride(1) != 1 or (w.shape[0] > 1 and w.stride(0) < w.shape[1]):
        w = w.contiguous()
    N, K = w.shape
    codes = torch.empty((N, kernels.round_up(K, W4_BLOCK) // 2), dtype=torch.uint8, device=w.device)
    scales = torch.empty((N, -(-K // group)), dtype=scale_dtype, device=w.device)
    with torch.cuda.device(w.device):
        kernels.w4_pack(w, group, codes, scales)
    _account(t0, 1)
    return codes, scales


def linear_w4(x, codes, scales, group, bias=None):
    """x [..., K] times a 4-bit weight (w4_pack) transposed, plus bias [N]: [..., N] in x's type (f32, bf16 or f16),
    summed in 32 bits and rounded once. Meant for the few rows of a decode step; any number is right."""
    t0 = _ready(x)
    y = _native.linear_w4(x, codes, scales, group, bias)
    if y is None:  # autograd records this call
        return torch.ops.xdna.linear_w4(x, codes, scales, group, bias)
    stats.macs[DEVICE] += x.numel() * len(codes)
    _account(t0)
    return y


def process_logits(logits, tokens=None, lens=None, prompt_lens=None, repetition=None, presence=None, frequency=None,
                   bias=None, mask=None):
    """Penalties, bias and grammar mask on the next token's logits [B, V] (f32, bf16 or f16; B up to 65535), in one pass.

    tokens [B, T] (int32 or int64): each row's tokens so far, the first lens[b] of them (all, unless given), of which
    the first prompt_lens[b] (none, unless given) are the prompt's; ids outside [0, V) count for nothing. Per row and
    f32 [B]: repetition (a seen token's positive logit is divided by it, another multiplied), presence and frequency
    (taken off a generated token's logit once, and once for each time it occurs). bias: f32 [V] or [B, V], added.
    mask: int32 [B, ceil(V / 32)] or [1, ...], bit v % 32 of word v / 32 set where v is allowed; others become -inf,
    whatever stood there. Each may be None. Returns new logits in the same type."""
    t0 = _ready(logits)
    out = _native.process_logits(logits, tokens, lens, prompt_lens, repetition, presence, frequency, bias, mask)
    if out is None:  # autograd records this call
        return torch.ops.xdna.process_logits(logits, tokens, lens, prompt_lens, repetition, presence, frequency, bias, mask)
    _account(t0)
    return out
