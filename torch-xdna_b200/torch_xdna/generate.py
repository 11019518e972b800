"""Generation on the B200: from packed prompts to the next token.

  packed_attention         causal attention over prompts of different lengths, packed into one [T, H, D]
  shared_prefix_attention  a decode step's attention for a batch that shares a prefix
  w4_pack, linear_w4       linears with 4-bit weights and group scales for the few rows of a decode step
  process_logits           penalties, bias and grammar mask on the next token's logits

The reference answers with the logits of whole sequences and has no counterpart of these. Each call
enqueues kernels of libxdna_b200.so on the current stream and neither synchronises nor reads device
values on the host; a bad argument raises XdnaError, CPU tensors and a missing GPU XdnaUnavailable.
Inference only. The same calls are the ops torch.ops.xdna.* of these names (without w4_pack).
"""

import time

import torch

from . import kernels
from .runtime import DEVICE, stats

ERR_INVALID, ERR_UNSUPPORTED = -1, -2
W4_BLOCK = 128          # columns per block of the stored codes
_HALF = (torch.bfloat16, torch.float16)
_FLOAT = (torch.float32, torch.bfloat16, torch.float16)


def _require(cond, name, message, status=ERR_INVALID):
    if not cond:
        raise kernels.XdnaError(name, status, message)


def _launch(name, tensors, launches, t0, fn_args):
    """Calls xdna_<name> with fn_args(stream) on the device of `tensors`, on its current stream."""
    dev = tensors[0].device
    for t in tensors:
        if t is not None and t.device != dev:
            raise kernels.XdnaError(name, ERR_INVALID, f"tensors on {dev} and {t.device}")
    kernels._cuda(tensors[0])
    fn = getattr(kernels.require(), "xdna_" + name)
    if dev.index != torch.cuda.current_device():
        with torch.cuda.device(dev):
            kernels._check(name, fn(*fn_args(torch.cuda.current_stream().cuda_stream)))
    else:
        kernels._check(name, fn(*fn_args(torch.cuda.current_stream().cuda_stream)))
    stats.calls[DEVICE] += 1
    stats.launches += launches
    stats.seconds[DEVICE] += time.perf_counter() - t0


def _ptr(t):
    return None if t is None else t.data_ptr()


def _rows(t):
    """t as the kernels read it: contiguous in the last dimension, every other stride a positive multiple of 8
    elements, 16-byte aligned; a copy where it is not. Strides of dimensions of one entry do not matter."""
    ok = t.stride(-1) == 1 and t.data_ptr() % 16 == 0
    for n, s in zip(t.shape[:-1], t.stride()[:-1]):
        ok = ok and (n <= 1 or (s > 0 and s % 8 == 0))
    return t if ok else t.clone(memory_format=torch.contiguous_format)


def _strides(t):
    """Strides of all but the last dimension, with a harmless one for dimensions of at most one entry."""
    return [s if n > 1 else 8 for n, s in zip(t.shape[:-1], t.stride()[:-1])]


def _check_heads(name, q, kv, scale):
    hq, d, hkv = q.shape[1], q.shape[2], kv.shape[-2]
    _require(q.dtype in _HALF, name, f"bf16 or f16, not {q.dtype}")
    _require(hq >= 1 and hkv >= 1 and hq % hkv == 0 and hq // hkv <= 128, name,
             f"{hq} query heads do not share {hkv} key heads evenly (at most 128 each)")
    _require(d in (64, 128), name, f"head dimension {d} (64 or 128)", ERR_UNSUPPORTED)
    scale = d ** -0.5 if scale is None else float(scale)
    _require(0.0 < scale < float("inf"), name, f"scale {scale} is not positive and finite")
    return scale


def packed_attention(q, k, v, cu_seqlens, scale=None):
    """Causal attention over packed sequences: softmax(scale q k^T) v per sequence and head, each token over the
    tokens of its sequence up to itself.

    q [T, Hq, D], k and v [T, Hkv, D] (bf16 or f16, D 64 or 128, Hq a multiple of Hkv; any strides, copied where the
    kernels cannot read them); cu_seqlens [N + 1] int32 on the GPU: sequence i is tokens cu_seqlens[i] ..
    cu_seqlens[i + 1] - 1. Tokens of no sequence (padding past the last one) give zeros. scale: 1 / sqrt(D) unless
    given. Returns [T, Hq, D]."""
    t0, name = time.perf_counter(), "packed_attention"
    _require(q.dim() == 3 and k.dim() == 3 and k.shape == v.shape and k.shape[0] == q.shape[0]
             and k.shape[2] == q.shape[2], name,
             f"q {tuple(q.shape)}, k {tuple(k.shape)}, v {tuple(v.shape)}: need [T, Hq, D] and [T, Hkv, D]")
    _require(k.dtype == q.dtype and v.dtype == q.dtype, name, f"q {q.dtype}, k {k.dtype}, v {v.dtype}")
    _require(cu_seqlens.dtype == torch.int32 and cu_seqlens.dim() == 1 and cu_seqlens.shape[0] >= 1
             and cu_seqlens.is_contiguous(), name, "cu_seqlens: int32 [N + 1], contiguous")
    scale = _check_heads(name, q, k, scale)
    kernels._cuda(q)
    T, hq, d = q.shape
    hkv, n = k.shape[1], cu_seqlens.shape[0] - 1
    q, k, v = _rows(q), _rows(k), _rows(v)
    out = torch.empty((T, hq, d), dtype=q.dtype, device=q.device)
    size = kernels.require().xdna_packed_attention_workspace(n, T, hq, hkv)
    ws = torch.empty(size, dtype=torch.uint8, device=q.device) if size else None
    _launch(name, (q, k, v, cu_seqlens), 1, t0, lambda s: (
        q.data_ptr(), *_strides(q), k.data_ptr(), *_strides(k), v.data_ptr(), *_strides(v), cu_seqlens.data_ptr(), n,
        T, hq, hkv, d, kernels.DTYPE_CODES[q.dtype], scale, out.data_ptr(), _ptr(ws), size, s))
    return out


def shared_prefix_attention(q, prefix_k, prefix_v, k_cache, v_cache, cache_lens, scale=None):
    """One decode step's attention for B sequences that share a prefix, read once for all of them.

    q [B, Hq, D]; prefix_k, prefix_v [P, Hkv, D]; k_cache, v_cache [B, S, Hkv, D], of which row b's first
    cache_lens[b] (int32 on the GPU, clamped to 0..S) are its own keys (bf16 or f16, D 64 or 128, Hq a multiple of
    Hkv; any strides, copied where the kernels cannot read them). Row b attends to the prefix and its own keys; with
    neither it is zero. scale: 1 / sqrt(D) unless given. Returns [B, Hq, D]."""
    t0, name = time.perf_counter(), "prefix_attention"
    _require(q.dim() == 3 and prefix_k.dim() == 3 and k_cache.dim() == 4 and prefix_k.shape == prefix_v.shape
             and k_cache.shape == v_cache.shape and k_cache.shape[0] == q.shape[0]
             and prefix_k.shape[1:] == k_cache.shape[2:] and prefix_k.shape[2] == q.shape[2], name,
             f"q {tuple(q.shape)}, prefix {tuple(prefix_k.shape)} / {tuple(prefix_v.shape)}, cache "
             f"{tuple(k_cache.shape)} / {tuple(v_cache.shape)}: need [B, Hq, D], [P, Hkv, D] and [B, S, Hkv, D]")
    _require(all(t.dtype == q.dtype for t in (prefix_k, prefix_v, k_cache, v_cache)), name, "operands of several types")
    _require(cache_lens.dtype == torch.int32 and cache_lens.shape == q.shape[:1] and cache_lens.is_contiguous(), name,
             "cache_lens: int32 [B], contiguous")
    scale = _check_heads(name, q, prefix_k, scale)
    kernels._cuda(q)
    B, hq, d = q.shape
    P, hkv = prefix_k.shape[:2]
    S = k_cache.shape[1]
    q, pk, pv, ck, cv = (_rows(t) for t in (q, prefix_k, prefix_v, k_cache, v_cache))
    out = torch.empty((B, hq, d), dtype=q.dtype, device=q.device)
    size = kernels.require().xdna_prefix_attention_workspace(B, P, S, hq, hkv, d)
    ws = torch.empty(size, dtype=torch.uint8, device=q.device) if size else None
    _launch(name, (q, pk, pv, ck, cv, cache_lens), 1, t0, lambda s: (
        q.data_ptr(), *_strides(q), pk.data_ptr(), *_strides(pk), pv.data_ptr(), *_strides(pv), ck.data_ptr(),
        *_strides(ck), cv.data_ptr(), *_strides(cv), cache_lens.data_ptr(), B, P, S, hq, hkv, d,
        kernels.DTYPE_CODES[q.dtype], scale, out.data_ptr(), _ptr(ws), size, s))
    return out


def w4_pack(w, group=128, scale_dtype=None):
    """A weight [N, K] (f32, bf16 or f16) in 4 bits: (codes uint8 [N, K' / 2], scales [N, ceil(K / group)]), K' = K
    rounded up to 128, w ~= (code - 8) * scale with scale = max |w| of the group / 7. group: 32, 64 or 128;
    scale_dtype: bf16 or f16, by default w's where it is one of them, else f16. The layout of the codes is described
    in include/xdna_b200.h."""
    t0, name = time.perf_counter(), "w4_pack"
    _require(w.dim() == 2 and w.shape[1] >= 1 and w.dtype in _FLOAT, name,
             f"a [N, K] weight in f32, bf16 or f16, not {tuple(w.shape)} {w.dtype}")
    _require(group in (32, 64, 128), name, f"group {group} (32, 64 or 128)")
    scale_dtype = scale_dtype or (w.dtype if w.dtype in _HALF else torch.float16)
    _require(scale_dtype in _HALF, name, f"scales in {scale_dtype} (bf16 or f16)")
    kernels._cuda(w)
    w = w.detach()
    if w.stride(1) != 1 or w.stride(0) < w.shape[1]:
        w = w.contiguous()
    N, K = w.shape
    codes = torch.empty((N, kernels.round_up(K, W4_BLOCK) // 2), dtype=torch.uint8, device=w.device)
    scales = torch.empty((N, -(-K // group)), dtype=scale_dtype, device=w.device)
    _launch(name, (w,), 1, t0, lambda s: (
        w.data_ptr(), kernels.DTYPE_CODES[w.dtype], N, K, max(w.stride(0), K), group, codes.data_ptr(),
        scales.data_ptr(), kernels.DTYPE_CODES[scale_dtype], s))
    return codes, scales


def linear_w4(x, codes, scales, group, bias=None):
    """x [..., K] times a 4-bit weight (w4_pack) transposed, plus bias [N]: [..., N] in x's type (f32, bf16 or f16),
    summed in 32 bits and rounded once. Meant for the few rows of a decode step; any number is right."""
    t0, name = time.perf_counter(), "linear_w4"
    _require(x.dim() >= 1 and x.dtype in _FLOAT, name, f"x {tuple(x.shape)} {x.dtype}: f32, bf16 or f16")
    K = x.shape[-1]
    _require(group in (32, 64, 128), name, f"group {group} (32, 64 or 128)")
    _require(codes.dim() == 2 and codes.dtype == torch.uint8 and codes.is_contiguous() and codes.data_ptr() % 16 == 0
             and K >= 1 and codes.shape[1] * 2 == kernels.round_up(K, W4_BLOCK), name,
             f"codes {tuple(codes.shape)} {codes.dtype} for K = {K}: need contiguous, aligned uint8 "
             f"[N, {kernels.round_up(max(K, 1), W4_BLOCK) // 2}]")
    N = codes.shape[0]
    _require(scales.shape == (N, -(-K // group)) and scales.dtype in _HALF and scales.is_contiguous(), name,
             f"scales {tuple(scales.shape)} {scales.dtype}: need contiguous bf16 or f16 [{N}, {-(-K // group)}]")
    _require(bias is None or (bias.shape == (N,) and bias.dtype in _FLOAT), name, "bias: [N] in f32, bf16 or f16")
    kernels._cuda(x)
    x2 = x if x.dim() == 2 else x.reshape(-1, K)
    if x2.stride(1) != 1 or (x2.shape[0] > 1 and x2.stride(0) < K):
        x2 = x2.contiguous()
    if bias is not None and not bias.is_contiguous():
        bias = bias.contiguous()
    M = x2.shape[0]
    y = torch.empty((M, N), dtype=x.dtype, device=x.device)
    _launch(name, (x2, codes, scales, bias), 1, t0, lambda s: (
        x2.data_ptr(), kernels.DTYPE_CODES[x.dtype], M, K, x2.stride(0) if M > 1 else K, codes.data_ptr(),
        scales.data_ptr(), kernels.DTYPE_CODES[scales.dtype], group, N, _ptr(bias),
        kernels.DTYPE_CODES[bias.dtype] if bias is not None else kernels.F32, y.data_ptr(), N, s))
    stats.macs[DEVICE] += M * N * K
    return y if x.dim() == 2 else y.view(*x.shape[:-1], N)


def process_logits(logits, tokens=None, lens=None, prompt_lens=None, repetition=None, presence=None, frequency=None,
                   bias=None, mask=None):
    """Penalties, bias and grammar mask on the next token's logits [B, V] (f32, bf16 or f16), in one pass.

    tokens [B, T] (int32 or int64): each row's tokens so far, the first lens[b] of them (all, unless given), of which
    the first prompt_lens[b] (none, unless given) are the prompt's; ids outside [0, V) count for nothing. Per row and
    f32 [B]: repetition (a seen token's positive logit is divided by it, another multiplied), presence and frequency
    (taken off a generated token's logit once, and once for each time it occurs). bias: f32 [V] or [B, V], added.
    mask: int32 [B, ceil(V / 32)] or [1, ...], bit v % 32 of word v / 32 set where v is allowed; others become -inf,
    whatever stood there. Each may be None. Returns new logits in the same type."""
    t0, name = time.perf_counter(), "process_logits"
    _require(logits.dim() == 2 and logits.dtype in _FLOAT, name,
             f"logits {tuple(logits.shape)} {logits.dtype}: [B, V] in f32, bf16 or f16")
    B, V = logits.shape
    T = 0
    if tokens is not None:
        _require(tokens.dim() == 2 and tokens.shape[0] == B and tokens.dtype in (torch.int32, torch.int64), name,
                 f"tokens {tuple(tokens.shape)} {tokens.dtype}: int32 or int64 [B, T]")
        T = tokens.shape[1]
        if tokens.stride(1) != 1 and T > 1:
            tokens = tokens.contiguous()
    for what, t, dt in (("lens", lens, torch.int32), ("prompt_lens", prompt_lens, torch.int32),
                        ("repetition", repetition, torch.float32), ("presence", presence, torch.float32),
                        ("frequency", frequency, torch.float32)):
        if t is not None:
            _require(tokens is not None, name, f"{what} without tokens")
            _require(t.shape == (B,) and t.dtype == dt and t.is_contiguous(), name, f"{what}: contiguous {dt} [B]")
    if bias is not None:
        _require(bias.dtype == torch.float32 and bias.shape in ((V,), (1, V), (B, V)), name, "bias: f32 [V] or [B, V]")
        if bias.stride(-1) != 1:
            bias = bias.contiguous()
    words = -(-V // 32)
    if mask is not None:
        _require(mask.dtype == torch.int32 and mask.shape in ((B, words), (1, words)), name,
                 f"mask: int32 [B, {words}] or [1, {words}]")
        if mask.stride(1) != 1:
            mask = mask.contiguous()
    kernels._cuda(logits)
    if logits.stride(1) != 1 or logits.stride(0) < 0:
        logits = logits.contiguous()
    out = torch.empty((B, V), dtype=logits.dtype, device=logits.device)
    _launch(name, (logits, tokens, lens, prompt_lens, repetition, presence, frequency, bias, mask), 1, t0, lambda s: (
        logits.data_ptr(), kernels.DTYPE_CODES[logits.dtype], B, V, logits.stride(0), _ptr(tokens),
        tokens.element_size() if tokens is not None else 4, T, tokens.stride(0) if tokens is not None else 0,
        _ptr(lens), _ptr(prompt_lens), _ptr(repetition), _ptr(presence), _ptr(frequency), _ptr(bias),
        bias.stride(0) if bias is not None and bias.dim() == 2 and bias.shape[0] > 1 else 0, _ptr(mask),
        mask.stride(0) if mask is not None and mask.shape[0] > 1 else 0, out.data_ptr(), V, s))
    return out
