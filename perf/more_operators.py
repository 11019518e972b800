"""What a decoder layer of torch_xdna does around its products, over a cache kept in pages and in 8 bits: the rotary
positions, appending keys and values to the cache, the attention that reads it, and the norms around a block.

Each case is one call as a serving loop makes it. The plain forms are elementary torch operations in 32 bits (angles
in 64), rounded once at the end; `exact` restates each definition in 64 bits.
"""

import math
import os
import random
import sys

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
ES = {"bf16": 2, "f16": 2, "f32": 4}
FORMATS = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}
EPS = 1e-6


def listed():
    return [
        # queries and keys of one decoded token with their norm, late in a context: latency
        dict(name="rotary_token", op="rotary", dtype="bf16", t=1, h=24, d=128, r=128, interleaved=False, norm=True,
             far=40000, stretch=1.0),
        # queries and keys of a prefill batch, with their norm
        dict(name="rotary_prompts", op="rotary", dtype="bf16", t=16384, h=24, d=128, r=128, interleaved=False, norm=True,
             far=16384, stretch=1.0),
        # a part of each head in the interleaved layout, at the far end of a stretched context
        dict(name="rotary_part", op="rotary", dtype="f16", t=4099, h=32, d=80, r=32, interleaved=True, norm=False,
             far=1000000, stretch=8.0),
        # the new token of one sequence: keys and values into the cache, queries rotated beside them; latency
        dict(name="append_one", op="append", dtype="bf16", hq=16, hkv=8, d=128, page=64, norm=True, starts="900"),
        # a decode batch with small pages
        dict(name="append_batch", op="append", dtype="bf16", hq=16, hkv=8, d=128, page=16, norm=True, b=128, s=700),
        # the keys and values of a prefill batch, some prompts behind a part that is in the cache already
        dict(name="append_prompts", op="append", dtype="bf16", hq=0, hkv=8, d=128, page=64, norm=True,
             lens="1900,1024,777,1333,128,999,1600,512,255,1801,640,1111,301,1450,96,1207",
             starts="0,0,64,300,0,1,0,77,128,0,0,63,500,0,0,130"),
        # one user's sequence: latency
        dict(name="paged_one", op="paged", dtype="bf16", hq=16, hkv=8, d=128, page=64, form="int8", b=1, s=764, t=1),
        # an ordinary decode batch of uneven lengths
        dict(name="paged_batch", op="paged", dtype="bf16", hq=16, hkv=8, d=128, page=64, form="e4m3", b=32, s=4700, t=1),
        # a few proposed tokens of each sequence checked at once, heads of 64, small pages
        dict(name="paged_checked", op="paged", dtype="f16", hq=14, hkv=2, d=64, page=16, form="int8", b=24, s=3001, t=4),
        # one very long document
        dict(name="paged_long", op="paged", dtype="bf16", hq=16, hkv=8, d=128, page=128, form="e4m3", b=1, s=131071, t=1),
        # between two blocks of one decoded token, residual stream in 32 bits: latency
        dict(name="norm_token", op="norm", xtype="f32", dtype="bf16", t=1, d=1024, post=False, gate="none", scale=1.0),
        # between two blocks of a prefill batch, with a norm behind the block and a gate for each token and entry
        dict(name="norm_rows", op="norm", xtype="bf16", dtype="bf16", t=8191, d=4096, post=True, gate="each", scale=0.7),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


HEADS = [(16, 8, 128), (16, 8, 128), (8, 8, 128), (12, 4, 128), (32, 4, 128), (16, 2, 64), (12, 12, 64), (14, 2, 64)]


def draw(rng):
    op = rng.choice(["rotary", "append", "append", "paged", "paged", "norm"])
    dtype = rng.choice(["bf16", "f16"])
    if op == "rotary":
        h, d, r = rng.choice([(24, 128, 128), (24, 128, 128), (40, 128, 64), (16, 64, 64), (32, 80, 32), (12, 96, 24),
                              (9, 256, 64), (_log(rng, 1, 64), 128, 2 * rng.randint(1, 64))])
        return dict(op=op, dtype=rng.choice(["bf16", "f16", "f32"]), t=_log(rng, 1, 6000), h=h, d=d, r=r,
                    interleaved=rng.random() < 0.4, norm=rng.random() < 0.5, far=_log(rng, 10, 2000000),
                    stretch=rng.choice([1.0, 1.0, 4.0, 32.0]))
    if op == "norm":
        return dict(op=op, xtype=rng.choice(["f32", "bf16", "f16"]), dtype=dtype, t=_log(rng, 1, 6000),
                    d=rng.choice([1024, 2048, 4096, _log(rng, 64, 5000)]), post=rng.random() < 0.5,
                    gate=rng.choice(["none", "all", "each"]), scale=rng.choice([1.0, 0.25, 1.4]))
    hq, hkv, d = rng.choice(HEADS)
    page = rng.choice([16, 32, 64, 128])
    if op == "append":
        if rng.random() < 0.6:
            return dict(op=op, dtype=dtype, hq=hq, hkv=hkv, d=d, page=page, norm=rng.random() < 0.7, b=_log(rng, 1, 200),
                        s=_log(rng, 1, 1000))
        n = _log(rng, 1, 24)
        lens = [_log(rng, 1, 14000 // n) for _ in range(n)]
        starts = [rng.choice([0, 0, rng.randint(0, 400)]) for _ in range(n)]
        return dict(op=op, dtype=dtype, hq=0, hkv=hkv, d=d, page=page, norm=rng.random() < 0.7,
                    lens=",".join(map(str, lens)), starts=",".join(map(str, starts)))
    b = _log(rng, 1, 100)
    t = rng.choice([1, 1, 1, 2, 3, 5])
    return dict(op=op, dtype=dtype, hq=hq, hkv=hkv, d=d, page=page, form=rng.choice(["e4m3", "int8"]), b=b,
                s=_log(rng, max(t, 2), 100000 // b), t=t)


# ------------------------------------------------------------------ inputs
def _ints(text):
    return [int(x) for x in text.split(",")]


def _append_lens(case):
    """(tokens in the cache before the call, new tokens) of each sequence."""
    if "lens" in case:
        return _ints(case["starts"]), _ints(case["lens"])
    if "b" not in case:
        starts = _ints(case["starts"])
    else:
        r = random.Random("%d.%d" % (case["b"], case["s"]))
        starts = [r.randint(0, case["s"]) for _ in range(case["b"])]
    return starts, [1] * len(starts)


def _paged_lens(case):
    """Tokens in the cache, the queries' own among them: a few far shorter than the longest."""
    r = random.Random("%d.%d.%d" % (case["b"], case["s"], case["t"]))
    return [case["s"]] + [max(case["t"], r.randint(case["s"] // 4, case["s"])) for _ in range(case["b"] - 1)]


def _frequencies(r, stretch):
    return (1e6 ** (-torch.arange(0, r, 2, dtype=torch.float64) / r) / stretch).float().cuda()


def _pages(lens, page, g):
    """A table of pages in no order, and how many there are."""
    counts = [-(-n // page) for n in lens]
    order = torch.randperm(sum(counts) + 3, generator=g, device="cuda").to(torch.int32)
    table = torch.full((len(lens), max(counts)), -1, dtype=torch.int32, device="cuda")
    at = 0
    for i, n in enumerate(counts):
        table[i, :n] = order[at:at + n]
        at += n
    return table, sum(counts) + 3


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def randn(*shape, scale=1.0, dtype=dt):
        return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)

    def weight(*shape):
        return 1 + randn(*shape, scale=0.2, dtype=torch.float32)

    def codes(form, *shape):
        if form == "int8":
            return torch.randn(*shape, generator=g, device="cuda").mul_(32).round_().clamp_(-127, 127).to(torch.int8)
        return torch.randn(*shape, generator=g, device="cuda").mul_(110).clamp_(-448, 448).to(torch.float8_e4m3fn)

    def scales(form, *shape):  # keys and values of about one, not every block as large as the next
        low = -5 if form == "int8" else -7
        return torch.exp2(torch.randint(low - 1, low + 1, shape, generator=g, device="cuda").float())

    state = dict(op=case["op"])
    if case["op"] == "rotary":
        t, h, d = case["t"], case["h"], case["d"]
        # the first heads of a projection's output, whose last ones are the values
        x = randn(t, h + max(1, h // 3), d, scale=1.5)[:, :h]
        state.update(x=x, positions=torch.randint(max(0, case["far"] - t - 100), case["far"] + 1, (t,), generator=g, device="cuda"),
                     inv_freq=_frequencies(case["r"], case["stretch"]), factor=1 + 0.1 * math.log(case["stretch"]),
                     interleaved=case["interleaved"], norm=weight(h, d) if case["norm"] else None)
    elif case["op"] == "append":
        hq, hkv, d, page = case["hq"], case["hkv"], case["d"], case["page"]
        starts, lens = _append_lens(case)
        qkv = randn(sum(lens), hq + 2 * hkv, d, scale=1.5)
        table, pages = _pages([a + b for a, b in zip(starts, lens)], page, g)
        state.update(
            q=qkv[:, :hq] if hq else None, k=qkv[:, hq:hq + hkv], v=qkv[:, hq + hkv:], table=table,
            starts=torch.tensor(starts, dtype=torch.int32).cuda(),
            cu=torch.tensor([0] + lens).cumsum(0).to(torch.int32).cuda() if "lens" in case else None,
            cache=(codes("e4m3", pages, hkv, page, d), codes("e4m3", pages, hkv, page, d),
                   scales("e4m3", pages, hkv), scales("e4m3", pages, hkv)),
            inv_freq=_frequencies(d, 1.0), q_norm=weight(d) if case["norm"] and hq else None,
            k_norm=weight(d) if case["norm"] else None)
    elif case["op"] == "paged":
        b, t, hq, hkv, d, page = (case[x] for x in ("b", "t", "hq", "hkv", "d", "page"))
        lens = _paged_lens(case)
        table, pages = _pages(lens, page, g)
        state.update(q=randn(*((b, hq, d) if t == 1 else (b, t, hq, d)), scale=1.2), table=table,
                     cache=(codes(case["form"], pages, hkv, page, d), codes(case["form"], pages, hkv, page, d),
                            scales(case["form"], pages, hkv), scales(case["form"], pages, hkv)),
                     lens=torch.tensor(lens, dtype=torch.int32).cuda())
    else:
        t, d = case["t"], case["d"]
        gate = dict(none=(), all=(d,), each=(t, d))[case["gate"]]
        state.update(x=randn(t, d, scale=2.0, dtype=DTYPES[case["xtype"]]), y=randn(t, d), weight=weight(d),
                     post=weight(d) if case["post"] else None, gate=randn(*gate, scale=0.5) if gate else None,
                     scale=case["scale"])
    return state


# ------------------------------------------------------------------ the plain forms
def _rms(x, w):
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * w


def _rotate(x, positions, inv_freq, factor, interleaved):
    """x [T, H, D] in 32 bits, its first entries rotated to the positions [T]."""
    n = len(inv_freq)
    angle = positions.double()[:, None] * inv_freq.double()
    c, s = (angle.cos() * factor).float()[:, None], (angle.sin() * factor).float()[:, None]
    if interleaved:
        a, b = x[..., 0:2 * n:2], x[..., 1:2 * n:2]
        turned = torch.stack((a * c - b * s, b * c + a * s), -1).flatten(-2)
    else:
        a, b = x[..., :n], x[..., n:2 * n]
        turned = torch.cat((a * c - b * s, b * c + a * s), -1)
    return torch.cat((turned, x[..., 2 * n:]), -1)


def _plain_rotary(x, positions, inv_freq, factor, interleaved, norm):
    y = x.float()
    return _rotate(y if norm is None else _rms(y, norm), positions, inv_freq, factor, interleaved).to(x.dtype)


def _plain_store(x, cache, scales, page, slot, pages):
    """x [T, Hkv, D] into slots of pages in e4m3. A block's scale is the least power of two with max |x| <= 448 times it;
    that of a page with older tokens grows where it has to, and their codes are rounded again."""
    new = torch.zeros_like(scales).index_reduce_(0, page, x.abs().amax(2), "amax")
    m, e = torch.frexp(new)
    new = torch.ldexp(torch.ones_like(new), (e - 9 + (m > 0.875)).clamp_min(-126))
    older = torch.full_like(scales[:, 0], cache.shape[2], dtype=torch.long).scatter_reduce_(0, page, slot, "amin")[pages, None]
    grown = torch.where(older == 0, new[pages], torch.maximum(new[pages], scales[pages]))
    less = (scales[pages] / grown)[..., None, None]
    older = torch.arange(cache.shape[2], device=x.device) < older
    old = cache[pages]
    cache[pages] = torch.where(older[:, None, :, None], old.float() * less, old.float()).to(cache.dtype)
    scales[pages] = grown
    cache[page, :, slot] = (x / scales[page][..., None]).to(cache.dtype)


def _plain_append(q, k, v, cache, table, starts, cu, inv_freq, q_norm, k_norm):
    token = torch.arange(len(k), device=k.device)
    seq = token if cu is None else torch.searchsorted(cu, token, right=True) - 1
    pos = starts.long()[seq] + (0 if cu is None else token - cu[seq])
    size = cache[0].shape[2]
    page, slot = table.long()[seq, pos // size], pos % size
    pages = torch.unique(page)
    kr = k.float() if k_norm is None else _rms(k.float(), k_norm)
    _plain_store(_rotate(kr, pos, inv_freq, 1.0, False), cache[0], cache[2], page, slot, pages)
    _plain_store(v.float(), cache[1], cache[3], page, slot, pages)
    return None if q is None else _plain_rotary(q, pos, inv_freq, 1.0, False, q_norm)


def _plain_paged(q, cache, table, lens):
    shape = q.shape
    q = q if q.dim() == 4 else q[:, None]
    b, t, hq, d = q.shape
    hkv, n = cache[0].shape[1], table.shape[1] * cache[0].shape[2]
    at = table.long().clamp_min(0)

    def whole(codes, scales):  # [B, Hkv, N, D]
        return (codes[at].float() * scales[at][..., None, None]).transpose(1, 2).reshape(b, hkv, n, d)

    scores = q.float().view(b, t, hkv, hq // hkv, d).permute(0, 2, 1, 3, 4).reshape(b, hkv, -1, d)
    scores = (scores @ whole(cache[0], cache[2]).transpose(2, 3)).view(b, hkv, t, -1, n) / math.sqrt(d)
    pos = torch.arange(n, device=q.device)
    last = lens[:, None] - t + torch.arange(t, device=q.device)
    scores = torch.where((pos <= last[..., None])[:, None, :, None], scores, -math.inf)
    e = torch.exp(scores - scores.amax(-1, keepdim=True))
    o = (e / e.sum(-1, keepdim=True)).view(b, hkv, -1, n) @ whole(cache[1], cache[3])
    return o.view(b, hkv, t, -1, d).permute(0, 2, 1, 3, 4).reshape(shape).to(q.dtype)


def _plain_norm(x, y, weight, post, gate, scale):
    z = y.float() if post is None else _rms(y.float(), post)
    z = z * scale if gate is None else z * gate.float() * scale
    z = x.float() + z
    return z.to(x.dtype), _rms(z, weight).to(y.dtype)


def _package():
    if "torch_xdna" not in sys.modules:
        here = os.path.join(os.getcwd(), "torch-xdna_b200")
        if here not in sys.path:
            sys.path.insert(0, here)
        import torch_xdna  # noqa: F401
    return sys.modules["torch_xdna"]


def run(state):
    s = state
    if s["op"] == "rotary":
        if own:
            return _package().rotary(s["x"], s["positions"], s["inv_freq"], factor=s["factor"], interleaved=s["interleaved"],
                                     norm=s["norm"], eps=EPS)
        return _plain_rotary(s["x"], s["positions"], s["inv_freq"], s["factor"], s["interleaved"], s["norm"])
    if s["op"] == "append":
        # the cache is returned as it stands: e4m3 values, and what each block of them is to be multiplied with
        if own:
            q = _package().cache_append(s["k"], s["v"], *s["cache"], s["table"], s["starts"], cu_seqlens=s["cu"],
                                        inv_freq=s["inv_freq"], k_norm=s["k_norm"], q=s["q"], q_norm=s["q_norm"], eps=EPS)
        else:
            q = _plain_append(s["q"], s["k"], s["v"], s["cache"], s["table"], s["starts"], s["cu"], s["inv_freq"],
                              s["q_norm"], s["k_norm"])
        return ([] if q is None else [q]) + list(s["cache"])
    if s["op"] == "paged":
        if own:
            return _package().paged_attention(s["q"], *s["cache"], s["table"], s["lens"])
        return _plain_paged(s["q"], s["cache"], s["table"], s["lens"])
    if own:
        return _package().add_norm(s["x"], s["y"], s["weight"], post=s["post"], gate=s["gate"], scale=s["scale"], eps=EPS)
    return _plain_norm(s["x"], s["y"], s["weight"], s["post"], s["gate"], s["scale"])


# ------------------------------------------------------------------ the work
def work(case):
    es = ES[case["dtype"]]
    if case["op"] == "rotary":
        n = case["t"] * case["h"] * case["d"]
        return {"bytes": 2 * n * es + 8 * case["t"], "flops": 8 * n}
    if case["op"] == "append":
        tokens, kv = sum(_append_lens(case)[1]), case["hkv"] * case["d"]
        return {"bytes": tokens * (2 * case["hq"] * case["d"] * es + 2 * kv * es + 2 * kv), "flops": 8 * tokens * kv}
    if case["op"] == "paged":
        keys, t = sum(_paged_lens(case)), case["t"]
        blocks = sum(-(-n // case["page"]) for n in _paged_lens(case))
        return {"bytes": 2 * keys * case["hkv"] * case["d"] + blocks * (8 * case["hkv"] + 4) + 2 * case["b"] * t * case["hq"] * case["d"] * es,
                "flops": 4 * keys * t * case["hq"] * case["d"]}
    n, xs = case["t"] * case["d"], ES[case["xtype"]]
    return {"bytes": 2 * n * (xs + es) + es * dict(none=0, all=case["d"], each=n)[case["gate"]], "flops": 10 * n}


# ------------------------------------------------------------------ the definitions in 64 bits
def _exact_norm(x, w):
    return x / (x.pow(2).sum(-1, keepdim=True) / x.shape[-1] + EPS).sqrt() * w.double()


def _exact_turn(x, positions, inv_freq, factor, interleaved):
    out = x.clone()
    for i, f in enumerate(inv_freq.double().tolist()):
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + len(inv_freq))
        z = torch.polar(torch.full_like(positions, factor, dtype=torch.float64), positions.double() * f)[:, None]
        z = torch.complex(x[..., a], x[..., b]) * z
        out[..., a], out[..., b] = z.real, z.imag
    return out


def _exact_blocks(x, cache, scales, pages, start):
    """New tokens x [n, Hkv, D] of one sequence from position `start` on; codes and scales in 64 bits, in place."""
    size, n = cache.shape[2], len(x)
    for j in range(start // size, -(-(start + n) // size)):
        page = int(pages[j])
        lo, hi = max(start, j * size), min(start + n, (j + 1) * size)
        block = x[lo - start:hi - start].transpose(0, 1)
        top = block.abs().amax((1, 2))
        e = torch.log2(top / 448).round()
        e = torch.where(448 * torch.exp2(e) < top, e + 1, e).clamp_min(-126)
        if lo > j * size:
            old = torch.log2(scales[page]).round()
            e = torch.maximum(e, old)
            kept = cache[page, :, :lo - j * size] * torch.exp2(old - e)[:, None, None]
            cache[page, :, :lo - j * size] = kept.float().to(torch.float8_e4m3fn).double()
        scales[page] = torch.exp2(e)
        cache[page, :, lo - j * size:hi - j * size] = (block / torch.exp2(e)[:, None, None]).float().to(torch.float8_e4m3fn).double()


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rotary":
        x = s["x"].double()
        return _exact_turn(x if s["norm"] is None else _exact_norm(x, s["norm"]), s["positions"], s["inv_freq"], s["factor"], s["interleaved"])
    if case["op"] == "append":
        starts, lens = _append_lens(case)
        pos = torch.cat([torch.arange(a, a + n) for a, n in zip(starts, lens)]).cuda()
        turned = [None if x is None else _exact_turn(x.double() if w is None else _exact_norm(x.double(), w), pos, s["inv_freq"], 1.0, False)
                  for x, w in ((s["q"], s["q_norm"]), (s["k"], s["k_norm"]))]
        cache = [x.double() for x in s["cache"]]
        at = 0
        for i, n in enumerate(lens):
            _exact_blocks(turned[1][at:at + n], cache[0], cache[2], s["table"][i].tolist(), starts[i])
            _exact_blocks(s["v"][at:at + n].double(), cache[1], cache[3], s["table"][i].tolist(), starts[i])
            at += n
        return ([] if turned[0] is None else [turned[0]]) + cache
    if case["op"] == "paged":
        q = s["q"].double().view(case["b"], case["t"], case["hq"], case["d"])
        rep, page, out = case["hq"] // case["hkv"], case["page"], torch.zeros_like(q)
        for i, n in enumerate(_paged_lens(case)):
            ids = s["table"][i, :-(-n // page)].long()
            for h in range(case["hkv"]):
                k, v = ((c[ids, h].double() * f[ids, h].double()[:, None, None]).flatten(0, 1)[:n] for c, f in zip(s["cache"][:2], s["cache"][2:]))
                for t in range(case["t"]):
                    seen = n - case["t"] + t + 1
                    w = torch.softmax(q[i, t, h * rep:(h + 1) * rep] @ k[:seen].t() * case["d"] ** -0.5, 1)
                    out[i, t, h * rep:(h + 1) * rep] = w @ v[:seen]
        return out.view(s["q"].shape)
    z = s["y"].double()
    z = z if s["post"] is None else _exact_norm(z, s["post"])
    z = s["x"].double() + case["scale"] * (z if s["gate"] is None else z * s["gate"].double())
    return z, _exact_norm(z, s["weight"])
