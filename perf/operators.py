"""What the generation operators of torch_xdna are measured on: the packed prompt attention, the shared-prefix
decode attention, the 4-bit linear and the logits processing.

Each case is one call as a serving loop makes it. The plain forms are elementary torch operations in 32 bits,
rounded once at the end; `exact` restates each definition in 64 bits.
"""

import math
import os
import random
import sys

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
ES = {"bf16": 2, "f16": 2, "f32": 4}
CODE_BLOCK = 128  # columns per block of the 4-bit codes


def listed():
    return [
        # a handful of short requests, one of a single token: the smallest prefill call of a server
        dict(name="packed_short", op="packed", dtype="bf16", hq=16, hkv=8, d=128, lens="1,17,64,130,33"),
        # a prefill batch of ordinary requests with ragged lengths
        dict(name="packed_ragged", op="packed", dtype="bf16", hq=16, hkv=8, d=128,
             lens="1900,1024,777,1333,128,999,1600,512,255,1801,640,1111,301,1450,96,1207"),
        # one long document
        dict(name="packed_long", op="packed", dtype="bf16", hq=16, hkv=8, d=128, lens="8191"),
        # heads of 64 with one key/value head each, in f16
        dict(name="packed_d64", op="packed", dtype="f16", hq=12, hkv=12, d=64, lens="2047,513,1280,700"),
        # one user behind a system prompt: latency
        dict(name="prefix_one", op="prefix", dtype="bf16", hq=16, hkv=8, d=128, b=1, p=700, s=64),
        # an ordinary batch behind a long system prompt
        dict(name="prefix_batch", op="prefix", dtype="bf16", hq=16, hkv=8, d=128, b=32, p=4096, s=600),
        # many samples of one long document, odd sizes
        dict(name="prefix_wide", op="prefix", dtype="f16", hq=16, hkv=8, d=128, b=190, p=16381, s=301),
        # q/k/v projection of one decoded token
        dict(name="w4_qkv_one", op="w4", dtype="bf16", m=1, n=4096, k=1024, group=128, bias=False),
        # the vocabulary head for a small batch
        dict(name="w4_head", op="w4", dtype="bf16", m=8, n=151936, k=1024, group=128, bias=False),
        # odd sizes, fine groups, a bias and 32-bit activations
        dict(name="w4_odd_f32", op="w4", dtype="f32", m=5, n=1001, k=2999, group=32, bias=True),
        # the next token of one sequence: latency
        dict(name="logits_one", op="logits", dtype="f32", b=1, v=151936, t=300, bias="row", mask=True),
        # a decode batch with grammar masks and long histories
        dict(name="logits_batch", op="logits", dtype="bf16", b=128, v=151936, t=2048, bias="shared", mask=True),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["packed", "prefix", "w4", "logits"])
    if op == "packed":
        hq, hkv, d = rng.choice([(16, 8, 128), (16, 8, 128), (8, 8, 128), (12, 4, 128), (16, 2, 64), (12, 12, 64),
                                 (14, 2, 64)])
        n = _log(rng, 1, 24)
        top = int(math.sqrt(16 * 6000.0 ** 2 / (n * hq)))  # the padded plain form stays below the longest listed case
        lens = [_log(rng, 1, top) for _ in range(n)]
        return dict(op=op, dtype=rng.choice(["bf16", "f16"]), hq=hq, hkv=hkv, d=d, lens=",".join(map(str, lens)))
    if op == "prefix":
        hq, hkv, d = rng.choice([(16, 8, 128), (16, 8, 128), (8, 8, 128), (12, 4, 128), (16, 2, 64), (14, 2, 64)])
        b = _log(rng, 1, 160)
        return dict(op=op, dtype=rng.choice(["bf16", "f16"]), hq=hq, hkv=hkv, d=d, b=b, p=_log(rng, 1, 12000),
                    s=_log(rng, 1, 300))
    if op == "w4":
        n, k = rng.choice([(4096, 1024), (1024, 2048), (6144, 1024), (_log(rng, 33, 20000), _log(rng, 65, 6000))])
        return dict(op=op, dtype=rng.choice(["bf16", "f16", "f32"]), m=_log(rng, 1, 48), n=n, k=k,
                    group=rng.choice([32, 64, 128]), bias=rng.random() < 0.3)
    return dict(op=op, dtype=rng.choice(["bf16", "f16", "f32"]), b=_log(rng, 1, 48), v=_log(rng, 1000, 152000),
                t=_log(rng, 1, 4000), bias=rng.choice(["none", "shared", "row"]), mask=rng.random() < 0.7)


# ------------------------------------------------------------------ inputs
def _packed_lens(case):
    return [int(x) for x in case["lens"].split(",")]


def _own_lens(case):
    """Own tokens of each sequence behind the shared prefix: from none to all of the cache."""
    r = random.Random("%d.%d.%d" % (case["b"], case["p"], case["s"]))
    return [r.randint(0, case["s"]) for _ in range(case["b"])]


def _history(case):
    """(tokens so far, of these the prompt's) of each row."""
    r = random.Random("%d.%d.%d" % (case["b"], case["v"], case["t"]))
    lens = [r.randint((case["t"] + 1) // 2, case["t"]) for _ in range(case["b"])]
    return lens, [r.randint(0, n) for n in lens]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def randn(*shape, scale=1.0, dtype=dt):
        return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)

    state = dict(op=case["op"])
    if case["op"] == "packed":
        lens = _packed_lens(case)
        t, hq, hkv, d = sum(lens), case["hq"], case["hkv"], case["d"]
        # queries and keys as they leave their norm and rotation; all three are views of one projection's output
        qkv = randn(t, hq + 2 * hkv, d, scale=1.2)
        state.update(q=qkv[:, :hq], k=qkv[:, hq:hq + hkv], v=qkv[:, hq + hkv:], max_len=max(lens),
                     cu=torch.tensor([0] + lens).cumsum(0).to(torch.int32).cuda())
    elif case["op"] == "prefix":
        b, p, s, hq, hkv, d = (case[x] for x in ("b", "p", "s", "hq", "hkv", "d"))
        state.update(q=randn(b, hq, d, scale=1.2), pk=randn(p, hkv, d, scale=1.2), pv=randn(p, hkv, d),
                     ck=randn(b, s, hkv, d, scale=1.2), cv=randn(b, s, hkv, d),
                     lens=torch.tensor(_own_lens(case), dtype=torch.int32).cuda())
    elif case["op"] == "w4":
        m, n, k, group = case["m"], case["n"], case["k"], case["group"]
        codes = torch.randn(n, k, generator=g, device="cuda").mul_(2.5).round_().clamp_(-8, 7).add_(8).to(torch.uint8)
        sdt = torch.bfloat16 if dt == torch.bfloat16 else torch.float16
        scales = (torch.rand(n, -(-k // group), generator=g, device="cuda") * 0.01 + 0.002).to(sdt)
        state.update(x=randn(m, k), codes=_pack(codes), scales=scales, group=group,
                     bias=randn(n, scale=0.1) if case["bias"] else None)
    else:
        b, v, t = case["b"], case["v"], case["t"]
        lens, prompts = _history(case)
        u = torch.rand(b, t, generator=g, device="cuda")
        bias = dict(none=(), shared=(v,), row=(b, v))[case["bias"]]
        words = -(-v // 32)
        state.update(
            logits=randn(b, v, scale=3.0),
            tokens=(float(v) ** u - 1).to(torch.int32).clamp_(0, v - 1),  # few frequent tokens, many rare ones
            lens=torch.tensor(lens, dtype=torch.int32).cuda(), prompts=torch.tensor(prompts, dtype=torch.int32).cuda(),
            rep=torch.rand(b, generator=g, device="cuda") * 0.3 + 1.0, pres=torch.rand(b, generator=g, device="cuda") * 0.5,
            freq=torch.rand(b, generator=g, device="cuda") * 0.2,
            bias=randn(*bias, scale=0.5, dtype=torch.float32) if bias else None,
            mask=torch.randint(-2 ** 31, 2 ** 31, (b, words), generator=g, device="cuda", dtype=torch.int64).to(
                torch.int32) if case["mask"] else None)
    return state


def _pack(codes):
    """Codes 0..15 [N, K] in the stored layout [N, K' / 2] (K' = K rounded up to 128, padded with 8): in a block of
    128 columns the 8-column runs are stored run 4 w + t at place 4 t + w, and in a run the eight 4-bit codes lie in
    the order 0, 2, 4, 6, 1, 3, 5, 7 from the lowest bits."""
    n, k = codes.shape
    blocks = -(-k // CODE_BLOCK)
    c = torch.nn.functional.pad(codes, (0, blocks * CODE_BLOCK - k), value=8)
    c = c.view(n, blocks, 4, 4, 8).transpose(2, 3)[..., [0, 2, 4, 6, 1, 3, 5, 7]].reshape(n, -1, 2)
    return (c[..., 0] | (c[..., 1] << 4)).contiguous()


def _unpack(packed, k):
    n = packed.shape[0]
    c = torch.stack((packed & 15, packed >> 4), -1).view(n, -1, 4, 4, 8)
    return c[..., [0, 4, 1, 5, 2, 6, 3, 7]].transpose(2, 3).reshape(n, -1)[:, :k]


# ------------------------------------------------------------------ the plain forms
def _softmax(scores, allowed):
    """exp(s - max) and its sum over the allowed places; rows that allow nothing give zeros."""
    scores = torch.where(allowed, scores, -math.inf)
    top = scores.amax(-1, keepdim=True)
    e = torch.exp(scores - torch.where(top == -math.inf, 0.0, top))
    total = e.sum(-1, keepdim=True)
    return e / torch.where(total == 0, 1.0, total)


def _plain_packed(q, k, v, cu, max_len):
    cu = cu.long()
    start, lens = cu[:-1], cu[1:] - cu[:-1]
    pos = torch.arange(max_len, device=q.device)
    inside = pos < lens[:, None]                                   # [B, L]
    at = torch.where(inside, start[:, None] + pos, 0)
    rep = q.shape[1] // k.shape[1]
    qp = q.float()[at].transpose(1, 2)                             # [B, Hq, L, D]
    kp = k.float()[at].transpose(1, 2).repeat_interleave(rep, 1)
    vp = v.float()[at].transpose(1, 2).repeat_interleave(rep, 1)
    scores = qp @ kp.transpose(2, 3) / math.sqrt(q.shape[2])
    allowed = (pos[:, None] >= pos) & inside[:, None, None, :]
    o = _softmax(scores, allowed) @ vp
    token = torch.arange(q.shape[0], device=q.device)
    seq = torch.searchsorted(cu, token, right=True) - 1
    return o[seq, :, token - start[seq]].to(q.dtype)


def _plain_prefix(q, pk, pv, ck, cv, lens):
    b, hq, d = q.shape
    hkv = pk.shape[1]
    qg = q.float().view(b, hkv, hq // hkv, d)
    shared = torch.einsum("bhgd,phd->bhgp", qg, pk.float())
    each = torch.einsum("bhgd,bshd->bhgs", qg, ck.float())
    p, s = pk.shape[0], ck.shape[1]
    allowed = torch.cat((torch.ones(b, p, dtype=torch.bool, device=q.device),
                         torch.arange(s, device=q.device) < lens[:, None]), 1)[:, None, None, :]
    w = _softmax(torch.cat((shared, each), -1) / math.sqrt(d), allowed)
    o = torch.einsum("bhgp,phd->bhgd", w[..., :p], pv.float()) + torch.einsum("bhgs,bshd->bhgd", w[..., p:], cv.float())
    return o.reshape(b, hq, d).to(q.dtype)


def _plain_w4(x, codes, scales, group, bias):
    k = x.shape[1]
    w = (_unpack(codes, k).float() - 8) * scales.float().repeat_interleave(group, 1)[:, :k]
    y = x.float() @ w.t()
    return (y if bias is None else y + bias.float()).to(x.dtype)


def _plain_logits(logits, tokens, lens, prompts, rep, pres, freq, bias, mask):
    b, v = logits.shape
    pos = torch.arange(tokens.shape[1], device=logits.device)
    in_history, in_prompt = pos < lens[:, None], pos < prompts[:, None]
    ids = tokens.long()
    seen = torch.zeros(b, v, device=logits.device).scatter_add_(1, ids, in_history.float()) > 0
    count = torch.zeros(b, v, device=logits.device).scatter_add_(1, ids, (in_history & ~in_prompt).float())
    y = logits.float()
    r = rep[:, None]
    y = torch.where(seen, torch.where(y > 0, y / r, y * r), y)
    y = y - freq[:, None] * count - pres[:, None] * (count > 0)
    if bias is not None:
        y = y + bias
    if mask is not None:
        bit = torch.arange(32, device=logits.device)
        allowed = ((mask[..., None] >> bit) & 1).view(b, -1)[:, :v] != 0
        y = torch.where(allowed, y, -math.inf)
    return y.to(logits.dtype)


def _package():
    if "torch_xdna" not in sys.modules:
        here = os.path.join(os.getcwd(), "torch-xdna_b200")
        if here not in sys.path:
            sys.path.insert(0, here)
        import torch_xdna  # noqa: F401
    return sys.modules["torch_xdna"]


def run(state):
    s = state
    if s["op"] == "packed":
        if own:
            return _package().packed_attention(s["q"], s["k"], s["v"], s["cu"])
        return _plain_packed(s["q"], s["k"], s["v"], s["cu"], s["max_len"])
    if s["op"] == "prefix":
        if own:
            return _package().shared_prefix_attention(s["q"], s["pk"], s["pv"], s["ck"], s["cv"], s["lens"])
        return _plain_prefix(s["q"], s["pk"], s["pv"], s["ck"], s["cv"], s["lens"])
    if s["op"] == "w4":
        if own:
            return _package().linear_w4(s["x"], s["codes"], s["scales"], s["group"], s["bias"])
        return _plain_w4(s["x"], s["codes"], s["scales"], s["group"], s["bias"])
    if own:
        return _package().process_logits(s["logits"], s["tokens"], s["lens"], s["prompts"], repetition=s["rep"],
                                         presence=s["pres"], frequency=s["freq"], bias=s["bias"], mask=s["mask"])
    return _plain_logits(s["logits"], s["tokens"], s["lens"], s["prompts"], s["rep"], s["pres"], s["freq"], s["bias"],
                         s["mask"])


# ------------------------------------------------------------------ the work
def work(case):
    es = ES[case["dtype"]]
    if case["op"] == "packed":
        lens = _packed_lens(case)
        return {"bytes": sum(lens) * case["d"] * es * 2 * (case["hq"] + case["hkv"]),
                "flops": sum(4 * case["hq"] * case["d"] * n * (n + 1) // 2 for n in lens)}
    if case["op"] == "prefix":
        own_tokens = sum(_own_lens(case))
        return {"bytes": 2 * es * case["d"] * (case["hkv"] * (case["p"] + own_tokens) + case["b"] * case["hq"]),
                "flops": 4 * case["hq"] * case["d"] * (case["b"] * case["p"] + own_tokens)}
    if case["op"] == "w4":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": n * ((k + 1) // 2 + 2 * -(-k // case["group"])) + es * (m * k + m * n + n * case["bias"]),
                "flops": 2 * m * n * k}
    b, v = case["b"], case["v"]
    extra = dict(none=0, shared=v, row=b * v)[case["bias"]]
    return {"bytes": 2 * b * v * es + 4 * extra + (b * -(-v // 32) * 4 if case["mask"] else 0) + 4 * sum(_history(case)[0]),
            "flops": 8 * b * v}


# ------------------------------------------------------------------ the definitions in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "packed":
        q, k, v = (s[x].double() for x in "qkv")
        rep, out, at = q.shape[1] // k.shape[1], [], 0
        for n in _packed_lens(case):
            heads = []
            for h in range(q.shape[1]):
                z = q[at:at + n, h] @ k[at:at + n, h // rep].t() * q.shape[2] ** -0.5
                z.masked_fill_(torch.ones(n, n, dtype=torch.bool, device=z.device).triu_(1), -math.inf)
                heads.append(torch.softmax(z, 1) @ v[at:at + n, h // rep])
            out.append(torch.stack(heads, 1))
            at += n
        return torch.cat(out)
    if case["op"] == "prefix":
        q = s["q"].double()
        rep, rows = case["hq"] // case["hkv"], []
        pk, pv = s["pk"].double(), s["pv"].double()
        for i, n in enumerate(_own_lens(case)):
            k = torch.cat((pk, s["ck"][i, :n].double())).repeat_interleave(rep, 1)
            v = torch.cat((pv, s["cv"][i, :n].double())).repeat_interleave(rep, 1)
            z = (k * q[i]).sum(2) * case["d"] ** -0.5
            rows.append((torch.softmax(z, 0)[..., None] * v).sum(0))
        return torch.stack(rows)
    if case["op"] == "w4":
        k, group = case["k"], case["group"]
        c = _unpack(s["codes"], k).double() - 8
        y = torch.zeros(case["m"], case["n"], dtype=torch.float64, device=c.device)
        for j in range(-(-k // group)):
            part = slice(j * group, min(k, (j + 1) * group))
            y += (s["x"][:, part].double() @ c[:, part].t()) * s["scales"][:, j].double()
        return y if s["bias"] is None else y + s["bias"].double()
    y = s["logits"].double()
    lens, prompts = _history(case)
    for i in range(case["b"]):
        r, f, p = (float(s[x][i].double()) for x in ("rep", "freq", "pres"))
        seen = torch.unique(s["tokens"][i, :lens[i]].long())
        y[i, seen] = torch.where(y[i, seen] > 0, y[i, seen] / r, y[i, seen] * r)
        ids, count = torch.unique(s["tokens"][i, prompts[i]:lens[i]].long(), return_counts=True)
        y[i, ids] -= f * count.double() + p
    if s["bias"] is not None:
        y += s["bias"].double()
    if s["mask"] is not None:
        place = torch.arange(case["v"], device=y.device)
        y[((s["mask"].long()[:, place // 32] >> (place % 32)) & 1) == 0] = -math.inf
    return y
