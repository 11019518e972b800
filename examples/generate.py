"""Greedy generation with the package's generation operators on a small Qwen3-shaped model with random weights.

    python examples/generate.py [--layers 4] [--prompts 6] [--tokens 16]

All prompts begin with the same system prompt. They are prefilled packed into one batch without padding
(packed_attention); the system prompt's keys and values are then kept once for all, and each prompt's own ones in a
cache of its own. Every further token runs its linears on 4-bit weights (linear_w4), attends to the shared prefix and
its own keys (shared_prefix_attention), and is chosen after penalties, a bias and a mask (process_logits).
"""

import argparse
import sys
import time
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parent.parent / "torch-xdna_b200"))
import torch_xdna  # noqa: E402
from torch_xdna import kernels  # noqa: E402

D, NH, NKV, DH, INTER, EPS = 1024, 16, 8, 128, 3072, 1e-6  # Qwen3-0.6B's widths
GROUP = 128


def norm(x, w):
    x = x.float()
    return (x * torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + EPS) * w).bfloat16()


def rope(x, pos):
    """Rotates x [T, H, DH] to the positions pos [T]."""
    freq = 1.0 / 1e6 ** (torch.arange(0, DH, 2, device=x.device).float() / DH)
    angle = (pos.float()[:, None] * freq)[:, None, :]
    c, s, (a, b) = angle.cos(), angle.sin(), x.float().chunk(2, -1)
    return torch.cat((a * c - b * s, b * c + a * s), -1).bfloat16()


class Linear4:
    """One weight in 4 bits for decoding, and what these bits stand for in bf16 for the prompts."""

    def __init__(self, n, k, gen, device):
        w = (torch.randn(n, k, generator=gen, device=device) * k ** -0.5).bfloat16()
        self.codes, self.scales = torch_xdna.w4_pack(w, GROUP)
        # the columns of the identity give the weight back, a hundred at a time
        eye = torch.eye(k, device=device, dtype=torch.bfloat16)
        self.w = torch.cat([self.few(eye[i:i + 96]) for i in range(0, k, 96)]).t().contiguous()

    def few(self, x):
        return torch_xdna.linear_w4(x, self.codes, self.scales, GROUP)

    def many(self, x):
        y = torch.empty(x.shape[0], self.w.shape[0], dtype=torch.bfloat16, device=x.device)
        kernels.gemm_bf16(x.contiguous(), self.w, kernels.GEMM_F32ACC, out=y)
        return y


class Model:
    def __init__(self, layers, vocab, device, seed=0):
        gen = torch.Generator(device=device).manual_seed(seed)
        self.layers = [dict(qkv=Linear4((NH + 2 * NKV) * DH, D, gen, device), o=Linear4(D, NH * DH, gen, device),
                            up=Linear4(2 * INTER, D, gen, device), down=Linear4(D, INTER, gen, device))
                       for _ in range(layers)]
        self.head = Linear4(vocab, D, gen, device)
        self.embed = torch.randn(vocab, D, generator=gen, device=device).bfloat16()
        self.ones = torch.ones(D, device=device)
        self.vocab = vocab

    def forward(self, tokens, pos, linear, attend):
        """Logits [T, vocab] of tokens [T] at positions pos; attend(layer, q, k, v) is the attention."""
        x = self.embed[tokens].float()
        for i, w in enumerate(self.layers):
            qkv = linear(w["qkv"], norm(x, self.ones)).unflatten(1, (-1, DH))
            q, k, v = qkv.split((NH, NKV, NKV), 1)
            q, k = rope(norm(q, self.ones[:DH]), pos), rope(norm(k, self.ones[:DH]), pos)
            x = x + linear(w["o"], attend(i, q, k, v).flatten(1)).float()
            gate, up = linear(w["up"], norm(x, self.ones)).float().chunk(2, 1)
            x = x + linear(w["down"], (torch.nn.functional.silu(gate) * up).bfloat16()).float()
        return linear(self.head, norm(x, self.ones))

    def prefill(self, prompts):
        """Packed logits of whole prompts (a list of token tensors), and each layer's keys and values."""
        lens = [len(p) for p in prompts]
        device = prompts[0].device
        cu = torch.tensor([0] + lens, device=device).cumsum(0).to(torch.int32)
        pos = torch.cat([torch.arange(n, device=device) for n in lens])
        kept = []

        def attend(i, q, k, v):
            kept.append((k, v))
            return torch_xdna.packed_attention(q, k, v, cu)

        return self.forward(torch.cat(prompts), pos, Linear4.many, attend), kept, cu


class Session:
    """Prompts that share their first `shared` tokens, and their continuations."""

    def __init__(self, model, prompts, shared, room):
        self.model, device = model, prompts[0].device
        logits, kept, cu = model.prefill(prompts)
        b = len(prompts)
        own = [len(p) - shared for p in prompts]
        size = max(own) + room
        self.prefix, self.cache = [], []
        for k, v in kept:
            self.prefix.append((k[:shared], v[:shared]))
            ck = torch.zeros(b, size, NKV, DH, dtype=torch.bfloat16, device=device)
            cv = torch.zeros_like(ck)
            for j in range(b):
                at = int(cu[j]) + shared
                ck[j, :own[j]], cv[j, :own[j]] = k[at:at + own[j]], v[at:at + own[j]]
            self.cache.append((ck, cv))
        self.shared = shared
        self.lens = torch.tensor(own, dtype=torch.int32, device=device)
        self.rows = torch.arange(b, device=device)
        # the tokens so far: prompt, then what is generated
        self.tokens = torch.full((b, shared + size), -1, dtype=torch.int32, device=device)
        for j, p in enumerate(prompts):
            self.tokens[j, :len(p)] = p.int()
        self.prompt_lens = self.lens + shared
        self.logits = logits[cu[1:].long() - 1]
        self.repetition = torch.full((b,), 1.3, device=device)
        self.presence = torch.full((b,), 0.2, device=device)
        self.frequency = torch.full((b,), 0.1, device=device)

    def choose(self, bias=None, mask=None):
        """The next token of each sequence, the likeliest after penalties, bias and mask."""
        scores = torch_xdna.process_logits(self.logits, self.tokens, self.lens + self.shared, self.prompt_lens,
                                           repetition=self.repetition, presence=self.presence,
                                           frequency=self.frequency, bias=bias, mask=mask)
        return scores.argmax(1)

    def step(self, token):
        """Takes each sequence's next token in; self.logits is then the one after it."""
        at = self.lens.long()
        self.tokens[self.rows, at + self.shared] = token.int()
        after = self.lens + 1

        def attend(i, q, k, v):
            ck, cv = self.cache[i]
            ck[self.rows, at], cv[self.rows, at] = k, v
            return torch_xdna.shared_prefix_attention(q, *self.prefix[i], ck, cv, after)

        self.logits = self.model.forward(token, at + self.shared, Linear4.few, attend)
        self.lens = after


def main():
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--layers", type=int, default=4)
    ap.add_argument("--prompts", type=int, default=6)
    ap.add_argument("--tokens", type=int, default=16)
    ap.add_argument("--vocab", type=int, default=8200)
    a = ap.parse_args()
    gen = torch.Generator().manual_seed(1)
    system = torch.randint(0, a.vocab, (300,), generator=gen)
    prompts = [torch.cat((system, torch.randint(0, a.vocab, (5 + 17 * i,), generator=gen))).cuda() for i in range(a.prompts)]
    with torch.no_grad():
        model = Model(a.layers, a.vocab, torch.device("cuda"))
        session = Session(model, prompts, len(system), a.tokens)
        bias = torch.zeros(a.vocab, device="cuda")
        bias[0] = -5.0                                              # discouraged
        mask = torch.full((1, -(-a.vocab // 32)), -1, dtype=torch.int32, device="cuda")
        mask[0, 0] &= ~0b1110                                       # tokens 1, 2 and 3 are not allowed
        torch.cuda.synchronize()
        t0 = time.perf_counter()
        for _ in range(a.tokens):
            session.step(session.choose(bias, mask))
        torch.cuda.synchronize()
        seconds = time.perf_counter() - t0
    for j in range(a.prompts):
        n = int(session.prompt_lens[j])
        print(f"prompt of {n} tokens ->", session.tokens[j, n:n + a.tokens].tolist())
    print(f"{a.prompts * a.tokens / seconds:.0f} tokens/s;", torch_xdna.report().splitlines()[-1].strip())


if __name__ == "__main__":
    main()
