"""Greedy generation over a paged cache in 8 bits, on the Qwen3-shaped model with random weights of generate.py.

    python examples/generate_paged.py [--layers 4] [--prompts 6] [--tokens 16] [--format int8]

The prompts are prefilled packed (rotary, packed_attention), their keys and values go into the pages of one pool per layer
(cache_append), and every further token runs on 4-bit weights (linear_w4), appends to the cache with the norm and the
rotation of queries and keys on the way, attends to the pages (paged_attention) and passes the norms between the blocks in
one call each (add_norm). The next token is chosen after penalties (process_logits).
"""

import argparse
import sys
import time
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parent))
from generate import D, DH, EPS, NH, NKV, Linear4, Model, norm, torch_xdna  # noqa: E402

PAGE = 64


class PagedSession:
    """Prompts and their continuations: a pool of pages per layer, and each sequence's pages."""

    def __init__(self, model, prompts, room, dtype=torch.int8):
        self.model, self.device = model, prompts[0].device
        lens = [len(p) for p in prompts]
        pages = [-(-(n + room) // PAGE) for n in lens]
        order = torch.randperm(sum(pages), generator=torch.Generator().manual_seed(0)).int()
        self.table = torch.full((len(prompts), max(pages)), -1, dtype=torch.int32)
        for i, p in enumerate(order.split(pages)):
            self.table[i, :len(p)] = p
        self.table = self.table.to(self.device)
        self.caches = [torch_xdna.paged_cache(sum(pages), NKV, DH, PAGE, dtype, self.device) for _ in model.layers]
        self.freq, self.factor = torch_xdna.rotary_frequencies(DH, 1e6, device=self.device)
        self.qk_norm = torch.ones(DH, device=self.device)
        self.lens = torch.zeros(len(prompts), dtype=torch.int32, device=self.device)
        cu = torch.tensor([0] + lens, device=self.device).cumsum(0).to(torch.int32)
        self.logits = self.forward(torch.cat(prompts), Linear4.many, cu)[cu[1:].long() - 1]
        self.tokens = torch.full((len(prompts), max(lens) + room), -1, dtype=torch.int32, device=self.device)
        for i, p in enumerate(prompts):
            self.tokens[i, :len(p)] = p.int()
        self.prompt_lens = self.lens.clone()
        self.repetition = torch.full((len(prompts),), 1.3, device=self.device)

    def attend(self, i, qkv, cu):
        """Attention of layer i's projections [T, NH + 2 NKV, DH], which are taken into its cache."""
        v, rotation = qkv[:, NH + NKV:], dict(inv_freq=self.freq, factor=self.factor, eps=EPS)
        if cu is None:  # one token of each sequence
            q = torch_xdna.cache_append(qkv[:, NH:NH + NKV], v, *self.caches[i], self.table, self.lens, k_norm=self.qk_norm,
                                        q=qkv[:, :NH], q_norm=self.qk_norm, **rotation)
            return torch_xdna.paged_attention(q, *self.caches[i], self.table, self.lens + 1)
        # whole prompts: the rotated keys are needed in 16 bits too
        pos = torch.cat([torch.arange(n, device=self.device) for n in (cu[1:] - cu[:-1]).tolist()])
        qk = torch_xdna.rotary(qkv[:, :NH + NKV], pos, self.freq, self.factor, norm=self.qk_norm, eps=EPS)
        torch_xdna.cache_append(qk[:, NH:], v, *self.caches[i], self.table, self.lens, cu)
        return torch_xdna.packed_attention(qk[:, :NH], qk[:, NH:], v, cu)

    def forward(self, tokens, linear, cu=None):
        """Logits of the sequences' next tokens (with cu: of packed prompts), which are taken in."""
        ones = self.model.ones
        x = self.model.embed[tokens].float()
        h = norm(x, ones)
        for i, w in enumerate(self.model.layers):
            o = self.attend(i, linear(w["qkv"], h).unflatten(1, (-1, DH)), cu)
            x, h = torch_xdna.add_norm(x, linear(w["o"], o.flatten(1)), ones, eps=EPS)
            gate, up = linear(w["up"], h).float().chunk(2, 1)
            x, h = torch_xdna.add_norm(x, linear(w["down"], (torch.nn.functional.silu(gate) * up).bfloat16()), ones, eps=EPS)
        self.lens = self.lens + (1 if cu is None else cu[1:] - cu[:-1])
        return linear(self.model.head, h)

    def choose(self):
        """The next token of each sequence, the likeliest after the penalty."""
        scores = torch_xdna.process_logits(self.logits, self.tokens, self.lens, self.prompt_lens, repetition=self.repetition)
        return scores.argmax(1)

    def step(self, token):
        """Takes each sequence's next token in; self.logits is then the one after it."""
        self.tokens.scatter_(1, self.lens.long()[:, None], token.int()[:, None])
        self.logits = self.forward(token, Linear4.few)


def main():
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--layers", type=int, default=4)
    ap.add_argument("--prompts", type=int, default=6)
    ap.add_argument("--tokens", type=int, default=16)
    ap.add_argument("--vocab", type=int, default=8200)
    ap.add_argument("--format", choices=["int8", "e4m3"], default="int8")
    a = ap.parse_args()
    gen = torch.Generator().manual_seed(1)
    prompts = [torch.randint(0, a.vocab, (40 + 97 * i,), generator=gen).cuda() for i in range(a.prompts)]
    with torch.no_grad():
        model = Model(a.layers, a.vocab, torch.device("cuda"))
        session = PagedSession(model, prompts, a.tokens, dict(int8=torch.int8, e4m3=torch.float8_e4m3fn)[a.format])
        torch.cuda.synchronize()
        t0 = time.perf_counter()
        for _ in range(a.tokens):
            session.step(session.choose())
        torch.cuda.synchronize()
        seconds = time.perf_counter() - t0
    for j, n in enumerate(session.prompt_lens.tolist()):
        print(f"prompt of {n} tokens ->", session.tokens[j, n:n + a.tokens].tolist())
    print(f"{a.prompts * a.tokens / seconds:.0f} tokens/s;", torch_xdna.report().splitlines()[-1].strip())


if __name__ == "__main__":
    main()
