"""Speculative decoding over paged caches: the serving calls together.

A small decoder (random weights) generates for a batch of sequences of different
lengths.  Each round a smaller one drafts a few tokens, a token at a time; the
target takes the last token and all drafts of every sequence in one pass;
``verify_draft`` settles how many stand and samples the next.  Every layer
stores its new keys and values with ``kv_write`` and attends with
``paged_attention``.  Drafts that did not stand leave nothing to undo: lengths
step back, and their slots are written again.

    python examples/speculative_decode.py --cache i8 --sequences 8 --rounds 20

The reference's own generation loop re-runs the whole prefix for each token
(run_gpt2.py:92-113).
"""

from __future__ import annotations

import argparse
import math
import pathlib
import sys

import torch

sys.path.insert(0, str(pathlib.Path(__file__).resolve().parents[1]))
import __graft_entry__  # noqa: E402

__graft_entry__.load_package()
from lbr_b200 import paged  # noqa: E402

CACHES = {"f32": torch.float32, "bf16": torch.bfloat16, "i8": torch.int8, "f8": torch.float8_e4m3fn}


class PagedCache:
    """Pages for all layers of one model, and which sequence has which of them."""

    def __init__(self, layers, heads, dim, dtype, sequences, longest, page_size=16, device="cuda"):
        per = -(-longest // page_size)
        shape = (sequences * per, page_size, heads, dim)
        self.page_size = page_size
        self.pages = [[torch.zeros(shape, dtype=dtype, device=device) for _ in "kv"] for _ in range(layers)]
        scaled = dtype in (torch.int8, torch.float8_e4m3fn)
        self.scales = [[torch.zeros(shape[:3], device=device) if scaled else None for _ in "kv"] for _ in range(layers)]
        # any page may be anywhere
        self.table = torch.randperm(shape[0], device=device).to(torch.int32).view(sequences, per)

    def slots(self, seq, pos):
        return self.table[seq, pos // self.page_size].long() * self.page_size + pos % self.page_size

    def write(self, layer, k, v, slots):
        (kp, vp), (ks, vs) = self.pages[layer], self.scales[layer]
        paged.kv_write(k, v, kp, vp, slots, k_scale=ks, v_scale=vs)

    def attend(self, layer, q, lens, cu, max_new, max_kv):
        (kp, vp), (ks, vs) = self.pages[layer], self.scales[layer]
        return paged.paged_attention(q, kp, vp, self.table, lens, cu, k_scale=ks, v_scale=vs, max_new=max_new, max_kv=max_kv)

    def read(self, layer, cu, total):
        (kp, vp), (ks, vs) = self.pages[layer], self.scales[layer]
        return paged.kv_read(kp, vp, self.table, None, cu, total, k_scale=ks, v_scale=vs)


class Decoder:
    """Pre-norm blocks with grouped heads; sine positions; tied embedding."""

    def __init__(self, vocab, width, layers, q_heads, heads, seed, device="cuda"):
        g = torch.Generator(device=device)
        g.manual_seed(seed)
        self.q_heads, self.heads, self.dim, self.width, self.layers = q_heads, heads, width // q_heads, width, layers
        rand = lambda a, b: torch.randn(a, b, generator=g, device=device) / math.sqrt(a)   # noqa: E731
        self.embed = torch.randn(vocab, width, generator=g, device=device)
        self.blocks = [(rand(width, (q_heads + 2 * heads) * self.dim), rand(width, width), rand(width, 4 * width), rand(4 * width, width))
                       for _ in range(layers)]
        self.freq = 10000.0 ** (-torch.arange(0, width, 2, device=device) / width)

    def __call__(self, tokens, pos, attend):
        """Logits of flat ``tokens`` at positions ``pos``; ``attend(layer, q, k, v)`` is the attention."""
        a = pos[:, None] * self.freq
        x = self.embed.to(a.dtype)[tokens] + torch.stack([a.sin(), a.cos()], -1).flatten(1)
        norm = lambda y: y * torch.rsqrt((y * y).mean(-1, keepdim=True) + 1e-6)   # noqa: E731
        for i, (wqkv, wo, w1, w2) in enumerate(self.blocks):
            qkv = (norm(x) @ wqkv.to(x.dtype)).unflatten(-1, (-1, self.dim))
            q, k, v = qkv.split([self.q_heads, self.heads, self.heads], 1)
            x = x + attend(i, q, k, v).reshape(len(x), -1) @ wo.to(x.dtype)
            x = x + torch.nn.functional.gelu(norm(x) @ w1.to(x.dtype)) @ w2.to(x.dtype)
        return norm(x) @ self.embed.to(x.dtype).T / math.sqrt(self.width)

    def step(self, cache, tokens, seq, pos, lens, cu, max_new, max_kv):
        slots = cache.slots(seq, pos)

        def attend(layer, q, k, v):
            cache.write(layer, k, v, slots)
            return cache.attend(layer, q, lens, cu, max_new, max_kv)
        return self(tokens, pos, attend)


class Generator:
    """State of a batch: tokens known so far, of which all but the last are in the target's cache."""

    def __init__(self, target, draft, prompts, cache="f32", drafts=4, rounds=8, seed=0, device="cuda"):
        self.target, self.draft, self.drafts = target, draft, drafts
        B, longest = len(prompts), max(map(len, prompts)) + (rounds + 1) * (drafts + 1)
        self.longest, self.B = longest, B
        self.rng = torch.Generator(device=device)
        self.rng.manual_seed(seed)
        self.tokens = torch.zeros(B, longest, dtype=torch.int64, device=device)
        for b, p in enumerate(prompts):
            assert len(p) >= 2
            self.tokens[b, :len(p)] = torch.tensor(p)
        self.n = torch.tensor([len(p) for p in prompts], device=device)
        self.caches = [PagedCache(m.layers, m.heads, m.dim, CACHES[cache], B, longest, device=device) for m in (target, draft)]
        # the prompts but for their last token, ragged, in one pass of each model
        own = self.n - 1
        cu = torch.nn.functional.pad(own.cumsum(0), (1, 0)).to(torch.int32)
        seq = torch.repeat_interleave(torch.arange(B, device=device), own)
        pos = torch.arange(len(seq), device=device) - cu[seq].long()
        for m, c in zip((target, draft), self.caches):
            m.step(c, self.tokens[seq, pos], seq, pos, own.to(torch.int32), cu, int(own.max()), longest)

    def _run(self, model, cache, first, count):
        """Probabilities [B, count, vocab] after tokens first .. first + count - 1 of every sequence."""
        dev = self.tokens.device
        seq = torch.arange(self.B, device=dev).repeat_interleave(count)
        pos = (first[:, None] + torch.arange(count, device=dev)).flatten()
        cu = torch.arange(0, self.B * count + 1, count, dtype=torch.int32, device=dev)
        self.logits = model.step(cache, self.tokens[seq, pos], seq, pos, (first + count).to(torch.int32), cu, count, self.longest)
        return torch.softmax(self.logits, -1).view(self.B, count, -1)

    def round(self):
        """Draft, check, sample: returns (tokens, accepted) of ``verify_draft``.  Nothing waits for the device."""
        K, B, dev = self.drafts, self.B, self.tokens.device
        q = []
        for i in range(K):   # the first pass takes two tokens: the last draft of a round has not been in the draft's cache
            p = self._run(self.draft, self.caches[1], self.n - 2, 2) if i == 0 else self._run(self.draft, self.caches[1], self.n + i - 1, 1)
            q.append(p[:, -1])
            x = torch.multinomial(q[-1], 1, generator=self.rng)
            self.tokens.scatter_(1, (self.n + i)[:, None], x)
        at = self.n[:, None] + torch.arange(K + 1, device=dev)
        p = self._run(self.target, self.caches[0], self.n - 1, K + 1)
        out, accepted = paged.verify_draft(p, torch.stack(q, 1), self.tokens.gather(1, at[:, :K]).to(torch.int32),
                                           torch.rand(B, K, generator=self.rng, device=dev), torch.rand(B, generator=self.rng, device=dev))
        self.tokens.scatter_(1, at, out.clamp(min=0).long())
        self.n = self.n + accepted + 1
        return out, accepted


def main():
    a = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    a.add_argument("--cache", choices=CACHES, default="i8")
    a.add_argument("--sequences", type=int, default=4)
    a.add_argument("--rounds", type=int, default=16)
    a.add_argument("--drafts", type=int, default=4)
    a = a.parse_args()
    target = Decoder(1000, 512, 4, 8, 4, seed=1)
    draft = Decoder(1000, 512, 4, 8, 4, seed=1)
    draft.blocks, draft.layers = draft.blocks[:2], 2      # the target's first half drafts for it
    prompts = [[(7 * b + 3 * i) % 1000 for i in range(5 + 40 * b)] for b in range(a.sequences)]
    run = Generator(target, draft, prompts, a.cache, a.drafts, a.rounds)
    kept = sum(run.round()[1].float().mean() for _ in range(a.rounds))
    paged.check_stream()
    for b, p in enumerate(prompts):
        print(f"sequence {b}: prompt {len(p)} tokens, then", run.tokens[b, len(p):int(run.n[b])].tolist()[:12], "...")
    print(f"{float(kept) / a.rounds:.2f} of {a.drafts} drafts kept per round")


if __name__ == "__main__":
    main()
