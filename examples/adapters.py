"""Adapters of several users on one quantized model: quantize, train, measure, serve.

A toy language model (embedding, one MLP block, head) gets its two projections quantized and packed by
the engine. Each user then has a next-token rule of their own, and their low-rank adapters are trained
together, every batch holding tokens of all of them: the packed projections with adapters forward and
backward, the inputs kept as 8-bit checkpoints, the loss over the vocabulary without its logits, each
user's gradients clipped to a norm of their own on the way to the 32-bit weights.
After that the perplexity of every user's text is measured, single tokens of all users, and of one
without adapters, are decoded in one batch, and short texts are written in which words of the users'
texts only may stand and repeated ones are penalized.

    python examples/adapters.py [--steps 60] [--width 512] [--vocab 4096] [--train-head] [--train-embed]
                                [--clip 1.0] [--dtype bf16]
"""
import argparse
import math
import os
import sys

import numpy as np
import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "cdcl-gptq_amd"))
import cdclq  # noqa: E402
from cdclq import tune  # noqa: E402


def quantized(ctx, w, x, bits, name):
    """w (m x n) quantized on inputs x (tokens x n), packed, and laid out for products."""
    m, n = w.shape
    xs = np.ascontiguousarray(x.float().cpu().numpy())
    h = np.zeros((n, n))
    cdclq.gram_accumulate(xs, xs, len(xs), n, h, ctx)
    cfg = cdclq.Config(bits=bits, group=128, passes=2)
    ql, stats = cdclq.quantize_layer(w.float().cpu().numpy(), m, n, (h / len(xs)).astype(np.float32), None, name, cfg,
                                     cdclq.PrepCache(ctx=ctx))
    print(f"{name}: {m} x {n}, {bits} bits, proxy loss {stats.loss_gptq:.4g} -> {stats.loss_final:.4g}")
    return tune.PackedLinear.from_tensors(ctx, cdclq.packed_tensors(name, ql, ctx), name)


class Model:
    """h = e + down(silu(up(e))), logits = h head^T, with adapters on both projections."""

    def __init__(self, ctx, width, vocab, users, rank, bits, dtype, seed):
        g = torch.Generator().manual_seed(seed)

        def normal(*shape, std):
            return (torch.randn(*shape, generator=g) * std).to(dtype).cuda()

        hidden = 4 * width
        self.ctx, self.users = ctx, users
        self.embed = normal(vocab, width, std=1.0)
        self.head = normal(vocab, width, std=width ** -0.5)
        up, down = normal(hidden, width, std=width ** -0.5), normal(width, hidden, std=0.5 * hidden ** -0.5)
        x = self.embed[torch.randint(vocab, (4 * hidden,), generator=g).cuda()]
        self.up = quantized(ctx, up, x, bits, "up")
        self.down = quantized(ctx, down, torch.nn.functional.silu(tune.adapter_linear(self.up, x)), bits, "down")

        def adapters(m, n):  # B = 0: an untrained adapter changes nothing
            a = normal(users, rank, n, std=n ** -0.5)
            return tune.Adapters(a.requires_grad_(), torch.zeros(users, m, rank, dtype=dtype, device="cuda",
                                                                 requires_grad=True),
                                 torch.full((users,), 2.0, device="cuda"))

        self.up_ad, self.down_ad = adapters(hidden, width), adapters(width, hidden)

    def weights(self):
        return [self.up_ad.a, self.up_ad.b, self.down_ad.a, self.down_ad.b]

    def states(self, tokens, user):
        """Hidden states for autograd."""
        e = tune.embedding(self.ctx, self.embed, tokens)
        u = torch.nn.functional.silu(tune.linear(self.up, e, self.up_ad, user))
        return e + tune.linear(self.down, u, self.down_ad, user)

    def decode(self, tokens, user, **constraints):
        """The likeliest next token of each request, under constraints as tune.constrain_logits takes them."""
        with torch.no_grad():
            e = tune.embed(self.ctx, self.embed, tokens)
            u = torch.nn.functional.silu(tune.adapter_linear(self.up, e, self.up_ad, user))
            h = e + tune.adapter_linear(self.down, u, self.down_ad, user)
            logits = h @ self.head.T
            if constraints:
                tune.constrain_logits(self.ctx, logits, out=logits, **constraints)
            return logits.argmax(1)

    def write(self, tokens, user, steps, words):
        """Texts of `steps` tokens after the first ones: a token's second use costs more than its first, and only
        `words` may stand in them."""
        r, v = len(tokens), self.head.shape[0]
        allowed = torch.zeros(-(-v // 32) * 32, dtype=torch.int64, device="cuda")
        allowed[words] = 1
        bits = (allowed.view(1, -1, 32) << torch.arange(32, device="cuda")).sum(2)
        mask = torch.where(bits >= 1 << 31, bits - (1 << 32), bits).int()
        history = torch.zeros(r, steps + 1, dtype=torch.int64, device="cuda")
        history[:, 0] = tokens
        lengths = torch.ones(r, dtype=torch.int32, device="cuda")
        limits = dict(history=history, lengths=lengths, prompts=torch.ones_like(lengths),
                      repetition=torch.full((r,), 1.1, device="cuda"), frequency=torch.full((r,), 0.5, device="cuda"),
                      mask=mask, mask_rows=torch.zeros_like(lengths))
        for i in range(steps):
            history[:, i + 1] = tokens = self.decode(tokens, user, **limits)
            lengths += 1
        return history

    def perplexity(self, tokens, user, targets):
        with torch.no_grad():
            loss, _ = tune.vocab_loss(self.ctx, self.states(tokens, user), self.head, targets)
        return [math.exp(loss[user == u].mean().item()) for u in range(self.users)]


def main(argv=None):
    p = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    p.add_argument("--steps", type=int, default=60)
    p.add_argument("--tokens", type=int, default=2048, help="tokens of a training step")
    p.add_argument("--width", type=int, default=512)
    p.add_argument("--vocab", type=int, default=4096)
    p.add_argument("--users", type=int, default=4)
    p.add_argument("--rank", type=int, default=16)
    p.add_argument("--bits", type=int, default=4)
    p.add_argument("--words", type=int, default=48, help="tokens of the vocabulary that the texts use")
    p.add_argument("--lr", type=float, default=5e-3)
    p.add_argument("--dtype", choices=["bf16", "f16"], default="bf16")
    p.add_argument("--train-head", action="store_true", help="train the head's weights as well")
    p.add_argument("--train-embed", action="store_true", help="train the embedding as well")
    p.add_argument("--clip", type=float, default=math.inf, help="largest norm of a user's gradients")
    p.add_argument("--seed", type=int, default=0)
    o = p.parse_args(argv)
    ctx = cdclq.Context(0)
    m = Model(ctx, o.width, o.vocab, o.users, o.rank, o.bits, torch.bfloat16 if o.dtype == "bf16" else torch.float16,
              o.seed)
    g = torch.Generator().manual_seed(o.seed + 1)
    words = torch.randperm(o.vocab, generator=g)[: o.words].cuda()
    rules = torch.stack([words[torch.randperm(o.words, generator=g).cuda()] for _ in range(o.users)])

    def batch(t):
        """t tokens, users one after another; a tenth of the targets is padding."""
        user = torch.arange(t).mul(o.users).div(t, rounding_mode="floor").int().cuda()
        at = torch.randint(o.words, (t,), generator=g).cuda()
        target = rules[user.long(), at]
        return words[at], user, target.masked_fill((torch.rand(t, generator=g) < 0.1).cuda(), -100)

    def text(t):
        tokens, user, target = batch(t)
        keep = target != -100
        return tokens[keep].contiguous(), user[keep].contiguous(), target[keep].contiguous()

    held = text(1000)
    before = m.perplexity(*held)
    # 32-bit copies of what is trained: small steps would vanish in 16 bits
    rest = ([m.head.requires_grad_()] if o.train_head else []) + ([m.embed.requires_grad_()] if o.train_embed else [])
    live = m.weights() + rest
    master = [w.detach().float().requires_grad_() for w in live]
    for w32 in master:
        w32.grad = torch.empty_like(w32)
    users = len(live) - len(rest)
    opt = torch.optim.Adam(master, lr=o.lr)
    for step in range(o.steps):
        tokens, user, target = batch(o.tokens)
        loss = tune.cross_entropy(ctx, m.states(tokens, user), m.head, target)
        loss.backward()
        # every user by the norm of their own gradients, what they share by its own
        for grads, out, adapters in (([w.grad for w in live[:users]], master[:users], o.users),
                                     ([w.grad for w in rest], master[users:], None)):
            tune.clip_grads(tune.Gradients(ctx, grads, out=[w32.grad for w32 in out], adapters=adapters), o.clip)
        for w in live:
            w.grad = None
        opt.step()
        with torch.no_grad():
            for w, w32 in zip(live, master):
                w.copy_(w32)
        if step % 10 == 0 or step == o.steps - 1:
            print(f"step {step}: loss {loss.item():.4f}", flush=True)
    after = m.perplexity(*held)
    for u, (b, a) in enumerate(zip(before, after)):
        print(f"user {u}: perplexity {b:.1f} -> {a:.2f}")
    # one decode step: a token of every user, and of a request without an adapter
    user = torch.tensor([*range(o.users), -1], dtype=torch.int32, device="cuda")
    right = 0
    for w in range(o.words):
        got = m.decode(words[w].expand(o.users + 1).contiguous(), user)
        right += (got[: o.users] == rules[:, w]).sum().item()
    accuracy = right / (o.users * o.words)
    print(f"decoded {o.users * o.words} tokens, {100 * accuracy:.1f}% by their user's rule")
    texts = m.write(words[torch.arange(o.users + 1, device="cuda") % o.words], user, 8, words)
    for u, text in enumerate(texts.tolist()):
        print(f"user {u if u < o.users else None}: {' '.join(map(str, text))}")
    ctx.clear_cache()
    return {"before": before, "after": after, "accuracy": accuracy, "texts": texts.tolist(), "words": words.tolist()}


if __name__ == "__main__":
    main()
