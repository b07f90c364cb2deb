"""Performance cases of the operators that train and serve low-rank adapters on a packed model.

Three kinds of work, over the sizes and options that their callers meet:
  checkpoint  a layer's input kept in 8 bits between forward and backward: saved, then restored.
  adapter     a packed (cdclq-v1) projection shared by all tokens, and the low-rank adapter of each
              token's request beside it. Serving is the forward pass alone; training is the forward
              pass, the 8-bit checkpoint of its input and the backward pass that reads it.
  loss        softmax cross entropy over a large vocabulary. Evaluation is the loss of each token;
              training adds the gradient of the hidden states and, unless the head is frozen, of
              the head's weights.
"""
import math
import os
import sys

import numpy as np
import torch

own = False

DEV = "cuda:0"
BLOCK = 128  # features per scale of an 8-bit checkpoint
IGNORE = -100
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
_ctx = None


def _tune():
    """The framework's operators and the context that a program keeps for them."""
    global _ctx
    root = os.path.join(os.getcwd(), "cdcl-gptq_amd")
    if root not in sys.path:
        sys.path.insert(0, root)
    import cdclq
    from cdclq import tune
    if _ctx is None:
        _ctx = cdclq.Context(0)
    return tune, _ctx


# ------------------------------------------------------------------------------------- the cases
def _checkpoint(t, n, dtype="bf16", **k):
    return dict(kind="checkpoint", t=t, n=n, dtype=dtype, **k)


def _adapter(t, n, m, bits=4, group=128, lead=0, adapters=1, rank=16, bare=0.0, train=False, dtype="bf16", **k):
    return dict(kind="adapter", t=t, n=n, m=m, bits=bits, group=group, lead=lead, adapters=adapters, rank=rank,
                bare=bare, train=train, dtype=dtype, **k)


def _loss(t, d, v, grad=False, head=False, ignored=0.0, dtype="bf16", **k):
    return dict(kind="loss", t=t, d=d, v=v, grad=grad, head=head, ignored=ignored, dtype=dtype, **k)


def listed():
    return [
        # one layer's input of a short training sequence: launches count
        _checkpoint(512, 4096, name="checkpoint_short"),
        # the widest input of a layer (its MLP's inner width) over a batch of long sequences
        _checkpoint(16384, 14336, name="checkpoint_long"),
        # one decode step of one user: every byte of the packed weights for a single token
        _adapter(1, 4096, 4096, adapters=4, name="serve_one"),
        # one decode step of 32 users, each with an adapter of its own, through the MLP's up projection
        _adapter(32, 4096, 14336, adapters=32, name="serve_batch"),
        # a few users of a small ragged layer: 3-bit codes, groups that are no multiple of the tiles,
        # some requests without an adapter
        _adapter(7, 1350, 1001, bits=3, group=48, adapters=3, rank=8, bare=0.3, dtype="f16", name="serve_ragged"),
        # prompts of several users in one batch, each token carrying its request's adapter
        _adapter(2000, 2048, 5632, bits=3, adapters=8, name="prefill"),
        # a training step of four small adapters on a 2-bit layer whose leading groups keep 8 bits
        _adapter(640, 2048, 2048, bits=2, group=64, lead=2, adapters=4, rank=8, train=True, dtype="f16",
                 name="train_small"),
        # a training step of one adapter on the MLP's up projection of an 8B model
        _adapter(4096, 4096, 14336, rank=64, train=True, name="train_mlp"),
        # perplexity of a quantized model: the loss of every token of a long window
        _loss(2048, 4096, 128256, name="loss_eval"),
        # training with the head frozen (adapters only): the hidden states' gradient, odd token count
        _loss(1001, 2048, 32000, grad=True, ignored=0.5, name="loss_frozen"),
        # training with the head: all of it, over a large vocabulary
        _loss(4096, 4096, 128256, grad=True, head=True, ignored=0.1, name="loss_train"),
        # sizes that no tile divides, in half precision
        _loss(77, 1000, 50001, grad=True, head=True, ignored=0.2, dtype="f16", name="loss_ragged"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _size(rng, lo, hi):
    """A size over the whole range; two of three are multiples of 64, as most models' are."""
    s = _log(rng, lo, hi)
    return s if rng.random() < 0.34 else max(64, s // 64 * 64)


def draw(rng):
    dtype = rng.choice(["bf16", "bf16", "f16"])
    kind = rng.choice(["checkpoint", "serve", "serve", "prefill", "train", "loss", "loss"])
    if kind == "checkpoint":
        return _checkpoint(_log(rng, 1, 16384), _size(rng, 64, 14336), dtype)
    if kind == "loss":
        grad = rng.random() < 0.6
        return _loss(_log(rng, 1, 4096), _size(rng, 64, 4096), _size(rng, 1000, 128256), grad,
                     grad and rng.random() < 0.5, rng.choice([0.0, 0.1, 0.6]), dtype)
    bits = rng.randint(2, 8)
    group = rng.choice([128, 128, 64, 32, 0, rng.randint(5, 200)])
    lead = rng.choice([0, 0, 2]) if group else 0
    n, m = _size(rng, 128, 14336), _size(rng, 128, 14336)
    rank = rng.choice([4, 8, 16, 16, 32, 64, rng.randint(1, 128)])
    t = {"serve": lambda: _log(rng, 1, 64), "prefill": lambda: _log(rng, 65, 4096),
         "train": lambda: _log(rng, 16, 4096)}[kind]()
    while t * n * m > 4096 * 4096 * 14336:
        t //= 2
    adapters = min(rng.choice([1, 2, 4, 8, 16, 32]), max(1, t), 1024 // rank)
    return _adapter(t, n, m, bits, group, lead, adapters, rank, rng.choice([0.0, 0.0, 0.3]), kind == "train", dtype)


# ------------------------------------------------------------------------------------- the inputs
def _widths(c):
    """Bits of each column group: the leading groups keep 8."""
    g = c["group"] if 0 < c["group"] < c["n"] else c["n"]
    ng = -(-c["n"] // g)
    return g, np.array([8 if i < c["lead"] else c["bits"] for i in range(ng)], np.uint8)


def _offsets(n, group, gbits):
    """Width and bit offset of each column of the permuted order within a row."""
    wid = gbits[np.arange(n) // group].astype(np.int64)
    return wid, np.cumsum(wid) - wid


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(int(seed))
    dt = TYPES[case["dtype"]]

    def normal(*shape, std=1.0, dtype=dt):
        return (torch.randn(*shape, generator=gen, device=DEV) * std).to(dtype)

    def tokens(t, n):
        """Activations with a few channels far above the rest, as a decoder's residual stream has."""
        big = torch.rand(n, generator=gen, device=DEV) < 0.01
        return (torch.randn(t, n, generator=gen, device=DEV) * torch.where(big, 10.0, 1.0)).to(dt)

    s = dict(case)
    if case["kind"] == "checkpoint":
        s["x"] = tokens(case["t"], case["n"])
        return s
    if case["kind"] == "loss":
        t, d, v = case["t"], case["d"], case["v"]
        s["x"], s["w"] = normal(t, d), normal(v, d, std=2.0 / math.sqrt(d))
        y = torch.randint(0, v, (t,), generator=gen, device=DEV)
        y[torch.rand(t, generator=gen, device=DEV) < case["ignored"]] = IGNORE
        s["y"] = y
        if case["grad"]:  # the mean over the tokens that count
            s["g"] = torch.full((t,), 1.0, device=DEV) / (y != IGNORE).sum().clamp(min=1)
        return s
    t, n, m, r, k = case["t"], case["n"], case["m"], case["adapters"], case["rank"]
    group, gbits = _widths(case)
    wid, off = _offsets(n, group, gbits)
    rb = (int(wid.sum()) + 7) // 8
    gw = torch.from_numpy(gbits.astype(np.int32)).to(DEV)
    ng = gbits.size
    # codes spread around their group's zero point, as round-to-nearest of normal weights gives
    w = torch.from_numpy(wid).to(DEV)
    top = (1 << w) - 1
    zeros = ((1 << gw) // 2 + torch.randint(-1, 1, (m, ng), generator=gen, device=DEV)).to(torch.uint8)
    z = zeros.long().float()[:, torch.arange(n, device=DEV) // group]
    codes = torch.randn(m, n, generator=gen, device=DEV).mul_((1 << w).float() / 5).add_(z).round_()
    codes = torch.minimum(codes.clamp_(min=0), top.float()).int()
    bits = torch.zeros(m, rb * 8, dtype=torch.uint8, device=DEV)
    o = torch.from_numpy(off).to(DEV)
    for b in range(8):
        has = (w > b).nonzero().flatten()
        if has.numel():
            bits[:, o[has] + b] = ((codes[:, has] >> b) & 1).to(torch.uint8)
    s["qweight"] = (bits.view(m, rb, 8) << torch.arange(8, device=DEV, dtype=torch.uint8)).sum(2, dtype=torch.uint8)
    del bits, codes, z
    spread = (torch.rand(m, ng, generator=gen, device=DEV) + 0.5) / math.sqrt(n) * 5
    s["scales"] = (spread / (1 << gw).float()).half()
    s["qzeros"] = zeros
    s["perm"] = torch.randperm(n, generator=gen, device=DEV).int()
    s["gbits"], s["gsize"] = gbits, group
    s["x"] = tokens(t, n)
    s["a"], s["b"] = normal(r, k, n, std=1.0 / math.sqrt(n)), normal(r, m, k, std=0.5 / math.sqrt(k))
    s["scaling"] = torch.rand(r, generator=gen, device=DEV) + 0.5
    if t <= 64:  # a decode step: one token of each request, in any order
        q = torch.randperm(t, generator=gen, device=DEV) % r
    else:  # prompts one after another
        q = torch.sort(torch.randint(0, r, (t,), generator=gen, device=DEV)).values
    q[torch.rand(t, generator=gen, device=DEV) < case["bare"]] = -1
    s["request"] = q.int()
    if case["train"]:
        s["dy"] = normal(t, m)
    if own:  # a served or trained model keeps its layers' handles
        tune, ctx = _tune()
        s["packed"] = tune.PackedLinear(ctx, s["qweight"], s["scales"], s["qzeros"], s["perm"], gbits, group)
        s["adapters_set"] = tune.Adapters(s["a"], s["b"], s["scaling"])
    return s


# ------------------------------------------------------------------------------------- one pass
def run(state):
    if state["kind"] == "checkpoint":
        return (_run_checkpoint_own if own else _run_checkpoint)(state)
    if state["kind"] == "loss":
        return (_run_loss_own if own else _run_loss)(state)
    return (_run_adapter_own if own else _run_adapter)(state)


def _run_checkpoint_own(s):
    tune, ctx = _tune()
    return tune.checkpoint_restore(ctx, tune.checkpoint_save(ctx, s["x"]))


def _run_adapter_own(s):
    tune, ctx = _tune()
    if not s["train"]:
        return tune.adapter_linear(s["packed"], s["x"], s["adapters_set"], s["request"])
    y, low = tune.adapter_linear(s["packed"], s["x"], s["adapters_set"], s["request"], return_low=True)
    saved = tune.checkpoint_save(ctx, s["x"])
    dx, da, db = tune.adapter_linear_backward(s["packed"], s["dy"], saved, low, s["adapters_set"], s["request"])
    return y, dx, da, db


def _run_loss_own(s):
    tune, ctx = _tune()
    loss, lse = tune.vocab_loss(ctx, s["x"], s["w"], s["y"], ignore_index=IGNORE)
    if not s["grad"]:
        return loss, lse
    dx, dw = tune.vocab_loss_backward(ctx, s["x"], s["w"], s["y"], lse, s["g"], ignore_index=IGNORE,
                                      need_dw=s["head"])
    return (loss, dx, dw) if s["head"] else (loss, dx)


def _plain_checkpoint(x):
    """The values that an 8-bit checkpoint of x holds, in 32 bits."""
    t, n = x.shape
    nb = -(-n // BLOCK)
    v = torch.nn.functional.pad(x.float(), (0, nb * BLOCK - n)).view(t, nb, BLOCK)
    scale = v.abs().amax(2, keepdim=True) / 127.0
    codes = torch.round(v / torch.where(scale > 0, scale, torch.ones_like(scale)))
    return (codes * scale).view(t, nb * BLOCK)[:, :n]


def _run_checkpoint(s):
    return _plain_checkpoint(s["x"]).to(s["x"].dtype)


def _plain_weight(s):
    """The packed layer's weights in the original column order, in 32 bits."""
    n, m = s["n"], s["m"]
    wid, off = _offsets(n, s["gsize"], s["gbits"])
    o = torch.from_numpy(off).to(DEV)
    q = torch.nn.functional.pad(s["qweight"], (0, 1))
    at = o >> 3
    word = q[:, at].int() | (q[:, at + 1].int() << 8)
    codes = (word >> (o & 7).int()) & torch.from_numpy((1 << wid) - 1).int().to(DEV)
    g = torch.arange(n, device=DEV) // s["gsize"]
    w = torch.empty(m, n, device=DEV)
    w[:, s["perm"].long()] = s["scales"].float()[:, g] * (codes.float() - s["qzeros"].float()[:, g])
    return w


def _run_adapter(s):
    r, k, n = s["a"].shape
    m, x = s["m"], s["x"].float()
    w = _plain_weight(s)
    a, b = s["a"].float().reshape(r * k, n), s["b"].float().permute(0, 2, 1).reshape(r * k, m)
    # a token's row of `of` is its request's scaling there and 0 at the other requests' places
    of = torch.where(s["request"].long()[:, None] == torch.arange(r, device=DEV), s["scaling"], 0.0)
    of = of.repeat_interleave(k, 1)
    low = x @ a.t() * of
    y = x @ w.t() + low @ b
    if not s["train"]:
        return y.to(s["x"].dtype)
    dy, dt = s["dy"].float(), s["x"].dtype
    up = dy @ b.t() * of
    dx = dy @ w + up @ a
    da = up.t() @ _plain_checkpoint(s["x"])
    db = (dy.t() @ low).view(m, r, k).permute(1, 0, 2)
    return y.to(dt), dx.to(dt), da.view(r, k, n).to(dt), db.to(dt).contiguous()


def _run_loss(s):
    x, w, y = s["x"].float(), s["w"].float(), s["y"]
    counts = y != IGNORE
    at = torch.where(counts, y, 0)[:, None]
    logits = x @ w.t()
    top = logits.amax(1, keepdim=True)
    logits -= top
    hit = logits.gather(1, at)
    total = logits.exp_().sum(1, keepdim=True)
    loss = torch.where(counts, (total.log() - hit)[:, 0], 0.0)
    if not s["grad"]:
        return loss, torch.where(counts, (total.log() + top)[:, 0], 0.0)
    d = logits.div_(total)
    d.scatter_add_(1, at, torch.full_like(at, -1, dtype=torch.float32))
    d *= torch.where(counts, s["g"], 0.0)[:, None]
    dx = (d @ w).to(s["x"].dtype)
    return (loss, dx, (d.t() @ x).to(s["w"].dtype)) if s["head"] else (loss, dx)


# ------------------------------------------------------------------------------------- the floors
def work(case):
    t = case["t"]
    if case["kind"] == "checkpoint":
        n = case["n"]
        # x read, the codes and scales written and read once more, the restored values written
        return {"bytes": 2 * t * n + 2 * (t * n + 4 * t * -(-n // BLOCK)) + 2 * t * n, "flops": 4 * t * n}
    if case["kind"] == "loss":
        d, v = case["d"], case["v"]
        parts = 1 + case["grad"] + case["head"]
        return {"bytes": 2 * (t * d + v * d) + 8 * t + 4 * t + case["grad"] * (2 * t * d + 4 * t) + case["head"] * 2 * v * d,
                "flops": parts * 2 * t * v * d}
    n, m, k = case["n"], case["m"], case["rank"]
    group, gbits = _widths(case)
    wid, _ = _offsets(n, group, gbits)
    used = min(case["adapters"], t) * k * (n + m) * 2
    low = 2 * t * k * (n + m)
    w = {"bytes": m * ((int(wid.sum()) + 7) // 8 + 3 * gbits.size) + 2 * t * (n + m) + used,
         "flops": 2 * t * m * n + low}
    if case["train"]:
        w["bytes"] += 2 * t * (n + m) + t * n + used
        w["flops"] += 2 * t * m * n + 2 * low
    return w


# ------------------------------------------------------------------------------------- in 64 bits
def _exact_saved(x):
    """Codes times scales of each block of 128 features; a scale is held in 32 bits."""
    t, n = x.shape
    out = torch.empty(t, n, dtype=torch.float64, device=x.device)
    for c in range(0, n, BLOCK):
        v = x[:, c:c + BLOCK].double()
        step = (v.abs().max(1, keepdim=True).values / 127).float().double()
        out[:, c:c + BLOCK] = step * torch.round(v / step.masked_fill(step == 0, 1))
    return out


def exact(case, seed):
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    if case["kind"] == "checkpoint":
        return _exact_saved(s["x"])
    if case["kind"] == "loss":
        x, w = s["x"].double(), s["w"].double()
        t, d = x.shape
        loss = torch.zeros(t, dtype=torch.float64, device=DEV)
        lse, dx, dw = loss.clone(), torch.zeros_like(x), torch.zeros_like(w) if case["head"] else None
        rows = (s["y"] != IGNORE).nonzero().flatten()
        for part in rows.split(1024):
            l = x[part] @ w.T
            lse[part] = torch.logsumexp(l, 1)
            loss[part] = lse[part] - l[torch.arange(len(part), device=DEV), s["y"][part]]
            if not case["grad"]:
                continue
            p = torch.softmax(l, 1)
            p[torch.arange(len(part), device=DEV), s["y"][part]] -= 1
            p *= s["g"][part].double()[:, None]
            dx[part] = p @ w
            if dw is not None:
                dw += p.T @ x[part]
        return (loss, lse) if not case["grad"] else (loss, dx, dw) if case["head"] else (loss, dx)
    m, n, dev = s["m"], s["n"], DEV
    w = torch.zeros(m, n, dtype=torch.float64, device=dev)
    flat = torch.stack([(s["qweight"] >> i) & 1 for i in range(8)], 2).view(m, -1)  # a row's bits, low first
    at = 0
    for g, width in enumerate(s["gbits"].tolist()):
        c0, c1 = g * s["gsize"], min((g + 1) * s["gsize"], n)
        field = flat[:, at:at + (c1 - c0) * width].view(m, c1 - c0, width).double()
        code = field @ (2.0 ** torch.arange(width, dtype=torch.float64, device=dev))
        w[:, s["perm"][c0:c1].long()] = s["scales"][:, g:g + 1].double() * (code - s["qzeros"][:, g:g + 1].double())
        at += (c1 - c0) * width
    x = s["x"].double()
    y = x @ w.T
    dy = s["dy"].double() if case["train"] else None
    if case["train"]:
        dx, kept = dy @ w, _exact_saved(s["x"])
        da, db = torch.zeros_like(s["a"], dtype=torch.float64), torch.zeros_like(s["b"], dtype=torch.float64)
    for i in range(case["adapters"]):
        sel = (s["request"] == i).nonzero().flatten()
        a, b, c = s["a"][i].double(), s["b"][i].double(), s["scaling"][i].double()
        y[sel] += c * (x[sel] @ a.T) @ b.T
        if case["train"]:
            up = c * (dy[sel] @ b)
            dx[sel] += up @ a
            da[i] = up.T @ kept[sel]
            db[i] = c * dy[sel].T @ (x[sel] @ a.T)
    return (y, dx, da, db) if case["train"] else y
