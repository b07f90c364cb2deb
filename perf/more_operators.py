"""Performance cases of the operators at the two ends of a training and of a decode step on a packed model.

Three kinds of work, over the sizes and options that their callers meet:
  embed      the embedding rows of a step's tokens, scaled; training adds the gradient of the whole
             table, which sums the rows of equal tokens.
  clip       the norm of all gradients of a step (of each user's, where several users' adapters train
             together) and the gradients clipped to it, most often into the 32-bit gradients of the
             master weights.
  constrain  penalties for tokens that a request has had, its biases and its grammar's mask on the
             logits of a decode step.
"""
import math
import os
import sys

import torch

own = False

DEV = "cuda:0"
IGNORE = -100
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
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
def _embed(t, d, v, grad=False, scale=1.0, ignored=0.0, dtype="bf16", **k):
    return dict(kind="embed", t=t, d=d, v=v, grad=grad, scale=scale, ignored=ignored, dtype=dtype, **k)


def _clip(layers, width, kv, inner, rank, users=1, each=False, head=0, limit=0.5, out="f32", dtype="bf16", **k):
    """Adapters of seven projections a layer. limit: the largest norm allowed, as a share of the expected
    one; out: where the clipped gradients go (f32, the gradients' own type, or in place)."""
    return dict(kind="clip", layers=layers, width=width, kv=kv, inner=inner, rank=rank, users=users, each=each, head=head,
                limit=limit, out=out, dtype=dtype, **k)


def _constrain(r, v, history=0, bias=0, masked=0.0, open=0.1, dtype="bf16", **k):
    """history: the longest one; masked: the share of requests with a grammar; open: of the tokens that it
    allows."""
    return dict(kind="constrain", r=r, v=v, history=history, bias=bias, masked=masked, open=open, dtype=dtype, **k)


def listed():
    return [
        # one decode step of 32 users: their tokens' rows, launches count
        _embed(32, 4096, 128256, name="embed_step"),
        # prompts of a batch, rows scaled by the root of the width
        _embed(16384, 4096, 128256, scale=64.0, name="embed_prompt"),
        # a short sequence over sizes that no tile divides, in half precision
        _embed(77, 1000, 50001, grad=True, ignored=0.2, dtype="f16", name="embed_ragged"),
        # a training step over a large vocabulary: most of its table's gradient is zeros
        _embed(4096, 4096, 128256, grad=True, ignored=0.1, name="embed_train"),
        # a batch of long sequences over a smaller vocabulary, where frequent tokens come by the thousand
        _embed(32768, 2048, 32000, grad=True, scale=45.25, name="embed_long"),
        # the adapters of two layers in place, with a norm that needs no clipping, as most steps have
        _clip(2, 2048, 2048, 5632, 8, limit=4.0, out="place", name="clip_small"),
        # four users' adapters, each user's gradients clipped to their own norm, in half precision
        _clip(4, 1350, 270, 1001, 8, users=4, each=True, out="f32", dtype="f16", name="clip_users"),
        # every adapter of an 8B model: 448 tensors
        _clip(32, 4096, 1024, 14336, 16, name="clip_adapters"),
        # adapters and the head's weights, clipped into a second set of the same type
        _clip(32, 4096, 1024, 14336, 64, head=128256, out="same", name="clip_head"),
        # one user's decode step: the 32-bit logits of a large vocabulary
        _constrain(1, 128256, history=1000, dtype="f32", name="constrain_one"),
        # seven requests over a ragged vocabulary, most with a grammar
        _constrain(7, 50001, history=300, bias=20, masked=0.7, dtype="f16", name="constrain_ragged"),
        # a full batch: long histories, some biases, half of the requests with a grammar
        _constrain(256, 128256, history=8192, bias=32, masked=0.5, name="constrain_batch"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _size(rng, lo, hi):
    """A size over the whole range; two of three are multiples of 64, as most models' are."""
    s = _log(rng, lo, hi)
    return s if rng.random() < 0.34 else max(64, s // 64 * 64)


def draw(rng):
    dtype = rng.choice(["bf16", "bf16", "f16"])
    kind = rng.choice(["embed", "embed_grad", "clip", "constrain"])
    if kind in ("embed", "embed_grad"):
        return _embed(_log(rng, 1, 32768), _size(rng, 64, 4096), _size(rng, 1000, 128256), kind == "embed_grad",
                      rng.choice([1.0, 1.0, rng.uniform(0.5, 64.0)]), rng.choice([0.0, 0.1, 0.6]), dtype)
    if kind == "constrain":
        return _constrain(_log(rng, 1, 256), _size(rng, 1000, 128256), rng.choice([0, _log(rng, 1, 8192), _log(rng, 1, 8192)]),
                          rng.choice([0, 1, _log(rng, 1, 300)]), rng.choice([0.0, 0.5, 1.0]),
                          rng.choice([0.001, 0.1, 0.9]), rng.choice([dtype, "f32"]))
    out = rng.choice(["f32", "f32", "same", "place"])
    width, inner = _size(rng, 64, 4096), _size(rng, 64, 14336)
    users = rng.choice([1, 1, rng.randint(2, 16)])
    layers, rank = _log(rng, 1, 32), _log(rng, 1, 64)
    while layers * rank * users > 2048:
        layers = max(1, layers // 2)
        rank = max(1, rank // 2)
    head = rng.choice([0, 0, 0, _log(rng, 1000, 32000)]) if users == 1 else 0
    return _clip(layers, width, max(8, width // rng.choice([1, 4])), inner, rank, users, users > 1 and rng.random() < 0.7, head,
                 rng.uniform(2.0, 8.0) if out == "place" else rng.choice([0.1, 0.7, 3.0]), out, rng.choice([dtype, "f32"]))


# ------------------------------------------------------------------------------------- the inputs
def _shapes(c):
    """(out, in) of a layer's seven projections."""
    w, kv, inner = c["width"], c["kv"], c["inner"]
    return [(w, w), (kv, w), (kv, w), (w, w), (inner, w), (inner, w), (w, inner)]


def _gradients(c):
    """Shapes of all gradients: A and B of each projection, users first, and the head's."""
    u, k = c["users"], c["rank"]
    layer = [s for m, n in _shapes(c) for s in ((u, k, n), (u, m, k))]
    return layer * c["layers"] + ([(c["head"], c["width"])] if c["head"] else [])


def _views(flat, shapes):
    sizes = [math.prod(s) for s in shapes]
    return [x.view(s) for x, s in zip(flat.split(sizes), shapes)]


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(int(seed))
    dt = TYPES[case["dtype"]]

    def normal(*shape, std=1.0, dtype=dt):
        return (torch.randn(*shape, generator=gen, device=DEV) * std).to(dtype)

    def tokens(v, *shape):
        """Ids as texts have them: the n-th most frequent about 1 / n as often as the first."""
        u = torch.rand(*shape, generator=gen, device=DEV, dtype=torch.float64)
        rank = (torch.exp(u * math.log(v + 1)) - 1).long().clamp(0, v - 1)
        return torch.randperm(v, generator=gen, device=DEV)[rank]

    s = dict(case)
    if case["kind"] == "embed":
        t, d, v = case["t"], case["d"], case["v"]
        s["table"] = normal(v, d, std=0.02)
        s["tokens"] = tokens(v, t)
        s["tokens"][torch.rand(t, generator=gen, device=DEV) < case["ignored"]] = IGNORE
        if case["grad"]:
            s["dy"] = normal(t, d, std=0.01)
        return s
    if case["kind"] == "clip":
        # gradients as a trainer's buckets hold them: one behind the other
        shapes = _gradients(case)
        n, u = sum(math.prod(x) for x in shapes), case["users"]
        s["flat"] = torch.empty(n, dtype=dt, device=DEV)
        for part in s["flat"].split(1 << 28):
            part.copy_(torch.randn(part.numel(), generator=gen, device=DEV) * 0.01)
        s["grads"] = _views(s["flat"], shapes)
        if u > 1 and case["out"] != "place":  # some users' gradients are far larger than others'
            by = torch.exp(torch.randn(u, generator=gen, device=DEV))
            for g in s["grads"]:
                g.copy_(g.float() * by[:, None, None])
        s["max_norm"] = case["limit"] * 0.01 * math.sqrt(n / (u if case["each"] else 1))
        if case["out"] != "place":
            s["to"] = torch.empty(n, dtype=torch.float32 if case["out"] == "f32" else dt, device=DEV)
            s["outs"] = _views(s["to"], shapes)
        if own:  # a trainer keeps the list of its gradients
            tune, ctx = _tune()
            s["set"] = tune.Gradients(ctx, s["grads"], out=s.get("outs"), adapters=u if case["each"] else None)
        return s
    r, v, h, b = case["r"], case["v"], case["history"], case["bias"]
    s["logits"] = normal(r, v, std=3.0)
    if h:
        s["tokens"] = tokens(v, r, h)
        s["lengths"] = torch.randint(h // 2, h + 1, (r,), generator=gen, device=DEV).int()
        s["prompts"] = (s["lengths"] * torch.rand(r, generator=gen, device=DEV)).int()
        s["repetition"] = torch.rand(r, generator=gen, device=DEV) * 0.4 + 1.0
        s["frequency"], s["presence"] = (torch.rand(r, generator=gen, device=DEV) * 0.5 for _ in range(2))
    if b:
        s["bias_tokens"] = torch.randint(0, v, (r, b), generator=gen, device=DEV)
        s["bias_tokens"][torch.rand(r, b, generator=gen, device=DEV) < 0.25] = -1  # requests have fewer
        s["biases"] = normal(r, b, std=5.0, dtype=torch.float32)
    if case["masked"]:
        words, some = -(-v // 32), max(1, round(r * case["masked"]))
        m = torch.zeros(some, words, dtype=torch.int64, device=DEV)
        for i in range(32):
            m |= (torch.rand(some, words, generator=gen, device=DEV) < case["open"]).long() << i
        s["mask"] = torch.where(m >= 1 << 31, m - (1 << 32), m).int()
        # the requests with a grammar, in any order; -1: without
        s["mask_rows"] = torch.full((r,), -1, dtype=torch.int32, device=DEV)
        s["mask_rows"][torch.randperm(r, generator=gen, device=DEV)[:some]] = torch.arange(some, device=DEV).int()
    return s


# ------------------------------------------------------------------------------------- one pass
def run(state):
    if state["kind"] == "embed":
        return (_run_embed_own if own else _run_embed)(state)
    if state["kind"] == "clip":
        return (_run_clip_own if own else _run_clip)(state)
    return (_run_constrain_own if own else _run_constrain)(state)


def _run_embed_own(s):
    tune, ctx = _tune()
    y = tune.embed(ctx, s["table"], s["tokens"], scale=s["scale"], ignore_index=IGNORE)
    if not s["grad"]:
        return y
    return y, tune.embed_backward(ctx, s["dy"], s["tokens"], s["v"], scale=s["scale"], ignore_index=IGNORE)


def _run_clip_own(s):
    tune, _ = _tune()
    norm = tune.clip_grads(s["set"], s["max_norm"])
    return norm, s["flat"] if s["out"] == "place" else s["to"]


def _run_constrain_own(s):
    tune, ctx = _tune()
    return tune.constrain_logits(ctx, s["logits"], history=s.get("tokens"), lengths=s.get("lengths"),
                                 prompts=s.get("prompts"), repetition=s.get("repetition"), frequency=s.get("frequency"),
                                 presence=s.get("presence"), bias_tokens=s.get("bias_tokens"), biases=s.get("biases"),
                                 mask=s.get("mask"), mask_rows=s.get("mask_rows"))


def _run_embed(s):
    counts = (s["tokens"] != IGNORE)[:, None]
    at = torch.where(counts[:, 0], s["tokens"], 0)
    dt = s["table"].dtype
    y = torch.where(counts, s["table"][at].float() * s["scale"], 0.0).to(dt)
    if not s["grad"]:
        return y
    dy = torch.where(counts, s["dy"].float(), 0.0)
    total = torch.zeros(s["v"], s["d"], dtype=torch.float32, device=DEV).index_add_(0, at, dy)
    return y, (total * s["scale"]).to(dt)


def _run_clip(s):
    parts = [g.float().flatten(1 if s["each"] else 0) for g in s["grads"]]
    square = torch.stack([p.square().sum(-1, dtype=torch.float64) for p in parts]).sum(0)
    norm = square.sqrt()
    by = torch.clamp(s["max_norm"] / (norm + 1e-6), max=1.0).float()
    by = by[:, None] if s["each"] else by
    [o.copy_((p * by).view_as(o)) for o, p in zip(s["grads"] if s["out"] == "place" else s["outs"], parts)]
    return norm.float(), s["flat"] if s["out"] == "place" else s["to"]


def _run_constrain(s):
    r, v = s["r"], s["v"]
    l = s["logits"].float()
    if s["history"]:
        at = torch.arange(s["history"], device=DEV)
        had = (at < s["lengths"][:, None]).float()
        made = had * (at >= s["prompts"][:, None])
        seen = torch.zeros(r, v, device=DEV).scatter_add_(1, s["tokens"], had) > 0
        count = torch.zeros(r, v, device=DEV).scatter_add_(1, s["tokens"], made)
        by = s["repetition"][:, None]
        l = torch.where(seen, torch.where(l > 0, l / by, l * by), l)
        l = l - (s["frequency"][:, None] * count + s["presence"][:, None] * (count > 0))
    if s["bias"]:
        use = s["bias_tokens"] >= 0
        l = l + torch.zeros(r, v, device=DEV).scatter_add_(1, s["bias_tokens"].clamp(min=0), torch.where(use, s["biases"], 0.0))
    if s["masked"]:
        token = torch.arange(v, device=DEV)
        bits = (s["mask"][s["mask_rows"].clamp(min=0).long()][:, token // 32] >> (token % 32).int()) & 1
        l = torch.where((bits > 0) | (s["mask_rows"][:, None] < 0), l, -math.inf)
    return l.to(s["logits"].dtype)


# ------------------------------------------------------------------------------------- the floors
def work(case):
    e = 4 if case["dtype"] == "f32" else 2
    if case["kind"] == "embed":
        t, d, v = case["t"], case["d"], case["v"]
        n = torch.arange(v, dtype=torch.float64)  # each id's share of the tokens, and the distinct ones expected
        rows = float((1 - (1 - torch.log1p(1 / (n + 1)) / math.log(v + 1)) ** t).sum())
        w = {"bytes": 8 * t + e * rows * d + e * t * d, "flops": t * d}
        if case["grad"]:
            w["bytes"] += e * t * d + e * v * d
            w["flops"] += 2 * t * d
        return w
    if case["kind"] == "clip":
        n = sum(math.prod(x) for x in _gradients(case))
        write = {"f32": 4, "same": e, "place": 0}[case["out"]]  # in place they need no clipping here
        return {"bytes": n * (e + write), "flops": n * (3 if write else 2)}
    r, v = case["r"], case["v"]
    return {"bytes": 2 * e * r * v + 8 * r * case["history"] * 3 // 4 + 12 * r * case["bias"] +
            (max(1, round(r * case["masked"])) * -(-v // 32) * 4 if case["masked"] else 0),
            "flops": r * (6 * case["history"] + case["bias"] + v)}


# ------------------------------------------------------------------------------------- in 64 bits
def exact(case, seed):
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    if case["kind"] == "embed":
        rows = (s["tokens"] != IGNORE).nonzero().flatten()
        ids = s["tokens"][rows]
        y = torch.zeros(case["t"], case["d"], dtype=torch.float64, device=DEV)
        y[rows] = s["table"].double()[ids] * s["scale"]
        if not case["grad"]:
            return y
        which, back = torch.unique(ids, return_inverse=True)
        sums = torch.zeros(len(which), case["d"], dtype=torch.float64, device=DEV)
        sums.index_put_((back,), s["dy"][rows].double() * s["scale"], accumulate=True)
        de = torch.zeros(case["v"], case["d"], dtype=torch.float64, device=DEV)
        de[which] = sums
        return y, de
    if case["kind"] == "clip":
        u = case["users"] if case["each"] else 1
        square = torch.zeros(u, dtype=torch.float64, device=DEV)
        for g in s["grads"]:
            x = g.reshape(u, -1)
            for i in range(u):
                square[i] += sum(torch.linalg.vector_norm(p.double()) ** 2 for p in x[i].split(1 << 26))
        norm = square.sqrt()
        by = (s["max_norm"] / (norm + 1e-6)).clamp(max=1.0)
        out = torch.empty(s["flat"].numel(), dtype=torch.float64, device=DEV)
        for g, o in zip(s["grads"], _views(out, _gradients(case))):
            o.view(u, -1).copy_(g.reshape(u, -1)).mul_(by[:, None])
        return (norm if case["each"] else norm[0]), out
    out = s["logits"].double()
    for i in range(case["r"]):
        l = out[i]
        if case["history"]:
            n, p = int(s["lengths"][i]), int(s["prompts"][i])
            had = torch.unique(s["tokens"][i, :n])
            l[had] = torch.where(l[had] > 0, l[had] / s["repetition"][i].double(), l[had] * s["repetition"][i].double())
            made, times = torch.unique(s["tokens"][i, p:n], return_counts=True)
            l[made] -= s["frequency"][i].double() * times + s["presence"][i].double()
        if case["bias"]:
            use = s["bias_tokens"][i] >= 0
            l.index_put_((s["bias_tokens"][i][use],), s["biases"][i][use].double(), accumulate=True)
        if case["masked"] and int(s["mask_rows"][i]) >= 0:
            words = s["mask"][int(s["mask_rows"][i])]
            allowed = ((words[:, None] >> torch.arange(32, device=DEV, dtype=torch.int32)) & 1).flatten()[:case["v"]]
            l[allowed == 0] = -math.inf
    return out
