"""GPU tests of cdclq.tune's embedding, loss, clipping and logit constraints as a training and a decode step use them
together, and of the example that does."""
import importlib.util
import math
import os

import pytest
import torch

import cdclq
from tests.test_gpu_adapters import make_adapters, make_layer, normal, rng

pytestmark = pytest.mark.gpu

EXAMPLE = os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "examples", "adapters.py")
U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
U32 = 2.0 ** -24


@pytest.fixture(scope="module")
def ctx():
    c = cdclq.Context(0)
    yield c
    c.close()


@pytest.fixture(scope="module")
def tune():
    from cdclq import tune
    return tune


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("t,d,v", [(60, 96, 500), (700, 256, 1000), (9000, 72, 300)])
def test_a_tied_table_in_a_training_step(ctx, tune, dtype, t, d, v):
    """loss = mean cross entropy of the logits e W^T, e = s W[tokens]: W's gradient is the head's plus the embedding's,
    then clipped into float32. The parts by the operators' own outputs, the joined gradient against autograd in 64
    bits: each of its two parts is held in 16 bits once (d of the loss is, too: u of each product's magnitude)."""
    s = 1.5
    w = normal(1, v, d, std=0.5, dtype=dtype)
    tokens = torch.randint(0, v, (t,), generator=rng(2), device="cuda")
    target = torch.randint(0, v, (t,), generator=rng(3), device="cuda")
    tokens[::9] = -100
    target[::9] = -100
    count = int((target != -100).sum())
    e = tune.embed(ctx, w, tokens, s)
    loss, lse = tune.vocab_loss(ctx, e, w, target)
    weight = torch.full((t,), 1.0 / count, device="cuda")
    dx, dw = tune.vocab_loss_backward(ctx, e, w, target, lse, weight)
    head = dw.clone()
    tune.embed_backward(ctx, dx, tokens, v, s, into=dw)

    on = (tokens != -100).nonzero().flatten()
    part = torch.zeros(v, d, dtype=torch.float64, device="cuda").index_put_((tokens[on],), dx[on].double() * s, accumulate=True)
    n = torch.bincount(tokens[on], minlength=v).double()[:, None]
    size = torch.zeros_like(part).index_put_((tokens[on],), dx[on].double().abs() * s, accumulate=True)
    joined = head.double() + part
    assert ((dw.double() - joined).abs() <= U[dtype] * joined.abs() + (n + 4) * U32 * (size + head.double().abs()) + 2.0 ** -24).all()

    x = w.double().cpu().requires_grad_()
    rows = on.cpu()
    full = torch.nn.functional.cross_entropy(s * x[tokens.cpu()[rows]] @ x.T, target.cpu()[rows])
    full.backward()
    assert abs(loss.double().sum().item() / count - full.item()) <= 8 * U[dtype] * full.item()
    gap = (dw.double().cpu() - x.grad).norm() / x.grad.norm()
    # e, d and dx are rounded once each and dw twice: five roundings of u of what they add up, which cancels in part
    assert gap <= 8 * U[dtype], gap.item()

    out = torch.empty(v, d, device="cuda")
    norm = tune.clip_grads(tune.Gradients(ctx, [dw], out=[out]), 0.01)
    want = dw.double().norm()
    assert abs(norm.double() - want) <= 1.01 * U32 * want
    by = min(1.0, 0.01 / (want.item() + 1e-6))
    assert ((out.double() - by * dw.double()).abs() <= 3.2 * U32 * by * dw.double().abs() + 2.0 ** -149).all()


def test_training_steps_in_a_graph(ctx, tune):
    """Embedding, packed projection with two users' adapters, loss, gradients and clipping captured once; every replay
    equals the eager step on the same inputs, bit for bit."""
    t, d, v, users, rank, b = 300, 256, 1000, 2, 8, torch.bfloat16
    packed, _, _ = make_layer(ctx, tune, 3, d, d, 4, 128)
    ad = make_adapters(tune, 2, users, rank, d, d, b)
    table, head = normal(1, v, d, std=0.5, dtype=b), normal(4, v, d, std=d ** -0.5, dtype=b)
    tokens, target = (torch.zeros(t, dtype=torch.int64, device="cuda") for _ in range(2))
    user = (torch.arange(t, device="cuda") * users // t).int()
    weight = torch.full((t,), 1.0 / t, device="cuda")
    outs = [torch.empty(x.shape, device="cuda") for x in (ad.a, ad.b)]

    def step(outs):
        e = tune.embed(ctx, table, tokens)
        y, low = tune.adapter_linear(packed, e, ad, user, return_low=True)
        loss, lse = tune.vocab_loss(ctx, y, head, target)
        dy, dhead = tune.vocab_loss_backward(ctx, y, head, target, lse, weight)
        dx, da, db = tune.adapter_linear_backward(packed, dy, tune.checkpoint_save(ctx, e), low, ad, user)
        tune.embed_backward(ctx, dx, tokens, v, into=dhead)
        norm = tune.clip_grads(tune.Gradients(ctx, [da, db], out=outs, adapters=users), 0.01)
        return loss, dhead, norm, *outs

    step(outs)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(outs)
    for i in range(4):
        tokens.copy_(torch.randint(0, v, (t,), generator=rng(i), device="cuda"))
        target.copy_(torch.randint(0, v, (t,), generator=rng(100 + i), device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        want = step([torch.empty_like(x) for x in outs])
        assert all(torch.equal(x, y) for x, y in zip(got, want))
        assert torch.isfinite(got[2]).all() and (got[2] > 0).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_a_decode_step(ctx, tune, dtype):
    """Tokens in, constrained logits out, for requests with and without adapters, histories and grammars: the chosen
    tokens are allowed, and the likeliest by the formulas on the step's own logits."""
    r, d, v, b = 33, 256, 2000, dtype
    packed, _, _ = make_layer(ctx, tune, 3, d, d, 4, 128)
    ad = make_adapters(tune, 2, 3, 8, d, d, b)
    table, head = normal(1, v, d, dtype=b), normal(4, v, d, std=d ** -0.5, dtype=b)
    tokens = torch.randint(0, v, (r,), generator=rng(5), device="cuda")
    user = torch.randint(-1, 3, (r,), generator=rng(6), device="cuda").int()
    h = tune.adapter_linear(packed, tune.embed(ctx, table, tokens, 2.0), ad, user)
    logits = h @ head.T
    history = torch.randint(0, v, (r, 40), generator=rng(7), device="cuda")
    lengths = torch.randint(0, 41, (r,), generator=rng(8), device="cuda").int()
    pres = torch.rand(r, generator=rng(9), device="cuda") * 8
    mask = torch.full((1, -(-v // 32)), 0x55555555, dtype=torch.int32, device="cuda")  # even tokens
    rows = (torch.arange(r, device="cuda") % 2 - 1).int()
    got = tune.constrain_logits(ctx, logits, history=history, lengths=lengths, presence=pres, mask=mask, mask_rows=rows)
    want = logits.double()
    for i in range(r):
        want[i, torch.unique(history[i, :int(lengths[i])])] -= pres[i].double()
        if rows[i] == 0:
            want[i, 1::2] = -math.inf
    pick = got.argmax(1)
    assert (pick[rows == 0] % 2 == 0).all()
    best = want.max(1).values
    assert (best - want.gather(1, pick[:, None])[:, 0] <= 2 * (U[dtype] + 2 * U32) * (best.abs() + pres.double())).all()


def test_example():
    spec = importlib.util.spec_from_file_location("adapters_example", EXAMPLE)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    r = mod.main(["--steps", "6", "--width", "256", "--tokens", "600", "--vocab", "1003", "--train-head", "--train-embed",
                  "--clip", "0.05"])
    assert all(math.isfinite(x) for x in r["before"] + r["after"])
    assert len(r["texts"]) == 5 and all(len(x) == 9 and set(x) <= set(r["words"]) for x in r["texts"])
