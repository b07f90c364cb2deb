"""GPU tests of the differentiable forms (cdclq.tune.linear, cross_entropy) and of the example that trains
and serves several users' adapters on one quantized model."""
import importlib.util
import os

import pytest
import torch

import cdclq
from tests.test_gpu_adapters import make_adapters, make_layer, normal, rng

pytestmark = pytest.mark.gpu

EXAMPLE = os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "examples", "adapters.py")


@pytest.fixture(scope="module")
def ctx():
    c = cdclq.Context(0)
    yield c
    c.close()


@pytest.fixture(scope="module")
def tune():
    from cdclq import tune
    return tune


@pytest.mark.parametrize("t", [0, 5, 100])
def test_linear_is_the_operators(ctx, tune, t):
    m, n, b = 130, 256, torch.bfloat16
    packed, _, _ = make_layer(ctx, tune, 3, m, n, 4, 128)
    ad = make_adapters(tune, 2, 3, 8, m, n, b)
    q = torch.randint(-1, 3, (t,), generator=rng(4), device="cuda").int()
    x, dy = normal(1, t, n, dtype=b).requires_grad_(), normal(2, t, m, dtype=b)
    live = tune.Adapters(ad.a.clone().requires_grad_(), ad.b.clone().requires_grad_(), ad.scaling)
    y = tune.linear(packed, x, live, q)
    y.backward(dy)
    y0, low = tune.adapter_linear(packed, x.detach(), ad, q, return_low=True)
    want = tune.adapter_linear_backward(packed, dy, tune.checkpoint_save(ctx, x.detach()), low, ad, q)
    assert torch.equal(y.detach(), y0)
    for got, w in zip((x.grad, live.a.grad, live.b.grad), want):
        assert torch.equal(got, w)
    bare = x.detach().clone().requires_grad_()
    tune.linear(packed, bare).backward(dy.t().contiguous().t())  # a gradient of another layout
    assert torch.equal(bare.grad, tune.adapter_linear_backward(packed, dy)[0])


def test_changed_adapters_are_refused(ctx, tune):
    m, n, b = 64, 128, torch.bfloat16
    packed, _, _ = make_layer(ctx, tune, 3, m, n, 4, 128)
    ad = make_adapters(tune, 2, 1, 8, m, n, b)
    q = torch.zeros(4, dtype=torch.int32, device="cuda")
    a = ad.a.clone().requires_grad_()
    y = tune.linear(packed, normal(1, 4, n, dtype=b), tune.Adapters(a, ad.b, ad.scaling), q)
    with torch.no_grad():
        a.add_(1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


@pytest.mark.parametrize("head", [False, True])
@pytest.mark.parametrize("ignored", [0.0, 0.3, 1.0])
def test_cross_entropy_is_the_operators(ctx, tune, head, ignored):
    t, d, v, b = 50, 96, 1000, torch.bfloat16
    x = normal(1, t, d, dtype=b).requires_grad_()
    w = normal(2, v, d, std=d ** -0.5, dtype=b).requires_grad_(head)
    y = torch.randint(0, v, (t,), generator=rng(3), device="cuda")
    y[: round(ignored * t)] = -100
    count = max(1, int((y != -100).sum()))
    loss = tune.cross_entropy(ctx, x, w, y)
    (2.0 * loss).backward()
    each, lse = tune.vocab_loss(ctx, x.detach(), w.detach(), y)
    assert abs(loss.item() - each.double().sum().item() / count) <= 1e-5 * max(1.0, loss.item())
    g = torch.full((t,), 2.0 / count, device="cuda")
    dx, dw = tune.vocab_loss_backward(ctx, x.detach(), w.detach(), y, lse, g, need_dw=head)
    assert torch.allclose(x.grad.float(), dx.float(), rtol=2.0 ** -6, atol=0)
    assert torch.allclose(w.grad.float(), dw.float(), rtol=2.0 ** -6, atol=1e-9) if head else w.grad is None


@pytest.mark.parametrize("args", [[], ["--dtype", "f16", "--train-head", "--bits", "3", "--vocab", "1003"]])
def test_example(args):
    spec = importlib.util.spec_from_file_location("adapters_example", EXAMPLE)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    r = mod.main(["--steps", "30", "--width", "256", "--tokens", "1024", *args])
    # untrained, the rules' tokens are as likely as any other: a perplexity near the vocabulary's size;
    # after 30 steps the users' texts are far more likely than that
    assert all(a < 0.25 * b for b, a in zip(r["before"], r["after"]))
    assert r["accuracy"] > 0.1
