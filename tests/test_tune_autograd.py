"""CPU tests of the differentiable forms of cdclq.tune (linear, cross_entropy): what they keep between the
passes, and what they refuse. The operators themselves are replaced by their formulas in torch; nothing is
launched."""
import pytest
import torch

from cdclq import tune


class Layer:
    """Stands for a packed layer: its weights and the place of a context."""

    def __init__(self, m, n):
        g = torch.Generator().manual_seed(1)
        self.w, self.ctx, self.d_out, self.d_in = torch.randn(m, n, generator=g), None, m, n


class Ads:
    """Stands for Adapters (which take 16-bit tensors only)."""

    def __init__(self, a, b, scaling):
        self.a, self.b, self.scaling = a, b, scaling
        self.count, self.rank, self.d_in = a.shape
        self.d_out = b.shape[1]


@pytest.fixture
def calls(monkeypatch):
    """The operators by their formulas (x kept as it is); counts the checkpoints."""
    made = []

    def of(ad, q):
        return torch.where(q >= 0, ad.scaling[q.long().clamp(min=0)], torch.zeros(()))

    def forward(packed, x, adapters=None, request=None, return_low=False):
        y = x @ packed.w.T
        if adapters is None:
            return y
        q = request.long().clamp(min=0)
        low = torch.einsum("tkn,tn->tk", adapters.a[q], x) * (request >= 0)[:, None]
        y = y + of(adapters, request)[:, None] * torch.einsum("tmk,tk->tm", adapters.b[q], low)
        return (y, low) if return_low else y

    def save(ctx, x):
        made.append(x.shape)
        return tune.Checkpoint(x.clone(), torch.ones(len(x), 1), x.dtype)

    def backward(packed, dy, saved=None, low=None, adapters=None, request=None):
        dx = dy @ packed.w
        if adapters is None:
            return dx, None, None
        q = request.long().clamp(min=0)
        up = of(adapters, request)[:, None] * torch.einsum("tmk,tm->tk", adapters.b[q], dy)
        dx = dx + torch.einsum("tkn,tk->tn", adapters.a[q], up)
        da, db = torch.zeros_like(adapters.a), torch.zeros_like(adapters.b)
        da.index_add_(0, q, torch.einsum("tk,tn->tkn", up, saved.codes))
        db.index_add_(0, q, torch.einsum("tm,tk->tmk", of(adapters, request)[:, None] * dy, low))
        return dx, da, db

    def loss(ctx, x, w, targets, ignore_index=-100):
        l = x @ w.T
        on = targets != ignore_index
        lse = torch.logsumexp(l, 1) * on
        return (lse - l.gather(1, targets.clamp(min=0)[:, None])[:, 0]) * on, lse

    def loss_backward(ctx, x, w, targets, lse, dloss, ignore_index=-100, need_dw=True):
        d = torch.softmax(x @ w.T, 1)
        d[torch.arange(len(x)), targets.clamp(min=0)] -= 1
        d = d * (dloss * (targets != ignore_index))[:, None]
        return d @ w, d.T @ x if need_dw else None

    for name, f in dict(adapter_linear=forward, checkpoint_save=save, adapter_linear_backward=backward,
                        vocab_loss=loss, vocab_loss_backward=loss_backward, Adapters=Ads).items():
        monkeypatch.setattr(tune, name, f)
    return made


def case(grad=True):
    g = torch.Generator().manual_seed(2)
    normal = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    a, b = normal(2, 3, 6).requires_grad_(grad), normal(2, 5, 3).requires_grad_(grad)
    return Layer(5, 6), normal(4, 6), Ads(a, b, torch.tensor([0.5, 2.0])), torch.tensor([0, 1, -1, 1], dtype=torch.int32)


def wanted(layer, x, a, b, scaling, q):
    """The same in torch, with autograd's own gradients."""
    i = q.long().clamp(min=0)
    low = torch.einsum("tkn,tn->tk", a[i], x)
    s = torch.where(q >= 0, scaling[i], torch.zeros(()))
    return x @ layer.w.T + s[:, None] * torch.einsum("tmk,tk->tm", b[i], low)


def test_linear_has_the_formulas_gradients(calls):
    layer, x, ad, q = case()
    dy = torch.randn(4, 5, generator=torch.Generator().manual_seed(3))
    x1, x2 = x.clone().requires_grad_(), x.clone().requires_grad_()
    got = torch.autograd.grad(tune.linear(layer, x1, ad, q), (x1, ad.a, ad.b), dy)
    want = torch.autograd.grad(wanted(layer, x2, ad.a, ad.b, ad.scaling, q), (x2, ad.a, ad.b), dy)
    for g, w in zip(got, want):
        assert torch.allclose(g, w, atol=1e-5)


def test_second_order_is_refused(calls):
    """The operators give no gradient of their gradients: a graph of them is refused, also where another path
    (a residual) or nothing at all would lead through it."""
    layer = Layer(6, 6)
    x = torch.randn(4, 6, generator=torch.Generator().manual_seed(3)).requires_grad_()
    w = torch.randn(9, 6, generator=torch.Generator().manual_seed(4))
    outputs = (lambda: tune.linear(layer, x),
               lambda: x * x + torch.nn.functional.silu(tune.linear(layer, x)),
               lambda: tune.cross_entropy(None, x, w, torch.tensor([1, 2, -100, 8])) + x.square().sum())
    for f in outputs:
        with pytest.raises(RuntimeError, match="first order only"):
            torch.autograd.grad(f().sum(), x, create_graph=True)
        (g,) = torch.autograd.grad(f().sum(), x)
        assert torch.isfinite(g).all() and g.any()


@pytest.mark.parametrize("what", ["a", "b", "scaling"])
def test_operands_changed_in_place_are_refused(calls, what):
    layer, x, ad, q = case()
    y = tune.linear(layer, x, ad, q)
    with torch.no_grad():
        getattr(ad, what).mul_(3.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


@pytest.mark.parametrize("what", ["a", "b", "scaling"])
def test_operands_replaced_do_not_reach_the_gradient(calls, what):
    """Another tensor put into the Adapters between the passes: the gradient is of what y was made with."""
    layer, x, ad, q = case()
    x = x.requires_grad_()
    a, b = ad.a, ad.b
    want = torch.autograd.grad(wanted(layer, x, a, b, ad.scaling, q).sum(), (x, a, b))
    y = tune.linear(layer, x, ad, q)
    setattr(ad, what, (getattr(ad, what).detach() * 3.0).requires_grad_(what != "scaling"))
    for g, w in zip(torch.autograd.grad(y.sum(), (x, a, b)), want):
        assert torch.allclose(g, w, atol=1e-5)


def test_a_scaling_that_asks_for_a_gradient_is_refused(calls):
    layer, x, ad, q = case()
    ad.scaling.requires_grad_()
    with pytest.raises(ValueError, match="scaling"):
        tune.linear(layer, x, ad, q)
    with torch.no_grad():  # no gradient is asked for
        assert torch.allclose(tune.linear(layer, x, ad, q), wanted(layer, x, ad.a, ad.b, ad.scaling, q), atol=1e-5)


def test_a_request_without_adapters_is_refused(monkeypatch):
    """As adapter_linear refuses it (before anything reaches the library)."""
    layer, x, _, q = case()
    monkeypatch.setattr(tune, "_matrix", lambda *_: 6)
    with pytest.raises(ValueError, match="request without adapters"):
        tune.linear(layer, x.bfloat16(), None, q)


def test_nothing_is_kept_where_no_gradient_is_asked_for(calls):
    layer, x, ad, q = case()
    want = wanted(layer, x, ad.a, ad.b, ad.scaling, q).detach()
    with torch.no_grad():
        assert torch.allclose(tune.linear(layer, x, ad, q), want, atol=1e-5)
    assert not calls
    layer, x, ad, q = case(grad=False)
    assert torch.allclose(tune.linear(layer, x, ad, q), want, atol=1e-5) and not calls
    layer, x, ad, q = case()
    tune.linear(layer, x, ad, q)
    assert len(calls) == 1
