"""CPU checks that the differentiable forms refuse tangents of forward-mode differentiation, for which they have no
formula, instead of dropping them (their operators by their formulas)."""
import pytest
import torch
import torch.autograd.forward_ad as fw

from cdclq import tune


class Packed:
    ctx, d_in, d_out = None, 5, 6
    weight = torch.randn(6, 5, generator=torch.Generator().manual_seed(1))


class Set:
    def __init__(self, a, b, scaling):
        self.a, self.b, self.scaling = a, b, scaling


@pytest.fixture(autouse=True)
def formulas(monkeypatch):
    def linear(packed, x, adapters=None, request=None, return_low=False):
        y = (x @ packed.weight.T).detach()
        return (y, x[:, :1].detach()) if return_low else y

    monkeypatch.setattr(tune, "embed", lambda ctx, table, tokens, *_: table.detach()[tokens])
    monkeypatch.setattr(tune, "adapter_linear", linear)
    monkeypatch.setattr(tune, "checkpoint_save", lambda ctx, x: tune.Checkpoint(x.detach(), x.detach(), x.dtype))


def adapters():
    return [torch.ones(1, 2, 5), torch.ones(1, 6, 2), torch.ones(1)]


def calls(which, dual):
    """A call with a tangent in one operand."""
    tokens, request = torch.tensor([1, 0, 1]), torch.zeros(3, dtype=torch.int32)
    x, parts = torch.ones(3, 5), adapters()
    if which == "embedding":
        return lambda: tune.embedding(None, dual(torch.ones(4, 5)), tokens)
    if which == "linear":
        return lambda: tune.linear(Packed, dual(x))
    if which == "linear x":
        return lambda: tune.linear(Packed, dual(x), Set(*parts), request)
    parts["abs".index(which[-1])] = dual(parts["abs".index(which[-1])])
    return lambda: tune.linear(Packed, x, Set(*parts), request)


@pytest.mark.parametrize("grad", [True, False])
@pytest.mark.parametrize("which", ["embedding", "linear", "linear x", "linear a", "linear b", "linear s"])
def test_tangents_are_refused(which, grad):
    """Under no_grad, too, which leaves forward mode on."""
    with fw.dual_level(), torch.set_grad_enabled(grad):
        with pytest.raises(NotImplementedError, match="jvp"):
            calls(which, lambda x: fw.make_dual(x, torch.ones_like(x)))()
        assert not calls(which, lambda x: x)().requires_grad  # no tangent: as ever
        with fw._set_fwd_grad_enabled(False):
            calls(which, lambda x: fw.make_dual(x, torch.ones_like(x)))()


@pytest.mark.parametrize("which", ["embedding", "linear", "linear x"])
def test_without_tangents_nothing_is_kept(which):
    assert calls(which, lambda x: x)().grad_fn is None
    assert calls(which, lambda x: x.requires_grad_())().requires_grad
    with torch.no_grad():
        assert calls(which, lambda x: x.requires_grad_())().grad_fn is None
