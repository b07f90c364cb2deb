"""GPU tests of cdclq.tune at the ends of the number range: sums near the largest numbers, weights of very
different sizes. Tolerances as in test_gpu_adapters.py and test_gpu_tune.py."""
import pytest
import torch

import cdclq
from tests.test_gpu_adapters import U, U32, check_backward, make_adapters, make_layer, make_request, near, normal, rng, \
    reference
from tests.test_gpu_tune import check_grad, logit_error, loss_inputs, loss_ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    c = cdclq.Context(0)
    yield c
    c.close()


@pytest.fixture(scope="module")
def tune():
    from cdclq import tune
    return tune


@pytest.mark.parametrize("mixed", [False, True])
def test_large_sums_beside_small_low_rank_vectors(ctx, tune, mixed):
    """bfloat16: projections of 2^106 and low-rank vectors of 2^-25 in one call. Dividing the former by the
    latter's power of two would pass the largest f32. A and B see eight features alone, whose x and dy are
    small; the others' weigh nothing in the low-rank terms."""
    m, n, t, rank, b = 150, 264, 300, 8, torch.bfloat16
    packed, w, _ = make_layer(ctx, tune, 5, m, n, 4, 64)
    ad = make_adapters(tune, 3, 2, rank, m, n, b)
    ad.a[:, :, 8:], ad.b[:, 8:] = 0, 0
    x, dy = normal(1, t, n, dtype=b), normal(2, t, m, dtype=b)
    q = make_request(4, t, 2, "any") if mixed else torch.zeros(t, dtype=torch.int32, device="cuda")
    x[:, :8] *= 2.0 ** -23
    x[:, 8:] *= 2.0 ** 107
    y, low = tune.adapter_linear(packed, x, ad, q, return_low=True)
    out, size = reference(w, ad, x, q)
    near(low, out["low"], size["low"] * n * U32, "low")
    near(y, out["y"], 1.01 * U[b] * out["y"].abs() + size["y"] * (U[b] + n * U32) + size["ylow"] * 2.0 ** -14, "y")
    # and the gradient of a large dy
    x = normal(1, t, n, dtype=b)
    dy[:, :8] *= 2.0 ** -23
    dy[:, 8:] *= 2.0 ** 107
    check_backward(packed, w, ad, x, q, dy, tune, ctx)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("t,d,v", [(60, 200, 3000), (300, 136, 5000), (2100, 64, 2000)])
def test_token_weights_of_very_different_sizes(ctx, tune, dtype, t, d, v):
    """A token's dx keeps its precision whatever the other tokens weigh: weights from 2^11 down to 2^-17 in one
    call, and head weights with a mean, of which dx = g (sum p w - w_y) has nothing only while the small p count.
    In float16 d is held scaled by 2^15 over its weight's power of two (half a subnormal step of it is
    2^-39 of the weight at most), and dw takes x scaled by the weight's power of two over the largest's, raised
    until its largest value is at float16's end: half a subnormal step there is, times the largest weight, at
    most 2^-39 of the largest x."""
    x, w, y = loss_inputs(t, t, d, v, dtype, ignored=0.1, std=1.5)
    w = (w.float() + 0.5).to(dtype)
    g = 2.0 ** (11.0 - torch.arange(t, device="cuda") % 29) * (1 + torch.rand(t, generator=rng(1), device="cuda")) / 2
    g *= torch.where(torch.arange(t, device="cuda") % 2 == 0, 1.0, -1.0)
    g[7], g[11] = 0.0, 0.0
    loss, lse = tune.vocab_loss(ctx, x, w, y)
    _, _, rdx, rdw, sx, sw = loss_ref(x, w, y, g)
    dx, dw = tune.vocab_loss_backward(ctx, x, w, y, lse, g)
    delta = 2 * logit_error(x, w, y) + 1e-6
    half = dtype == torch.float16
    # half a subnormal step of the token's own d (scaled by 2^15 over its weight's power of two), and of the output
    each = g.abs().double()[:, None] * 2.0 ** -38 * w.double().abs().sum(0) if half else 0.0
    out = 2.0 ** -25 if half else 0.0
    check_grad(dx, rdx, sx, dtype, delta, v, each + out)
    on = y != -100
    parts = 0.0
    if half:
        p = torch.softmax(x[on].double() @ w.double().T, 1)
        p[torch.arange(len(p), device="cuda"), y[on]] -= 1
        parts = (p.abs().sum(0) * g.abs().max() * x[on].double().abs().max() * 2.0 ** -38)[:, None]
        parts = parts + g.abs().max().item() * 2.0 ** -38 * x.double().abs().sum(0)
    check_grad(dw, rdw, sw, dtype, delta, t, parts + out)
    alone, _ = tune.vocab_loss_backward(ctx, x, w, y, lse, g, need_dw=False)
    assert torch.equal(alone, dx)
    assert not dx[7].any() and not dx[11].any()


def test_weights_that_are_not_finite_stay_at_their_token(ctx, tune):
    """An infinite or NaN weight makes its token's dx and dw not finite; the other tokens' dx do not change."""
    for dtype in (torch.bfloat16, torch.float16):
        x, w, y = loss_inputs(3, 40, 64, 700, dtype)
        lse = tune.vocab_loss(ctx, x, w, y)[1]
        g = torch.rand(40, generator=rng(2), device="cuda") * 2.0 ** -(torch.arange(40, device="cuda") % 9)
        g[0] = 2.0  # the largest stays
        want = tune.vocab_loss_backward(ctx, x, w, y, lse, g)[0]
        bad = g.clone()
        bad[3], bad[9] = float("inf"), float("nan")
        keep = torch.ones(40, dtype=torch.bool, device="cuda")
        keep[3] = keep[9] = False
        dx, dw = tune.vocab_loss_backward(ctx, x, w, y, lse, bad)
        assert torch.equal(dx[keep], want[keep])
        assert not torch.isfinite(dx[~keep]).any() and not torch.isfinite(dw).any()
        every = tune.vocab_loss_backward(ctx, x, w, y, lse, torch.full_like(g, float("inf")))[0]
        assert not torch.isfinite(every).any()
