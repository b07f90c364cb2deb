"""GPU tests of the tile shapes that large and narrow calls of cdclq.tune take, with enough stages that the
tiles' main loop runs, and of strides, streams and graphs in the forms of many tokens.

Tolerances as in test_gpu_tune.py and test_gpu_adapters.py; in addition the root mean square of an expanded
product's error: each weight is rounded once (relative error at most u, independent of the others), the
output once, so it stays below u (rms of the output + rms of sqrt(sum (w x)^2)). A column left out or
taken twice would move it by several times that."""
import pytest
import torch

import cdclq
from tests.test_gpu_adapters import U, U32, make_adapters, make_layer, make_request, near, normal, reference, rng, \
    saved_values
from tests.test_gpu_tune import check_grad, check_loss, logit_error, loss_inputs, loss_ref

pytestmark = pytest.mark.gpu

FEW, FEW_GRAD = 192, 128  # tokens up to which the weights are exact; up to which the gradient's dots are in f32
TYPES = [torch.bfloat16, torch.float16]


@pytest.fixture(scope="module")
def ctx():
    c = cdclq.Context(0)
    yield c
    c.close()


@pytest.fixture(scope="module")
def tune():
    from cdclq import tune
    return tune


# ---------------------------------------------------------------- the vocabulary loss
# Logits of a standard deviation of 6, so that a token's probability lies on a few entries: a piece of the
# vocabulary left out shows in the tokens that look there. Tiles of the logits, of dx and of dw:
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("t,d,v", [
    (1, 512, 128256),    # 256 x 16 and 256 x 16
    (10, 200, 128256),   # 256 x 16, 128 x 16
    (10, 201, 128256),   # the same on rows of W that are not aligned
    (17, 512, 128256),   # 256 x 32 and 256 x 32
    (30, 201, 128256),   # 256 x 32, 128 x 32, not aligned
    (60, 200, 128256),   # 256 x 64, 256 x 192
    (60, 201, 128256),   # 256 x 64 and 256 x 64, not aligned
    (9, 513, 50001),     # 128 x 16 and 128 x 16, not aligned
    (50, 513, 50001),    # 256 x 64, 128 x 64, not aligned
    (64, 256, 32000),    # 128 x 64, 128 x 128
    (77, 1000, 50001),   # 128 x 128, 256 x 192
    (200, 512, 32000),   # 128 x 128, 256 x 192, dw 256 x 256
    (513, 200, 32000),   # 256 x 192, 128 x 128
    (1200, 520, 12000),  # 256 x 256, 256 x 192
    (1000, 2048, 32000),  # 256 x 256 all
])
def test_loss_tiles(ctx, tune, dtype, t, d, v):
    x, w, y = loss_inputs(t + d + v, t, d, v, dtype, ignored=0.1, std=6.0)
    if t == 1:
        y[0] = v - 1
    g = torch.rand(t, generator=rng(7), device="cuda") / t
    rl, rs, rdx, rdw, sx, sw = loss_ref(x, w, y, g)
    loss, lse = tune.vocab_loss(ctx, x, w, y)
    check_loss(loss, rl, x, w, y)
    check_loss(lse, rs, x, w, y)
    dx, dw = tune.vocab_loss_backward(ctx, x, w, y, lse, g)
    delta = 2 * logit_error(x, w, y) + 1e-6
    half = dtype == torch.float16
    small = g.max().item() * 2.0 ** -40 if half else 0.0  # half a subnormal step of d, which is scaled by 2^15 / max g
    out = 2.0 ** -25 if half else 0.0
    check_grad(dx, rdx, sx, dtype, delta, v, small * w.double().abs().sum(0).max().item() + out)
    check_grad(dw, rdw, sw, dtype, delta, t, small * x.double().abs().sum(0).max().item() + out)


# ---------------------------------------------------------------- the projection
def rms(x):
    return x.double().square().mean().sqrt().item()


def forward(packed, w, big, ad, x, q, tune):
    y, low = tune.adapter_linear(packed, x, ad, q, return_low=True)
    out, size = reference(w, ad, x, q)
    u, n, t, k = U[x.dtype], w.shape[1], len(x), ad.rank
    tiny = 2.0 ** -25 if x.dtype == torch.float16 else 0.0
    exact = t <= FEW
    base = (x.double().abs() @ big.T) * (n + 8) * U32 if exact else size["y"] * (u + n * U32)
    near(low, out["low"], size["low"] * n * U32 + 1e-30, "low")
    near(y, out["y"], 1.01 * u * out["y"].abs() + base + size["ylow"] * (n * U32 + 2.0 ** -15 + k * U32) + tiny, "y")
    if not exact:
        each = (x.double().square() @ w.square().T).sqrt()
        assert rms(y.double() - out["y"]) <= u * (rms(out["y"]) + rms(each)) + 2.0 ** -15 * rms(size["ylow"])
    return y, low


def backward(packed, w, ad, x, q, dy, tune, ctx):
    low = tune.adapter_linear(packed, x, ad, q, return_low=True)[1]
    ck = tune.checkpoint_save(ctx, x)
    dx, da, db = tune.adapter_linear_backward(packed, dy, ck, low, ad, q)
    out, size = reference(w, ad, x, q, dy, saved_values(ck))
    u, (m, n), t, k = U[x.dtype], w.shape, len(x), ad.rank
    tiny = 2.0 ** -25 if x.dtype == torch.float16 else 0.0
    near(dx, out["dx"], 1.01 * u * out["dx"].abs() + size["dx"] * (u + m * U32) +
         size["dxlow"] * (m * U32 + 2.0 ** -15 + k * U32) + tiny, "dx")
    each = (dy.double().square() @ w.square()).sqrt()
    assert rms(dx.double() - out["dx"]) <= u * (rms(out["dx"]) + rms(each)) + 2.0 ** -15 * rms(size["dxlow"]) + tiny
    near(da, out["da"], 1.01 * u * out["da"].abs() + size["da"] * (m * U32 + 2.0 ** -15 + t * U32) + tiny, "da")
    near(db, out["db"], 1.01 * u * out["db"].abs() + size["db"] * (n * U32 + 2.0 ** -15 + t * U32) +
         tiny * (1 + dy.double().abs().sum(0).max().item()), "db")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n,t", [
    (500, 250, 200),    # 128 x 32
    (500, 1000, 193),   # 128 x 32, split in k
    (500, 2000, 260),   # 128 x 64, split
    (2000, 250, 520),   # 128 x 64
    (4000, 250, 520),   # 128 x 128
    (1000, 2000, 520),  # 128 x 128, split
    (12000, 250, 260),  # 256 x 64
    (6000, 250, 2000),  # 256 x 256
    (16000, 250, 520),  # 256 x 192
])
def test_forward_tiles(ctx, tune, dtype, m, n, t):
    packed, w, big = make_layer(ctx, tune, m + t, m, n, 4, 128)
    ad = make_adapters(tune, 3, 3, 12, m, n, dtype)
    for order in ("sorted", "any"):
        forward(packed, w, big, ad, normal(1, t, n, dtype=dtype), make_request(t, t, 3, order), tune)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n,t", [
    (200, 4090, 3000),    # 256 x 256
    (200, 4090, 1500),    # 128 x 64
    (203, 4090, 700),     # 128 x 128
    (4000, 1020, 300),    # 128 x 128, split in k
    (1000, 510, 150),     # 128 x 32, split
    (201, 131000, 10),    # 256 x 16
    (201, 131000, 30),    # 256 x 32
    (201, 131000, 60),    # 256 x 64
])
def test_gradient_tiles(ctx, tune, dtype, m, n, t):
    packed, w, _ = make_layer(ctx, tune, m + t, m, n, 4, 128)
    ad = make_adapters(tune, 3, 2, 12, m, n, dtype)
    backward(packed, w, ad, normal(1, t, n, dtype=dtype), make_request(t, t, 2, "any"), normal(2, t, m, dtype=dtype),
             tune, ctx)


@pytest.mark.parametrize("bits,group,lead", [(2, 64, 0), (3, 128, 0), (4, 128, 0), (8, 32, 0), (5, 48, 0), (4, 64, 2)])
@pytest.mark.parametrize("dtype", TYPES)
def test_weights_are_exact_up_to_the_limit(ctx, tune, dtype, bits, group, lead):
    m, n = 203, 393
    packed, w, big = make_layer(ctx, tune, bits * 100 + group, m, n, bits, group, lead)
    ad = make_adapters(tune, 5, 3, 8, m, n, dtype)
    for t in (65, 128, FEW):
        forward(packed, w, big, ad, normal(t, t, n, dtype=dtype), make_request(t, t, 3, "any"), tune)


# ---------------------------------------------------------------- many tokens: strides, no adapters, streams
def step(tune, ctx, packed, ad, x, dy, q):
    y, low = tune.adapter_linear(packed, x, ad, q, return_low=True)
    return (y, low) + tune.adapter_linear_backward(packed, dy, tune.checkpoint_save(ctx, x), low, ad, q)


@pytest.mark.parametrize("rank", [8, 16])
def test_strides_and_alignment_of_many_tokens(ctx, tune, rank):
    m, n, t, b = 100, 256, 230, torch.bfloat16
    packed, _, _ = make_layer(ctx, tune, 8, m, n, 4, 128)
    ad = make_adapters(tune, 2, 2, rank, m, n, b)
    shifted = lambda z: torch.empty(z.numel() + 1, dtype=b, device="cuda")[1:].view_as(z).copy_(z)  # noqa: E731
    odd = tune.Adapters(shifted(ad.a), shifted(ad.b), ad.scaling)
    big, up = normal(1, 500, 300, dtype=b), normal(2, 500, 120, dtype=b)
    q = make_request(4, t, 2, "any")
    for x, dy in ((big[:t, :256], up[:t, :100]), (big[: 2 * t: 2, 1:257], up[: 2 * t: 2, 3:103]),
                  (big[5: t + 5, 7:263], up[1: t + 1, 20:]), (big[:t, 8:264], up[:t, 8:108])):
        want = step(tune, ctx, packed, ad, x.contiguous(), dy.contiguous(), q)
        for which in (ad, odd):
            for a, c in zip(step(tune, ctx, packed, which, x, dy, q), want):
                assert torch.equal(a, c)


def test_many_tokens_without_adapters(ctx, tune):
    m, n, t, b = 90, 200, 300, torch.bfloat16
    packed, w, _ = make_layer(ctx, tune, 12, m, n, 4, 128)
    x, dy = normal(1, t, n, dtype=b), normal(2, t, m, dtype=b)
    y = tune.adapter_linear(packed, x)
    dx, da, db = tune.adapter_linear_backward(packed, dy)
    assert da is None and db is None
    near(y, x.double() @ w.T, 1.01 * U[b] * (x.double() @ w.T).abs() + (x.double().abs() @ w.abs().T) * (U[b] + n * U32), "y")
    near(dx, dy.double() @ w, 1.01 * U[b] * (dy.double() @ w).abs() + (dy.double().abs() @ w.abs()) * (U[b] + m * U32), "dx")
    ad = make_adapters(tune, 1, 3, 8, m, n, b)
    none = torch.full((t,), -1, dtype=torch.int32, device="cuda")
    y2, low, dx2, da, db = step(tune, ctx, packed, ad, x, dy, none)
    assert torch.equal(y, y2) and not low.any() and torch.equal(dx, dx2) and not da.any() and not db.any()
    live = x.clone().requires_grad_()
    out = tune.linear(packed, live)
    out.backward(dy)
    assert torch.equal(out.detach(), y) and torch.equal(live.grad, dx)


@pytest.mark.parametrize("t", [230, 700])
def test_many_tokens_in_a_graph(ctx, tune, t):
    m, n, b = 200, 384, torch.bfloat16
    packed, _, _ = make_layer(ctx, tune, 6, m, n, 4, 128)
    ad = make_adapters(tune, 2, 3, 24, m, n, b)
    held_in = [normal(1, t, n, dtype=b), normal(2, t, m, dtype=b), make_request(3, t, 3, "any")]
    step(tune, ctx, packed, ad, *held_in)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step(tune, ctx, packed, ad, *held_in)
    for seed in (11, 12, 13):
        new = normal(seed, t, n, dtype=b), normal(seed + 50, t, m, dtype=b), make_request(seed, t, 3, "any")
        for h, z in zip(held_in, new):
            h.copy_(z)
        graph.replay()
        torch.cuda.synchronize()
        for u, v in zip(held, step(tune, ctx, packed, ad, *new)):
            assert torch.equal(u, v)


def test_two_streams_at_once(ctx, tune):
    """Steps of two layers and two losses enqueued in turn on two streams, without a wait between them."""
    m, n, v, b = 300, 384, 5000, torch.bfloat16
    jobs = []
    for i, t in enumerate((700, 500)):
        packed, _, _ = make_layer(ctx, tune, 6 + i, m, n, 4, 128)
        ad = make_adapters(tune, 2 + i, 3, 24, m, n, b)
        args = (packed, ad, normal(i, t, n, dtype=b), normal(9 + i, t, m, dtype=b), make_request(i, t, 3, "any"))
        jobs.append((args, loss_inputs(i, t, n, v, b, ignored=0.1), torch.rand(t, generator=rng(i), device="cuda")))

    def run(job):
        args, (x, w, y), g = job
        loss, lse = tune.vocab_loss(ctx, x, w, y)
        return step(tune, ctx, *args) + (loss, lse) + tune.vocab_loss_backward(ctx, x, w, y, lse, g)

    want = [run(j) for j in jobs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in jobs]
    got = [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(run(jobs[i]))
    torch.cuda.synchronize()
    for i, w in enumerate(want):
        for g in got[i]:
            for a, c in zip(g, w):
                assert torch.equal(a, c)
