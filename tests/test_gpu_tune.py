"""GPU tests of cdclq.tune: 8-bit activation checkpoints and the cross entropy over a large
vocabulary, against their definitions in 64 bits.

Tolerances follow from the number formats. u is the unit roundoff of the 16-bit type (2^-8 for
bfloat16, 2^-11 for float16; f32 2^-24). A product of two 16-bit values is exact in f32, so a sum of
k of them is off by at most k 2^-24 sum |a| |b|. What is rounded to 16 bits on the way adds u times
its magnitude, and an output rounded once adds u |out|."""
import ctypes as C

import numpy as np
import pytest
import torch

import cdclq

pytestmark = pytest.mark.gpu

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
U32 = 2.0 ** -24
IGNORE = -100


@pytest.fixture(scope="module")
def ctx():
    c = cdclq.Context(0)
    yield c
    c.close()


@pytest.fixture(scope="module")
def tune():
    from cdclq import tune
    return tune


def normal(seed, *shape, std=1.0, dtype=torch.float32):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * std).to(dtype)


# ---------------------------------------------------------------- 8-bit checkpoints
def saved_values(x):
    """codes and scales of the definition: one f32 division gives a block's scale, one f32 division
    and rint its codes."""
    x = x.float().cpu().numpy()
    t, n = x.shape
    nb = -(-n // 128)
    v = np.zeros((t, nb * 128), np.float32)
    v[:, :n] = x
    v = v.reshape(t, nb, 128)
    with np.errstate(invalid="ignore", over="ignore"):
        scale = np.abs(v).max(2) / np.float32(127)
        scale[~np.isfinite(v).all(2)] = np.nan
        ok = scale > 0
        codes = np.where(ok[:, :, None], np.rint(v / np.where(ok, scale, 1)[:, :, None]), 0)
    return codes.reshape(t, -1)[:, :n].astype(np.int8), scale


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("t,n", [(1, 1), (1, 128), (3, 127), (5, 129), (64, 1350), (130, 4096), (2, 28672)])
def test_checkpoint_matches_its_definition(ctx, tune, dtype, t, n):
    x = normal(t * 1000 + n, t, n, std=3.0, dtype=dtype)
    x[0, : n // 2] *= 50
    ck = tune.checkpoint_save(ctx, x)
    codes, scales = saved_values(x)
    assert np.array_equal(ck.codes.cpu().numpy(), codes)
    assert np.array_equal(ck.scales.cpu().numpy(), scales)
    want = torch.from_numpy(codes.astype(np.float32) * np.repeat(scales, 128, 1)[:, :n]).to(dtype)
    assert torch.equal(tune.checkpoint_restore(ctx, ck).cpu(), want)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_checkpoint_special_values(ctx, tune, dtype):
    """Zero blocks, the type's smallest and largest values, NaN and infinities (their block alone)."""
    x = torch.zeros(6, 300, dtype=dtype, device="cuda")
    tiny = torch.finfo(dtype).smallest_normal * 2.0 ** (-7 if dtype == torch.bfloat16 else -10)
    x[1, 5] = tiny
    x[2, :128] = torch.finfo(dtype).max
    x[2, 1] = torch.finfo(dtype).min
    x[3, 128] = float("nan")
    x[4, 299] = float("inf")
    x[5, 0], x[5, 200] = -float("inf"), 1.0
    ck = tune.checkpoint_save(ctx, x)
    codes, scales = saved_values(x)
    assert np.array_equal(ck.codes.cpu().numpy(), codes)
    assert np.array_equal(ck.scales.cpu().numpy(), scales, equal_nan=True)
    out = tune.checkpoint_restore(ctx, ck).float().cpu()
    assert torch.isnan(out[3, 128:256]).all() and torch.isfinite(out[3, :128]).all()
    assert torch.isnan(out[4, 256:]).all() and torch.isnan(out[5, :128]).all()
    assert out[5, 200] == 1.0 and not out[0].any()


def test_checkpoint_takes_any_row_stride_and_alignment(ctx, tune):
    big = normal(3, 40, 520, dtype=torch.bfloat16)
    for x in (big[:, :512], big[::2, 1:301], big[3:4, 7:], big[:, 4:260]):
        ck, own = tune.checkpoint_save(ctx, x), tune.checkpoint_save(ctx, x.contiguous())
        assert torch.equal(ck.codes, own.codes) and torch.equal(ck.scales, own.scales)
    assert tune.checkpoint_restore(ctx, tune.checkpoint_save(ctx, big[:0])).shape == (0, 520)


# ---------------------------------------------------------------- cross entropy
def loss_inputs(seed, t, d, v, dtype, ignored=0.0, std=2.0):
    x, w = normal(seed, t, d, dtype=dtype), normal(seed + 1, v, d, std=std / d ** 0.5, dtype=dtype)
    g = torch.Generator(device="cuda").manual_seed(seed + 2)
    y = torch.randint(0, v, (t,), generator=g, device="cuda")
    y[torch.rand(t, generator=g, device="cuda") < ignored] = IGNORE
    return x, w, y


def loss_ref(x, w, y, g=None):
    """loss, lse, d, dx, dw in 64 bits over the tokens that count; ignored rows are 0."""
    on = (y != IGNORE).nonzero().flatten()
    xd, wd = x[on].double(), w.double()
    l = xd @ wd.T
    lse_on = torch.logsumexp(l, 1) if len(on) else l.new_zeros(0)
    loss, lse = (torch.zeros(len(y), dtype=torch.float64, device="cuda") for _ in range(2))
    lse[on] = lse_on
    loss[on] = lse_on - l.gather(1, y[on][:, None])[:, 0]
    if g is None:
        return loss, lse
    d = torch.exp(l - lse_on[:, None])
    d[torch.arange(len(on), device="cuda"), y[on]] -= 1
    d *= g[on].double()[:, None]
    dx = torch.zeros_like(x, dtype=torch.float64)
    dx[on] = d @ wd
    sx = torch.zeros_like(dx)
    sx[on] = d.abs() @ wd.abs()
    return loss, lse, dx, d.T @ xd, sx, d.abs().T @ xd.abs()


def logit_error(x, w, y):
    """Largest error of a logit: d products summed in f32."""
    on = y != IGNORE
    big = (x[on].double().abs() @ w.double().abs().T).max().item() if on.any() else 0.0
    return x.shape[1] * U32 * big


def check_loss(got, want, x, w, y):
    # two logits, the rounding of the result and of the sum of exponentials' logarithm, exp and log
    # (a few ulp of values below 2^5 each)
    tol = 2 * logit_error(x, w, y) + 4 * U32 * want.abs().max().item() + 1e-5
    assert torch.isfinite(got).all()
    assert (got.double() - want).abs().max().item() <= tol


def check_grad(got, want, size, dtype, delta, k, extra):
    """size = sum |d| |b|: d is rounded to 16 bits (u), its exponent is off by delta + 4 ulp, the sum of
    k terms is in f32; extra covers what the 16-bit type cannot hold of d."""
    u = U[dtype]
    tol = u * want.abs() * 1.01 + size * (1.01 * u + 2 * delta + 8 * U32 + k * U32) + extra
    bad = (got.double() - want).abs() > tol
    assert torch.isfinite(got).all() and not bad.any(), ((got.double() - want).abs() / tol).max().item()


LOSS_SIZES = [(1, 1, 1), (1, 64, 1000), (2, 8, 257), (7, 1000, 5001), (16, 63, 999), (17, 512, 640), (33, 128, 4096),
              (64, 2048, 2000), (65, 72, 513), (129, 320, 1111), (300, 200, 8000), (257, 1350, 3001)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("t,d,v", LOSS_SIZES)
def test_vocab_loss_and_gradient(ctx, tune, dtype, t, d, v):
    x, w, y = loss_inputs(t + d + v, t, d, v, dtype, ignored=0.2)
    loss, lse = tune.vocab_loss(ctx, x, w, y)
    g = torch.rand(t, device="cuda") / t
    rl, rs, rdx, rdw, sx, sw = loss_ref(x, w, y, g)
    check_loss(loss, rl, x, w, y)
    check_loss(lse, rs, x, w, y)
    dx, dw = tune.vocab_loss_backward(ctx, x, w, y, lse, g)
    delta = 2 * logit_error(x, w, y) + 1e-6
    small = g.max().item() * 2.0 ** -15 * 2.0 ** -25 if dtype == torch.float16 else 0.0  # half a subnormal step of d
    out = 2.0 ** -25 if dtype == torch.float16 else 0.0  # and of the output
    check_grad(dx, rdx, sx, dtype, delta, v, small * w.double().abs().sum(0).max().item() + out)
    check_grad(dw, rdw, sw, dtype, delta, t, small * x.double().abs().sum(0).max().item() + out)
    alone, none = tune.vocab_loss_backward(ctx, x, w, y, lse, g, need_dw=False)
    assert none is None and torch.equal(alone, dx)


def test_vocab_loss_many_pieces_and_splits(ctx, tune):
    """More tokens than one piece of the vocabulary takes, and few tokens whose dx is split."""
    for t, d, v in ((4096, 64, 70001), (20, 128, 40000)):
        x, w, y = loss_inputs(5, t, d, v, torch.bfloat16, ignored=0.05)
        loss, lse = tune.vocab_loss(ctx, x, w, y)
        g = torch.full((t,), 1.0 / t, device="cuda")
        rl, rs, rdx, rdw, sx, sw = loss_ref(x, w, y, g)
        check_loss(loss, rl, x, w, y)
        dx, dw = tune.vocab_loss_backward(ctx, x, w, y, lse, g)
        delta = 2 * logit_error(x, w, y) + 1e-6
        check_grad(dx, rdx, sx, torch.bfloat16, delta, v, 0.0)
        check_grad(dw, rdw, sw, torch.bfloat16, delta, t, 0.0)
        del rdw, sw, dw


def test_vocab_loss_large_logits(ctx, tune):
    """Logits of hundreds: the running maximum keeps the exponentials in range."""
    x, w, y = loss_inputs(9, 40, 256, 3000, torch.bfloat16, std=60.0)
    loss, lse = tune.vocab_loss(ctx, x, w, y)
    want, wl = loss_ref(x, w, y)
    check_loss(loss, want, x, w, y)
    check_loss(lse, wl, x, w, y)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_ignored_tokens_reach_nothing(ctx, tune, dtype):
    """NaN and infinities at ignored tokens (and NaN weights of theirs) change no bit of the rest."""
    t, d, v = 70, 128, 900
    x, w, y = loss_inputs(21, t, d, v, dtype, ignored=0.4)
    off = y == IGNORE
    g = torch.rand(t, device="cuda")
    loss, lse = tune.vocab_loss(ctx, x, w, y)
    dx, dw = tune.vocab_loss_backward(ctx, x, w, y, lse, g)
    x2, g2 = x.clone(), g.clone()
    x2[off] = float("nan")
    x2[off.nonzero()[0, 0]] = float("inf")
    g2[off] = float("nan")
    loss2, lse2 = tune.vocab_loss(ctx, x2, w, y)
    dx2, dw2 = tune.vocab_loss_backward(ctx, x2, w, y, lse2, g2)
    assert torch.equal(loss, loss2) and torch.equal(lse, lse2) and torch.equal(dx, dx2) and torch.equal(dw, dw2)
    assert not loss[off].any() and not lse[off].any() and not dx[off].any()


def test_all_ignored_empty_and_outside(ctx, tune):
    t, d, v = 20, 64, 500
    x, w, y = loss_inputs(31, t, d, v, torch.bfloat16)
    none = torch.full_like(y, IGNORE)
    loss, lse = tune.vocab_loss(ctx, x, w, none)
    dx, dw = tune.vocab_loss_backward(ctx, x, w, none, lse, torch.ones(t, device="cuda"))
    assert not loss.any() and not lse.any() and not dx.any() and not dw.any()
    loss, lse = tune.vocab_loss(ctx, x[:0], w, y[:0])
    dx, dw = tune.vocab_loss_backward(ctx, x[:0], w, y[:0], lse, lse)
    assert loss.numel() == 0 and dx.shape == (0, d) and not dw.any()
    y[3], y[4] = v, -1
    loss, lse = tune.vocab_loss(ctx, x, w, y)
    assert torch.isnan(loss[3:5]).all() and torch.isfinite(loss[:3]).all() and torch.isfinite(loss[5:]).all()
    dx, _ = tune.vocab_loss_backward(ctx, x, w, y, lse, torch.ones(t, device="cuda"), need_dw=False)
    assert torch.isnan(dx[3:5]).all() and torch.isfinite(dx[5:]).all()
    # weights of zero give a gradient of zero
    y[3:5] = 0
    loss, lse = tune.vocab_loss(ctx, x, w, y)
    dx, dw = tune.vocab_loss_backward(ctx, x, w, y, lse, torch.zeros(t, device="cuda"))
    assert not dx.any() and not dw.any()


def test_vocab_loss_strides(ctx, tune):
    big, wide = normal(41, 50, 400, dtype=torch.bfloat16), normal(42, 700, 300, std=0.1, dtype=torch.bfloat16)
    y = torch.randint(0, 700, (25,), device="cuda")
    for x, w in ((big[::2, :256], wide[:, :256]), (big[::2, 3:203], wide[:, 1:201]), (big[25:, 8:264], wide[:, 40:296])):
        loss, lse = tune.vocab_loss(ctx, x, w, y)
        g = torch.ones(25, device="cuda")
        grads = tune.vocab_loss_backward(ctx, x, w, y, lse, g)
        xc, wc = x.contiguous(), w.contiguous()
        l2, s2 = tune.vocab_loss(ctx, xc, wc, y)
        assert torch.equal(loss, l2) and torch.equal(lse, s2)
        for a, b in zip(grads, tune.vocab_loss_backward(ctx, xc, wc, y, s2, g)):
            assert torch.equal(a, b)


def test_gradient_against_differences(ctx, tune):
    """(f(x + h u) - f(x - h u)) / 2 h of the kernel's losses against its gradient, along steps that
    bfloat16 holds exactly. The difference quotient's own error is taken from 64 bits."""
    t, d, v, h = 24, 64, 400, 2.0 ** -4
    gen = torch.Generator(device="cuda").manual_seed(5)
    grid = lambda *s: torch.randint(-15, 16, s, generator=gen, device="cuda").double() / 16  # noqa: E731
    x, w = grid(t, d), grid(v, d) / 2
    y = torch.randint(0, v, (t,), generator=gen, device="cuda")
    sign = lambda *s: torch.randint(0, 2, s, generator=gen, device="cuda").double() * 2 - 1  # noqa: E731
    b = torch.bfloat16
    g = torch.rand(t, device="cuda")
    _, lse = tune.vocab_loss(ctx, x.to(b), w.to(b), y)
    dx, dw = tune.vocab_loss_backward(ctx, x.to(b), w.to(b), y, lse, g)
    for which, grad in (("x", dx), ("w", dw)):
        u = sign(*(x.shape if which == "x" else w.shape)) * (torch.rand(t if which == "x" else v, 1, device="cuda") < 0.2)
        step = u * (h if which == "x" else h / 4)
        at = lambda s: (x + s * step, w) if which == "x" else (x, w + s * step)  # noqa: E731
        for s in (1, -1):
            for z in at(s):
                assert torch.equal(z.to(b).double(), z)  # representable
        kernel = sum(s * (tune.vocab_loss(ctx, *(z.to(b) for z in at(s)), y)[0].double() * g).sum() for s in (1, -1)) / 2
        exact = sum(s * (loss_ref(*at(s), y)[0] * g).sum() for s in (1, -1)) / 2
        inner = (grad.double() * step).sum()
        r = loss_ref(x, w, y, g)
        truth = (r[2 if which == "x" else 3] * step).sum()
        noise = t * 4e-6  # f32 losses below 2^4, a few ulp each, on both sides
        rounding = ((U[b] * 2.1 + 1e-5) * (r[4 if which == "x" else 5] * step.abs())).sum()
        assert (kernel - inner).abs() <= (exact - truth).abs() + noise + rounding
        assert (kernel - exact).abs() <= noise


def test_loss_repeats_bit_for_bit_on_streams_and_in_a_graph(ctx, tune):
    x, w, y = loss_inputs(51, 90, 256, 3000, torch.bfloat16, ignored=0.1)
    g = torch.rand(90, device="cuda")

    def step(x, y):
        loss, lse = tune.vocab_loss(ctx, x, w, y)
        return (loss, lse) + tune.vocab_loss_backward(ctx, x, w, y, lse, g)

    first = step(x, y)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step(x, y)
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(first, other):
        assert torch.equal(a, b)
    sx, sy = x.clone(), y.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step(sx, sy)
    for seed in (52, 53, 54):
        x2, _, y2 = loss_inputs(seed, 90, 256, 3000, torch.bfloat16, ignored=0.3)
        sx.copy_(x2)
        sy.copy_(y2)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(held, step(x2, y2)):
            assert torch.equal(a, b)


def test_refusals(ctx, tune):
    x, w, y = loss_inputs(61, 8, 64, 100, torch.bfloat16)
    with pytest.raises(TypeError):
        tune.vocab_loss(ctx, x.float(), w, y)
    with pytest.raises(TypeError):
        tune.vocab_loss(ctx, x, w.half(), y)
    with pytest.raises(TypeError):
        tune.vocab_loss(ctx, x, w, y.int())
    with pytest.raises(ValueError):
        tune.vocab_loss(ctx, x, w[:, :32], y)
    with pytest.raises(ValueError):
        tune.vocab_loss(ctx, x, w, y[:4])
    with pytest.raises(ValueError):
        tune.vocab_loss(ctx, x.t(), w, y)
    with pytest.raises(ValueError):
        tune.vocab_loss(ctx, x.cpu(), w, y)
    with pytest.raises(ValueError):
        tune.checkpoint_save(ctx, x[0])
    with pytest.raises(TypeError):
        tune.checkpoint_save(ctx, x.float())
    with pytest.raises(cdclq.CdclqError) as e:
        tune.vocab_loss(ctx, x, w[:0], y)
    assert "vocabulary" in str(e.value)
    L = cdclq.lib()
    out = torch.empty(16, device="cuda")
    args = [ctx.ptr, x.data_ptr(), 64, w.data_ptr(), 64, 8, 64, 100, cdclq.DTYPE_BF16, y.data_ptr(), IGNORE,
            out.data_ptr(), out[8:].data_ptr(), None, 0, None]
    assert L.cdclq_vocab_loss_device(*args) == cdclq.INVALID_ARG
    assert b"workspace" in L.cdclq_last_error(ctx.ptr)
    need = L.cdclq_vocab_work_bytes(8, 64, 100, w.data_ptr(), 64, 0)
    work = torch.empty(need + 256, dtype=torch.uint8, device="cuda")
    args[13:15] = [work.data_ptr() + 16, need]
    assert L.cdclq_vocab_loss_device(*args) == cdclq.INVALID_ARG
    args[13:15] = [work.data_ptr(), need - 1]
    assert L.cdclq_vocab_loss_device(*args) == cdclq.INVALID_ARG
    args[13:15] = [work.data_ptr(), need]
    for at, bad in ((2, 63), (4, 8), (8, cdclq.DTYPE_F32), (9, None), (11, None), (5, 1 << 40)):
        wrong = list(args)
        wrong[at] = bad
        assert L.cdclq_vocab_loss_device(*wrong) == cdclq.INVALID_ARG, at
    assert L.cdclq_vocab_loss_device(*args) == cdclq.OK
    assert L.cdclq_vocab_loss_device(None, *args[1:]) == cdclq.INVALID_ARG
    torch.cuda.synchronize()
