"""GPU tests of cdclq.tune's embedding, clipping and logit constraints beyond those of the operators' own files: sets of
gradients whose tensors change at their place, factors and norms at the ends of f32, tensors that autograd has saved,
gradients of the embedding through the C entry point, rows that lie between each other.

Tolerances are those of the operators' own files: u is the unit roundoff of the output's type, a sum of n rows in f32 is
off by at most n 2^-24 of the sum of their magnitudes, each other rounding to f32 by 2^-24."""
import math

import pytest
import torch

import cdclq

pytestmark = pytest.mark.gpu

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
TINY = {torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24, torch.float32: 2.0 ** -149}
U32 = 2.0 ** -24
TYPES = [torch.bfloat16, torch.float16, torch.float32]


@pytest.fixture(scope="module")
def ctx():
    c = cdclq.Context(0)
    yield c
    c.close()


@pytest.fixture(scope="module")
def tune():
    from cdclq import tune
    return tune


def rng(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def normal(seed, *shape, std=1.0, dtype=torch.float32):
    return (torch.randn(shape, generator=rng(seed), device="cuda") * std).to(dtype)


# ---------------------------------------------------------------- a set of gradients that is kept
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("count", [1, 200])
def test_a_gradient_changed_at_its_place(ctx, tune, dtype, count):
    """Shorter, longer and of another type in a buffer that others use, too: what lies outside stays."""
    flat = normal(1, 4000, dtype=dtype)
    rest = [normal(2 + i, 30) for i in range(count - 1)]
    x = flat[100:3100]
    g = tune.Gradients(ctx, [x, *rest])
    tune.clip_grads(g, math.inf)
    for dt, n in ((dtype, 10), (dtype, 3500), (torch.float32 if dtype != torch.float32 else torch.bfloat16, 100), (dtype, 0)):
        x.data = flat[100:].view(dt)[:n] if dt != dtype else flat[100:100 + n]
        x.copy_(normal(n, n))
        before, others = flat.clone(), [r.double().norm() ** 2 for r in rest]
        want = (x.double().norm() ** 2 + sum(others)).sqrt()
        old = x.double()
        got = tune.clip_grads(g, 0.5)
        assert abs(got.double() - want) <= 1.01 * U32 * want
        e = old * min(1.0, 0.5 / (want.item() + 1e-6))
        assert ((x.double() - e).abs() <= (U[dt] + 2.1 * U32) * e.abs() + TINY[dt]).all()
        end = 100 + n * x.element_size() // flat.element_size()
        now, before = flat.view(torch.uint8), before.view(torch.uint8)  # bits: halves of a wider type may be NaN
        at, end = 100 * flat.element_size(), end * flat.element_size()
        assert torch.equal(now[:at], before[:at]) and torch.equal(now[end:], before[end:])


def test_gradients_freed_and_allocated_again(ctx, tune):
    """set_to_none and a smaller gradient in the block that became free."""
    x = normal(1, 100_000)
    g = tune.Gradients(ctx, [x])
    tune.grad_norm(g)
    for n in (90_000, 5000, 100_000):
        x.data = torch.empty(0, device="cuda")
        x.data = normal(n, n)
        want = x.double().norm()
        assert abs(tune.grad_norm(g).double() - want) <= 1.01 * U32 * want


# ---------------------------------------------------------------- factors and norms at the ends of f32
def clipped(tensors, want, most, out):
    """Against min(1, most / (norm + 1e-6)) x in 64 bits: the factor, the product and the result rounded to f32, the
    result to its type; half a step of the smallest numbers."""
    by = min(1.0, most / (want + 1e-6))
    for o, x in zip(out, tensors):
        e = by * x.double()
        assert ((o.double() - e).abs() <= (U[o.dtype] + 2.1 * U32) * e.abs() + TINY[o.dtype]).all()
        # something is left of it, unless all is below the type's least number (half of it rounds to 0)
        assert e.abs().max() < TINY[o.dtype] or o.any()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("size,most", [(1e30, 1e-8), (1e30, 1e-16), (1e36, 1e-2), (1e36, 1e-30), (1e28, 1e-9)])
@pytest.mark.parametrize("n", [5, 70_001])
def test_factors_below_the_normal_numbers_of_f32(ctx, tune, dtype, size, most, n):
    """The factor is 1e-40 or 1e-70, its products are ordinary numbers; in place, into the same type and into float32."""
    tensors = [normal(1, n, dtype=dtype) * size, normal(2, 3, 1001, dtype=dtype) * size]
    want = sum(x.double().norm() ** 2 for x in tensors).sqrt().item()
    for kind in (dtype, torch.float32):
        out = [torch.full(x.shape, math.nan, dtype=kind, device="cuda") for x in tensors]
        tune.clip_grads(tune.Gradients(ctx, tensors, out=out), most)
        clipped(tensors, want, most, out)
    place = [x.clone() for x in tensors]
    tune.clip_grads(tune.Gradients(ctx, place), most)
    clipped(tensors, want, most, place)


def test_small_factors_of_half_precision(ctx, tune):
    """Float16 gradients into float32: factors of 1e-40, results of 1e-36."""
    x = normal(1, 3, 5000, std=1000.0, dtype=torch.float16)
    out = torch.empty(3, 5000, device="cuda")
    norm = tune.clip_grads(tune.Gradients(ctx, [x], out=[out], adapters=3), 1e-34)
    for i in range(3):
        clipped([x[i]], x[i].double().norm().item(), 1e-34, [out[i]])
    assert norm.shape == (3,)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("size,most", [(3e37, 1e38), (3e37, 1.0), (3e37, 1e-6), (5e37, 1e-40)])
def test_norms_above_f32_clip(ctx, tune, dtype, size, most):
    """Finite gradients whose norm is a number of f64 but not of f32: infinite where it is returned, and the gradients are
    clipped by what it is; another adapter's norm is as ever."""
    x = normal(1, 2, 70_001, dtype=dtype)
    x[0] *= size
    assert torch.isfinite(x).all()
    want = x.double().norm(dim=1)
    assert want[0] > torch.finfo(torch.float32).max
    out, place = torch.empty(2, 70_001, device="cuda"), x.clone()
    for n in (tune.clip_grads(tune.Gradients(ctx, [x], out=[out], adapters=2), most),
              tune.clip_grads(tune.Gradients(ctx, [place], adapters=2), most)):
        assert n[0] == math.inf and abs(n[1].double() - want[1]) <= 1.01 * U32 * want[1]
    for i in range(2):
        clipped([x[i], x[i]], want[i].item(), most, [out[i], place[i]])
    whole = [torch.empty_like(x)]
    assert tune.clip_grads(tune.Gradients(ctx, [x], out=whole), most) == math.inf
    clipped([x], want.norm().item(), most, whole)


# ---------------------------------------------------------------- tensors that autograd has saved
def writes(ctx, tune, x):
    """Each call that writes a tensor of its caller's (x: 4 x 40 float32), by name."""
    other, tokens = normal(1, 4, 40), torch.zeros(4, dtype=torch.int64, device="cuda")
    dy = normal(2, 4, 40, dtype=torch.bfloat16)
    return {"clip in place": lambda: tune.clip_grads(tune.Gradients(ctx, [other, x]), 1e-3),
            "clip into": lambda: tune.clip_grads(tune.Gradients(ctx, [other], out=[x]), 1e-3),
            "embed into": lambda: tune.embed_backward(ctx, dy, tokens, 4, into=x),
            "embed nothing into": lambda: tune.embed_backward(ctx, dy[:0], tokens[:0], 4, into=x),
            "constrain in place": lambda: tune.constrain_logits(ctx, x, out=x, history=tokens[:, None],
                                                                presence=torch.ones(4, device="cuda")),
            "constrain into": lambda: tune.constrain_logits(ctx, other, out=x)}


@pytest.mark.parametrize("call", ["clip in place", "clip into", "embed into", "embed nothing into", "constrain in place",
                                  "constrain into"])
def test_what_autograd_has_saved_and_a_call_writes_is_an_error(ctx, tune, call):
    x, w = normal(3, 4, 40), normal(4, 4, 40).requires_grad_()
    y = (x * w).sum()  # keeps x
    writes(ctx, tune, x)[call]()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
    y = (x * w).sum()
    tune.grad_norm(tune.Gradients(ctx, [x]))  # reads only
    tune.constrain_logits(ctx, x)
    y.backward()
    assert torch.equal(w.grad, x)


@pytest.mark.parametrize("call", ["clip in place", "clip into", "embed into", "constrain in place", "constrain into"])
def test_refused_calls_and_inference_tensors(ctx, tune, call):
    """A refused call leaves the counter alone; tensors of inference mode have none."""
    x = normal(3, 4, 40)
    before = x._version
    with pytest.raises((cdclq.CdclqError, ValueError)):
        tune.constrain_logits(ctx, x[:, :39], out=x[:, 1:])
    with pytest.raises(cdclq.CdclqError):
        tune.clip_grads(tune.Gradients(ctx, [x]), -1.0)
    assert x._version == before
    with torch.inference_mode():
        y = x.clone()
        writes(ctx, tune, y)[call]()
    writes(ctx, tune, x)[call]()
    assert torch.equal(x, y)


# ---------------------------------------------------------------- rows between each other
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("r,v,gap", [(1, 40, 0), (5, 33, 0), (5, 1000, 7), (70, 20_000, 1)])
@pytest.mark.parametrize("first", [True, False])
def test_logits_and_results_side_by_side(ctx, tune, dtype, r, v, gap, first):
    """Two halves of one buffer's columns share no memory."""
    buf = normal(1, r, 2 * v + gap, dtype=dtype)
    logits, out = (buf[:, :v], buf[:, v + gap:]) if first else (buf[:, v + gap:], buf[:, :v])
    k = dict(history=torch.randint(0, v, (r, 30), generator=rng(2), device="cuda"), presence=normal(3, r))
    before, want = buf.clone(), tune.constrain_logits(ctx, logits, **k)
    assert tune.constrain_logits(ctx, logits, out=out, **k) is out
    assert torch.equal(out, want)
    out.copy_(before[:, v + gap:] if first else before[:, :v])
    assert torch.equal(buf, before)
    for wrong in (buf[:, 1:v + 1], buf[:, v - 1:2 * v - 1], buf[:, v + gap - 1:2 * v + gap - 1]):
        if r > 1 and wrong.data_ptr() not in (logits.data_ptr(), out.data_ptr()):
            with pytest.raises(cdclq.CdclqError, match="overlaps"):
                tune.constrain_logits(ctx, buf[:, :v] if wrong.data_ptr() < buf.data_ptr() + v * buf.element_size() else
                                      buf[:, v + gap:], out=wrong)
    assert torch.equal(buf, before)


def test_rows_of_a_table_beside_its_gradient(ctx, tune):
    """dy and the gradient that it is added to in one buffer."""
    b, t, v, d = torch.bfloat16, 9, 9, 24
    buf = normal(1, t, 2 * d, dtype=b)
    tokens = torch.randint(0, v, (t,), generator=rng(2), device="cuda")
    want = tune.embed_backward(ctx, buf[:, :d].clone(), tokens, v, into=buf[:, d:].clone())
    before = buf.clone()
    tune.embed_backward(ctx, buf[:, :d], tokens, v, into=buf[:, d:])
    assert torch.equal(buf[:, d:], want) and torch.equal(buf[:, :d], before[:, :d])
    for wrong in (buf[:, :d], buf[:, 1:d + 1], buf[:, d - 1:2 * d - 1]):
        with pytest.raises(cdclq.CdclqError, match="overlaps"):
            tune.embed_backward(ctx, buf[:, :d], tokens, v, into=wrong)
    with pytest.raises(cdclq.CdclqError, match="overlaps"):  # strides of their own: by their ranges
        flat = buf.view(-1)
        tune.embed_backward(ctx, buf[:, :d], tokens, v, into=flat[d: d + v * d].view(v, d))


# ---------------------------------------------------------------- the embedding's gradient
def ids(seed, t, v):
    """Tokens, of which the first ones of the vocabulary come more often than the last."""
    u = torch.rand(t, generator=rng(seed), device="cuda", dtype=torch.float64)
    return (u * u * v).long().clamp(max=v - 1)


def summed(dy, tokens, v, scale):
    """The gradient in 64 bits, and the bound of its sums' errors: n additions, the scale and its product."""
    on = (tokens != -100).nonzero().flatten()
    rows, x = tokens[on], dy[on].double() * scale
    de, size = (torch.zeros(v, dy.shape[1], dtype=torch.float64, device="cuda").index_put_((rows,), y, accumulate=True)
                for y in (x, x.abs()))
    n = torch.zeros(v, dtype=torch.float64, device="cuda").index_put_((rows,), torch.ones_like(rows).double(), accumulate=True)
    return de, (n + 3)[:, None] * U32 * size, n > 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("into", ["same", "f32"])
@pytest.mark.parametrize("t,d,v", [(1, 9, 5), (2, 9, 5), (7, 1, 3), (64, 130, 77), (65, 2056, 20), (100, 4099, 9), (127, 8, 2),
                                   (128, 65, 300)])
@pytest.mark.parametrize("pad", [0, 3])
def test_few_tokens_added_to_a_gradient(ctx, tune, dtype, into, t, d, v, pad):
    """Some of them ignored, most ids several times."""
    kind = dtype if into == "same" else torch.float32
    tokens, dy = ids(1, t, v), normal(2, t, d, std=0.1, dtype=dtype)
    tokens[1::7] = -100
    buf = normal(3, v, d + pad, std=0.5, dtype=kind)
    before = buf.clone()
    got = tune.embed_backward(ctx, dy, tokens, v, 0.75, into=buf[:, :d])
    want, bound, on = summed(dy, tokens, v, 0.75)
    old = before[:, :d].double()
    assert on.any() and not torch.equal(got, before[:, :d])
    e = want + old
    assert ((got.double() - e).abs() <= bound + U32 * (want.abs() + old.abs()) + U[kind] * (e.abs() + bound) + TINY[kind]).all()
    assert torch.equal(got[~on], before[:, :d][~on]) and torch.equal(buf[:, d:], before[:, d:])


def grad_by_entry_point(ctx, tune, dy, tokens, v, scale, de, add=0):
    """cdclq_embed_backward_device itself: a new gradient of any type and row stride."""
    L, (t, d) = cdclq.lib(), dy.shape
    codes = {torch.float32: cdclq.DTYPE_F32, torch.float16: cdclq.DTYPE_F16, torch.bfloat16: cdclq.DTYPE_BF16}
    n = L.cdclq_embed_work_bytes(t, d, v)
    work = torch.empty(max(n, 1), dtype=torch.uint8, device="cuda")
    ctx.check(L.cdclq_embed_backward_device(ctx.ptr, dy.data_ptr(), d, t, d, v, codes[dy.dtype], tokens.data_ptr(), scale, -100,
                                            add, de.data_ptr(), de.stride(0), codes[de.dtype], work.data_ptr(), n,
                                            tune._stream(ctx)))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("into", ["same", "f32"])
@pytest.mark.parametrize("pad", [0, 3])
@pytest.mark.parametrize("d,v", [(33, 50), (65, 1000), (521, 70), (9, 20_000)])
@pytest.mark.parametrize("t", [0, 1, 77, 600, 9000])
def test_new_gradients_of_any_type_and_stride(ctx, tune, dtype, into, pad, d, v, t):
    """Rows without tokens are cleared, what lies between the rows stays."""
    kind = dtype if into == "same" else torch.float32
    tokens, dy = ids(1, t, v), normal(2, t, d, std=0.1, dtype=dtype)
    tokens[1::7] = -100
    buf = torch.full((v + 1, d + pad), 7.0, dtype=kind, device="cuda")
    de = buf[:v, :d]
    grad_by_entry_point(ctx, tune, dy, tokens, v, 1.25, de)
    want, bound, on = summed(dy, tokens, v, 1.25)
    assert ((de.double() - want).abs() <= bound + U[kind] * (want.abs() + bound) + TINY[kind]).all()
    assert not de[~on].any() and (buf[:v, d:] == 7).all() and (buf[v] == 7).all()
    if t:
        tokens[t // 2] = v
        for add in (0, 1):
            buf[:] = 7.0
            grad_by_entry_point(ctx, tune, dy, tokens, v, 1.25, de, add)
            assert de.isnan().all() and (buf[:v, d:] == 7).all() and (buf[v] == 7).all()
