"""GPU tests of cdclq.tune's gradient norms and clipping, against their definitions in 64 bits.

Tolerances. The squares of the elements are exact in 64 bits but for float32 ones (2^-53), a sum of n of them is off by
at most n 2^-53 of itself: the norm is the float32 next to the exact one, or the one beside it: 2^-24 and n 2^-54 of it
(1.01 2^-24 here, n < 2^26). The factor is rounded to f32 (2^-24), its product with x again and once more to the output's
type (u): (u + 2 2^-24 + the norm's n 2^-54) |out|, and half a step of the smallest numbers."""
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


def norms(tensors, parts=None):
    p = parts or 1
    return sum((x.double().reshape(p, -1) ** 2).sum(1) for x in tensors).sqrt()


def close_norm(got, want):
    assert got.dtype == torch.float32
    assert ((got.double() - want).abs() <= 1.01 * U32 * want).all(), (got, want)


def check_clipped(got, tensors, want, most, parts=None):
    p = parts or 1
    by = torch.clamp(most / (want + 1e-6), max=1.0)
    for o, x in zip(got, tensors):
        e = by.view(-1, 1) * x.double().reshape(p, -1)
        err = (o.double().reshape(p, -1) - e).abs()
        assert (err <= (U[o.dtype] + 2.1 * U32) * e.abs() + TINY[o.dtype]).all(), err.max().item()


SHAPES = [[()], [(1,)], [(7,), (8, 3), (0,), (1000, 17)], [(4096,), (4097,), (4095,)], [(300, 300)] * 5 + [(2, 3, 5)],
          [(1 << 20,), (5,)], [(3000, 3000), (1,), (70, 1)]]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shapes", SHAPES)
@pytest.mark.parametrize("share", [0.25, 2.0])
def test_norm_and_clipping(ctx, tune, dtype, shapes, share):
    """In place, into the same type and into float32; above the limit and below it (nothing changes a bit)."""
    tensors = [normal(i, *s, std=0.3, dtype=dtype) for i, s in enumerate(shapes)]
    want = norms(tensors)[0]
    most = share * want.item()
    close_norm(tune.grad_norm(tune.Gradients(ctx, tensors)), want)
    for kind in (dtype, torch.float32):
        out = [torch.full(x.shape, math.nan, dtype=kind, device="cuda") for x in tensors]
        before = [x.clone() for x in tensors]
        close_norm(tune.clip_grads(tune.Gradients(ctx, tensors, out=out), most), want)
        check_clipped(out, tensors, want, most)
        assert all(torch.equal(x, b) for x, b in zip(tensors, before))
        if share > 1:
            assert all(torch.equal(o, x.to(kind)) for o, x in zip(out, tensors))
    place = [x.clone() for x in tensors]
    n = tune.clip_grads(tune.Gradients(ctx, place), most)
    assert n.shape == ()
    close_norm(n, want)
    check_clipped(place, tensors, want, most)
    if share > 1:
        assert all(torch.equal(x, b) for x, b in zip(place, tensors))


@pytest.mark.parametrize("count", [149, 150, 151, 300, 301, 448])
def test_many_tensors(ctx, tune, count):
    """More than one launch's tables hold; the three types side by side."""
    tensors = [normal(i, 3 + 37 * i % 901, 5, std=1 + i % 5, dtype=TYPES[i % 3]) for i in range(count)]
    want = norms(tensors)[0]
    out = [torch.empty(x.shape, device="cuda") for x in tensors]
    g = tune.Gradients(ctx, tensors, out=out)
    close_norm(tune.grad_norm(g), want)
    close_norm(tune.clip_grads(g, 1.0), want)
    check_clipped(out, tensors, want, 1.0)
    first = [o.clone() for o in out]
    tune.clip_grads(g, 1.0)
    assert all(torch.equal(a, b) for a, b in zip(first, out))


@pytest.mark.parametrize("count", [229, 230, 231, 460, 461])
def test_tables_of_several_launches(ctx, tune, count):
    """Sets at the ends of the launches that write the table; tensors of one and of several chunks, and adapters."""
    tensors = [normal(i, 2, (7 + 7 * i % 77) * (1 + 613 * (i % 2)), std=1 + i % 5, dtype=TYPES[i % 3])
               for i in range(count)]
    for adapters in (None, 2):
        out = [torch.empty(x.shape, device="cuda") for x in tensors]
        g = tune.Gradients(ctx, tensors, out=out, adapters=adapters)
        want = norms(tensors, adapters)
        close_norm(tune.clip_grads(g, 1.0), want if adapters else want[0])
        check_clipped(out, tensors, want, 1.0, adapters)


@pytest.mark.parametrize("count", [3, 448])
def test_a_norm_does_not_look_at_outputs(ctx, tune, count):
    tensors = [normal(i, 40 + i, dtype=TYPES[i % 3]) for i in range(count)]
    g = tune.Gradients(ctx, tensors)
    g.table["out"] = 2**64 - 2
    close_norm(tune.grad_norm(g), norms(tensors)[0])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("users", [1, 2, 5, 300])
def test_each_adapter_by_its_own_norm(ctx, tune, dtype, users):
    """Users' adapters in the first dimension: one above the limit is clipped, its neighbours are not touched."""
    tensors = [normal(i, users, *s, std=0.1, dtype=dtype) for i, s in enumerate([(8, 33), (77, 8), (1,), (3, 1001)])]
    loud = users // 2
    for x in tensors:
        x[loud] *= 50
    want = norms(tensors, users)
    most = 10.0  # the quiet ones' norms are about 6
    assert want[loud] > most and (users == 1 or want[0] < most)
    g = tune.Gradients(ctx, [x.clone() for x in tensors], adapters=users)
    close_norm(tune.grad_norm(g), want)
    n = tune.clip_grads(g, most)
    assert n.shape == (users,)
    close_norm(n, want)
    check_clipped(g.tensors, tensors, want, most, users)
    for x, b in zip(g.tensors, tensors):
        rest = [i for i in range(users) if i != loud]
        assert torch.equal(x[rest], b[rest])
        assert torch.equal(torch.isfinite(x).all(), torch.tensor(True, device="cuda"))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("size", [1e-30, 1e30])
def test_squares_outside_f32(ctx, tune, dtype, size):
    x = normal(1, 5000, std=size, dtype=dtype)
    want = norms([x])[0]
    close_norm(tune.grad_norm(tune.Gradients(ctx, [x])), want)
    out = torch.empty(5000, device="cuda")
    tune.clip_grads(tune.Gradients(ctx, [x], out=[out]), 1.0)
    check_clipped([out], [x], want, 1.0)


@pytest.mark.parametrize("dtype", TYPES)
def test_norms_that_are_not_finite_clip_nothing(ctx, tune, dtype):
    """A user whose gradients overflowed: their norm says so, they stay, and the others are clipped as ever."""
    x = normal(1, 3, 5000, dtype=dtype)
    x[1, 17] = math.inf
    x[2, 4999] = math.nan
    g = tune.Gradients(ctx, [x.clone()], adapters=3)
    n = tune.clip_grads(g, 1.0)
    assert torch.isfinite(n[0]) and n[1] == math.inf and n[2].isnan()
    got = g.tensors[0]
    assert torch.equal(got[1], x[1]) and torch.equal(got[2].nan_to_num(9), x[2].nan_to_num(9))
    check_clipped([got[:1]], [x[:1]], norms([x[:1]], 1), 1.0)
    out = [torch.empty(3, 5000, device="cuda")]
    tune.clip_grads(tune.Gradients(ctx, [x], out=out, adapters=3), 1.0)
    assert torch.equal(out[0][1], x[1].float()) and torch.equal(out[0][0].to(dtype), got[0])


def test_limits_of_max_norm(ctx, tune):
    x = normal(1, 1000)
    for most, share in ((0.0, 0.0), (math.inf, 1.0), (1e-300, 0.0)):
        out = [torch.empty_like(x)]
        tune.clip_grads(tune.Gradients(ctx, [x], out=out), most)
        assert torch.equal(out[0], x * share)
    zero = torch.zeros(5, device="cuda")
    assert tune.clip_grads(tune.Gradients(ctx, [zero]), 0.0).item() == 0.0 and not zero.any()


@pytest.mark.parametrize("adapters", [None, 4])
def test_nothing_to_clip(ctx, tune, adapters):
    for tensors in ([], [torch.empty(4, 0, device="cuda")]):
        g = tune.Gradients(ctx, tensors, adapters=adapters)
        for n in (tune.grad_norm(g), tune.clip_grads(g, 1.0)):
            assert n.shape == (() if adapters is None else (4,)) and not n.any()


@pytest.mark.parametrize("dtype", TYPES)
def test_tensors_of_any_alignment(ctx, tune, dtype):
    """Views one behind the other in a bucket, at odd elements; what lies between them stays."""
    flat = normal(1, 40_000, dtype=dtype)
    at, tensors, held = 1, [], torch.zeros(40_000, dtype=torch.bool, device="cuda")
    for n in (1, 3, 4097, 8, 12_345, 15):
        tensors.append(flat[at:at + n])
        held[at:at + n] = True
        at += n + (n & 2)
    before = flat.clone()
    want = norms(tensors)[0]
    close_norm(tune.clip_grads(tune.Gradients(ctx, tensors), 1.0), want)
    by = min(1.0, 1.0 / (want.item() + 1e-6))
    e = before.double() * by
    assert torch.equal(flat[~held], before[~held])
    assert ((flat.double() - e).abs()[held] <= ((U[dtype] + 2.1 * U32) * e.abs() + TINY[dtype])[held]).all()


def test_large_tensors(ctx, tune):
    """Past 2^31 elements: pieces of 2^30, more than 2^32 bytes from the start."""
    x = torch.full(((1 << 31) + 12_345,), 2.0 ** -10, dtype=torch.bfloat16, device="cuda")
    x[-1] = 3.0
    g = tune.Gradients(ctx, [x])
    want = torch.tensor(math.sqrt((len(x) - 1) * 2.0 ** -20 + 9.0), dtype=torch.float64, device="cuda")
    close_norm(tune.grad_norm(g), want)
    close_norm(tune.clip_grads(g, want.item() / 2), want)
    assert x[0] == 2.0 ** -11 and x[1 << 30] == 2.0 ** -11 and x[-2] == 2.0 ** -11 and x[-1] == 1.5
    assert (x[:-1] == 2.0 ** -11).all()


def test_a_set_follows_its_tensors(ctx, tune):
    """A kept set whose tensors got other memory."""
    x = normal(1, 1000)
    g = tune.Gradients(ctx, [x])
    a = tune.grad_norm(g)
    x.data = normal(2, 1000, std=3.0)
    b = tune.grad_norm(g)
    close_norm(b, norms([x])[0])
    assert a != b
    for n, dtype in ((10, torch.float32), (50_000, torch.float32), (0, torch.float32)):  # of other sizes, too
        x.data = normal(3, n, dtype=dtype)
        close_norm(tune.grad_norm(g), norms([x])[0])
        before = x.clone()
        tune.clip_grads(g, 1.0)
        check_clipped([x], [before], norms([before])[0], 1.0)
    x.data = normal(4, 20, 30).t()
    with pytest.raises(ValueError, match="contiguous"):
        tune.grad_norm(g)
    out = normal(5, 100)
    h = tune.Gradients(ctx, [normal(6, 100)], out=[out])
    out.data = normal(5, 99)
    with pytest.raises(ValueError, match="shape"):
        tune.clip_grads(h, 1.0)


def test_captured_and_replayed(ctx, tune):
    tensors = [normal(i, 4, 500 + i, dtype=torch.bfloat16) for i in range(250)]
    out = [torch.empty(x.shape, device="cuda") for x in tensors]
    sets = tune.Gradients(ctx, tensors, out=out, adapters=4), tune.Gradients(ctx, tensors, adapters=4)
    for s in sets:
        tune.clip_grads(s, 1e9)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        n = tune.clip_grads(sets[0], 3.0)
        m = tune.clip_grads(sets[1], 2.0)
    for i in range(4):
        for k, x in enumerate(tensors):
            x.copy_(normal(1000 * i + k, *x.shape, std=0.1 + i))
        before = [x.clone() for x in tensors]
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(n, m)
        close_norm(n, norms(before, 4))
        check_clipped(out, before, norms(before, 4), 3.0, 4)
        check_clipped(tensors, before, norms(before, 4), 2.0, 4)
        eager = [x.clone() for x in before]
        tune.clip_grads(tune.Gradients(ctx, eager, adapters=4), 2.0)
        assert all(torch.equal(a, b) for a, b in zip(eager, tensors))


def test_two_streams_at_once(ctx, tune):
    streams = [torch.cuda.Stream() for _ in range(2)]
    data = [[normal(10 * i + k, 100_000 + k) for k in range(5)] for i in range(2)]
    outs = [[torch.empty_like(x) for x in d] for d in data]
    sets = [tune.Gradients(ctx, d, out=o) for d, o in zip(data, outs)]
    want = [norms(d)[0] for d in data]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(tune.clip_grads(sets[i], 1.0 + i))
    torch.cuda.synchronize()
    for i in range(2):
        for n in got[i]:
            close_norm(n, want[i])
        check_clipped(outs[i], data[i], want[i], 1.0 + i)


def test_refusals(ctx, tune):
    x, y = normal(1, 4, 6), normal(2, 4, 6)
    for e, f in [(TypeError, lambda: tune.Gradients(ctx, [x.double()])),
                 (TypeError, lambda: tune.Gradients(ctx, [x.long()])),
                 (ValueError, lambda: tune.Gradients(ctx, [x.cpu()])),
                 (ValueError, lambda: tune.Gradients(ctx, [x.t()])),
                 (ValueError, lambda: tune.Gradients(ctx, [x], out=[])),
                 (ValueError, lambda: tune.Gradients(ctx, [x], out=[y[:3]])),
                 (TypeError, lambda: tune.Gradients(ctx, [x], out=[y.half()])),
                 (ValueError, lambda: tune.Gradients(ctx, [x], adapters=3)),
                 (ValueError, lambda: tune.Gradients(ctx, [x], adapters=0)),
                 (ValueError, lambda: tune.Gradients(ctx, [x.sum()], adapters=1)),
                 (cdclq.CdclqError, lambda: tune.clip_grads(tune.Gradients(ctx, [x]), -1.0)),
                 (cdclq.CdclqError, lambda: tune.clip_grads(tune.Gradients(ctx, [x]), math.nan)),
                 (TypeError, lambda: tune.clip_grads([x], 1.0)),
                 (cdclq.CdclqError, lambda: tune.clip_grads(tune.Gradients(ctx, [x, x]), 1.0)),
                 (cdclq.CdclqError, lambda: tune.clip_grads(tune.Gradients(ctx, [x, x[1:]]), 1.0)),
                 (cdclq.CdclqError, lambda: tune.clip_grads(tune.Gradients(ctx, [x, y], out=[y, x]), 1.0)),
                 (cdclq.CdclqError, lambda: tune.clip_grads(tune.Gradients(ctx, [x[:2]], out=[x[1:3]]), 1.0))]:
        with pytest.raises(e):
            f()
    g, n = tune.Gradients(ctx, [x]), torch.empty((), device="cuda")
    for work, size in ((0, 0), (torch.empty(1024, dtype=torch.uint8, device="cuda").data_ptr(), g.work_bytes - 1)):
        for call in (lambda: cdclq.lib().cdclq_grad_norm_device(ctx.ptr, g.ptr, 1, 1, n.data_ptr(), work, size, 0),
                     lambda: cdclq.lib().cdclq_clip_grads_device(ctx.ptr, g.ptr, 1, 1, 1.0, n.data_ptr(), work, size, 0)):
            assert call() == cdclq.INVALID_ARG and b"workspace" in cdclq.lib().cdclq_last_error(ctx.ptr)
    assert cdclq.lib().cdclq_grad_norm_device(ctx.ptr, g.ptr, 1, 7, n.data_ptr(), 0, 0, 0) == cdclq.INVALID_ARG  # parts
    assert torch.equal(x, normal(1, 4, 6)) and torch.equal(y, normal(2, 4, 6))
    close_norm(tune.grad_norm(tune.Gradients(ctx, [x, x])), norms([x, x])[0])  # nothing is written: twice is twice
