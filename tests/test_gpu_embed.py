"""GPU tests of cdclq.tune's token embedding and the gradient of its table, against their definitions in 64 bits.

Tolerances. u is the unit roundoff of the output's type (2^-8 for bfloat16, 2^-11 for float16, 2^-24 for float32). The
forward pass rounds scale and scale * x to f32 and then to the type: (u + 2 2^-24) |y|, and half a step of the smallest
numbers. A sum of n rows in f32 is off by at most n 2^-24 sum |dy|, times scale; scale, the product and the addition to a
gradient that exists are rounded to f32 each, and the result once more: u |dE|."""
import numpy as np
import pytest
import torch

import cdclq

pytestmark = pytest.mark.gpu

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
TINY = {torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24, torch.float32: 2.0 ** -149}
U32 = 2.0 ** -24
TYPES = [torch.bfloat16, torch.float16]
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


def rng(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def normal(seed, *shape, std=1.0, dtype=torch.float32):
    return (torch.randn(shape, generator=rng(seed), device="cuda") * std).to(dtype)


def make_tokens(seed, t, v, kind):
    """Ids: all over the vocabulary, a few frequent ones beside rare ones, one alone, every one once, the last ones."""
    g = rng(seed)
    if kind == "any":
        x = torch.randint(0, v, (t,), generator=g, device="cuda")
    elif kind == "frequent":
        u = torch.rand(t, generator=g, device="cuda", dtype=torch.float64)
        x = (torch.exp(u * np.log(v + 1)) - 1).long().clamp(0, v - 1)
        x = torch.randperm(v, generator=g, device="cuda")[x]
    elif kind == "one":
        x = torch.full((t,), v // 2, device="cuda")
    elif kind == "once":
        x = torch.randperm(max(t, v), generator=g, device="cuda")[:t] % v
    else:
        x = torch.randint(max(0, v - 3), v, (t,), generator=g, device="cuda")
    return x.long()


def table_gradient(dy, tokens, v, scale):
    """dE and the bound of its sum's error, in 64 bits."""
    on = (tokens != IGNORE).nonzero().flatten()
    ids, x = tokens[on], dy[on].double()
    d = dy.shape[1]
    de = torch.zeros(v, d, dtype=torch.float64, device="cuda").index_put_((ids,), x * scale, accumulate=True)
    size = torch.zeros(v, d, dtype=torch.float64, device="cuda").index_put_((ids,), x.abs() * abs(scale), accumulate=True)
    n = torch.bincount(ids, minlength=v).double() if len(ids) else torch.zeros(v, dtype=torch.float64, device="cuda")
    return de, (n + 3)[:, None] * U32 * size


def check(got, want, bound, dtype):
    err = (got.double() - want).abs()
    assert (err <= bound * 1.0001 + U[dtype] * want.abs() * 1.0001 + TINY[dtype]).all(), err.max().item()


# ---------------------------------------------------------------- rows
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("t,d,v", [(0, 8, 4), (1, 1, 1), (1, 4096, 100), (3, 7, 5), (5, 64, 1000), (33, 1000, 77),
                                   (257, 4104, 50), (1000, 129, 3001), (4, 40000, 9)])
@pytest.mark.parametrize("scale", [1.0, 0.37])
def test_rows(ctx, tune, dtype, t, d, v, scale):
    table, tokens = normal(1, v, d, dtype=dtype), make_tokens(2, t, v, "any")
    if t > 2:
        tokens[1] = IGNORE
    y = tune.embed(ctx, table, tokens, scale)
    assert y.shape == (t, d) and y.dtype == dtype
    want = table.double()[tokens.clamp(min=0)] * scale * (tokens != IGNORE)[:, None]
    if scale == 1.0:
        assert torch.equal(y.double(), want)
    check(y, want, 2 * U32 * want.abs(), dtype)  # scale and the product in f32


@pytest.mark.parametrize("dtype", TYPES)
def test_rows_of_strange_ids(ctx, tune, dtype):
    """Ids outside the vocabulary (past 32 bits among them) give NaN, the ignored one zeros, also where it is an id
    of the vocabulary; NaN and infinities of the table come through."""
    v, d = 10, 100
    table = normal(1, v, d, dtype=dtype)
    table[3, 5], table[3, 6] = float("nan"), float("-inf")
    ids = [0, 3, -1, v, v + 1, 1 << 32, (1 << 32) + 3, -(1 << 63), (1 << 63) - 1, IGNORE, 9]
    y = tune.embed(ctx, table, torch.tensor(ids, device="cuda"), 2.0)
    for i, k in enumerate(ids):
        if 0 <= k < v:
            assert torch.equal(y[i].nan_to_num(7.0), (table[k].float() * 2.0).to(dtype).nan_to_num(7.0))
        elif k == IGNORE:
            assert torch.equal(y[i], torch.zeros_like(y[i]))
        else:
            assert y[i].isnan().all()
    y = tune.embed(ctx, table, torch.tensor([0, 1, 0], device="cuda"), ignore_index=0)
    assert not y[0].any() and not y[2].any() and torch.equal(y[1], table[1])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("offset,ld", [(0, 72), (1, 71), (3, 70), (8, 65)])
def test_rows_of_strided_tables(ctx, tune, dtype, offset, ld):
    t, d, v = 40, 65, 30
    buf = normal(1, v * ld + offset, dtype=dtype)
    table = buf[offset:].view(v, ld)[:, :d]
    tokens = make_tokens(2, t, v, "any")
    assert torch.equal(tune.embed(ctx, table, tokens), table[tokens])


# ---------------------------------------------------------------- gradient
SIZES = [(1, 1, 1), (1, 8, 3), (7, 33, 20), (64, 100, 50), (65, 4096, 70), (128, 72, 50), (129, 72, 50), (511, 72, 1000), (512, 130, 20),
         (513, 130, 20), (600, 2056, 300), (1025, 65, 5000), (4096, 64, 257), (8192, 40, 999), (8193, 40, 999),
         (12289, 24, 100), (20000, 520, 70000), (70001, 8, 300), (530_001, 8, 70_000), (1_100_000, 16, 500)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("t,d,v", SIZES)
@pytest.mark.parametrize("kind", ["any", "frequent", "one", "once", "last"])
def test_gradient(ctx, tune, dtype, t, d, v, kind):
    tokens = make_tokens(t + v, t, v, kind)
    tokens[torch.rand(t, generator=rng(4), device="cuda") < 0.1] = IGNORE
    dy = normal(5, t, d, std=0.1, dtype=dtype)
    want, bound = table_gradient(dy, tokens, v, 1.25)
    got = tune.embed_backward(ctx, dy, tokens, v, 1.25)
    assert got.dtype == dtype and got.shape == (v, d)
    check(got, want, bound, dtype)
    none = torch.ones(v, dtype=torch.bool, device="cuda")
    none[tokens[tokens != IGNORE]] = False
    assert not got[none].any()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("into", ["same", "f32"])
@pytest.mark.parametrize("t,d,v", [(1, 9, 5), (300, 130, 77), (2000, 130, 77), (9000, 65, 1234)])
def test_gradient_added_to_one_that_exists(ctx, tune, dtype, into, t, d, v):
    """A tied head's gradient: rows without tokens keep their bits."""
    kind = dtype if into == "same" else torch.float32
    tokens = make_tokens(3, t, v, "frequent")
    tokens[::7] = IGNORE
    dy, old = normal(5, t, d, std=0.1, dtype=dtype), normal(6, v, d, std=0.5, dtype=kind)
    buf = torch.cat([old, normal(7, v, 3, dtype=kind)], 1)
    got = tune.embed_backward(ctx, dy, tokens, v, 0.75, into=buf[:, :d])
    assert got.data_ptr() == buf.data_ptr()
    want, bound = table_gradient(dy, tokens, v, 0.75)
    check(got, want + old.double(), bound + U32 * (want.abs() + old.double().abs()), kind)
    assert torch.equal(buf[:, d:], normal(7, v, 3, dtype=kind))
    none = torch.ones(v, dtype=torch.bool, device="cuda")
    none[tokens[tokens != IGNORE]] = False
    assert torch.equal(got[none], old[none])


@pytest.mark.parametrize("t", [0, 5, 600, 9000])
def test_gradient_without_tokens(ctx, tune, t):
    dy, tokens = normal(1, t, 40, dtype=torch.bfloat16), torch.full((t,), IGNORE, device="cuda")
    dy[:] = float("nan")
    assert not tune.embed_backward(ctx, dy, tokens, 100).any()
    old = normal(2, 100, 40)
    assert torch.equal(tune.embed_backward(ctx, dy, tokens, 100, into=old.clone()), old)


@pytest.mark.parametrize("t", [3, 600, 9000])
@pytest.mark.parametrize("wrong", [-1, 50, 1 << 40])
@pytest.mark.parametrize("add", [False, True])
def test_gradient_of_wrong_ids_is_nan(ctx, tune, t, wrong, add):
    dy, tokens = normal(1, t, 72, dtype=torch.bfloat16), make_tokens(2, t, 50, "any")
    tokens[t // 2] = wrong
    into = torch.zeros(50, 72, device="cuda") if add else None
    assert tune.embed_backward(ctx, dy, tokens, 50, into=into).isnan().all()


@pytest.mark.parametrize("t", [100, 700, 9000])
def test_gradient_keeps_to_its_rows(ctx, tune, t):
    """NaN and infinities of a token's dy reach its own row alone, an ignored token's nothing."""
    v, d = 40, 24
    tokens = make_tokens(1, t, v, "any")
    dy = normal(2, t, d, dtype=torch.bfloat16)
    dy[10], dy[20, 3], dy[30] = float("nan"), float("inf"), float("nan")
    tokens[10], tokens[20], tokens[30] = 5, 6, IGNORE
    got = tune.embed_backward(ctx, dy, tokens, v)
    clean = dy.clone()
    clean[10], clean[20, 3], clean[30] = 0, 0, 0
    want = tune.embed_backward(ctx, clean, tokens, v)
    assert got[5].isnan().all() and got[6, 3] == float("inf")
    got[5], got[6, 3] = want[5], want[6, 3]
    assert torch.equal(got, want)


@pytest.mark.parametrize("t", [300, 3000, 20000])
def test_gradient_is_the_same_every_time(ctx, tune, t):
    tokens, dy = make_tokens(1, t, 500, "frequent"), normal(2, t, 264, dtype=torch.float16)
    first = tune.embed_backward(ctx, dy, tokens, 500)
    for _ in range(5):
        assert torch.equal(tune.embed_backward(ctx, dy, tokens, 500), first)


@pytest.mark.parametrize("t", [100, 2000, 9000])
@pytest.mark.parametrize("offset,ld", [(0, 48), (1, 41), (5, 43)])
def test_gradient_of_strided_rows(ctx, tune, t, offset, ld):
    d, v = 40, 60
    buf = normal(1, t * ld + offset, dtype=torch.bfloat16)
    dy, tokens = buf[offset:].view(t, ld)[:, :d], make_tokens(2, t, v, "frequent")
    assert torch.equal(tune.embed_backward(ctx, dy, tokens, v), tune.embed_backward(ctx, dy.contiguous(), tokens, v))


def test_gradient_of_many_ids(ctx, tune):
    """Vocabularies whose ids take one, two and three passes of the sort."""
    for v in (300, 1 << 18, (1 << 24)):
        t, d = 10000, 8
        tokens, dy = make_tokens(v % 97, t, v, "any"), normal(2, t, d, dtype=torch.bfloat16)
        tokens[0], tokens[1] = 0, v - 1
        got = tune.embed_backward(ctx, dy, tokens, v)
        want, bound = table_gradient(dy, tokens, v, 1.0)
        check(got, want, bound, torch.bfloat16)


def test_gradient_against_differences(ctx, tune):
    """d / dE of sum(y * c) by steps that bfloat16 holds exactly."""
    t, d, v = 50, 16, 12
    table = (torch.randint(-8, 9, (v, d), generator=rng(1), device="cuda") / 8).to(torch.bfloat16)
    tokens, c = make_tokens(2, t, v, "any"), torch.randint(-4, 5, (t, d), generator=rng(3), device="cuda").float()
    de = tune.embed_backward(ctx, c.to(torch.bfloat16), tokens, v, 2.0)

    def objective(e):
        return (tune.embed(ctx, e, tokens, 2.0).double() * c.double()).sum().item()

    for r, k in ((0, 0), (3, 7), (v - 1, d - 1)):
        up, down = table.clone(), table.clone()
        up[r, k] += 0.5
        down[r, k] -= 0.5
        assert objective(up) - objective(down) == de[r, k].item()


def test_differentiable(ctx, tune):
    t, d, v = 100, 64, 30
    table = normal(1, v, d, dtype=torch.float16).requires_grad_()
    tokens, dy = make_tokens(2, t, v, "any"), normal(3, t, d, dtype=torch.float16)
    y = tune.embedding(ctx, table, tokens, 3.0)
    y.backward(dy.t().contiguous().t())
    assert torch.equal(y.detach(), tune.embed(ctx, table.detach(), tokens, 3.0))
    assert torch.equal(table.grad, tune.embed_backward(ctx, dy, tokens, v, 3.0))


# ---------------------------------------------------------------- streams, graphs, refusals
@pytest.mark.parametrize("t", [200, 3000, 10000])
def test_captured_and_replayed(ctx, tune, t):
    d, v = 136, 700
    table, dy, tokens = normal(1, v, d, dtype=torch.bfloat16), normal(2, t, d, dtype=torch.bfloat16), make_tokens(3, t, v, "any")
    tune.embed_backward(ctx, dy, tokens, v)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        tune.embed_backward(ctx, dy, tokens, v, into=None)
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y, de = tune.embed(ctx, table, tokens), tune.embed_backward(ctx, dy, tokens, v)
    for i in range(4):
        tokens.copy_(make_tokens(10 + i, t, v, "frequent"))
        dy.copy_(normal(20 + i, t, d, dtype=torch.bfloat16))
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, table[tokens])
        assert torch.equal(de, tune.embed_backward(ctx, dy, tokens, v))


def test_a_captured_differentiable_step(ctx, tune):
    """Forward and backward by autograd in one graph; nothing made outside it refers to the table when it is captured."""
    t, d, v = 300, 72, 500
    start, dy, tokens = normal(1, v, d, dtype=torch.bfloat16), normal(2, t, d, dtype=torch.bfloat16), make_tokens(3, t, v, "any")
    table = start.clone().requires_grad_()

    def step():
        y = tune.embedding(ctx, table, tokens, 2.0)
        return y.detach(), torch.autograd.grad(y, table, dy)[0]

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y, de = step()
    for i in range(4):
        tokens.copy_(make_tokens(10 + i, t, v, "any"))
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, tune.embed(ctx, start, tokens, 2.0))
        assert torch.equal(de, tune.embed_backward(ctx, dy, tokens, v, 2.0))


def test_two_streams_at_once(ctx, tune):
    v, d, streams = 900, 256, [torch.cuda.Stream() for _ in range(2)]
    jobs = [(make_tokens(i, t, v, "frequent"), normal(i, t, d, dtype=torch.bfloat16)) for i, t in enumerate((9000, 1500))]
    want = [tune.embed_backward(ctx, dy, tok, v) for tok, dy in jobs]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(tune.embed_backward(ctx, jobs[i][1], jobs[i][0], v))
    torch.cuda.synchronize()
    for g, w in zip(got, want):
        assert all(torch.equal(x, w) for x in g)


def test_refusals(ctx, tune):
    b = torch.bfloat16
    table, tok = normal(1, 10, 16, dtype=b), torch.zeros(4, dtype=torch.int64, device="cuda")
    dy = normal(2, 4, 16, dtype=b)
    for e, f in [(TypeError, lambda: tune.embed(ctx, table.float(), tok)),
                 (TypeError, lambda: tune.embed(ctx, table, tok.int())),
                 (ValueError, lambda: tune.embed(ctx, table, tok.view(2, 2))),
                 (ValueError, lambda: tune.embed(ctx, table, tok.cpu())),
                 (ValueError, lambda: tune.embed(ctx, table.t(), tok)),
                 (ValueError, lambda: tune.embed(ctx, table.cpu(), tok)),
                 (cdclq.CdclqError, lambda: tune.embed(ctx, table[:0], tok)),
                 (cdclq.CdclqError, lambda: tune.embed(ctx, table[:, :0], tok)),
                 (TypeError, lambda: tune.embed_backward(ctx, dy.float(), tok, 10)),
                 (ValueError, lambda: tune.embed_backward(ctx, dy, tok[:3], 10)),
                 (cdclq.CdclqError, lambda: tune.embed_backward(ctx, dy, tok, 0)),
                 (cdclq.CdclqError, lambda: tune.embed_backward(ctx, dy[:, :0], tok, 10)),
                 (TypeError, lambda: tune.embed_backward(ctx, dy, tok, 10, into=table.half())),
                 (ValueError, lambda: tune.embed_backward(ctx, dy, tok, 10, into=table[:9])),
                 (cdclq.CdclqError, lambda: tune.embed_backward(ctx, dy, tok, 4, into=dy))]:
        with pytest.raises(e):
            f()
    L = cdclq.lib()
    big = torch.empty(1000, 8, dtype=b, device="cuda")
    ids = torch.zeros(1000, dtype=torch.int64, device="cuda")
    rc = L.cdclq_embed_backward_device(ctx.ptr, big.data_ptr(), 8, 1000, 8, 10, cdclq.DTYPE_BF16, ids.data_ptr(), 1.0, -100, 0,
                                       table.data_ptr(), 16, cdclq.DTYPE_BF16, 0, 0, 0)
    assert rc == cdclq.INVALID_ARG and b"workspace" in L.cdclq_last_error(ctx.ptr)
    rc = L.cdclq_embed_device(ctx.ptr, table.data_ptr(), 16, 10, 16, cdclq.DTYPE_BF16, tok.data_ptr(), 4, 1.0, -100,
                              table.data_ptr(), 16, 0)
    assert rc == cdclq.INVALID_ARG and b"overlaps" in L.cdclq_last_error(ctx.ptr)
