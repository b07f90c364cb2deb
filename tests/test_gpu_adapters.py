"""GPU tests of the packed projection with low-rank adapters and its gradient (cdclq.tune), against the
definition in 64 bits.

Tolerances: u is the unit roundoff of the 16-bit type (2^-8 for bfloat16, 2^-11 for float16), f32 2^-24.
A sum of k exact products in f32 is off by at most k 2^-24 sum |.|. Up to 64 tokens the weights are exact
(2^b + code, of at most 34 times the size of code - zero, and sum x are summed instead); beyond, each
weight is rounded to 16 bits (u); from 65 to 192 tokens the first form runs under the second's bound. The
low-rank vectors lose at most 2^-15 of their largest element."""
import numpy as np
import pytest
import torch

import cdclq

pytestmark = pytest.mark.gpu

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


def rng(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def normal(seed, *shape, std=1.0, dtype=torch.float32):
    return (torch.randn(*shape, generator=rng(seed), device="cuda") * std).to(dtype)


def make_layer(ctx, tune, seed, m, n, bits, group, lead=0):
    """A packed layer of random codes through the framework's own packing, and its weights in 64 bits."""
    r = np.random.default_rng(seed)
    g = n if group == 0 or group >= n else group
    ng = -(-n // g)
    gbits = np.array([8 if i < lead else bits for i in range(ng)], np.uint8)
    wid = gbits[np.arange(n) // g].astype(int)
    codes = r.integers(0, 1 << wid, (m, n)).astype(np.uint8)
    zeros = r.integers(0, (1 << gbits.astype(int)), (m, ng)).astype(np.float32)
    scales = (r.uniform(0.5, 1.5, (m, ng)) / (1 << gbits.astype(int)) / n ** 0.5).astype(np.float16).astype(np.float32)
    ql = cdclq.QLayer(m, n, g, r.permutation(n).astype(np.uint32), gbits, codes, scales, zeros)
    packed = tune.PackedLinear.from_tensors(ctx, cdclq.packed_tensors("l", ql, ctx), "l")
    gi = np.arange(n) // g
    w = np.zeros((m, n))
    w[:, ql.perm.astype(int)] = scales.astype(np.float64)[:, gi] * (codes - zeros.astype(np.float64)[:, gi])
    big = np.zeros((m, n))  # what the exact operands 2^b + code and the offset weigh, with their scale
    big[:, ql.perm.astype(int)] = scales.astype(np.float64)[:, gi] * (2.0 * (1 << wid) + 272 + zeros[:, gi])
    return packed, torch.from_numpy(w).cuda(), torch.from_numpy(big).cuda()


def make_adapters(tune, seed, r, k, m, n, dtype):
    a, b = normal(seed, r, k, n, std=n ** -0.5, dtype=dtype), normal(seed + 1, r, m, k, std=k ** -0.5, dtype=dtype)
    return tune.Adapters(a, b, torch.rand(r, generator=rng(seed + 2), device="cuda") + 0.5)


def make_request(seed, t, r, order):
    q = torch.randint(-1, r, (t,), generator=rng(seed), device="cuda").int()
    return torch.sort(q).values if order == "sorted" else q


def reference(w, ad, x, q, dy=None, kept=None):
    """y, low (and dx, da, db) in 64 bits, and the magnitudes sum |.| that the tolerances need."""
    x = x.double()
    n, m, dev = w.shape[1], w.shape[0], w.device
    r, k = (ad.count, ad.rank) if ad else (0, 0)
    out = {"y": x @ w.T, "low": torch.zeros(len(x), k, dtype=torch.float64, device=dev)}
    size = {"y": x.abs() @ w.abs().T, "ylow": torch.zeros_like(out["y"]), "low": torch.zeros_like(out["low"])}
    if dy is not None:
        dy = dy.double()
        out |= {"dx": dy @ w, "da": torch.zeros(r, k, n, dtype=torch.float64, device=dev),
                "db": torch.zeros(r, m, k, dtype=torch.float64, device=dev)}
        size |= {"dx": dy.abs() @ w.abs(), "dxlow": torch.zeros_like(out["dx"]), "da": out["da"].clone(),
                 "db": out["db"].clone()}
    for i in range(r):
        s = (q == i).nonzero().flatten()
        a, b, c = ad.a[i].double(), ad.b[i].double(), ad.scaling[i].double()
        out["low"][s] = x[s] @ a.T
        size["low"][s] = x[s].abs() @ a.abs().T
        out["y"][s] += c * out["low"][s] @ b.T
        # a low-rank vector's error goes by its largest element
        size["ylow"][s] = c * size["low"][s] @ b.abs().T + c * out["low"][s].abs().amax(1, True) * b.abs().sum(1)
        if dy is not None:
            up = c * dy[s] @ b
            upsize = c * dy[s].abs() @ b.abs()
            out["dx"][s] += up @ a
            size["dxlow"][s] = upsize @ a.abs() + up.abs().amax(1, True) * a.abs().sum(0) if len(s) else 0
            out["da"][i], size["da"][i] = up.T @ kept[s], upsize.T @ kept[s].abs()
            out["db"][i] = c * dy[s].T @ out["low"][s]
            size["db"][i] = c * dy[s].abs().T @ size["low"][s]
    return out, size


def near(got, want, tol, what):
    bad = (got.double() - want).abs() > tol
    assert got.shape == want.shape and torch.isfinite(got).all(), what
    assert not bad.any(), (what, ((got.double() - want).abs() / tol.clamp(min=1e-300)).max().item())


def check_forward(packed, w, big, ad, x, q, tune):
    y, low = tune.adapter_linear(packed, x, ad, q, return_low=True)
    out, size = reference(w, ad, x, q)
    u, n, t = U[x.dtype], w.shape[1], len(x)
    tiny = 2.0 ** -25 if x.dtype == torch.float16 else 0.0
    base = size["y"] * (u + n * U32) if t > 64 else (x.double().abs() @ big.T) * (n + 8) * U32
    k = low.shape[1]
    # low: n products in f32; then 2^-15 of its largest element and k products
    lowtol = size["ylow"] * (n * U32 + 2.0 ** -15 + k * U32) if k else 0
    near(low, out["low"], size["low"] * n * U32 + 1e-30, "low")
    near(y, out["y"], 1.01 * u * out["y"].abs() + base + lowtol + tiny, "y")
    return y, low


SHAPES = [(1, 1), (16, 32), (17, 100), (128, 128), (130, 257), (1001, 1350), (512, 2048)]


@pytest.mark.parametrize("bits,group", [(2, 64), (3, 128), (4, 128), (8, 32), (5, 48), (1, 17), (6, 0), (7, 128)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_widths_and_groups(ctx, tune, dtype, bits, group):
    m, n = 203, 393
    packed, w, big = make_layer(ctx, tune, bits * 100 + group, m, n, bits, group)
    ad = make_adapters(tune, 5, 3, 8, m, n, dtype)
    for t in (1, 20, 50, 70, 150):
        x = normal(t, t, n, dtype=dtype)
        check_forward(packed, w, big, ad, x, make_request(t, t, 3, "any"), tune)


@pytest.mark.parametrize("m,n", SHAPES)
def test_shapes_and_token_counts(ctx, tune, m, n):
    packed, w, big = make_layer(ctx, tune, m + n, m, n, 4, 128)
    ad = make_adapters(tune, 7, 2, 16, m, n, torch.bfloat16)
    for t in (1, 2, 16, 17, 32, 33, 64, 65, 129, 300):
        x = normal(t + 1, t, n, dtype=torch.bfloat16)
        check_forward(packed, w, big, ad, x, make_request(t, t, 2, "any"), tune)


@pytest.mark.parametrize("lead", [1, 2, 3])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_mixed_widths(ctx, tune, dtype, lead):
    """Leading 8-bit groups that share blocks of 128 slots with narrow ones, and a group over blocks."""
    for bits, group, n in ((2, 64, 520), (3, 200, 900), (4, 32, 333)):
        packed, w, big = make_layer(ctx, tune, 31 + group, 65, n, bits, group, lead)
        ad = make_adapters(tune, 9, 2, 4, 65, n, dtype)
        for t in (1, 40, 80):
            check_forward(packed, w, big, ad, normal(t, t, n, dtype=dtype), make_request(3, t, 2, "any"), tune)


@pytest.mark.parametrize("rank", [1, 7, 8, 16, 20, 33, 64, 100, 128])
def test_ranks(ctx, tune, rank):
    m, n = 150, 264
    packed, w, big = make_layer(ctx, tune, 77, m, n, 4, 64)
    ad = make_adapters(tune, rank, 5, rank, m, n, torch.bfloat16)
    for t in (3, 70):
        check_forward(packed, w, big, ad, normal(t, t, n, dtype=torch.bfloat16), make_request(2, t, 5, "any"), tune)


def test_many_rows_take_two_tiles_a_wavefront(ctx, tune):
    packed, w, big = make_layer(ctx, tune, 3, 16400, 128, 4, 128)
    x = normal(1, 33, 128, dtype=torch.bfloat16)
    check_forward(packed, w, big, make_adapters(tune, 4, 2, 4, 16400, 128, torch.bfloat16), x,
                  make_request(1, 33, 2, "any"), tune)


def saved_values(ck):
    n = ck.codes.shape[1]
    return ck.codes.double() * ck.scales.double().repeat_interleave(128, 1)[:, :n]


def check_backward(packed, w, ad, x, q, dy, tune, ctx):
    y, low = tune.adapter_linear(packed, x, ad, q, return_low=True)
    ck = tune.checkpoint_save(ctx, x)
    dx, da, db = tune.adapter_linear_backward(packed, dy, ck, low, ad, q)
    out, size = reference(w, ad, x, q, dy, saved_values(ck))
    u, (m, n), t, k = U[x.dtype], w.shape, len(x), ad.rank
    tiny = 2.0 ** -25 if x.dtype == torch.float16 else 0.0
    near(dx, out["dx"], 1.01 * u * out["dx"].abs() + size["dx"] * (u + m * U32) +
         size["dxlow"] * (m * U32 + 2.0 ** -15 + k * U32) + tiny, "dx")
    # u and low enter as two 16-bit values, 2^-15 of the element
    near(da, out["da"], 1.01 * u * out["da"].abs() + size["da"] * (m * U32 + 2.0 ** -15 + t * U32) + tiny, "da")
    near(db, out["db"], 1.01 * u * out["db"].abs() + size["db"] * (n * U32 + 2.0 ** -15 + t * U32) +
         tiny * (1 + dy.double().abs().sum(0).max().item()), "db")
    return dx, da, db


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("t,m,n,bits,group,r,rank,order",
                         [(1, 64, 128, 4, 128, 1, 8, "any"), (40, 130, 257, 3, 48, 3, 5, "any"),
                          (100, 201, 1350, 4, 128, 4, 16, "any"), (300, 512, 512, 2, 64, 2, 64, "sorted"),
                          (700, 96, 264, 4, 32, 7, 33, "any"), (1300, 128, 256, 8, 128, 1, 128, "sorted"),
                          (65, 1001, 72, 5, 0, 40, 3, "any"),
                          # long sums: the low-rank vectors by tiles of 128 tokens of one adapter
                          (1300, 96, 8192, 4, 128, 3, 128, "any"), (1301, 8200, 100, 4, 128, 5, 120, "any"),
                          (2100, 72, 9000, 3, 128, 2, 60, "sorted")])
def test_gradient(ctx, tune, dtype, t, m, n, bits, group, r, rank, order):
    packed, w, _ = make_layer(ctx, tune, t + m, m, n, bits, group)
    ad = make_adapters(tune, 3, r, rank, m, n, dtype)
    q = make_request(t, t, r, order)
    check_backward(packed, w, ad, normal(1, t, n, dtype=dtype), q, normal(2, t, m, dtype=dtype), tune, ctx)


@pytest.mark.parametrize("size,factor", [(1e-4, 1), (1e4, 16)])
def test_half_precision_gradient_of_small_and_large_low_rank_vectors(ctx, tune, size, factor):
    """low beyond float16's range on both sides (up to 1e6, down to 1e-7): B's gradient keeps its precision
    where its own values are in range."""
    t, m, n, rank = 700, 96, 256, 16
    packed, w, _ = make_layer(ctx, tune, 4, m, n, 4, 64)
    ad = make_adapters(tune, 3, 2, rank, m, n, torch.float16)
    ad.a.mul_(factor)
    x = normal(1, t, n, std=size, dtype=torch.float16)
    x[300:] *= 2.0 ** -6
    assert torch.isfinite(x).all()
    check_backward(packed, w, ad, x, make_request(t, t, 2, "any"), normal(2, t, m, std=1e-3, dtype=torch.float16), tune, ctx)


def test_no_adapters_unused_adapters_and_no_tokens(ctx, tune):
    packed, w, big = make_layer(ctx, tune, 12, 90, 200, 4, 128)
    b = torch.bfloat16
    for t in (5, 100):
        x, dy = normal(1, t, 200, dtype=b), normal(2, t, 90, dtype=b)
        y = tune.adapter_linear(packed, x)
        dx, da, db = tune.adapter_linear_backward(packed, dy)
        assert da is None and db is None
        ad = make_adapters(tune, 1, 3, 8, 90, 200, b)
        none = torch.full((t,), -1, dtype=torch.int32, device="cuda")
        y2, low = tune.adapter_linear(packed, x, ad, none, return_low=True)
        assert torch.equal(y, y2) and not low.any()
        dx2, da, db = tune.adapter_linear_backward(packed, dy, tune.checkpoint_save(ctx, x), low, ad, none)
        assert torch.equal(dx, dx2) and not da.any() and not db.any()
    x = x[:0]
    y, low = tune.adapter_linear(packed, x, ad, none[:0], return_low=True)
    assert y.shape == (0, 90)
    dx, da, db = tune.adapter_linear_backward(packed, dy[:0], tune.checkpoint_save(ctx, x), low, ad, none[:0])
    assert dx.shape == (0, 200) and not da.any() and not db.any()


@pytest.mark.parametrize("t", [40, 200])
def test_tokens_and_adapters_stay_apart(ctx, tune, t):
    """NaN and infinities of one token, or of one adapter's weights, change no bit of the others; a
    request outside the adapters gives a NaN row."""
    m, n, b = 100, 256, torch.bfloat16
    packed, _, _ = make_layer(ctx, tune, 8, m, n, 4, 128)
    ad = make_adapters(tune, 2, 3, 16, m, n, b)
    q = make_request(4, t, 3, "any")
    x, dy = normal(1, t, n, dtype=b), normal(2, t, m, dtype=b)

    def step(x, ad, q):
        y, low = tune.adapter_linear(packed, x, ad, q, return_low=True)
        return (y,) + tune.adapter_linear_backward(packed, dy, tune.checkpoint_save(ctx, x), low, ad, q)

    y, dx, da, db = step(x, ad, q)
    x2 = x.clone()
    bad = (q == 1).nonzero()[0, 0]
    x2[bad, 3], x2[bad, 200] = float("nan"), float("inf")
    y2, dx2, da2, db2 = step(x2, ad, q)
    keep = torch.arange(t, device="cuda") != bad
    assert torch.equal(y[keep], y2[keep]) and torch.equal(dx, dx2) and not torch.isfinite(y2[bad]).any()
    for i in (0, 2):
        assert torch.equal(da[i], da2[i]) and torch.equal(db[i], db2[i])
    assert torch.isnan(da2[1]).any() and not torch.isfinite(db2[1]).all()
    sick = tune.Adapters(ad.a.clone(), ad.b.clone(), ad.scaling)
    sick.a[2], sick.b[2] = float("nan"), float("inf")
    y3, dx3, da3, db3 = step(x, sick, q)
    other = q != 2
    assert torch.equal(y[other], y3[other]) and torch.equal(dx[other], dx3[other])
    for i in (0, 1):
        assert torch.equal(da[i], da3[i]) and torch.equal(db[i], db3[i])
    q4 = q.clone()
    q4[0], q4[1] = 3, -2
    y4, low4 = tune.adapter_linear(packed, x, ad, q4, return_low=True)
    assert torch.isnan(y4[:2]).all() and torch.equal(y4[2:], y[2:])
    dx4, _, _ = tune.adapter_linear_backward(packed, dy, tune.checkpoint_save(ctx, x), low4, ad, q4)
    assert torch.isnan(dx4[:2]).all() and torch.equal(dx4[2:], dx[2:])


def test_order_of_requests_changes_no_token(ctx, tune):
    m, n, b = 300, 384, torch.bfloat16
    packed, _, _ = make_layer(ctx, tune, 6, m, n, 3, 128)
    ad = make_adapters(tune, 2, 9, 16, m, n, b)
    for t in (50, 333):
        q, x = make_request(4, t, 9, "any"), normal(1, t, n, dtype=b)
        y = tune.adapter_linear(packed, x, ad, q)
        p = torch.randperm(t, generator=rng(1), device="cuda")
        assert torch.equal(tune.adapter_linear(packed, x[p].contiguous(), ad, q[p].contiguous()), y[p])


@pytest.mark.parametrize("bits,group", [(2, 64), (3, 128), (4, 128), (8, 32), (5, 48), (1, 17), (6, 0), (7, 128)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_expanded_widths_and_groups(ctx, tune, dtype, bits, group):
    m, n = 203, 393
    for lead in (0, 2):
        packed, w, big = make_layer(ctx, tune, bits * 100 + group, m, n, bits, group, lead if group else 0)
        ad = make_adapters(tune, 5, 3, 8, m, n, dtype)
        x = normal(4, 210, n, dtype=dtype)
        check_forward(packed, w, big, ad, x, make_request(3, 210, 3, "sorted"), tune)


@pytest.mark.parametrize("rank", [1, 7, 16, 17, 33, 64, 100, 128])
@pytest.mark.parametrize("order", ["any", "sorted"])
def test_expanded_ranks(ctx, tune, rank, order):
    m, n, t = 290, 512, 1100
    packed, w, big = make_layer(ctx, tune, rank, m, n, 4, 128)
    for dtype in (torch.bfloat16, torch.float16):
        ad = make_adapters(tune, rank, 4, rank, m, n, dtype)
        check_forward(packed, w, big, ad, normal(2, t, n, dtype=dtype), make_request(t, t, 4, order), tune)


@pytest.mark.parametrize("t", [127, 128, 129, 191, 192, 193])
@pytest.mark.parametrize("rank", [4, 64, 128])
def test_token_counts_where_the_form_changes(ctx, tune, t, rank):
    m, n, b = 150, 264, torch.bfloat16
    packed, w, big = make_layer(ctx, tune, t, m, n, 4, 128)
    ad = make_adapters(tune, 3, 3, rank, m, n, b)
    x, q = normal(1, t, n, dtype=b), make_request(t, t, 3, "any")
    check_forward(packed, w, big, ad, x, q, tune)
    check_backward(packed, w, ad, x, q, normal(2, t, m, dtype=b), tune, ctx)


@pytest.mark.parametrize("t", [130, 700])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_neighbours_change_no_token(ctx, tune, dtype, t):
    """The same tokens of one adapter alone, with tokens of no adapter among them, with tokens of other
    adapters, and with an adapter whose weights are not finite: the same bits."""
    m, n = 300, 384
    packed, _, _ = make_layer(ctx, tune, 6, m, n, 3, 128)
    ad = make_adapters(tune, 2, 3, 40, m, n, dtype)
    x = normal(1, t, n, dtype=dtype)
    x[::7] *= 2.0 ** -9  # several exponents of the low-rank vectors
    one = torch.zeros(t, dtype=torch.int32, device="cuda")
    some, mixed = one.clone(), one.clone()
    some[1::3], mixed[2::5] = -1, 1
    y0, y1, y2 = (tune.adapter_linear(packed, x, ad, q) for q in (one, some, mixed))
    assert torch.equal(y0[some == 0], y1[some == 0]) and torch.equal(y0[mixed == 0], y2[mixed == 0])
    bare = tune.adapter_linear(packed, x, ad, torch.full_like(one, -1))
    assert torch.equal(y1[some == -1], bare[some == -1])
    sick = tune.Adapters(ad.a, ad.b.clone(), ad.scaling)
    sick.b[0, 5], sick.b[0, 290] = float("inf"), float("nan")
    y3 = tune.adapter_linear(packed, x, sick, some)
    assert torch.equal(y3[some == -1], y1[some == -1])
    fine = torch.ones(m, dtype=torch.bool, device="cuda")
    fine[5] = fine[290] = False
    assert torch.equal(y3[some == 0][:, fine], y1[some == 0][:, fine])
    assert not torch.isfinite(y3[some == 0][:, ~fine]).any()


def test_strides_and_alignment(ctx, tune):
    m, n, b = 100, 256, torch.bfloat16
    packed, _, _ = make_layer(ctx, tune, 8, m, n, 4, 128)
    ad = make_adapters(tune, 2, 2, 8, m, n, b)
    flat = torch.empty(ad.a.numel() + 1, dtype=b, device="cuda")
    odd = tune.Adapters(flat[1:].view_as(ad.a).copy_(ad.a), ad.b, ad.scaling)
    big, up = normal(1, 400, 300, dtype=b), normal(2, 400, 120, dtype=b)
    for t in (30, 90):
        q = make_request(4, t, 2, "any")
        for x, dy in ((big[:t, :256], up[:t, :100]), (big[: 2 * t : 2, 1:257], up[: 2 * t : 2, 3:103]), (big[5 : t + 5, 7:263], up[1 : t + 1, 20:])):
            y, low = tune.adapter_linear(packed, x, ad, q, return_low=True)
            xc, dyc = x.contiguous(), dy.contiguous()
            y2, low2 = tune.adapter_linear(packed, xc, ad, q, return_low=True)
            # the few-token sums of low take another order where rows are not aligned
            assert torch.equal(y, y2) if t > 64 else torch.allclose(y.float(), y2.float(), rtol=2.0 ** -7, atol=1e-6)
            ck = tune.checkpoint_save(ctx, xc)
            for a, c in zip(tune.adapter_linear_backward(packed, dy, ck, low2, ad, q),
                            tune.adapter_linear_backward(packed, dyc, ck, low2, ad, q)):
                assert torch.equal(a, c)
            yo = tune.adapter_linear(packed, xc, odd, q)
            assert torch.equal(yo, y2) if t > 64 else torch.allclose(yo.float(), y2.float(), rtol=2.0 ** -7, atol=1e-6)


def test_gradient_against_differences(ctx, tune):
    """y is linear in x, in A and in B: differences of the kernel's y along steps that the type holds
    exactly, contracted with dy, against its gradients. Exact but for the outputs' roundings."""
    t, m, n, r, k, b = 80, 48, 64, 2, 4, torch.bfloat16
    packed, w, _ = make_layer(ctx, tune, 8, m, n, 4, 32)
    g = rng(3)
    grid = lambda *s: (torch.randint(-8, 9, s, generator=g, device="cuda") / 8).to(b)  # noqa: E731
    x, dy = grid(t, n), grid(t, m)
    ad = tune.Adapters(grid(r, k, n), grid(r, m, k), torch.rand(r, generator=g, device="cuda") + 0.5)
    q = make_request(1, t, r, "any")
    y, low = tune.adapter_linear(packed, x, ad, q, return_low=True)
    ck = tune.checkpoint_save(ctx, x)
    dx, da, db = tune.adapter_linear_backward(packed, dy, ck, low, ad, q)
    for part, grad in (("x", dx), ("a", da), ("b", db)):
        step = grid(*grad.shape)
        at = lambda s: (x + s * step if part == "x" else x,  # noqa: E731
                        tune.Adapters(ad.a + s * step if part == "a" else ad.a,
                                      ad.b + s * step if part == "b" else ad.b, ad.scaling))
        ys = [tune.adapter_linear(packed, *at(s), q).double() for s in (1, -1)]
        slope = ((ys[0] - ys[1]) / 2 * dy.double()).sum()
        inner = (grad.double() * step.double()).sum()
        # roundings of both y and of the weights; of the gradient and its operands; x in 8 bits (half a
        # step of 1 / 127 of the block's maximum, 1) for A
        tol = sum((yy.abs() * dy.double().abs()).sum() * 2 * U[b] for yy in ys)
        xx, _ = at(1)
        tol += ((xx.double().abs() @ w.abs().T) * dy.double().abs()).sum() * 2 * U[b]
        tol += (grad.double() * step.double()).abs().sum() * 4 * U[b]
        tol += (dy.double().abs() @ w.abs() * step.double().abs()).sum() * 2 * U[b] if part == "x" else 0
        if part == "a":
            up = (dy.double().abs()[:, None, :] @ ad.b.double().abs()[q.clamp(min=0).long()])[:, 0] * 1.5
            tol += (up[:, :, None] * step.double().abs()[q.clamp(min=0).long()]).sum() / 254
        assert (slope - inner).abs() <= tol, part


def test_repeats_bit_for_bit_on_streams_and_in_a_graph(ctx, tune):
    m, n, b = 200, 384, torch.bfloat16
    packed, _, _ = make_layer(ctx, tune, 6, m, n, 4, 128)
    ad = make_adapters(tune, 2, 3, 16, m, n, b)
    for t in (20, 150):
        def step(x, dy, q):
            y, low = tune.adapter_linear(packed, x, ad, q, return_low=True)
            ck = tune.checkpoint_save(ctx, x)
            return (y,) + tune.adapter_linear_backward(packed, dy, ck, low, ad, q)

        x, dy, q = normal(1, t, n, dtype=b), normal(2, t, m, dtype=b), make_request(3, t, 3, "any")
        first = step(x, dy, q)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            other = step(x, dy, q)
        torch.cuda.current_stream().wait_stream(side)
        for u, v in zip(first, other):
            assert torch.equal(u, v)
        held_in = [z.clone() for z in (x, dy, q)]
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held = step(*held_in)
        for seed in (11, 12, 13):
            new = normal(seed, t, n, dtype=b), normal(seed + 50, t, m, dtype=b), make_request(seed, t, 3, "any")
            for h, z in zip(held_in, new):
                h.copy_(z)
            graph.replay()
            torch.cuda.synchronize()
            for u, v in zip(held, step(*new)):
                assert torch.equal(u, v)


def test_refusals(ctx, tune):
    m, n, b = 32, 64, torch.bfloat16
    packed, _, _ = make_layer(ctx, tune, 6, m, n, 4, 32)
    ad = make_adapters(tune, 2, 2, 4, m, n, b)
    x, q = normal(1, 4, n, dtype=b), make_request(1, 4, 2, "any")
    dy = normal(1, 4, m, dtype=b)
    for bad in (x.float(), x.half()):
        with pytest.raises(TypeError):
            tune.adapter_linear(packed, bad, ad, q)
    for args in ((x[:, :32], ad, q), (x, ad, q[:2]), (x, ad, None), (x, None, q), (x.cpu(), ad, q), (x.t(), ad, q)):
        with pytest.raises(ValueError):
            tune.adapter_linear(packed, *args)
    with pytest.raises(TypeError):
        tune.adapter_linear(packed, x, ad, q.long())
    with pytest.raises(ValueError):
        tune.adapter_linear(packed, x, make_adapters(tune, 2, 2, 4, m, 32, b), q)
    with pytest.raises(ValueError):
        tune.Adapters(ad.a, ad.b[:, :, :2], ad.scaling)
    with pytest.raises(TypeError):
        tune.Adapters(ad.a, ad.b.half(), ad.scaling)
    with pytest.raises(ValueError):
        tune.Adapters(ad.a, ad.b, ad.scaling[:1])
    with pytest.raises(ValueError):
        tune.adapter_linear_backward(packed, dy, None, None, ad, q)
    wide = make_adapters(tune, 2, 1, 129, m, n, b)
    with pytest.raises(cdclq.CdclqError) as e:
        tune.adapter_linear(packed, x, wide, q)
    assert "rank 129" in str(e.value)
    u8 = lambda *s: torch.zeros(*s, dtype=torch.uint8, device="cuda")  # noqa: E731
    s16, perm = torch.ones(m, 2, dtype=torch.float16, device="cuda"), torch.arange(n, dtype=torch.int32, device="cuda")
    ok = dict(qweight=u8(m, 32), scales=s16, qzeros=u8(m, 2), perm=perm, gbits=[4, 4], group=32)
    tune.PackedLinear(ctx, **ok).close()
    for key, value in (("perm", perm.clone().fill_(0)), ("perm", perm + 1), ("qweight", u8(m, 31)), ("gbits", [4, 9]),
                       ("group", 0), ("group", 31), ("qweight", u8(0, 32))):
        args = dict(ok)
        args[key] = value
        if key == "qweight" and len(value) == 0:
            args |= dict(scales=s16[:0], qzeros=u8(0, 2))
        with pytest.raises(cdclq.CdclqError):
            tune.PackedLinear(ctx, **args)
    with pytest.raises(ValueError):
        tune.PackedLinear(ctx, **(ok | dict(scales=s16[:, :1])))
    with pytest.raises(TypeError):
        tune.PackedLinear(ctx, **(ok | dict(perm=perm.long())))
    L = cdclq.lib()
    y = torch.empty(4, m, dtype=b, device="cuda")
    need = L.cdclq_adapter_work_bytes(packed.ptr, x.data_ptr(), n, 4, ad.a.data_ptr(), ad.b.data_ptr(), 2, 4, 0)
    work = torch.empty(need, dtype=torch.uint8, device="cuda")
    args = [ctx.ptr, packed.ptr, x.data_ptr(), n, 4, cdclq.DTYPE_BF16, ad.a.data_ptr(), ad.b.data_ptr(),
            ad.scaling.data_ptr(), 2, 4, q.data_ptr(), y.data_ptr(), m, None, work.data_ptr(), need, None]
    for at, value in ((1, None), (2, None), (3, n - 1), (5, cdclq.DTYPE_F32), (6, None), (8, None), (9, 0), (10, 0),
                      (11, None), (12, None), (13, m - 1), (15, None), (16, need - 1)):
        wrong = list(args)
        wrong[at] = value
        assert L.cdclq_adapter_linear_device(*wrong) == cdclq.INVALID_ARG, at
        assert L.cdclq_last_error(ctx.ptr)
    assert L.cdclq_adapter_linear_device(*args) == cdclq.OK
    torch.cuda.synchronize()
