"""GPU tests of what cdclq.tune and the container calls beside it take and refuse at the ends of their ranges:
layouts that do not fit their tensors, views of one row, sizes whose launches pass 2^32 work-items."""
import numpy as np
import pytest
import torch

import cdclq
from tests.test_gpu_adapters import make_adapters, make_layer, make_request, normal

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


def test_the_largest_group_is_one_group_of_any_width(ctx):
    """A group of 2^64 - 1 (a signed caller's -1) over layers of one shape and several widths: the tables of one
    are not taken for the next."""
    n, m = 40, 6
    r = np.random.default_rng(1)
    for bits in (4, 8, 3):
        ql = cdclq.QLayer(m, n, n, np.arange(n, dtype=np.uint32), np.array([bits], np.uint8),
                          r.integers(0, 1 << bits, (m, n)).astype(np.uint8), np.ones((m, 1), np.float32),
                          np.zeros((m, 1), np.float32))
        qw, s16, qz, p32 = cdclq.pack_layer(ctx, ql)
        got = cdclq.dequantize_packed(ctx, qw, s16, qz, p32, ql.gbits, (1 << 64) - 1)
        assert np.array_equal(got, ql.codes.astype(np.float32))
        assert np.array_equal(cdclq.dequantize_layer(ctx, cdclq.QLayer(m, n, (1 << 64) - 1, ql.perm, ql.gbits, ql.codes,
                                                                       ql.scales, ql.zeros)), got)


@pytest.mark.parametrize("extra", [1, 8, -1])
def test_rows_of_another_width_are_refused(ctx, tune, extra):
    """qweight rows wider than the layout's (a layout of another layer, rows padded for alignment) are not read
    one into the next."""
    ql = cdclq.QLayer(6, 64, 32, np.arange(64, dtype=np.uint32), np.array([4, 3], np.uint8),
                      np.random.default_rng(1).integers(0, 8, (6, 64)).astype(np.uint8), np.ones((6, 2), np.float32),
                      np.zeros((6, 2), np.float32))
    qw, s16, qz, p32 = cdclq.pack_layer(ctx, ql)
    tune.PackedLinear(ctx, qw, s16, qz, p32, ql.gbits, 32).close()
    wrong = np.zeros((6, qw.shape[1] + extra), np.uint8)
    with pytest.raises(cdclq.CdclqError, match="qweight"):
        tune.PackedLinear(ctx, wrong, s16, qz, p32, ql.gbits, 32)
    with pytest.raises(cdclq.CdclqError, match="qweight"):
        cdclq.dequantize_packed(ctx, wrong, s16, qz, p32, ql.gbits, 32)


def test_views_of_one_row_are_contiguous(ctx, tune):
    """One token's row of larger tensors (its stride is of no meaning): low and a checkpoint of it are taken."""
    m, n, rank = 48, 256, 8
    packed, _, _ = make_layer(ctx, tune, 3, m, n, 4, 128)
    ad = make_adapters(tune, 2, 2, rank, m, n, torch.bfloat16)
    q = torch.ones(1, dtype=torch.int32, device="cuda")
    x, dy = normal(1, 1, n, dtype=torch.bfloat16), normal(2, 1, m, dtype=torch.bfloat16)
    low = tune.adapter_linear(packed, x, ad, q, return_low=True)[1]
    ck = tune.checkpoint_save(ctx, x)
    want = tune.adapter_linear_backward(packed, dy, ck, low, ad, q)

    def row(z):
        out = torch.zeros(1, z.shape[1] + 24, dtype=z.dtype, device="cuda")[:, : z.shape[1]].copy_(z)
        assert out.is_contiguous() and out.stride(0) > out.shape[1]
        return out

    ck2 = tune.Checkpoint(row(ck.codes), row(ck.scales), ck.dtype)
    assert torch.equal(tune.checkpoint_restore(ctx, ck2), tune.checkpoint_restore(ctx, ck))
    for a, b in zip(tune.adapter_linear_backward(packed, dy, ck2, row(low), ad, q), want):
        assert torch.equal(a, b)
    two = torch.zeros(2, n + 8, dtype=torch.int8, device="cuda")[:, :n]
    with pytest.raises(ValueError, match="contiguous"):
        tune.checkpoint_restore(ctx, tune.Checkpoint(two, torch.zeros(2, 2, device="cuda"), torch.bfloat16))


def test_gradient_of_more_adapters_than_work_items_along_x(ctx, tune):
    """32768 adapters of rank 128 on 769 columns: 2^24 and some workgroups of 256 write dA and dB. Three of the
    adapters have a token each; they have to get what a call with those three alone gives, the others zeros."""
    r, rank, m, n, b = 32768, 128, 4, 769, torch.bfloat16
    packed, _, _ = make_layer(ctx, tune, 3, m, n, 4, 128)
    few = make_adapters(tune, 2, 3, rank, m, n, b)
    at = torch.tensor([5, 20000, r - 1], device="cuda")
    a, bb = torch.zeros(r, rank, n, dtype=b, device="cuda"), torch.zeros(r, m, rank, dtype=b, device="cuda")
    a[at], bb[at] = few.a, few.b
    scaling = torch.ones(r, device="cuda")
    scaling[at] = few.scaling
    x, dy = normal(1, 3, n, dtype=b), normal(2, 3, m, dtype=b)
    results = []
    for ad, q in ((tune.Adapters(a, bb, scaling), at.int()), (few, torch.arange(3, dtype=torch.int32, device="cuda"))):
        y, low = tune.adapter_linear(packed, x, ad, q, return_low=True)
        results.append((y,) + tune.adapter_linear_backward(packed, dy, tune.checkpoint_save(ctx, x), low, ad, q))
    (y, dx, da, db), (y3, dx3, da3, db3) = results
    assert torch.equal(y, y3) and torch.equal(dx, dx3)
    assert torch.equal(da[at], da3) and torch.equal(db[at], db3)
    da[at], db[at] = 0, 0
    assert not da.any() and not db.any()
    del a, bb, ad, results, y, dx, da, db
    torch.cuda.empty_cache()


def test_loss_of_more_tiles_than_work_items_along_x(ctx, tune):
    """2^22 tokens over 2^17 entries: 2^23 tiles of 512 threads. The losses of tokens from all over are compared
    with 64 bits (8 products of values up to 8 in f32, and a few ulp of values below 2^5)."""
    t, d, v, b = 1 << 22, 8, 1 << 17, torch.bfloat16
    x, w = normal(1, t, d, dtype=b), normal(2, v, d, dtype=b)
    y = torch.randint(0, v, (t,), generator=torch.Generator(device="cuda").manual_seed(3), device="cuda")
    y[::5] = -100
    loss, lse = tune.vocab_loss(ctx, x, w, y)
    on = y != -100
    assert not loss[~on].any() and not lse[~on].any() and torch.isfinite(loss).all() and (loss[on] > 0).all()
    for rows in torch.arange(1, t, 1999, device="cuda").split(512):
        rows = rows[on[rows]]
        l = x[rows].double() @ w.double().T
        want = torch.logsumexp(l, 1)
        assert (lse[rows].double() - want).abs().max() <= 1e-4
        assert (loss[rows].double() - (want - l.gather(1, y[rows][:, None])[:, 0])).abs().max() <= 1e-4
    del x, w, y, loss, lse, on
    torch.cuda.empty_cache()
