"""GPU tests of cdclq.tune at the ends of the number range: sums near the largest numbers, weights of very
different sizes. Tolerances as in test_gpu_adapters.py and test_gpu_tune.py."""
import pytest
import torch

import cdclq
from tests.test_gpu_adapters import U, U32, check_backward, make_adapters, make_layer, make_request, near, normal, \
    reference

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
