"""CPU checks of the embedding, clipping and logit entry points: workspace sizes over edge sizes (pure host
arithmetic), null handles, and what the differentiable embedding keeps and refuses (its operators by their formulas)."""
import numpy as np
import pytest
import torch

import cdclq
from cdclq import tune

L = cdclq.lib()
GRAD = tune._GRAD


@pytest.mark.parametrize("d,v", [(1, 1), (8, 510), (64, 511), (1000, 50001), (4096, 128256), (1 << 20, 64), (64, 1 << 24)])
def test_embed_workspace_sizes(d, v):
    for t in (0, 1, 128, 129, 512, 8192, 8193, 100_000, 1 << 22):
        n = L.cdclq_embed_work_bytes(t, d, v)
        assert n % 256 == 0
        assert n == 0 if t <= 128 else n >= 8 * t  # ids and places of the sorted tokens
        # two sets of those, the runs that pass a chunk's end (two rows of float32 for eight tokens, padded to eight
        # columns), the counts of 512 digits for 2048 tokens
        assert n <= 17 * t + (d + 7) // 8 * 8 * (t // 8 + 1) * 8 + 2048 * (t // 2048 + 1) + 4096


def test_sizes_outside_the_limits_ask_for_nothing():
    for t, d, v in ((1 << 23, 64, 100), (4, 0, 100), (4, 64, 0), (4, 1 << 21, 100), (4, 64, 1 << 25)):
        assert L.cdclq_embed_work_bytes(t, d, v) == 0
    g = np.zeros(1, GRAD)
    assert L.cdclq_grad_work_bytes(g.ctypes.data, 1, 0) == 0
    assert L.cdclq_grad_work_bytes(g.ctypes.data, 1, 1 << 16) == 0
    assert L.cdclq_grad_work_bytes(None, 1, 1) == 0
    g["count"] = 1 << 41
    assert L.cdclq_grad_work_bytes(g.ctypes.data, 1, 1) == 0
    g = np.zeros(5, GRAD)  # together
    g["count"] = 1 << 38
    assert L.cdclq_grad_work_bytes(g.ctypes.data, 4, 1) and L.cdclq_grad_work_bytes(g.ctypes.data, 5, 1) == 0


@pytest.mark.parametrize("parts", [1, 8, 32768])
def test_grad_workspace_holds_few_sums(parts):
    """64-bit sums, 4096 or one for each part, and of more than 150 tensors a table and 4 bytes for 4096 elements of a
    part, over any sizes."""
    for counts in ([0], [1] * 150, [1] * 300, [1 << 20, 17, 0, 4096], [1 << 30] * 3, [(1 << 33) + 5, 1]):
        g = np.zeros(len(counts), GRAD)
        g["count"] = np.array(counts, np.uint64) // (1 if parts == 1 else 512) * parts
        n = L.cdclq_grad_work_bytes(g.ctypes.data, len(counts), parts)
        chunks = sum(-(-int(c) // parts // 4096) + 1 for c in g["count"])
        assert n % 256 == 0 and 8 * parts <= n <= 8 * max(4096, parts) + 256 + (len(counts) > 150) * (
            32 * len(counts) + 4 * chunks + 512)


def test_null_handles_are_refused():
    bad = cdclq.INVALID_ARG
    assert L.cdclq_embed_device(None, 0, 8, 4, 8, cdclq.DTYPE_BF16, 0, 1, 1.0, -100, 0, 8, 0) == bad
    assert L.cdclq_embed_backward_device(None, 0, 8, 1, 8, 4, cdclq.DTYPE_BF16, 0, 1.0, -100, 0, 0, 8, cdclq.DTYPE_BF16, 0,
                                         0, 0) == bad
    assert L.cdclq_grad_norm_device(None, 0, 0, 1, 0, 0, 0, 0) == bad
    assert L.cdclq_clip_grads_device(None, 0, 0, 1, 1.0, 0, 0, 0, 0) == bad
    assert L.cdclq_constrain_logits_device(None, 0, 8, 1, 8, cdclq.DTYPE_F32, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0,
                                           8, 0, 0, 0) == bad


# ---------------------------------------------------------------- the differentiable embedding
@pytest.fixture
def formulas(monkeypatch):
    def embed(ctx, table, tokens, scale=1.0, ignore_index=-100):
        on = tokens != ignore_index
        return scale * table[tokens.clamp(min=0)] * on[:, None]

    def backward(ctx, dy, tokens, vocab, scale=1.0, ignore_index=-100, into=None):
        on = tokens != ignore_index
        return torch.zeros(vocab, dy.shape[1]).index_add_(0, tokens[on], scale * dy[on])

    monkeypatch.setattr(tune, "embed", embed)
    monkeypatch.setattr(tune, "embed_backward", backward)


def test_embedding_has_the_formulas_gradient(formulas):
    g = torch.Generator().manual_seed(1)
    table, dy = torch.randn(7, 5, generator=g).requires_grad_(), torch.randn(4, 5, generator=g)
    tokens = torch.tensor([2, -100, 2, 6])
    (got,) = torch.autograd.grad(tune.embedding(None, table, tokens, 1.5), table, dy)
    on = torch.tensor([0, 2, 3])
    (want,) = torch.autograd.grad(1.5 * table[tokens[on]], table, dy[on])
    assert torch.allclose(got, want)


def test_embedding_of_a_frozen_table_keeps_nothing(formulas):
    table = torch.zeros(7, 5)
    assert not tune.embedding(None, table, torch.tensor([1])).requires_grad
    with torch.no_grad():
        assert tune.embedding(None, table.requires_grad_(), torch.tensor([1])).grad_fn is None


def test_second_order_is_refused(formulas):
    table = torch.ones(7, 5).requires_grad_()
    with pytest.raises(RuntimeError, match="first order only"):
        torch.autograd.grad(tune.embedding(None, table, torch.tensor([1, 1])).sum(), table, create_graph=True)


def test_tokens_changed_in_place_are_refused(formulas):
    table, tokens = torch.ones(7, 5).requires_grad_(), torch.tensor([1, 2])
    y = tune.embedding(None, table, tokens)
    tokens.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
