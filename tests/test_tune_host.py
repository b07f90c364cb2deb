"""CPU checks of the adapter, checkpoint and vocabulary loss entry points: workspace sizes over edge
sizes (pure host arithmetic) and the refusals that need no GPU."""
import pytest

import cdclq

L = cdclq.lib()
TOKENS = (0, 1, 2, 15, 16, 17, 63, 64, 65, 511, 512, 2048, 2049, 1 << 22)


@pytest.mark.parametrize("d,v", [(1, 1), (7, 1000), (64, 17), (1350, 50001), (4096, 128256), (1 << 20, 64)])
def test_vocab_workspace_sizes(d, v):
    for w, ldw in ((0, d), (2, d), (0, d + 1)):
        for grad in (0, 1):
            sizes = [L.cdclq_vocab_work_bytes(t, d, v, w, ldw, grad) for t in TOKENS]
            assert all(s > 0 and s % 256 == 0 for s in sizes)
            # the tokens' packed copy is part of it; a padded head too, where its rows need one for many tokens
            assert all(s >= 2 * t * d for s, t in zip(sizes, TOKENS))
            if (w or d % 8 or ldw % 8) and TOKENS[-1] > 64:
                assert sizes[-1] >= 2 * v * d


def test_vocab_workspace_has_no_logits():
    """4096 tokens over 128256 entries: 1 GB of 16-bit logits, of which a piece's gradient takes 256 MB."""
    t, d, v = 4096, 4096, 128256
    assert L.cdclq_vocab_work_bytes(t, d, v, 0, d, 0) < 128 << 20
    assert L.cdclq_vocab_work_bytes(t, d, v, 0, d, 1) < 512 << 20


def test_sizes_outside_the_limits_ask_for_nothing():
    for t, d, v in ((1 << 23, 64, 100), (4, 0, 100), (4, 64, 0), (4, 1 << 21, 100), (4, 64, 1 << 25)):
        assert L.cdclq_vocab_work_bytes(t, d, v, 0, d, 0) == 0
    assert L.cdclq_adapter_work_bytes(None, 0, 64, 4, 0, 0, 1, 4, 0) == 0


def test_null_handles_are_refused():
    assert L.cdclq_checkpoint_save_device(None, 0, 8, 1, 8, cdclq.DTYPE_BF16, 0, 0, 0) == cdclq.INVALID_ARG
    assert L.cdclq_checkpoint_restore_device(None, 0, 0, 1, 8, cdclq.DTYPE_BF16, 0, 8, 0) == cdclq.INVALID_ARG
    assert L.cdclq_packed_open_device(None, 1, 8, 8, 0, 1, 0, 8, 0, 0, 0, None) == cdclq.INVALID_ARG
    L.cdclq_packed_close(None)
    assert L.cdclq_packed_bytes(None) == 0


def test_widths_are_checked_for_any_group_size():
    """d_in + group - 1 passes the end of size_t: the widths were not looked at (-1 of a signed caller)."""
    assert cdclq.row_bytes(10, (1 << 64) - 1, [4]) == cdclq.row_bytes(10, 10, [4]) == 5
    for group in (10, 1 << 40, (1 << 64) - 9, (1 << 64) - 1):
        for gbits in ([9], [0], []):
            with pytest.raises(cdclq.CdclqError):
                cdclq.row_bytes(10, group, gbits)
