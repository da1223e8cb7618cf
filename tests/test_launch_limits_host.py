"""Calls whose second kernel would pass a launch's 2^32 threads are refused on
the host, before the first kernel is queued (no GPU)."""

import pytest

from minitp import _native as N
from tests.test_beam_host import attention, select


def _most_rows(d):
    """Query rows that the join of partial results takes: d / 4 threads each,
    in whole blocks of 256."""
    return ((1 << 32) - 256) // (d // 4)


@pytest.mark.parametrize("dtype", [N.BF16, N.F32])
@pytest.mark.parametrize("d", [16, 32, 64, 128])
def test_attention_with_a_join_of_too_many_threads(d, dtype):
    """Rows of 65 tokens, one head, on a long prefix: parts of their own, joined
    by a second launch."""
    size = N.lib().minitp_shared_prefix_attention_workspace_bytes
    for b, fits in ((_most_rows(d) // 65 // 4, True), (_most_rows(d) // 65 + 1, False)):
        if b * 65 >= (1 << 31) - 256:
            continue  # (past the bound on query rows)
        shape = dict(b=b, g=1, t=65, hq=1, hkv=1, d=d, p=1500, c=0)
        need = size(dtype, *shape.values())
        if fits:
            assert need > 0
            assert attention(dtype, s=65, **shape, nbytes=need - 1) == N.ERR_ARG  # (refused for its scratch alone)
        else:
            assert need == -1
            assert attention(dtype, s=65, **shape, nbytes=1 << 62) == N.ERR_UNSUPPORTED and "too many" in N.last_error()


def test_rows_of_65_tokens_behind_one_prefix():
    """2^21 of them: 2^27 query rows of 128, a thread of the join for four elements."""
    assert attention(b=1 << 21, g=1, t=65, hq=1, hkv=1, d=128, p=1500, c=0, s=65, nbytes=1 << 62) == N.ERR_UNSUPPORTED


def test_rows_that_one_launch_takes_are_not_refused():
    """Without a second launch the bound is that of the query rows."""
    size = N.lib().minitp_shared_prefix_attention_workspace_bytes
    assert size(N.BF16, 1 << 17, 1, 2048, 4, 4, 128, 0, 0) == 0  # 2^30 rows, no prefix


@pytest.mark.parametrize("dtype", [N.BF16, N.F32])
def test_selection_of_too_many_groups(dtype):
    """A block of 1,024 threads a group."""
    for g in (1 << 22, (1 << 24) - 1):
        assert select(dtype, g=g, w=1, nbytes=1 << 62) == N.ERR_UNSUPPORTED and "too many" in N.last_error()
    assert select(dtype, g=(1 << 22) - 1, w=1, nbytes=64) == N.ERR_ARG  # (refused for its scratch alone)
