"""What lies behind the arrays of a packed attention call, and rows far apart."""

import math

import pytest
import torch

from tests.test_gpu_packed import BOTH, DEV, FORMS, bounds_of, check, make, offsets_of

pytestmark = pytest.mark.gpu


def behind(x, rows, value, by_heads):
    """x [N, H, D] in front of `rows` more rows of a value, in the same array."""
    n, h, d = x.shape
    store = torch.full((h, n + rows, d) if by_heads else (n + rows, h, d), value, dtype=x.dtype, device=DEV)
    view = (store.transpose(0, 1) if by_heads else store)[:n]
    return view.copy_(x)


@pytest.mark.parametrize("by_heads", [True, False])
@pytest.mark.parametrize("dtype,heads,lens", FORMS, ids=lambda x: f"{len(x)}x{x[0]}" if isinstance(x, list) else str(x))
def test_rows_behind_the_arrays_are_not_read(dtype, heads, lens, by_heads):
    """K and V rows behind the last one, which belong to something else, change no
    bit: as NaN they would show, or send a tile's rows through another sum."""
    from minitp import kernels as K

    lens = lens + [1]  # (the last tiles of keys hold a few rows, and one)
    q, k, v = make(sum(lens), *heads, dtype)
    want = K.packed_attention(q, k, v, offsets_of(lens))
    assert torch.isfinite(want).all()
    for value in (0.0, math.nan, math.inf):
        kk, vv = behind(k, 400, value, by_heads), behind(v, 400, value, by_heads)
        assert torch.equal(want, K.packed_attention(q, kk, vv, offsets_of(lens))), value
