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


@pytest.mark.parametrize("dtype,heads,lens", [
    (torch.bfloat16, (4, 2, 64), [250, 9]),           # four sets, tiles of 128 keys
    (torch.bfloat16, (28, 4, 128), [13] * 20),        # tiles of 64 keys, one stage of V
    (torch.bfloat16, (14, 2, 64), [13] * 20),         # ... and two
    (torch.float32, (4, 2, 64), [250, 9]), (torch.float32, (28, 4, 128), [13] * 20),
], ids=lambda x: f"{len(x)}x{x[0]}" if isinstance(x, list) else str(x))
def test_rows_as_far_apart_as_they_may_be(dtype, heads, lens):
    """K/V rows 2^24 elements apart (fp32 2^23), the most that a call takes: a tile
    of 128 keys spans all but 32 MiB of 4 GiB, and what lies between the rows is
    NaN where it is near them."""
    from minitp import kernels as K

    hq, hkv, d = heads
    step, n = (1 << 24) // (1 if dtype == torch.bfloat16 else 2), sum(lens)
    store = torch.empty(n * step, dtype=dtype, device=DEV).view(n, step)
    store[:, :8192], store[:, -4096:] = math.nan, math.nan
    q, k, v = make(n, hq, hkv, d, dtype)
    kk, vv = (store[:, at:at + hkv * d].view(n, hkv, d) for at in (0, 4096))
    kk.copy_(k)
    vv.copy_(v)
    out = K.packed_attention(q, kk, vv, offsets_of(lens))
    assert torch.equal(out, K.packed_attention(q, k, v, offsets_of(lens)))
    check(out, q, k, v, bounds_of(lens))
    del store, kk, vv
    torch.cuda.empty_cache()
