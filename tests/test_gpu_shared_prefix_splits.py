"""Several tokens whose own keys split over blocks: every split's causal
border, splits that no early token sees, rows of other lengths and idle ones,
and a hidden value that is not finite, against the formula in 64 bits (the
bars of test_gpu_shared_prefix.py)."""

import pytest
import torch

from tests.test_gpu_shared_prefix import bars, check, make, reference

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _own_splits(dtype, b, groups, t, hq, hkv, d, p, c):
    """Splits of the own part, from the scratch that the call asks for: a
    partial result a query row, split and part."""
    from minitp import _native as N

    size = N.lib().minitp_shared_prefix_attention_workspace_bytes
    code = N.dtype_code(dtype)
    row = b * t * hq * (d + 2) * 4
    total = size(code, b, groups, t, hq, hkv, d, p, c) // row
    if p == 0:
        return total
    return total - size(code, b, groups, t, hq, hkv, d, p, 0) // row + 1  # (one own split at c = 0 and few tokens)


# t query tokens, c cached rows, p prefix rows
SIZES = [(2, 700, 0), (5, 1000, 1500), (17, 1001, 0), (17, 763, 1500), (65, 830, 0), (65, 959, 1500), (130, 900, 1500)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("hq,hkv,d", [(4, 2, 64), (7, 1, 128), (2, 2, 16)])
@pytest.mark.parametrize("t,c,p", SIZES)
def test_own_keys_over_several_blocks(t, c, p, hq, hkv, d, dtype):
    from minitp import kernels as K

    b, groups = 4, 2
    assert _own_splits(dtype, b, groups, t, hq, hkv, d, p, c) > 1
    x = make(b, groups, t, hq, hkv, d, p, c, dtype)
    check(K.shared_prefix_attention(*x[:5], p, c), *x)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("hq,hkv,d", [(4, 2, 64), (7, 1, 128), (2, 2, 16)])
@pytest.mark.parametrize("t,c,p", SIZES)
def test_unequal_rows_over_several_blocks(t, c, p, hq, hkv, d, dtype):
    """Rows that leave the later splits empty, an idle one, prefixes cut short."""
    from minitp import kernels as K

    plens, clens = [p // 3, p], [c, 5, -1, c - 70, 0, c // 2]
    x = make(6, 2, t, hq, hkv, d, p, c, dtype, plens, clens)
    out = K.shared_prefix_attention(*x[:5], p, c, torch.tensor(plens, device=DEV), torch.tensor(clens, device=DEV))
    check(out, *x)
    assert (out[2] == 0).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("hq,hkv,d", [(4, 2, 64), (7, 1, 128), (2, 2, 16)])
@pytest.mark.parametrize("t,c,p", [(5, 1000, 1500), (17, 763, 0), (130, 900, 1500)])
def test_hidden_values_that_are_not_finite_in_a_split(t, c, p, hq, hkv, d, dtype):
    """A late token's value is infinite, another row's K and V are NaN: the
    tokens before it keep their results, those that see it are not finite."""
    from minitp import kernels as K

    n = t // 2
    x = make(4, 2, t, hq, hkv, d, p, c, dtype)
    kc, vc = x[3], x[4]
    clean = K.shared_prefix_attention(*x[:5], p, c)
    check(clean, *x)
    vc[1, :, c + n] = float("inf")
    kc[2, :, c + n] = float("nan")
    vc[2, :, c + n] = float("nan")
    out = K.shared_prefix_attention(*x[:5], p, c)
    assert torch.equal(out[0], clean[0]) and torch.equal(out[3], clean[3])
    seen = torch.where(torch.isfinite(vc), vc, 0.0)
    ref, mag = reference(*x[:3], torch.where(torch.isfinite(kc), kc, 0.0), seen, *x[5:])
    bar = bars(ref, mag, dtype, d)
    got = out.view(4, t, hq, d).double().cpu()
    for i in (1, 2):
        assert ((got[i, :n] - ref[i, :n]).abs() <= bar[i, :n] + 1e-9).all()
        assert not torch.isfinite(got[i, n:]).any()
