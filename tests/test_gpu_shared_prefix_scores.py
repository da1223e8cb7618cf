"""Attention behind a shared prefix where scores are large and close together:
only their differences matter, and parts of the keys that are computed apart
have to be weighed as exactly as keys within one part.

Every score is a number of at most 23 bits that the kernels form without
rounding (two products of few bits each, a scale of 1/4 or 1/8), its
distance to the largest one too. Bars, in steps of 2^-24 of the
attention-weighted |V|: an exponential 2, the sum over a part's keys (a tile, in
chains of 64 and 16) 80, at most 29 parts joined with 3 roundings each 87, once
above and once below the fraction, and the output's own: 340. bf16 adds half a
step of the output and of the probabilities, 2^-8 of the value and of the
attention-weighted |V|.
"""

import pytest
import torch

from tests.test_gpu_shared_prefix import reference

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("d", [16, 64])
@pytest.mark.parametrize("t,p,c", [(1, 1500, 40), (1, 900, 700), (5, 1500, 90), (3, 60, 5)])
def test_large_scores_close_together(t, p, c, d, dtype):
    from minitp import kernels as K

    b, groups, hq, hkv = 4, 2, 4, 2
    g = torch.Generator(device=DEV).manual_seed(t + p + c + d)
    q = torch.zeros(b, t, hq, d, dtype=dtype, device=DEV)
    q[..., 0], q[..., 1] = 128 * d ** 0.5, d ** 0.5  # score: 128 k[0] + k[1]

    def keys(*shape):
        k = torch.zeros(*shape, d, dtype=dtype, device=DEV)
        k[..., 0] = 96  # 12,288, and 0 to 7 in steps of 1/16
        k[..., 1] = torch.randint(0, 113, shape, generator=g, device=DEV) / 16
        return k, torch.randn(*shape, d, generator=g, device=DEV).to(dtype)

    (kp, vp), (kc, vc) = keys(groups, hkv, p), keys(b, hkv, c + t)
    out = K.shared_prefix_attention(q, kp, vp, kc, vc, p, c).view(b, t, hq, d).double().cpu()
    ref, mag = reference(q, kp, vp, kc, vc, [p] * groups, [c] * b)
    bar = mag * 340 * 2 ** -24
    if dtype == torch.bfloat16:
        bar = bar + (ref.abs() + mag) * 2 ** -8
    assert ((out - ref).abs() <= bar).all(), ((out - ref).abs() / bar).max()
