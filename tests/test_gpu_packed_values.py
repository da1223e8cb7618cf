"""Packed attention over values that are infinite or NaN: what a query sees of
them is in its result as the formula has it, what it does not see is not, and
neither takes a call out of its usual time."""

import math

import pytest
import torch

from tests.test_gpu_packed import BOTH, DEV, FORMS, bars, make, offsets_of, sampled

pytestmark = pytest.mark.gpu


def agree(out, rows, q, k, v, lens):
    """NaN and infinities where the formula has them in 64 bits (each visible key
    has a weight there, and here too: scores are within 30 of each other), all
    else within the bars."""
    dtype, d = q.dtype, q.shape[2]
    ref, _ = sampled(q, k, v, lens, rows)
    _, mag = sampled(q, k, v.nan_to_num(0.0, 0.0, 0.0), lens, rows)
    got = out.view(q.shape)[rows].double()
    assert torch.equal(torch.isnan(got), torch.isnan(ref))
    there = torch.isfinite(ref)
    assert torch.equal(torch.where(torch.isinf(ref), got, 0.0), torch.where(torch.isinf(ref), ref, 0.0))
    err, bar = (got - ref).abs()[there], (bars(ref, mag, dtype, d) + 1e-9)[there]
    assert (err <= bar).all(), (err / bar).max()


@pytest.mark.parametrize("dtype,heads,lens", FORMS, ids=lambda x: f"{len(x)}x{x[0]}" if isinstance(x, list) else str(x))
def test_values_that_are_seen_and_hidden(dtype, heads, lens):
    """In the first and the last text: one dim infinite from an early key on, one
    infinite both ways, one NaN in the middle, and later keys of the tiles that
    are bad in dims of their own."""
    from minitp import kernels as K

    lens = [7] + lens if lens[0] > 7 else lens
    n = sum(lens)
    q, k, v = make(n, *heads, dtype, "heads", seed=9)
    starts = offsets_of(lens).tolist()
    rows = set()
    for i in {1 % len(lens), len(lens) - 1}:
        lo, hi = starts[i], starts[i + 1]
        at = sorted({lo + min(x, hi - lo - 1) for x in (1, (hi - lo) // 3, (hi - lo) // 2, (hi - lo) * 2 // 3)})
        v[at[0], :, 3] = math.inf
        v[at[1 % len(at)], :, 5] = -math.inf
        v[at[-1], :, 3] = -math.inf
        v[at[2 % len(at)], :, 7] = math.nan
        rows |= {r for a in at + [lo, hi - 1] for r in range(a - 3, a + 4) if lo <= r < hi}
        rows |= {r for a in at for r in (a - 130, a - 40, a + 40, a + 130) if lo <= r < hi}
        rows |= {r for r in (lo - 1, hi) if 0 <= r < n}
    out = K.packed_attention(q, k, v, offsets_of(lens))
    agree(out, sorted(rows), q, k, v, lens)


@pytest.mark.parametrize("dtype", BOTH)
def test_values_near_the_types_end(dtype):
    """Finite values whose weighted sums pass float32 on the way in bf16 tiles,
    where a weight may be up to 2^8 before the division."""
    from minitp import kernels as K

    lens = [90, 300]
    q, k, v = make(390, 4, 2, 64, dtype)
    q = (q * 0 + torch.linspace(-1, 1, 64, device=DEV).to(dtype)).contiguous()
    ramp = torch.linspace(0, 1, 390, device=DEV)[:, None, None]
    k = (q[:, :2] * ramp.to(dtype) * 1.5).contiguous()  # scores rise with the keys, by less than 8 in base 2
    v = (v.clamp(-2, 2) * 2.0 ** 117).to(dtype)
    rows = list(range(0, 390, 13))
    out = K.packed_attention(q, k, v, offsets_of(lens))
    ref, mag = sampled(q, k, v, lens, rows)
    assert ((out.view(390, 4, 64)[rows].double() - ref).abs() <= bars(ref, mag, dtype, 64)).all()


@pytest.mark.parametrize("dtype,heads,length", [(torch.bfloat16, (28, 4, 128), 4000), (torch.bfloat16, (14, 2, 64), 5900),
                                                (torch.float32, (14, 2, 64), 3000)])
def test_an_early_infinity_takes_no_longer(dtype, heads, length):
    """A text whose rows nearly all see an infinite value takes about the time of
    any other (30 to 165 times as long if those rows are computed again, one by
    one; the bound leaves room for a busy machine)."""
    from minitp import kernels as K

    q, k, v = make(length, *heads, dtype, "heads")
    bad = v.clone()
    bad[5, :, 3] = math.inf
    offsets = offsets_of([length])

    def time(values):
        best = math.inf
        for _ in range(5):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            K.packed_attention(q, k, values, offsets)
            b.record()
            b.synchronize()
            best = min(best, a.elapsed_time(b))
        return best

    time(v)
    assert time(bad) <= 8 * time(v)


@pytest.mark.parametrize("power", [20, 31, 36, 44, 90])
@pytest.mark.parametrize("dtype,heads,lens", [
    (torch.bfloat16, (28, 4, 128), [300]), (torch.bfloat16, (14, 2, 64), [2500, 333]), (torch.bfloat16, (28, 4, 128), [60] * 300),
    (torch.bfloat16, (14, 2, 64), [60] * 300), (torch.bfloat16, (4, 2, 16), [60] * 300), (torch.float32, (28, 4, 128), [300]),
    (torch.float32, (14, 2, 64), [60] * 300), (torch.float32, (8, 2, 32), [20] * 600),
], ids=lambda x: f"{len(x)}x{x[0]}" if isinstance(x, list) else str(x))
def test_far_scores(dtype, heads, lens, power):
    """Scores up to 2^power / sqrt(D) of either sign, past what a rounded maximum
    in powers of two holds to a step of one. They are products of two numbers of
    eight bits, so exact, and apart by at least |q|: at 2^20 and above another
    key's probability is e^-2 of the greatest or less, known to 2^-15 (256 such
    steps are the whole range, each score off by 2^-24 of itself)."""
    from minitp import kernels as K

    hq, hkv, d = heads
    n = sum(lens)
    g = torch.Generator(device=DEV).manual_seed(power + n)

    def whole(h):
        return torch.randint(-255, 256, (n, h), generator=g, device=DEV).float()

    q, k = torch.zeros(n, hq, d, device=DEV), torch.zeros(n, hkv, d, device=DEV)
    q[..., d // 2], k[..., d // 2] = whole(hq) * 2.0 ** (power - 16), whole(hkv)
    q, k = q.to(dtype), k.to(dtype)
    v = torch.randn(n, hkv, d, generator=g, device=DEV).to(dtype)
    rows = sorted(set(range(0, n, max(n // 60, 1))) | {n - 1})
    ref, mag = sampled(q, k, v, lens, rows)
    got = K.packed_attention(q, k, v, offsets_of(lens)).view(n, hq, d)
    assert torch.isfinite(got).all()
    bar = bars(ref, mag, dtype, d) + mag * 2 ** -14 + 1e-9
    err = (got[rows].double() - ref).abs()
    assert (err <= bar).all(), (err / bar).max()


@pytest.mark.parametrize("heads", [(14, 2, 64), (28, 4, 128), (4, 2, 16)])
def test_an_infinity_beside_values_near_the_types_end(heads):
    """Rows of a bf16 tile that see an infinite value in one dim, while the others'
    weighted sums pass float32 on the way: scores rise by 7.5 in base 2 over the
    text, which moves no maximum, so that some 400 weights of up to 2^6 meet values
    of 2^117 and more."""
    from minitp import kernels as K

    hq, hkv, d = heads
    lens = [390] * 60
    n = sum(lens)
    _, _, v = make(n, hq, hkv, d, torch.bfloat16)
    rise = torch.linspace(0, 7.5 * math.log(2), 390, device=DEV).repeat(60)
    q, k = torch.zeros(n, hq, d, device=DEV), torch.zeros(n, hkv, d, device=DEV)
    q[..., 0], k[..., 0] = math.sqrt(d), rise[:, None]
    q, k = q.bfloat16(), k.bfloat16()
    v = (v.abs().clamp(max=1) + 1).mul(2.0 ** 117).to(torch.bfloat16)
    v[391, :, 3], v[390 * 7 + 5, :, 3] = math.inf, -math.inf
    rows = [r for t in (0, 1, 7, 59) for r in (390 * t, 390 * t + 4, 390 * t + 200, 390 * t + 300, 390 * t + 389)]
    out = K.packed_attention(q, k, v, offsets_of(lens))
    agree(out, rows, q, k, v, lens)
