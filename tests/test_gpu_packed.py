"""Attention over packed sequences (csrc/packed.hip) against the formula in 64
bits: every head shape, both types, lengths around the tiles' edges, empty
sequences, rows of none, and values of other sequences that are not finite.

Bars. bf16: the output's own rounding, half a step (2^-8 of the value), and the
probabilities rounded to bf16 for the product (2^-8 of the attention-weighted
|V|, the sum they are divided by unrounded). fp32: a score is at most four chains of
D / 4 products and three more sums, each off by at most 2^-24 of the sum of the
products' magnitudes, which is below 20 here (1.5 x 0.64 sqrt(D) = 11 at D = 128 for
normal rows, its spread below 1.5); a score's error is its probability's
relative error, once above and once below the fraction; exponentials and sums
over tiles add less than 64 steps.
"""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
BOTH = [torch.bfloat16, torch.float32]
HEADS = [(14, 2, 64), (28, 4, 128), (4, 2, 16), (4, 4, 32), (8, 1, 128), (3, 1, 64), (9, 3, 16), (16, 8, 32), (33, 1, 32)]


def make(n, hq, hkv, d, dtype, layout="tokens", seed=0):
    """q [N, Hq, D], k and v [N, Hkv, D] as contiguous rows, K and V kept by
    heads, or slices of one projection's rows."""
    g = torch.Generator(device=DEV).manual_seed(seed + n * 3 + hq * 7 + d)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=DEV).to(dtype)

    if layout == "together":
        qkv = normal(n, (hq + 2 * hkv) * d)
        q, k, v = qkv.view(n, -1, d).split([hq, hkv, hkv], 1)
        q *= 1.5
        return q, k, v
    q = normal(n, hq, d) * 1.5
    if layout == "heads":
        return q, normal(hkv, n, d).transpose(0, 1), normal(hkv, n, d).transpose(0, 1)
    return q, normal(n, hkv, d), normal(n, hkv, d)


def reference(q, k, v, bounds):
    """(out, the attention-weighted |V|) [N, Hq, D] in float64 on the device;
    bounds: (first row, end) of each sequence."""
    n, hq, d = q.shape
    per = hq // k.shape[1]
    out = torch.zeros(n, hq, d, dtype=torch.float64, device=DEV)
    mag = torch.zeros_like(out)
    for lo, hi in bounds:
        if hi <= lo:
            continue
        hidden = torch.ones(hi - lo, hi - lo, dtype=torch.bool, device=DEV).triu(1)
        for h in range(hq):
            kh, vh = k[lo:hi, h // per].double(), v[lo:hi, h // per].double()
            s = q[lo:hi, h].double() @ kh.t().contiguous() / math.sqrt(d)
            p = torch.softmax(s.masked_fill(hidden, -math.inf), -1)
            out[lo:hi, h], mag[lo:hi, h] = p @ vh, p @ vh.abs()
    return out, mag


def bars(ref, mag, dtype, d):
    if dtype == torch.bfloat16:
        return (ref.abs() + mag) * 2 ** -8
    return mag * (2 * 20 * (d / 4 + 3) + 64) * 2 ** -24


def check(got, q, k, v, bounds):
    ref, mag = reference(q, k, v, bounds)
    got = got.view(ref.shape).double()
    assert torch.isfinite(got).all()
    bar = bars(ref, mag, q.dtype, q.shape[2]) + 1e-9
    assert ((got - ref).abs() <= bar).all(), ((got - ref).abs() / bar).max()


def offsets_of(lens, first=0):
    return torch.tensor([first] + lens, device=DEV).cumsum(0)


def bounds_of(lens, first=0):
    ends = [first]
    for n in lens:
        ends.append(ends[-1] + n)
    return list(zip(ends, ends[1:]))


LENS = [[1], [2, 1, 1], [16], [17, 64, 65, 1, 0, 130], [0, 0, 5, 0], [31, 33, 32, 63, 2, 127, 129, 128], [300, 1, 77],
        [1] * 50, [700]]


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("layout", ["tokens", "heads", "together"])
@pytest.mark.parametrize("hq,hkv,d", HEADS)
@pytest.mark.parametrize("lens", LENS, ids=lambda x: f"{len(x)}x{max(x)}")
def test_lengths(lens, hq, hkv, d, layout, dtype):
    from minitp import kernels as K

    x = make(sum(lens), hq, hkv, d, dtype, layout)
    check(K.packed_attention(*x, offsets_of(lens)), *x, bounds_of(lens))


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("hq,hkv,d", [(14, 2, 64), (28, 4, 128), (4, 2, 16), (4, 4, 32)])
def test_rows_of_no_sequence(hq, hkv, d, dtype):
    """Rows in front of the first sequence and behind the last, NaN all over,
    come out as zeros and change nothing else; int32 offsets."""
    from minitp import kernels as K

    lens, first = [40, 0, 130, 3], 37
    q, k, v = make(first + sum(lens) + 200, hq, hkv, d, dtype)
    end = first + sum(lens)
    for t in (q, k, v):
        t[:first], t[end:] = math.nan, math.nan
    out = K.packed_attention(q, k, v, offsets_of(lens, first).int())
    check(out[first:end], q[first:end], k[first:end], v[first:end], bounds_of(lens))
    assert (out[:first] == 0).all() and (out[end:] == 0).all()
    for none in (torch.zeros(1, device=DEV, dtype=torch.long), torch.tensor([5], device=DEV),
                 torch.zeros(4, device=DEV, dtype=torch.long)):
        assert (K.packed_attention(q, k, v, none) == 0).all()


@pytest.mark.parametrize("value", [math.nan, math.inf])
@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("hq,hkv,d", [(14, 2, 64), (28, 4, 128), (4, 2, 16), (4, 4, 32)])
def test_values_that_are_not_finite_stay_in_their_rows(hq, hkv, d, dtype, value):
    """A bad key or value row of one sequence shows in that sequence's rows from
    it on, and nowhere else."""
    from minitp import kernels as K

    lens = [50, 70, 1, 140, 33]
    for which in (1, 2):
        x = make(sum(lens), hq, hkv, d, dtype, seed=which)
        # (of the clean rows: the product's own zeros times the bad value are no zeros)
        ref, mag = reference(*x, bounds_of(lens))
        bad = 50 + 70 + 1 + 60  # row 60 of the fourth sequence
        x[which][bad, :, d - 1] = value
        out = K.packed_attention(*x, offsets_of(lens))
        touched = torch.zeros(sum(lens), dtype=torch.bool, device=DEV)
        touched[bad:50 + 70 + 1 + 140] = True
        mine = out.view(-1, hq, d)
        if which == 2:
            assert not torch.isfinite(mine[touched][..., d - 1]).any()
        elif math.isnan(value):
            assert torch.isnan(mine[touched]).all()
        bar = bars(ref, mag, dtype, d) + 1e-9
        assert ((mine.double() - ref).abs() <= bar)[~touched].all()


@pytest.mark.parametrize("dtype", BOTH)
def test_a_query_that_is_no_number_shows(dtype):
    from minitp import kernels as K

    lens = [20, 90]
    x = make(110, 14, 2, 64, dtype)
    x[0][33, 5, 7] = math.nan
    out = K.packed_attention(*x, offsets_of(lens)).view(110, 14, 64)
    assert torch.isnan(out[33, 5]).all()
    out[33, 5] = 0
    assert torch.isfinite(out).all()


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("scale", [60.0, 1e4])
def test_large_scores(dtype, scale):
    """Scores far apart: probabilities of nearly zero and one."""
    from minitp import kernels as K

    lens = [130, 64]
    q, k, v = make(194, 4, 2, 64, dtype)
    q = (q * scale).to(dtype)
    out = K.packed_attention(q, k, v, offsets_of(lens)).view(194, 4, 64).double()
    ref, mag = reference(q, k, v, bounds_of(lens))
    # a score's error is a step of its products' magnitudes' sum (fp32 sums)
    size = (q.double().abs()[:, :, None] * k.double().abs().amax(0).repeat_interleave(2, 0)[None, :, None]).sum(-1) / 8
    rel = 2 * size * (64 / 4 + 3 + 2) * 2 ** -24
    bar = (ref.abs() + mag) * 2 ** -8 if dtype == torch.bfloat16 else mag * 64 * 2 ** -24
    assert ((out - ref).abs() <= bar + rel.clamp(max=1.0) * v.double().abs().max() + 1e-9).all()


@pytest.mark.parametrize("dtype", BOTH)
def test_many_short_sequences(dtype):
    """More sequences than a block holds boundaries of, empty ones among them."""
    from minitp import kernels as K

    g = torch.Generator().manual_seed(4)
    lens = torch.randint(0, 4, (5000,), generator=g).tolist()
    lens[100:900] = [0] * 800
    n = sum(lens)
    x = make(n, 4, 2, 16, dtype)
    out = K.packed_attention(*x, offsets_of(lens)).view(n, 4, 16).double()
    # a sequence of up to three rows at a time: all starts at once
    start = torch.repeat_interleave(offsets_of(lens)[:-1], torch.tensor(lens, device=DEV))
    rows = torch.arange(n, device=DEV)
    idx = (rows[:, None] - torch.arange(3, device=DEV)).clamp(min=0)
    there = idx >= start[:, None]
    there &= rows[:, None] - torch.arange(3, device=DEV) >= 0
    q, k, v = (t.double() for t in x)
    kk, vv = (t.repeat_interleave(2, 1)[idx] for t in (k, v))
    s = (q[:, None] * kk).sum(-1) / 4
    p = torch.softmax(s.masked_fill(~there[:, :, None], -math.inf), 1)
    ref, mag = (p[..., None] * vv).sum(1), (p[..., None] * vv.abs()).sum(1)
    assert ((out - ref).abs() <= bars(ref, mag, dtype, 16) + 1e-9).all()


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("hq,hkv,d", [(14, 2, 64), (28, 4, 128)])
def test_long_sequences(hq, hkv, d, dtype):
    from minitp import kernels as K

    lens = [2500, 333, 1700]
    x = make(sum(lens), hq, hkv, d, dtype, "heads")
    check(K.packed_attention(*x, offsets_of(lens)), *x, bounds_of(lens))


def sampled(q, k, v, lens, rows):
    """reference() for some rows: (out, mag) [rows, Hq, D] in float64."""
    hq, d, hkv = q.shape[1], q.shape[2], k.shape[1]
    starts = offsets_of(lens).tolist()
    outs, mags = [], []
    for r in rows:
        lo = max(s for s in starts[:-1] if s <= r)
        kk, vv = (t[lo:r + 1].double().transpose(0, 1).contiguous() for t in (k, v))  # [Hkv, n, D]
        s = (kk @ q[r].double().view(hkv, -1, d).transpose(1, 2).contiguous()).transpose(1, 2) / math.sqrt(d)
        p = torch.softmax(s, -1).contiguous()
        outs.append((p @ vv).reshape(hq, d))
        mags.append((p @ vv.abs()).reshape(hq, d))
    return torch.stack(outs), torch.stack(mags)


# shapes for each form of the kernels: sets of waves a row, keys of a tile, waves of a block
FORMS = [
    (torch.bfloat16, (14, 2, 64), [500]), (torch.bfloat16, (28, 4, 128), [150, 90]),      # 4 sets
    (torch.bfloat16, (8, 2, 32), [900, 300]), (torch.bfloat16, (4, 2, 16), [1500, 700]),
    (torch.bfloat16, (14, 2, 64), [2500, 333, 1700]), (torch.bfloat16, (28, 4, 128), [600, 500]),  # 2 sets
    (torch.bfloat16, (8, 2, 32), [2500] * 6), (torch.bfloat16, (4, 2, 16), [16000, 15000]),
    (torch.bfloat16, (28, 4, 128), [3000, 2400]),                                         # 128 keys, 8 waves
    (torch.bfloat16, (14, 2, 64), [5900]),                                                # 2 sets of 8 waves
    (torch.bfloat16, (14, 2, 64), [8191]), (torch.bfloat16, (14, 2, 64), [4000, 3000]),   # 128 keys
    (torch.bfloat16, (14, 2, 64), [60] * 300), (torch.bfloat16, (28, 4, 128), [60] * 300),
    (torch.bfloat16, (8, 2, 32), [60] * 300), (torch.bfloat16, (4, 2, 16), [60] * 300),
    (torch.float32, (14, 2, 64), [500]), (torch.float32, (28, 4, 128), [700]), (torch.float32, (14, 2, 64), [3000]),
    (torch.float32, (28, 4, 128), [60] * 300), (torch.float32, (8, 2, 32), [2500] * 6), (torch.float32, (4, 2, 16), [90] * 400),
    (torch.float32, (28, 4, 128), [1500]), (torch.float32, (4, 2, 16), [5000, 4900]),     # two strips a wave
    (torch.float32, (14, 2, 64), [100] * 60), (torch.float32, (28, 4, 128), [300] * 10),  # 2 sets
    (torch.float32, (14, 2, 64), [20] * 600), (torch.float32, (8, 2, 32), [20] * 600),    # 1 set
    (torch.float32, (4, 2, 16), [3] * 6000), (torch.float32, (8, 2, 32), [40, 30, 20]),
]


@pytest.mark.parametrize("dtype,heads,lens", FORMS, ids=lambda x: f"{len(x)}x{x[0]}" if isinstance(x, list) else str(x))
def test_forms(dtype, heads, lens):
    """Each form over whole calls: sampled rows, rows behind the last sequence,
    and a value row that is not finite in one of the sequences."""
    from minitp import kernels as K

    hq, hkv, d = heads
    n, pad = sum(lens), 45
    x = make(n + pad, hq, hkv, d, dtype, "heads")
    for t in x:
        t[n:] = math.nan
    g = torch.Generator().manual_seed(n)
    ends = offsets_of(lens).tolist()
    rows = sorted(set(torch.randint(0, n, (50,), generator=g).tolist() + [0, n - 1, ends[1] - 1, ends[-2]]
                      + [r for r in (15, 16, 31, 32, 63, 64, 127, 128, 255, 256) if r < n]))
    ref, mag = sampled(*x, lens, rows)
    bar = bars(ref, mag, dtype, d) + 1e-9
    out = K.packed_attention(*x, offsets_of(lens)).view(n + pad, hq, d)
    assert torch.isfinite(out).all() and (out[n:] == 0).all()
    err = (out[rows].double() - ref).abs()
    assert (err <= bar).all(), (err / bar).max()
    bad = ends[1] - lens[0] // 3  # in the first sequence
    x[2][bad, :, 3] = math.inf
    again = K.packed_attention(*x, offsets_of(lens)).view(n + pad, hq, d)
    assert not torch.isfinite(again[bad:ends[1], :, 3]).any()
    assert torch.isfinite(again[:bad]).all() and torch.isfinite(again[ends[1]:]).all()
    err = (again[rows].double() - ref).abs()
    clean = torch.tensor([not bad <= r < ends[1] for r in rows], device=DEV)
    assert (err <= bar)[clean].all(), (err / bar)[clean].max()


@pytest.mark.parametrize("dtype,heads,lens", [FORMS[i] for i in (0, 4, 8, 9, 10, 12, 16, 18, 19, 22, 24)],
                         ids=lambda x: f"{len(x)}x{x[0]}" if isinstance(x, list) else str(x))
def test_a_text_of_nan(dtype, heads, lens):
    """Keys, values and queries that are no numbers from a row on, as a token
    outside the vocabulary leaves them: NaN from there to the sequence's end."""
    from minitp import kernels as K

    hq, hkv, d = heads
    n = sum(lens)
    x = make(n, hq, hkv, d, dtype, "heads", seed=3)
    want = K.packed_attention(*x, offsets_of(lens)).view(n, hq, d)
    bad, end = lens[0] // 3, lens[0]
    for t in x:
        t[bad:end] = math.nan
    out = K.packed_attention(*x, offsets_of(lens)).view(n, hq, d)
    assert torch.isnan(out[bad:end]).all()
    rest = torch.arange(n, device=DEV)
    rest = rest[(rest < bad) | (rest >= end)]
    _, mag = sampled(*make(n, hq, hkv, d, dtype, "heads", seed=3), lens, rest[::97].tolist())
    bar = mag * (4 * 2 ** -8 if dtype == torch.bfloat16 else 2 * (2 * 20 * (d / 4 + 3) + 64) * 2 ** -24) + 1e-9
    assert torch.isfinite(out[rest]).all()
    assert ((out[rest[::97]].double() - want[rest[::97]].double()).abs() <= bar).all()


@pytest.mark.parametrize("first,pad", [(0, 0), (37, 0), (0, 50), (333, 1000)])
@pytest.mark.parametrize("dtype,heads,most", [(torch.bfloat16, (28, 4, 128), 0), (torch.bfloat16, (28, 4, 128), 300),
                                              (torch.bfloat16, (14, 2, 64), 600), (torch.float32, (14, 2, 64), 300),
                                              (torch.float32, (9, 3, 16), 500)])
def test_order_of_the_tiles(dtype, heads, most, first, pad):
    """Up to 31 sequences take their tiles by the number of keys, more of them in
    the order of the stream (an empty one behind the others makes one more): every
    row is computed once, to the same bits."""
    from minitp import kernels as K

    g = torch.Generator().manual_seed(most + first)
    lens = torch.randint(-most // 6, most, (31,), generator=g).clamp(min=0).tolist() if most else [1900, 0, 1400]
    n = first + sum(lens) + pad
    x = make(n, *heads, dtype)
    offsets = offsets_of(lens) + first
    more = torch.cat([offsets, offsets[-1:].repeat(32 - len(lens))])
    for _ in range(2):
        torch.full((n, heads[0] * heads[2]), math.nan, dtype=dtype, device=DEV)  # (what the result's memory held)
        out = K.packed_attention(*x, offsets)
        assert torch.isfinite(out).all()
        assert torch.equal(out, K.packed_attention(*x, more))
    down = offsets.flip(0).contiguous()  # in disorder: as many rows as ever, no access outside
    assert K.packed_attention(*x, down).shape == out.shape
    torch.cuda.synchronize()


def test_sequences_equal_prompts_on_their_own():
    """As far as the two kernels round alike: the model's prompt attention."""
    from minitp import kernels as K

    lens = [130, 17, 64]
    q, k, v = make(sum(lens), 14, 2, 64, torch.bfloat16, "heads")
    out = K.packed_attention(q, k, v, offsets_of(lens))
    for lo, hi in bounds_of(lens):
        alone = K.attention(q[None, lo:hi], k[lo:hi].transpose(0, 1)[None].contiguous(),
                            v[lo:hi].transpose(0, 1)[None].contiguous(), 0)[0]
        _, mag = reference(q[lo:hi], k[lo:hi], v[lo:hi], [(0, hi - lo)])
        bar = mag.view(hi - lo, -1) * 4 * 2 ** -8
        assert ((alone.double() - out[lo:hi].double()).abs() <= bar + 1e-9).all()


def test_results_are_the_same_bits_each_time():
    from minitp import kernels as K

    lens = [500, 3, 0, 800]
    for dtype in BOTH:
        x = make(sum(lens), 14, 2, 64, dtype)
        first = K.packed_attention(*x, offsets_of(lens))
        for _ in range(3):
            assert torch.equal(first, K.packed_attention(*x, offsets_of(lens)))


def test_odd_views_are_copied():
    """Unaligned rows, another element order, K and V of different layouts."""
    from minitp import kernels as K

    lens = [70, 9]
    q, k, v = make(79, 4, 2, 32, torch.bfloat16)
    want = K.packed_attention(q, k, v, offsets_of(lens))
    shifted = torch.empty(79 * 4 * 32 + 1, dtype=torch.bfloat16, device=DEV)[1:].view(79, 4, 32).copy_(q)
    assert torch.equal(want, K.packed_attention(shifted, k, v, offsets_of(lens)))
    by_dim = k.transpose(1, 2).contiguous().transpose(1, 2)
    assert torch.equal(want, K.packed_attention(q, by_dim, v, offsets_of(lens)))
    by_head = v.transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(want, K.packed_attention(q, k, by_head, offsets_of(lens)))
    # one K/V row for all heads and one for all tokens
    one = k[:, :1].expand(79, 2, 32)
    assert torch.equal(K.packed_attention(q, one, one, offsets_of(lens)),
                       K.packed_attention(q, one.contiguous(), one.contiguous(), offsets_of(lens)))
    same = k[:1].expand(79, 2, 32)
    assert torch.equal(K.packed_attention(q, same, same, offsets_of(lens)),
                       K.packed_attention(q, same.contiguous(), same.contiguous(), offsets_of(lens)))


def test_graph_streams_and_changed_offsets():
    """A captured call takes other offsets at each replay; a second stream runs
    at the same time."""
    from minitp import kernels as K

    n = 400
    x = make(n, 14, 2, 64, torch.bfloat16)
    offsets = offsets_of([100, 200, 50])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        K.packed_attention(*x, offsets)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = K.packed_attention(*x, offsets)
    for lens in ([100, 200, 50], [1, 398, 1], [0, 0, 0], [399, 0, 0], [133, 133, 134]):
        offsets.copy_(offsets_of(lens))
        with torch.cuda.stream(side):
            side.wait_stream(torch.cuda.current_stream())
            beside = K.packed_attention(*x, offsets)
        graph.replay()
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        assert torch.equal(out, beside)
        assert torch.equal(out, K.packed_attention(*x, offsets))


def test_offsets_in_disorder_stay_inside():
    """Values that no caller should pass: nothing outside the arrays is read,
    and sequences that are in order hold."""
    from minitp import kernels as K

    x = make(200, 14, 2, 64, torch.bfloat16)
    for bad in ([50, 20, 90, 60], [-7, 1 << 40], [-(1 << 62), 300, 10], [199, 0], [1 << 40, 1 << 41]):
        assert torch.isfinite(K.packed_attention(*x, torch.tensor(bad, device=DEV))).all()
    check(K.packed_attention(*x, torch.tensor([-100, 200], device=DEV)), *x, [(0, 200)])
    check(K.packed_attention(*x, torch.tensor([0, 1 << 40], device=DEV)), *x, [(0, 200)])


@pytest.mark.parametrize("dtype", BOTH)
def test_rows_past_four_gib(dtype):
    """K/V rows far apart: offsets past 32 bits, in bytes and in elements."""
    from minitp import kernels as K

    step = 1 << 17
    n = (1 << 32) // step + 200  # elements past 2^32
    store = torch.zeros(n * step, dtype=dtype, device=DEV).view(n, step)
    q, k, v = make(n, 4, 2, 64, dtype)
    kk, vv = store[:, :128].view(n, 2, 64), store[:, 256:384].view(n, 2, 64)
    kk.copy_(k)
    vv.copy_(v)
    offsets = offsets_of([n - 300, 300])
    out, near = K.packed_attention(q, kk, vv, offsets), K.packed_attention(q, k, v, offsets)
    assert torch.equal(out, near)
    check(out[-300:], q[-300:], k[-300:], v[-300:], [(0, 300)])


def test_nothing():
    from minitp import kernels as K

    x = make(0, 4, 2, 64, torch.bfloat16)
    assert K.packed_attention(*x, torch.tensor([0], device=DEV)).shape == (0, 256)
    assert K.packed_attention(*x, torch.tensor([0, 0], device=DEV)).shape == (0, 256)
