"""Attention of batches that share prefixes (csrc/shared_prefix.hip) against the
formula in 64 bits: every head shape, both types, lengths around the tiles'
edges, unequal and idle rows, rows that no length covers poisoned.

Bars. bf16: the output's own rounding, half a step (2^-8 of the value), and the
probabilities rounded to bf16 for the product (2^-8 of the attention-weighted
|V|, the sum they are divided by unrounded). fp32: a score is four chains of D / 4
products and three more sums, each off by at most 2^-24 of the sum of the
products' magnitudes, which is below 20 here (1.5 x 0.64 sqrt(D) = 11 at D = 128 for
normal rows, its spread below 1.5); a score's error is its probability's
relative error, once above and once below the fraction; exponentials and sums
over tiles and splits add less than 64 steps.
"""

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


def reference(q, kp, vp, kc, vc, plens, clens):
    """(out, the attention-weighted |V|), both [B, T, Hq, D] in float64."""
    b, t, hq, d = q.shape
    groups, hkv = kp.shape[:2]
    out = torch.zeros(b, t, hq, d, dtype=torch.float64)
    mag = torch.zeros_like(out)
    for i in range(b):
        if clens[i] < 0:
            continue
        g = i // (b // groups)
        for h in range(hq):
            kv = h // (hq // hkv)
            k = torch.cat([kp[g, kv, :plens[g]], kc[i, kv, :clens[i] + t]]).double().cpu()
            v = torch.cat([vp[g, kv, :plens[g]], vc[i, kv, :clens[i] + t]]).double().cpu()
            for n in range(t):
                m = plens[g] + clens[i] + n + 1
                p = torch.softmax(k[:m] @ q[i, n, h].double().cpu() / d ** 0.5, 0)
                out[i, n, h] = p @ v[:m]
                mag[i, n, h] = p @ v[:m].abs()
    return out, mag


def make(b, groups, t, hq, hkv, d, p, c, dtype, plens=None, clens=None, seed=0, room=5):
    g = torch.Generator(device=DEV).manual_seed(seed + b * 7 + t * 31 + p + 3 * c + d)
    plens = [p] * groups if plens is None else plens
    clens = [c] * b if clens is None else clens

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=DEV).to(dtype)

    q = normal(b, t, hq, d) * 1.5
    kp, vp = normal(groups, hkv, p + room, d), normal(groups, hkv, p + room, d)
    kc, vc = normal(b, hkv, c + t + room, d), normal(b, hkv, c + t + room, d)
    for i in range(groups):
        kp[i, :, plens[i]:] = float("nan")
        vp[i, :, plens[i]:] = float("nan")
    for i in range(b):
        end = clens[i] + t if clens[i] >= 0 else 0
        kc[i, :, end:] = float("nan")
        vc[i, :, end:] = float("nan")
    return q, kp, vp, kc, vc, plens, clens


def bars(ref, mag, dtype, d):
    if dtype == torch.bfloat16:
        return (ref.abs() + mag) * 2 ** -8
    return mag * (2 * 20 * (d / 4 + 3) + 64) * 2 ** -24


def check(out, q, kp, vp, kc, vc, plens, clens):
    ref, mag = reference(q, kp, vp, kc, vc, plens, clens)
    b, t, hq, d = q.shape
    got = out.view(b, t, hq, d).double().cpu()
    assert torch.isfinite(got).all()
    bar = bars(ref, mag, q.dtype, d)
    assert ((got - ref).abs() <= bar + 1e-9).all(), ((got - ref).abs() / (bar + 1e-9)).max()


HEADS = [(14, 2, 64), (28, 4, 128), (4, 2, 16), (4, 4, 32), (8, 1, 128), (3, 1, 64)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("hq,hkv,d", HEADS)
@pytest.mark.parametrize("p,c", [(1, 0), (63, 1), (64, 63), (200, 70), (513, 130)])
def test_one_token(p, c, hq, hkv, d, dtype):
    from minitp import kernels as K

    x = make(6, 2, 1, hq, hkv, d, p, c, dtype)
    check(K.shared_prefix_attention(*x[:5], p, c), *x)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("hq,hkv,d", [(14, 2, 64), (4, 1, 128), (4, 2, 16), (2, 2, 32)])
@pytest.mark.parametrize("t,p,c", [(2, 0, 0), (3, 130, 0), (17, 40, 47), (65, 66, 3)])
def test_several_tokens(t, p, c, hq, hkv, d, dtype):
    from minitp import kernels as K

    x = make(4, 2, t, hq, hkv, d, p, c, dtype)
    check(K.shared_prefix_attention(*x[:5], p, c), *x)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("t", [1, 5])
@pytest.mark.parametrize("hq,hkv,d", [(14, 2, 64), (28, 4, 128), (4, 2, 16)])
@pytest.mark.parametrize("p", [300, 1500])  # both parts by one block, or by blocks of their own
def test_unequal_empty_and_idle_rows(p, hq, hkv, d, t, dtype):
    """Prefixes of length 0 and 1, rows without cached tokens, idle rows."""
    from minitp import kernels as K

    plens, clens = [p, 0, 1], [0, 90, -1, 17, 64, -1, 90, 1, 33]
    x = make(9, 3, t, hq, hkv, d, p, 90, dtype, plens, clens)
    out = K.shared_prefix_attention(*x[:5], p, 90, prefix_lens=torch.tensor(plens, device=DEV),
                                    cache_lens=torch.tensor(clens, device=DEV, dtype=torch.int32))
    check(out, *x)
    assert (out[2] == 0).all() and (out[5] == 0).all()


def test_lengths_past_the_bounds_are_the_bounds():
    from minitp import kernels as K

    x = make(4, 2, 1, 14, 2, 64, 100, 20, torch.bfloat16)
    out = K.shared_prefix_attention(*x[:5], 100, 20, prefix_lens=torch.tensor([10 ** 12, 100], device=DEV),
                                    cache_lens=torch.tensor([21, 20, 10 ** 15, 20], device=DEV))
    assert torch.equal(out, K.shared_prefix_attention(*x[:5], 100, 20))
    none = K.shared_prefix_attention(*x[:5], 100, 20, prefix_lens=torch.tensor([-5, 0], device=DEV))
    check(none, *x[:5], [0, 0], x[6])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("d", [64, 16])
def test_hidden_values_that_are_not_finite_stay_hidden(d, dtype):
    """A later token's K and V are infinite or NaN: the tokens before it are
    untouched, those that see it are not finite."""
    from minitp import kernels as K

    x = make(4, 2, 40, 4, 2, d, 70, 9, dtype)
    kc, vc = x[3], x[4]
    clean = K.shared_prefix_attention(*x[:5], 70, 9)
    vc[1, :, 9 + 30] = float("inf")
    kc[2, :, 9 + 20] = float("nan")
    vc[2, :, 9 + 20] = float("nan")
    out = K.shared_prefix_attention(*x[:5], 70, 9)
    assert torch.equal(out[0], clean[0]) and torch.equal(out[3], clean[3])
    ref, mag = reference(*x[:4], torch.where(torch.isfinite(vc), vc, 0.0), *x[5:])
    bar = bars(ref, mag, dtype, d).flatten(2).to(DEV) * 2  # (two results of one form each)
    for i, n in ((1, 30), (2, 20)):
        assert ((out[i, :n].double() - clean[i, :n].double()).abs() <= bar[i, :n] + 1e-9).all()
    assert not torch.isfinite(out[1, 30:]).any() and not torch.isfinite(out[2, 20:]).any()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("p", [100, 1500])
@pytest.mark.parametrize("hq,hkv,d,t", [(14, 2, 64, 1), (28, 4, 128, 40), (4, 2, 16, 3)])
def test_a_query_that_is_no_number_shows(hq, hkv, d, t, p, dtype):
    """Its own output is NaN, as its softmax is; no other row changes."""
    from minitp import kernels as K

    x = make(6, 2, t, hq, hkv, d, p, 33, dtype)
    clean = K.shared_prefix_attention(*x[:5], p, 33).view(6, t, hq, d)
    x[0][1, t - 1, 2, 5] = float("nan")
    out = K.shared_prefix_attention(*x[:5], p, 33).view(6, t, hq, d)
    assert torch.isnan(out[1, t - 1, 2]).all()
    out[1, t - 1, 2] = clean[1, t - 1, 2]
    assert torch.equal(out, clean)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_a_prefix_equals_the_same_rows_in_every_cache(dtype):
    """The prefix's rows copied in front of each row's own: the plain
    attention of the framework gives the same within both forms' bars."""
    from minitp import kernels as K

    x = make(6, 2, 1, 14, 2, 64, 130, 21, dtype)
    q, kp, vp, kc, vc, plens, clens = x
    k = torch.cat([kp[:, :, :130].repeat_interleave(3, 0), kc[:, :, :22]], 2)
    v = torch.cat([vp[:, :, :130].repeat_interleave(3, 0), vc[:, :, :22]], 2)
    _, mag = reference(*x)
    got = K.shared_prefix_attention(*x[:5], 130, 21).view(6, 1, 14, 64).double().cpu()
    plain = K.attention(q, k.contiguous(), v.contiguous(), 151).view(6, 1, 14, 64).double().cpu()
    # (both forms are within the bar of the formula)
    assert ((got - plain).abs() <= 2 * bars(mag, mag, dtype, 64)).all()


def test_cache_views_streams_and_graph():
    """Layer views of KVCache buffers, a side stream, and a captured call that is
    replayed with other contents and lengths between the program's own work."""
    from minitp import kernels as K
    from minitp.kv_cache import KVCache

    pre = KVCache(2, 2, 2, 64, 300, torch.bfloat16, torch.device(DEV), init="zeros")
    own = KVCache(2, 6, 2, 64, 50, torch.bfloat16, torch.device(DEV), init="zeros")
    for c in (pre, own):
        c.k_buf.normal_()
        c.v_buf.normal_()
    q = torch.randn(6, 1, 14, 64, device=DEV).bfloat16()
    plens, clens = torch.tensor([300, 211], device=DEV), torch.tensor([49, 0, 3, 17, 49, 30], device=DEV)

    def call():
        return K.shared_prefix_attention(q, pre.k[1], pre.v[1], own.k[1], own.v[1], 300, 49, plens, clens)

    def wanted():
        return reference(q, pre.k[1], pre.v[1], own.k[1], own.v[1], plens.tolist(), clens.tolist())

    def near(out):
        ref, mag = wanted()
        assert ((out.view(6, 1, 14, 64).double().cpu() - ref).abs() <= bars(ref, mag, q.dtype, 64) + 1e-9).all()

    eager = call()
    near(eager)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = call()
    side.synchronize()
    assert torch.equal(other, eager)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for step in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, call())
        near(out)
        q.normal_()
        clens.copy_((clens + 7) % 50)
        plens.copy_((plens + 41) % 301)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("hq,hkv,d", [(8, 8, 64), (28, 4, 128)])
def test_prompts_that_fill_the_chip(hq, hkv, d, dtype):
    """Rows whose own queries fill whole query tiles (one block over both
    parts), unequal, one idle."""
    from minitp import kernels as K

    b, t, p, c = 36, 130 * hkv // hq if hq > hkv else 130, 200, 70
    plens, clens = [p, 131], [c - i % 9 * 7 for i in range(b)]
    clens[5] = -1
    q, kp, vp, kc, vc, _, _ = make(b, 2, t, hq, hkv, d, p, c, dtype, plens, clens)
    out = K.shared_prefix_attention(q, kp, vp, kc, vc, p, c, torch.tensor(plens, device=DEV),
                                    torch.tensor(clens, device=DEV)).view(b, t, hq, d).double()
    assert (out[5] == 0).all()
    for i in range(b):
        if clens[i] < 0:
            continue
        g, per = i // (b // 2), hq // hkv
        k, v = (torch.cat([x[g, :, :plens[g]], y[i, :, :clens[i] + t]], 1).double().repeat_interleave(per, 0)
                for x, y in ((kp, kc), (vp, vc)))
        s = q[i].double().transpose(0, 1) @ k.transpose(-1, -2).contiguous() / d ** 0.5
        last = plens[g] + clens[i] + torch.arange(t, device=DEV)
        pr = s.masked_fill(torch.arange(k.shape[1], device=DEV) > last[:, None], float("-inf")).softmax(-1)
        ref, mag = (pr @ v).transpose(0, 1), (pr @ v.abs()).transpose(0, 1)
        assert ((out[i] - ref).abs() <= bars(ref, mag, dtype, d) + 1e-9).all(), i


def test_many_keys_and_rows():
    """A prefix and rows whose keys split over many blocks: against the product
    in 64 bits on the device."""
    from minitp import kernels as K

    for b, groups, p, c, dtype in ((40, 1, 5003, 333, torch.bfloat16), (6, 2, 3001, 1200, torch.float32),
                                   (24, 3, 777, 5, torch.bfloat16)):
        q, kp, vp, kc, vc, _, _ = x = make(b, groups, 1, 14, 2, 64, p, c, dtype)
        out = K.shared_prefix_attention(*x[:5], p, c).view(b, 14, 64).double()
        k = torch.cat([kp[:, :, :p].repeat_interleave(b // groups, 0), kc[:, :, :c + 1]], 2).double()
        v = torch.cat([vp[:, :, :p].repeat_interleave(b // groups, 0), vc[:, :, :c + 1]], 2).double()
        s = q.double().view(b, 2, 7, 64) @ k.transpose(-1, -2).contiguous() / 8
        pr = s.softmax(-1)
        ref, mag = (pr @ v).view(b, 14, 64), (pr @ v.abs()).view(b, 14, 64)
        assert ((out - ref).abs() <= bars(ref, mag, dtype, 64) + 1e-9).all()


@pytest.mark.parametrize("own", [False, True])
def test_keys_past_four_gib_of_a_head(own):
    """2^24 rows and some of 256 bytes, all zeros but for the last ones: one of
    those takes nearly all of a query's weight."""
    from minitp import kernels as K

    d, n = 128, (1 << 24) + 200
    long_k, long_v = (torch.zeros(1, 1, n + 8, d, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    short = torch.zeros(1, 1, 8, d, dtype=torch.bfloat16, device=DEV)
    q = torch.zeros(1, 1, 2, d, dtype=torch.bfloat16, device=DEV)
    for h, row in enumerate((n - 1, n - 150)):  # (256 n bytes are past 2^32)
        q[0, 0, h, h], long_k[0, 0, row, h] = 16.0, 20.0
        long_v[0, 0, row] = torch.arange(d, device=DEV) * (1 + h) / 64
    args = (short, short, long_k, long_v, 3, n - 1) if own else (long_k, long_v, short, short, n, 2)
    out = K.shared_prefix_attention(q, *args).view(2, d).double().cpu()
    weight = torch.tensor(16.0 * 20.0 / d ** 0.5, dtype=torch.float64).exp()
    ref = torch.stack([long_v[0, 0, r].double().cpu() for r in (n - 1, n - 150)]) * weight / (weight + n + 2)
    # the product's and the output's rounding, 2^-8 each; sums of 600 tiles of 32 and less in a row
    assert ((out - ref).abs() <= ref.abs() * (2 * 2 ** -8 + 2 * 600 * 32 * 2 ** -24)).all()
