"""Log-probabilities of given tokens (csrc/logprobs.hip) against float64 and a
stable sort.

Bars. The sum of exponentials runs in fp32 chains of at most 8 terms joined in
two more additions, then one addition and at most one rescaling (an exponential of 2
steps and a product) for each 4,096 logits; a term's exponential is off by 2
steps and by the rounding of its exponent, a step of x - m that weighs at most
log V < 14 steps in the sum. log turns the sum's relative error into an absolute
one. The result is rounded once, and log2(e) in fp32 is off by 2^-26 of itself.
The entropy's second sum carries the same steps of its own size, A = sum p (m - x).
Ranks and tokens have to be equal.
"""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
BOTH = [torch.bfloat16, torch.float32]
STEP = 2.0 ** -24


def reference(logits, tokens, top):
    """By rows, in float64 on the device: log-probabilities, entropy, ranks, the
    first tokens and theirs, A."""
    vocab = logits.shape[-1]
    x, t = logits.reshape(-1, vocab).double(), tokens.reshape(-1)
    order = torch.where(torch.isnan(x), math.inf, x)
    # NaN before plus infinity: sorted by (is NaN, value), both stable
    first = order.sort(dim=-1, descending=True, stable=True).indices
    nan_first = torch.isnan(x).gather(1, first).to(torch.int8).sort(dim=-1, descending=True, stable=True).indices
    places = first.gather(1, nan_first)
    inside = (t >= 0) & (t < vocab)
    tt = t.clamp(0, vocab - 1)
    ranks = (places == tt[:, None]).int().argmax(-1)
    lp = torch.log_softmax(x, -1)
    m = x.amax(-1, keepdim=True)
    p = lp.exp()
    entropy = -torch.where(p > 0, p * lp, torch.zeros_like(p)).sum(-1)
    entropy = torch.where(torch.isnan(lp).any(-1), math.nan, entropy)
    spread = torch.where(p > 0, p * (m - x), torch.zeros_like(p)).sum(-1)
    best = places[:, :top]
    nan = torch.full_like(lp[:, 0], math.nan)
    return (torch.where(inside, lp.gather(1, tt[:, None])[:, 0], nan), entropy, torch.where(inside, ranks, -1), best,
            lp.gather(1, best), spread)


def close(got, ref, bar):
    got = got.double().reshape(ref.shape)
    assert torch.equal(torch.isnan(got), torch.isnan(ref))
    there = torch.isfinite(ref)
    assert torch.equal(got[~there & ~torch.isnan(ref)], ref[~there & ~torch.isnan(ref)])
    err = (got - ref).abs()
    assert (err <= bar)[there].all(), (err / bar)[there].max()


def check(r, logits, tokens, top):
    vocab = logits.shape[-1]
    lp, entropy, ranks, best, best_lp, spread = reference(logits, tokens, top)
    steps = (8 + 2 + 2 + 14 + 4 * math.ceil(vocab / 4096)) * STEP
    assert r.logprobs.dtype == r.entropy.dtype == r.top_logprobs.dtype == torch.float32
    assert r.ranks.dtype == r.top_tokens.dtype == torch.long
    assert r.logprobs.shape == r.entropy.shape == r.ranks.shape == tokens.shape
    assert r.top_tokens.shape == r.top_logprobs.shape == (*tokens.shape, top)
    assert torch.equal(r.ranks.reshape(-1), ranks)
    assert torch.equal(r.top_tokens.reshape(best.shape), best)
    close(r.logprobs, lp, steps + lp.abs() * 1.5 * STEP)
    close(r.top_logprobs, best_lp, steps + best_lp.abs() * 1.5 * STEP)
    close(r.entropy, entropy, steps * (2 + 2 * spread) + entropy.abs() * 1.5 * STEP)


def make(rows, vocab, dtype, seed=0, std=2.5):
    g = torch.Generator(device=DEV).manual_seed(seed + rows * 31 + vocab)
    logits = (torch.randn(rows, vocab, generator=g, device=DEV) * std).to(dtype)
    tokens = torch.randint(0, vocab, (rows,), generator=g, device=DEV)
    tokens[::3] = logits[::3].float().argmax(-1)
    return logits, tokens


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("vocab", [1, 2, 7, 63, 64, 65, 1000, 4096, 4097, 8192, 20011, 151936, 152064])
@pytest.mark.parametrize("rows,top", [(1, 1), (3, 0), (5, 20), (2, 32), (33, 5)])
def test_rows(rows, top, vocab, dtype):
    from minitp import kernels as K

    x = make(rows, vocab, dtype)
    top = min(top, vocab)
    check(K.token_logprobs(*x, top=top), *x, top)


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("rows,vocab", [(700, 1000), (2100, 8193), (3000, 64), (513, 50007)])
def test_many_rows(rows, vocab, dtype):
    from minitp import kernels as K

    x = make(rows, vocab, dtype)
    for top in (0, 7, 32):
        check(K.token_logprobs(*x, top=top), *x, top)


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("vocab", [3, 33, 255, 1017, 1021, 1022, 1025, 2040, 2041, 2042, 2049])
def test_small_vocabularies(vocab, dtype):
    """Around the sizes that one turn of a chunk a thread takes, rows at every
    alignment."""
    from minitp import kernels as K

    for rows in (9, 700):
        logits, tokens = make(rows, vocab, dtype)
        for top in (0, 1, min(5, vocab), min(32, vocab)):
            check(K.token_logprobs(logits, tokens, top=top), logits, tokens, top)
        flat = torch.zeros_like(logits)
        check(K.token_logprobs(flat, tokens, top=min(32, vocab)), flat, tokens, min(32, vocab))


@pytest.mark.parametrize("rows", [1, 40, 600])
@pytest.mark.parametrize("dtype", BOTH)
def test_equal_logits_go_to_the_lower_token(dtype, rows):
    """All equal, few values, signed zeros, one slope up and one down."""
    from minitp import kernels as K

    g = torch.Generator(device=DEV).manual_seed(6)
    vocab = 9001
    tokens = torch.randint(0, vocab, (rows,), generator=g, device=DEV)
    for logits in (torch.zeros(rows, vocab, device=DEV), torch.full((rows, vocab), -1e30, device=DEV),
                   torch.randint(0, 3, (rows, vocab), generator=g, device=DEV).float(),
                   torch.where(torch.rand(rows, vocab, generator=g, device=DEV) < 0.5, 0.0, -0.0),
                   torch.linspace(-8, 8, vocab, device=DEV).repeat(rows, 1),
                   torch.linspace(8, -8, vocab, device=DEV).repeat(rows, 1)):
        logits = logits.to(dtype)
        check(K.token_logprobs(logits, tokens, top=32), logits, tokens, 32)


@pytest.mark.parametrize("rows", [6, 600])
@pytest.mark.parametrize("dtype", BOTH)
def test_masked_infinite_and_nan_logits(dtype, rows):
    from minitp import kernels as K

    vocab = 5003
    logits, tokens = make(rows, vocab, dtype, seed=3)
    low = torch.finfo(dtype).min
    logits[0, 100:] = -math.inf            # masked
    logits[1, 3:] = low                    # masked by the lowest value
    logits[2] = -math.inf                  # nothing left
    logits[3, 4000] = math.inf
    logits[4, 17] = math.nan
    logits[4, 4999] = math.nan
    logits[5] = low
    tokens[0], tokens[1], tokens[3], tokens[4] = 101, 2, 4000, 4999
    check(K.token_logprobs(logits, tokens, top=32), logits, tokens, 32)
    tokens[0], tokens[1], tokens[3], tokens[4] = 99, 5002, 0, 5
    check(K.token_logprobs(logits, tokens, top=5), logits, tokens, 5)
    logits[4] = math.nan
    logits[3] = math.inf
    check(K.token_logprobs(logits, tokens, top=32), logits, tokens, 32)


@pytest.mark.parametrize("dtype", BOTH)
def test_tokens_outside_the_vocabulary(dtype):
    from minitp import kernels as K

    logits, tokens = make(6, 3001, dtype)
    tokens[0], tokens[2], tokens[4] = -1, 3001, 1 << 40
    tokens[5] = -(1 << 40)
    check(K.token_logprobs(logits, tokens, top=3), logits, tokens, 3)


@pytest.mark.parametrize("dtype", BOTH)
def test_flat_peaked_and_far_logits(dtype):
    from minitp import kernels as K

    for std, shift in ((0.0, 5.0), (1e-3, 0.0), (40.0, 0.0), (2.0, 1000.0), (2.0, -30000.0), (1e4, 0.0)):
        logits, tokens = make(9, 20011, torch.float32, seed=8, std=std)
        logits = (logits + shift).to(dtype)
        check(K.token_logprobs(logits, tokens, top=4), logits, tokens, 4)


@pytest.mark.parametrize("dtype", BOTH)
def test_shapes_and_strides(dtype):
    """[..., V] of any leading shape; rows apart, odd widths, one row for all,
    columns in another order."""
    from minitp import kernels as K

    logits, tokens = make(24, 3001, dtype)
    want = K.token_logprobs(logits, tokens, top=6)
    for shape in ((2, 12), (4, 1, 6), (24, 1), (1, 24)):
        r = K.token_logprobs(logits.view(*shape, 3001), tokens.view(shape), top=6)
        for a, b in zip(r, want):
            assert torch.equal(a.reshape(b.shape), b)
    one = K.token_logprobs(logits[3], tokens[3], top=6)
    assert one.logprobs.shape == () and torch.equal(one.top_tokens, want.top_tokens[3])
    wide = torch.full((24, 3777), math.nan, dtype=dtype, device=DEV)
    for shift in range(9):
        wide[:, shift:shift + 3001] = logits
        r = K.token_logprobs(wide[:, shift:shift + 3001], tokens, top=6)
        check(r, logits, tokens, 6)
        wide[:, shift:shift + 3001] = math.nan
    last = torch.stack([logits, logits * 0], 1)
    check(K.token_logprobs(last[:, 0], tokens, top=6), logits, tokens, 6)
    check(K.token_logprobs(last[:, :1], tokens[:, None], top=6), logits[:, None], tokens[:, None], 6)
    same = logits[5].expand(24, 3001)
    check(K.token_logprobs(same, tokens, top=6), same.contiguous(), tokens, 6)
    turned = logits.t().contiguous().t()
    check(K.token_logprobs(turned, tokens, top=6), logits, tokens, 6)
    assert all(torch.equal(a, b) for a, b in zip(K.token_logprobs(logits, tokens.view(24, 1).expand(24, 2)[:, 0], top=6), want))


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("rows", [2, 520])
def test_best_sets_in_few_threads(dtype, rows):
    """A long row in which only sets of 64 logits that an eighth of the threads
    look through stand out, so that more of them pass than the list of a block
    holds (1,953 of 15,625 at a million logits)."""
    from minitp import kernels as K

    vocab = 1_000_000
    g = torch.Generator(device=DEV).manual_seed(12)
    one = torch.randn(2, vocab, generator=g, device=DEV)
    sets = torch.arange(0, vocab, 64, device=DEV)
    sets = sets[sets // 64 % 256 < 32]
    one[0, sets] += 20 + torch.rand(sets.numel(), generator=g, device=DEV)
    one[1, sets + 17] += 20
    logits = one.to(dtype)
    tokens = torch.tensor([64 * 5, 3], device=DEV)
    r = K.token_logprobs(logits.repeat(rows // 2, 1), tokens.repeat(rows // 2), top=32)
    for i in (0, rows - 2):
        check(type(r)(*(t[i:i + 2] for t in r)), logits, tokens, 32)


def test_rank_zero_is_the_greedy_pick():
    from minitp import kernels as K

    for rows in (3, 700):
        logits, _ = make(rows, 9001, torch.bfloat16)
        r = K.token_logprobs(logits, K.argmax(logits), top=1)
        assert (r.ranks == 0).all() and torch.equal(r.top_tokens[:, 0], K.argmax(logits))
        assert torch.equal(r.top_logprobs[:, 0], r.logprobs)


def test_graph_and_streams():
    from minitp import kernels as K

    a, b = make(4, 20011, torch.bfloat16, seed=1), make(4, 20011, torch.bfloat16, seed=2)
    many = make(700, 5000, torch.float32, seed=3)
    logits, tokens = a[0].clone(), a[1].clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        K.token_logprobs(logits, tokens, top=9)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        r = K.token_logprobs(logits, tokens, top=9)
    for i in range(6):
        x = (a, b)[i % 2]
        logits.copy_(x[0])
        tokens.copy_(x[1])
        with torch.cuda.stream(side):
            beside = K.token_logprobs(*many, top=5)
        graph.replay()
        want = K.token_logprobs(*x, top=9)
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(r, want))
        check(beside, *many, 5)
    check(r, *b, 9)


def test_offsets_past_32_bits():
    """Rows that begin past 2^32 elements, and a long row."""
    from minitp import kernels as K

    for dtype in BOTH:
        store = torch.zeros(3 << 31, dtype=dtype, device=DEV).view(3, 1 << 31)
        x, t = make(3, 5001, dtype)
        rows = store[:, (1 << 31) - 6000:(1 << 31) - 999]
        rows.copy_(x)
        check(K.token_logprobs(rows, t, top=4), x, t, 4)
        del store, rows
    x, t = make(2, 3_000_017, torch.float32)
    check(K.token_logprobs(x, t, top=11), x, t, 11)


def test_nothing():
    from minitp import kernels as K

    r = K.token_logprobs(torch.empty(0, 100, device=DEV), torch.empty(0, dtype=torch.long, device=DEV), top=3)
    assert r.logprobs.shape == (0,) and r.top_tokens.shape == (0, 3)
