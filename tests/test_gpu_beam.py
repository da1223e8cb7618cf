"""Beam selection and cache reordering (csrc/beam.hip) against plain forms: the
selection by a full stable sort in 64 bits, the reordering by indexing.

Bar of a score: its sum over the vocabulary is off by at most 20 steps (chains of
8 terms and 2 more additions in fp32, two exponentials of 2 steps each, a
wave's and its part's weight, the rest in 64 bits), which the logarithm turns
into as much of an absolute error; the result is rounded once.
Tokens, parents, flags and lengths have to be equal.
"""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


def reference(logits, scores, finished, lengths, eos, alpha):
    """(tokens, parents, scores, finished, lengths) as lists [G][W], from the
    definition."""
    groups, beams, vocab = logits.shape
    out = ([], [], [], [], [])
    for g in range(groups):
        done = [bool(f) for f in finished[g]] if finished is not None else [False] * beams
        lens = lengths[g].tolist() if lengths is not None else [0] * beams
        lp = torch.full((beams, vocab), -math.inf, dtype=torch.float64)
        for w in range(beams):
            s, x = float(scores[g, w]), logits[g, w].double().cpu()
            if s == -math.inf:
                continue
            if done[w]:
                lp[w, eos] = s
            elif (x == -math.inf).all():
                continue
            else:
                lp[w] = s + torch.log_softmax(x, -1)
        norm = torch.tensor([max(1, n + (not d)) for n, d in zip(lens, done)], dtype=torch.float64) ** alpha
        key = (lp / norm[:, None]).flatten()
        key = torch.where(torch.isnan(key), math.inf, key) if torch.isnan(key).any() else key
        rank = [f for f in key.sort(descending=True, stable=True).indices[:beams].tolist() if key[f] > -math.inf]
        slots, late = [None] * beams, []
        for f in rank:
            if slots[f // vocab] is None:
                slots[f // vocab] = f
            else:
                late.append(f)
        for i in range(beams):
            if slots[i] is None and late:
                slots[i] = late.pop(0)
        row = [[], [], [], [], []]
        for i, f in enumerate(slots):
            p = i if f is None else f // vocab
            row[0].append(max(eos, 0) if f is None else f % vocab)
            row[1].append(g * beams + p)
            row[2].append(-math.inf if f is None else float(lp[p, f % vocab]))
            row[3].append(True if f is None else done[p] or f % vocab == eos)
            row[4].append(lens[p] + (f is not None and not done[p]))
        for o, r in zip(out, row):
            o.append(r)
    return out


def compare(step, want):
    tokens, parents, scores, finished, lengths = want
    assert step.tokens.tolist() == tokens
    assert step.parents.tolist() == parents
    assert step.finished.tolist() == finished
    assert step.lengths.tolist() == lengths
    got, ref = step.scores.double().cpu(), torch.tensor(scores, dtype=torch.float64)
    assert torch.equal(torch.isnan(got), torch.isnan(ref))
    there = torch.isfinite(ref)
    assert torch.equal(got[~there & ~torch.isnan(ref)], ref[~there & ~torch.isnan(ref)])
    assert ((got - ref)[there].abs() <= 20 * 2 ** -24 + ref[there].abs() * 2 ** -24).all()


def make(groups, beams, vocab, dtype, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed + groups * 31 + beams * 7 + vocab)
    logits = (torch.randn(groups, beams, vocab, generator=g, device=DEV) * 2.5).to(dtype)
    scores = -torch.rand(groups, beams, generator=g, device=DEV) * 3 - 5
    return logits, scores, g


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("beams", [1, 2, 3, 5, 8, 16, 17, 32])
@pytest.mark.parametrize("vocab", [1, 7, 33, 1000, 4096, 4097, 20011])
def test_selection(vocab, beams, dtype):
    from minitp import kernels as K

    logits, scores, _ = make(3, beams, vocab, dtype)
    compare(K.beam_select(logits, scores), reference(logits, scores, None, None, -1, 0.0))


@pytest.mark.parametrize("alpha", [0.0, 0.7, 1.0, -0.5, 16.0])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_finished_beams_lengths_and_empty_slots(dtype, alpha):
    from minitp import kernels as K

    logits, scores, g = make(5, 8, 3001, dtype, seed=5)
    finished = torch.rand(5, 8, generator=g, device=DEV) < 0.4
    finished[2], finished[3] = True, False
    lengths = torch.randint(0, 60, (5, 8), generator=g, device=DEV)
    scores[0, 3:], scores[4], scores[3, 0] = -math.inf, -math.inf, 0.0
    logits[1, 2] = -math.inf  # nothing may follow this beam
    logits[3, :, 50:] = -math.inf
    logits[3, :, 11] = 30.0  # the end token, far ahead
    step = K.beam_select(logits, scores, finished, lengths, eos_token_id=11, length_penalty=alpha)
    compare(step, reference(logits, scores, finished, lengths, 11, alpha))
    # (the outputs are the next call's inputs)
    again = K.beam_select(logits, step.scores, step.finished, step.lengths, eos_token_id=11, length_penalty=alpha)
    compare(again, reference(logits, step.scores, step.finished, step.lengths, 11, alpha))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_equal_keys_go_to_the_lower_beam_and_token(dtype):
    from minitp import kernels as K

    # everything equal; equal beams; a few values over a long row; signed zeros
    flat = torch.zeros(2, 32, 9001, device=DEV, dtype=dtype)
    scores = torch.full((2, 32), -1.0, device=DEV)
    scores[1, :7] = -2.0
    compare(K.beam_select(flat, scores), reference(flat, scores, None, None, -1, 0.0))
    g = torch.Generator(device=DEV).manual_seed(3)
    coarse = torch.randint(0, 3, (2, 1, 9001), generator=g, device=DEV).to(dtype).expand(2, 32, 9001)
    compare(K.beam_select(coarse, scores), reference(coarse, scores, None, None, -1, 0.0))
    zeros = torch.where(torch.rand(1, 4, 5000, generator=g, device=DEV) < 0.5, 0.0, -0.0).to(dtype)
    compare(K.beam_select(zeros, torch.zeros(1, 4, device=DEV)),
            reference(zeros, torch.zeros(1, 4), None, None, -1, 0.0))


def test_sorted_rows_and_one_beam_ahead():
    """The best tokens side by side in one slice, all from one beam."""
    from minitp import kernels as K

    up = torch.linspace(-8, 8, 30000, device=DEV).expand(1, 32, 30000).contiguous()
    scores = -torch.arange(32, device=DEV, dtype=torch.float32)[None] * 20
    compare(K.beam_select(up, scores), reference(up, scores, None, None, -1, 0.0))
    down = up.flip(-1).contiguous()
    compare(K.beam_select(down, scores), reference(down, scores, None, None, -1, 0.0))


def test_nan_and_infinite_logits():
    from minitp import kernels as K

    logits, scores, _ = make(4, 4, 5003, torch.float32, seed=9)
    logits[0, 2, 4999] = math.nan
    logits[1, 1, 17] = math.inf
    scores[2, 3] = math.nan
    logits[3, :, ::3] = -math.inf
    step = K.beam_select(logits, scores)
    # a beam whose sum is no number: its lowest tokens, above every number
    assert torch.isnan(step.scores[:3]).all()
    assert sorted(step.tokens[0].tolist()) == sorted(step.tokens[1].tolist()) == [0, 1, 2, 3]
    assert (step.parents[0] == 2).all() and (step.parents[1] == 4 + 1).all() and (step.parents[2] == 8 + 3).all()
    want = reference(logits[3:], scores[3:], None, None, -1, 0.0)
    assert step.tokens[3:].tolist() == want[0] and (step.parents[3:] - 12).tolist() == want[1]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_logits_masked_by_the_lowest_value(dtype):
    """Masks of the type's lowest value and far below the rest; a row of
    nothing else is an even choice, as its softmax is."""
    from minitp import kernels as K

    logits, scores, _ = make(3, 5, 6007, dtype, seed=11)
    low = torch.finfo(dtype).min
    logits[0, :, 1::2] = low
    logits[1, 2] = low
    logits[1, 3, 9:] = low
    logits[2, :, 40:6000] = -1e30
    compare(K.beam_select(logits, scores), reference(logits, scores, None, None, -1, 0.0))


def test_scores_far_beyond_the_logits():
    """Scores so large that neighbouring logits give equal keys in 64 bits:
    the lower token of them wins."""
    from minitp import kernels as K

    logits, scores, _ = make(4, 6, 9001, torch.float32, seed=21)
    scores[0] *= 1e12
    scores[1] = -2.0 ** 50
    scores[2, 1:] = -2.0 ** 45
    scores[3] = 2.0 ** 40
    step, want = K.beam_select(logits, scores), reference(logits, scores, None, None, -1, 0.0)
    # a key of 2^50 has steps of 2^-3: the two forms' sums of three may round one step apart
    for g in range(4):
        key = logits[g].double().log_softmax(-1).cpu() + scores[g].double().cpu()[:, None]
        picked = [key[p - 6 * g, t].item() for t, p in zip(step.tokens[g].tolist(), step.parents[g].tolist())]
        best = [key[p - 6 * g, t].item() for t, p in zip(want[0][g], want[1][g])]
        step_of = 2.0 ** -52 * max(abs(b) for b in best)
        assert all(abs(a - b) <= 2 * step_of for a, b in zip(sorted(picked), sorted(best)))
        assert len(set(zip(step.tokens[g].tolist(), step.parents[g].tolist()))) == 6


def test_outputs_over_the_inputs():
    """The C entry's outputs may be its inputs."""
    from minitp import _native as N
    from minitp import kernels as K

    logits, scores, g = make(4, 7, 2000, torch.bfloat16, seed=3)
    finished = torch.rand(4, 7, generator=g, device=DEV) < 0.3
    lengths = torch.randint(0, 9, (4, 7), generator=g, device=DEV)
    want = K.beam_select(logits, scores, finished, lengths, eos_token_id=3, length_penalty=1.0)
    size = N.lib().minitp_beam_select_workspace_bytes(4, 7, 2000)
    ws = torch.empty(size, dtype=torch.uint8, device=DEV)
    tokens, parents = (torch.empty(4, 7, dtype=torch.long, device=DEV) for _ in range(2))
    N.check(N.lib().minitp_beam_select(N.stream(), N.BF16, logits.data_ptr(), 7 * 2000, 2000, 4, 7, 2000, scores.data_ptr(),
                                       finished.data_ptr(), lengths.data_ptr(), 3, 1.0, tokens.data_ptr(),
                                       parents.data_ptr(), scores.data_ptr(), finished.data_ptr(), lengths.data_ptr(),
                                       ws.data_ptr(), size), "beam_select")
    for got, w in zip((tokens, parents, scores, finished, lengths), want):
        assert torch.equal(got, w)


def test_first_step_from_one_row_and_strided_rows():
    from minitp import kernels as K

    logits, scores, _ = make(3, 1, 4099, torch.bfloat16)
    start = torch.full((3, 6), -math.inf, device=DEV)
    start[:, 0] = 0.0
    rows = logits.expand(3, 6, 4099)
    step = K.beam_select(rows, start)
    compare(step, reference(rows, start, None, None, -1, 0.0))
    assert (step.parents == torch.arange(3, device=DEV)[:, None] * 6).all()  # every beam continues the prompt
    wide = torch.randn(6, 5000, device=DEV)
    cut = wide[:, 3:4102]  # rows that start at odd addresses
    got = K.beam_select(cut, torch.zeros(2, 3, device=DEV))
    compare(got, reference(cut.reshape(2, 3, -1), torch.zeros(2, 3), None, None, -1, 0.0))
    turned = torch.randn(1000, 4, device=DEV).t().unflatten(0, (2, 2))
    compare(K.beam_select(turned, torch.zeros(2, 2, device=DEV)),
            reference(turned, torch.zeros(2, 2), None, None, -1, 0.0))


@pytest.mark.parametrize("beams", [2, 6, 16, 17, 32])
@pytest.mark.parametrize("vocab", [500, 70001, 151936])
def test_few_open_beams(vocab, beams):
    """One open beam a group (a search's first step), a few, and one beside
    finished ones, over short and long rows."""
    from minitp import kernels as K

    logits, scores, g = make(4, beams, vocab, torch.bfloat16)
    finished = torch.zeros(4, beams, dtype=torch.bool, device=DEV)
    scores[0, 1:] = -math.inf
    scores[1, : beams - 1] = -math.inf
    finished[2] = True
    finished[2, beams // 2] = False
    scores[2, beams // 2] += 4.0
    scores[3, beams // 3 :] = -math.inf
    lengths = torch.full((4, beams), 3, device=DEV)
    step = K.beam_select(logits, scores, finished, lengths, eos_token_id=7, length_penalty=0.5)
    compare(step, reference(logits, scores, finished, lengths, 7, 0.5))


def test_large_vocabulary():
    from minitp import kernels as K

    logits, scores, g = make(2, 8, 151936, torch.bfloat16)
    finished = torch.zeros(2, 8, dtype=torch.bool, device=DEV)
    finished[1, 4] = True
    lengths = torch.full((2, 8), 6, device=DEV)
    step = K.beam_select(logits.view(16, -1), scores, finished, lengths, eos_token_id=151643, length_penalty=1.0)
    compare(step, reference(logits, scores, finished, lengths, 151643, 1.0))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("groups,beams", [(1, 1), (1, 4), (2, 8), (3, 5), (1, 13), (2, 32)])
@pytest.mark.parametrize("hkv,s,d,rows", [(2, 64, 64, 15), (1, 33, 128, 33), (2, 40, 16, 1), (3, 300, 32, 257)])
def test_reorder(hkv, s, d, rows, groups, beams, dtype):
    """Any parents: permutations, a beam for all, chains, rows that stay."""
    from minitp import kernels as K

    g = torch.Generator(device=DEV).manual_seed(beams * 100 + rows)
    base = torch.arange(groups, device=DEV)[:, None] * beams
    turn = (torch.arange(beams, device=DEV) + 1) % beams
    for parents in (torch.randint(0, beams, (groups, beams), generator=g, device=DEV),
                    turn.expand(groups, beams), torch.full((groups, beams), beams - 1, device=DEV),
                    torch.arange(beams, device=DEV).expand(groups, beams)):
        k = torch.randn(2, groups * beams, hkv, s, d, generator=g, device=DEV).to(dtype)
        v = torch.randn(2, groups * beams, hkv, s, d, generator=g, device=DEV).to(dtype)
        p = parents + base
        want = [x.clone() for x in (k, v)]
        for w, x in zip(want, (k, v)):
            w[:, :, :, :rows] = x[:, p.flatten(), :, :rows]
        K.kv_reorder(k, v, p, rows)
        assert torch.equal(k, want[0]) and torch.equal(v, want[1])


def test_reorder_leaves_rows_with_foreign_parents():
    from minitp import kernels as K

    k, v = torch.randn(2, 2, 6, 2, 16, 16, device=DEV).unbind(0)
    k, v = k.contiguous(), v.contiguous()
    want = [x.clone() for x in (k, v)]
    parents = torch.tensor([[1, 5, -1], [4, 2, 10 ** 12]], device=DEV)  # rows 0 and 3 have parents in their group
    for x in want:
        new = x.clone()
        new[:, 0, :, :9] = x[:, 1, :, :9]
        new[:, 3, :, :9] = x[:, 4, :, :9]
        x.copy_(new)
    K.kv_reorder(k, v, parents, 9)
    assert torch.equal(k, want[0]) and torch.equal(v, want[1])


def test_reorder_of_no_rows_and_the_cache_method():
    from minitp.kv_cache import KVCache

    kv = KVCache(2, 6, 2, 64, 40, torch.bfloat16, torch.device(DEV), init="zeros")
    kv.k_buf.normal_()
    kv.v_buf.normal_()
    k, v = kv.k_buf.clone(), kv.v_buf.clone()
    parents = torch.tensor([[0, 0, 2], [5, 4, 4]], device=DEV)
    kv.reorder(parents)  # nothing cached yet
    assert torch.equal(kv.k_buf, k) and torch.equal(kv.v_buf, v)
    kv.advance(11)
    kv.reorder(parents)
    k[:, :, :, :11] = k[:, parents.flatten(), :, :11]
    v[:, :, :, :11] = v[:, parents.flatten(), :, :11]
    assert torch.equal(kv.k_buf, k) and torch.equal(kv.v_buf, v)


def test_selection_and_reorder_in_a_graph_and_on_a_side_stream():
    """The two calls of a step captured together; the replays follow the logits
    that they find, beside the program's own eager work."""
    from minitp import kernels as K

    logits, scores, _ = make(2, 4, 9001, torch.bfloat16)
    k, v = torch.randn(2, 2, 8, 2, 32, 64, device=DEV).bfloat16().unbind(0)
    k, v = k.contiguous(), v.contiguous()

    def step():
        s = K.beam_select(logits, scores)
        K.kv_reorder(k, v, s.parents, 20)
        return s

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        first = step()
    side.synchronize()
    compare(first, reference(logits, scores, None, None, -1, 0.0))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        s = step()
    for _ in range(3):
        logits.normal_(0, 2.5)
        before = k.clone()
        graph.replay()
        torch.cuda.synchronize()
        compare(s, reference(logits, scores, None, None, -1, 0.0))
        want = before.clone()
        want[:, :, :, :20] = before[:, s.parents.flatten(), :, :20]
        assert torch.equal(k, want)
        eager = K.beam_select(logits, scores)
        assert all(torch.equal(a, b) for a, b in zip(eager, s))


def test_offsets_past_32_bits():
    """Rows of logits 2^31 elements apart, caches of more than 4 GiB a beam row."""
    from minitp import kernels as K

    far = (1 << 31) + 24
    flat = torch.empty(far + 8000, dtype=torch.bfloat16, device=DEV)
    logits = flat.as_strided((2, 4, 2000), (far, 2000, 1))
    src, scores, g = make(2, 4, 2000, torch.bfloat16, seed=4)
    logits.copy_(src)
    compare(K.beam_select(logits, scores), reference(src, scores, None, None, -1, 0.0))
    del flat, logits
    k, v = (torch.empty(1, 3, 2, (1 << 23) + 16, 128, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    for x in (k, v):
        x[:, :, :, :40] = torch.randn(1, 3, 2, 40, 128, generator=g, device=DEV)
    parents = torch.tensor([[2, 0, 1]], device=DEV)
    want = [x[:, [2, 0, 1], :, :33] for x in (k, v)]
    rest = [x[:, :, :, 33:40].clone() for x in (k, v)]
    K.kv_reorder(k, v, parents, 33)
    for x, w, r in zip((k, v), want, rest):
        assert torch.equal(x[:, :, :, :33], w) and torch.equal(x[:, :, :, 33:40], r)


def test_calls_on_two_streams_at_once():
    """Selections and attention queued on two streams: scratch of their own."""
    from minitp import kernels as K

    logits, scores, g = make(6, 8, 20000, torch.float32)
    q = torch.randn(12, 1, 8, 64, generator=g, device=DEV)
    pre, own = torch.randn(2, 2, 900, 64, generator=g, device=DEV), torch.randn(12, 2, 60, 64, generator=g, device=DEV)
    calls = (lambda: list(K.beam_select(logits, scores)), lambda: [K.shared_prefix_attention(q, pre, pre, own, own, 900, 59)])
    want = [c() for c in calls]
    streams = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    outs = []
    for i in range(12):
        with torch.cuda.stream(streams[i % 2]):
            outs.append([c() for c in calls])
    torch.cuda.synchronize()
    for out in outs:
        assert all(torch.equal(a, b) for got, ref in zip(out, want) for a, b in zip(got, ref))
