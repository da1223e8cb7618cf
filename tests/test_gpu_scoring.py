"""Scoring of texts (minitp.scoring, TPQwen2ForCausalLM.forward_packed): packed
forwards against the oracle and against prompts on their own.

Bars. The suite's bar on logits (fp32 1e-3, bf16 0.5 on the device against the
oracle) carries over to a log-probability, a logit less a log sum of them, at
most twice. Two device paths on the same inputs: fp32 1e-5 of logits of at most
some units, bf16 0.05 and 2 % (the suite's bar for module against native).
"""

import torch

import pytest

from tests.conftest import ROOT  # noqa: F401  (puts the package on the path)

pytestmark = pytest.mark.gpu
DEV = "cuda"
BOTH = [torch.float32, torch.bfloat16]


def build(name, dtype, layers=None):
    import dataclasses

    from minitp.synthetic import SHAPES, build_synthetic_model

    cfg = SHAPES[name]
    if layers is not None:
        cfg = dataclasses.replace(cfg, num_hidden_layers=layers)
    return build_synthetic_model(cfg, dtype, DEV)


def texts_of(lens, vocab, seed=1):
    g = torch.Generator().manual_seed(seed)
    return [torch.randint(0, vocab, (n,), generator=g) for n in lens]


def alone(model, text):
    """float64 log-probabilities [T - 1, V] of a prompt on its own."""
    return torch.log_softmax(model(text[None].to(DEV))[0, :-1].double(), -1)


LENS = [5, 1, 40, 0, 130, 2, 17]


@pytest.mark.parametrize("dtype", BOTH)
def test_tiny_against_the_oracle(dtype):
    from minitp.scoring import score_tokens
    from oracle import qwen2_ref

    model = build("tiny", dtype)
    shape = qwen2_ref.TINY
    ref = qwen2_ref.OracleQwen2(shape, qwen2_ref.synthetic_state(shape, 0, dtype))
    bar = 2e-3 if dtype == torch.float32 else 1.0
    texts = texts_of(LENS, 1000)
    for text, r in zip(texts, score_tokens(model, texts, top=3)):
        if len(text) < 2:
            assert r.logprobs.numel() == 0
            continue
        lp = torch.log_softmax(ref.forward(text[None])[0, :-1].double(), -1)
        want = lp.gather(1, text[1:, None])[:, 0]
        assert ((r.logprobs.double().cpu() - want).abs() <= bar).all()
        assert ((r.entropy.double().cpu() + (lp.exp() * lp).sum(-1)).abs() <= bar).all()


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("name,layers", [("tiny", None), ("qwen2.5-0.5b", 2), ("qwen2.5-7b", 1)])
def test_against_prompts_on_their_own(name, layers, dtype):
    from minitp.scoring import score_tokens

    model = build(name, dtype, layers)
    texts = texts_of(LENS, model.cfg.vocab_size)
    got = score_tokens(model, texts, top=4)
    assert len(got) == len(texts)
    bar = 2e-3 if dtype == torch.float32 else 1.0
    for text, r in zip(texts, got):
        n = max(len(text) - 1, 0)
        assert r.logprobs.shape == r.entropy.shape == r.ranks.shape == (n,)
        assert r.top_tokens.shape == r.top_logprobs.shape == (n, 4)
        if n == 0:
            continue
        lp = alone(model, text)
        want = lp.gather(1, text[1:, None].to(DEV))[:, 0]
        assert ((r.logprobs.double() - want).abs() <= bar).all()
        assert ((r.top_logprobs.double() - lp.topk(4, -1).values).abs() <= bar).all()
        entropy = -(lp.exp() * lp).sum(-1)
        assert ((r.entropy.double() - entropy).abs() <= bar).all()
        # ranks and tokens fit the log-probabilities that came with them
        assert ((r.ranks == 0) == (r.top_tokens[:, 0] == text[1:].to(DEV))).all()
        for j in range(4):
            mine = r.ranks == j
            assert (r.top_tokens[mine, j] == text[1:].to(DEV)[mine]).all()
            assert torch.equal(r.top_logprobs[mine, j], r.logprobs[mine])


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("name,layers", [("tiny", None), ("qwen2.5-0.5b", 2)])
def test_module_path_and_native_program_agree(name, layers, dtype):
    model = build(name, dtype, layers)
    for lens in ([3], [1], [2, 1], [5, 1, 40, 0, 130], [256, 200] if layers is None else [700, 300]):
        ids = torch.cat(texts_of(lens, model.cfg.vocab_size)).to(DEV)
        native = model.forward_packed(ids, lens)
        model.model.layers[0].self_attn.use_fused_qkv = False
        assert not model.native_path()
        module = model.forward_packed(ids, lens)
        model.model.layers[0].self_attn.use_fused_qkv = True
        a, b = model.lm_head(native).double(), model.lm_head(module).double()
        bar = 1e-5 if dtype == torch.float32 else 0.05 + 0.02 * b.abs()
        assert ((a - b).abs() <= bar).all(), (a - b).abs().max()


def test_no_cached_rotary_tables():
    model = build("tiny", torch.float32)
    ids = torch.cat(texts_of([9, 4], 1000)).to(DEV)
    want = model.forward_packed(ids, [9, 4])
    model.use_rotary_cache = False
    got = model.forward_packed(ids, [9, 4])
    assert ((model.lm_head(want) - model.lm_head(got)).abs() <= 1e-5).all()


def test_greedy_texts_rank_first():
    """What generate_greedy picked is what the scores rank first."""
    from minitp.generation import generate_greedy
    from minitp.scoring import score_tokens

    model = build("qwen2.5-0.5b", torch.float32, 2)
    prompts = torch.stack(texts_of([20, 20, 20], model.cfg.vocab_size))
    out = generate_greedy(model, prompts.to(DEV), 12, early_stop=False)
    for r in score_tokens(model, list(out), top=2, starts=[20] * 3):
        assert r.ranks.shape == (12,)
        close = (r.top_logprobs[:, 0] - r.top_logprobs[:, 1]) <= 2e-3
        assert ((r.ranks == 0) | close).all()


def test_starts_batches_and_kinds_of_input():
    from minitp.scoring import score_tokens

    model = build("tiny", torch.float32)
    texts = texts_of(LENS, 1000)
    whole = score_tokens(model, texts, top=2)
    starts = [2, 1, 30, 1, 130, 5, 16]
    lists = [t.tolist() if i % 3 == 0 else t.to(DEV) if i % 3 == 1 else t.int() for i, t in enumerate(texts)]
    for limit in (16384, 130, 50, 1):
        part = score_tokens(model, lists, top=2, starts=starts, max_tokens=limit)
        for w, p, s in zip(whole, part, starts):
            n = max(w.logprobs.numel() - (s - 1), 0)
            assert p.logprobs.shape == (n,) and p.top_tokens.shape == (n, 2)
            if n:
                assert ((p.logprobs - w.logprobs[s - 1:]).abs() <= 2e-3).all()
    assert score_tokens(model, []) == []
    assert [r.logprobs.numel() for r in score_tokens(model, [[], [3]], top=1)] == [0, 0]


def test_many_rows_of_logits(monkeypatch):
    """More scored rows than go through the LM head at a time."""
    from minitp import scoring

    model = build("tiny", torch.float32)
    texts = texts_of([200, 3, 150], 1000)
    want = scoring.score_tokens(model, texts, top=3)
    monkeypatch.setattr(scoring, "LOGIT_ROWS", 64)
    for a, b in zip(want, scoring.score_tokens(model, texts, top=3)):
        assert ((a.logprobs - b.logprobs).abs() <= 2e-3).all() and a.top_tokens.shape == b.top_tokens.shape


def test_ids_outside_the_vocabulary():
    from minitp.scoring import score_tokens

    model = build("tiny", torch.float32)
    a, b = score_tokens(model, [[5, 6, 1000, 7, 8], [5, 6, 7]])
    assert torch.isfinite(a.logprobs[:1]).all() and torch.isnan(a.logprobs[1:]).all() and a.ranks[1] == -1
    assert torch.isfinite(b.logprobs).all()


def test_two_streams_at_once():
    from minitp.scoring import score_tokens

    model = build("qwen2.5-0.5b", torch.bfloat16, 2)
    x, y = texts_of([300, 20, 77], model.cfg.vocab_size, 1), texts_of([9, 500], model.cfg.vocab_size, 2)
    want = [score_tokens(model, t, top=3) for t in (x, y)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(3):
        got = []
        for s, t in zip(streams, (x, y)):
            with torch.cuda.stream(s):
                got.append(score_tokens(model, t, top=3))
        torch.cuda.synchronize()
        for g, w in zip(got, want):
            for p, q in zip(g, w):
                assert all(torch.equal(u, v) for u, v in zip(p, q))


def test_refusals():
    from minitp.scoring import score_tokens

    model = build("tiny", torch.float32)
    limit = model.cfg.max_position_embeddings
    score_tokens(model, [list(range(limit))])
    with pytest.raises(IndexError):
        score_tokens(model, [[1] * (limit + 1)])
    with pytest.raises(IndexError):
        model.forward_packed(torch.zeros(limit + 1, dtype=torch.long, device=DEV), [limit + 1])
    ids = torch.zeros(3, dtype=torch.long, device=DEV)
    for bad in ([1, 1], [7], [4, -1]):
        with pytest.raises(ValueError):
            model.forward_packed(ids, bad)
    with pytest.raises(ValueError):
        model.forward_packed(ids[None], [3])
    assert model.forward_packed(ids[:0], []).shape == (0, 64)
    assert model.forward_packed(ids[:0], [0, 0]).shape == (0, 64)
    for kw in (dict(top=-1), dict(top=33), dict(starts=[1]), dict(starts=[0, 1]), dict(max_tokens=0)):
        with pytest.raises(ValueError):
            score_tokens(model, [[1, 2], [3]], **kw)
    for bad in (torch.zeros(2, 3, dtype=torch.long), torch.zeros(3)):
        with pytest.raises(ValueError):
            score_tokens(model, [bad])


def test_no_capture():
    """Texts and lengths come from the host: refused inside a captured graph,
    which goes on without them, and right before and after."""
    from minitp.scoring import score_tokens

    model = build("tiny", torch.bfloat16)
    text = texts_of([40], 1000)[0]
    ids, x = text.to(DEV), torch.ones(8, device=DEV)
    before = score_tokens(model, [text])[0]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = x + 1
        with pytest.raises(RuntimeError, match="captured"):
            model.forward_packed(ids, [40])
        with pytest.raises(RuntimeError, match="captured"):
            score_tokens(model, [text])
        y = y * 3
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert (y == 6).all()
        after = score_tokens(model, [text])[0]
        assert all(torch.equal(a, b) for a, b in zip(before, after))
