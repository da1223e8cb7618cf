"""Beam search and generation under a shared prefix, whole: the tiny and the
2-layer 0.5B-shaped model against the oracle run over the full sequences (no
cache, no sharing), and the shared forms against the plain ones."""

import dataclasses

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _pair(name, dtype=torch.float32):
    """(model, oracle) of the same seeded weights."""
    from minitp import synthetic
    from oracle import qwen2_ref

    cfg = synthetic.SHAPES[name]
    cfg = dataclasses.replace(cfg, num_hidden_layers=2, max_position_embeddings=256)
    shape = qwen2_ref.Qwen2Shape(**dataclasses.asdict(cfg))
    model = synthetic.build_synthetic_model(cfg, dtype=dtype, device=DEV, seed=0)
    state = {k: v.cpu() for k, v in model.state_dict().items()}
    if "lm_head.weight" not in state:
        state["lm_head.weight"] = state["model.embed_tokens.weight"]
    return model, qwen2_ref.OracleQwen2(shape, state)


def _reference_beams(oracle, prompt, steps, beams, eos, alpha):
    """[(score, tokens)] best first for one prompt: every step runs the whole
    sequence of every beam and sorts every continuation."""
    live = [(0.0, [], False)]
    for _ in range(steps):
        grown = []
        for score, toks, done in live:
            if done:
                grown.append((score, toks + [eos], True, max(1, toks.index(eos) + 1)))
                continue
            ids = torch.cat([prompt, torch.tensor(toks, dtype=torch.long)])[None]
            lp = torch.log_softmax(oracle.forward(ids)[0, -1].double(), -1)
            best = lp.sort(descending=True, stable=True)
            for v, i in zip(best.values[:beams].tolist(), best.indices[:beams].tolist()):
                grown.append((score + v, toks + [i], i == eos, len(toks) + 1))
        grown.sort(key=lambda c: -c[0] / c[3] ** alpha)
        live = [c[:3] for c in grown[:beams]]
    return live


@pytest.mark.parametrize("alpha", [0.0, 1.0])
@pytest.mark.parametrize("name,beams,steps", [("tiny", 4, 9), ("tiny", 1, 5), ("qwen2.5-0.5b", 3, 5)])
def test_beam_search_matches_the_oracle(name, beams, steps, alpha):
    from minitp.generation import generate_beam

    model, oracle = _pair(name)
    g = torch.Generator().manual_seed(beams + steps)
    prompts = torch.randint(0, model.cfg.vocab_size, (2, 11), generator=g)
    eos = None
    for _ in range(2):
        ids, scores = generate_beam(model, prompts.to(DEV), steps, beams, eos_token_id=eos, length_penalty=alpha,
                                    early_stop=False)
        assert ids.shape == (2, beams, 11 + steps)
        for b in range(2):
            want = _reference_beams(oracle, prompts[b], steps, beams, eos, alpha)
            assert (ids[b, :, :11].cpu() == prompts[b]).all()
            assert ids[b, :, 11:].tolist() == [w[1] for w in want]
            # logits of a few units in fp32, each step's score within some 1e-5
            ref = torch.tensor([w[0] for w in want], dtype=torch.float64)
            assert (scores[b].double().cpu() - ref).abs().max() <= steps * 1e-5
        eos = int(ids[0, 0, 11 + 1])  # again, with an end token that a good beam meets early


def test_early_stop_trims_to_the_longest_beam():
    from minitp.generation import generate_beam

    model, _ = _pair("tiny")
    prompts = torch.randint(0, 1000, (2, 7), generator=torch.Generator().manual_seed(3)).to(DEV)
    free, _ = generate_beam(model, prompts, 1, 4)
    # the first selection's favourite ends a beam at once; one beam a prompt is then finished
    eos = int(free[0, 0, 7])
    whole, s0 = generate_beam(model, prompts[:1], 30, 1, eos_token_id=eos, early_stop=False)
    short, s1 = generate_beam(model, prompts[:1], 30, 1, eos_token_id=eos)
    assert short.shape[2] == 8 and whole.shape[2] == 37 and (whole[0, 0, 7:] == eos).all()
    assert torch.equal(s0, s1) and torch.equal(whole[:, :, :8], short)


def test_one_beam_is_greedy():
    from minitp.generation import generate_beam, generate_greedy

    model, _ = _pair("qwen2.5-0.5b")
    prompts = torch.randint(0, 151936, (3, 20), generator=torch.Generator().manual_seed(1)).to(DEV)
    ids, _ = generate_beam(model, prompts, 12, 1)
    assert torch.equal(ids[:, 0], generate_greedy(model, prompts, 12))


def test_more_beams_than_continuations_and_limits():
    from minitp import synthetic
    from minitp.generation import generate_beam

    cfg = dataclasses.replace(synthetic.TINY, vocab_size=8, max_position_embeddings=16)
    model = synthetic.build_synthetic_model(cfg, dtype=torch.float32, device=DEV, seed=0)
    prompts = torch.tensor([[1, 2, 3]], device=DEV)
    ids, scores = generate_beam(model, prompts, 1, 20)
    assert torch.isfinite(scores[0, :8]).all() and (scores[0, 8:] == float("-inf")).all()
    assert sorted(ids[0, :8, 3].tolist()) == list(range(8))
    ids, scores = generate_beam(model, prompts, 14, 20)
    assert torch.isfinite(scores).all() and len({tuple(r) for r in ids[0].tolist()}) == 20
    with pytest.raises(IndexError):
        generate_beam(model, prompts, 15, 2)
    with pytest.raises(ValueError):
        generate_beam(model, prompts, 2, 33)
    with pytest.raises(ValueError):
        generate_beam(model, prompts, 0, 2)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_greedy_under_a_shared_prefix(dtype):
    """Questions [B, T] behind cached system prompts give what the whole
    prompts give: the same ids in fp32, logits within bf16's steps."""
    from minitp.generation import generate_greedy, make_kv_cache

    model, _ = _pair("qwen2.5-0.5b", dtype)
    g = torch.Generator().manual_seed(2)
    system = torch.randint(0, 151936, (2, 70), generator=g).to(DEV)
    asks = torch.randint(0, 151936, (6, 9), generator=g).to(DEV)

    def caches():
        pre = make_kv_cache(model, 2, 70)
        model(system, kv_cache=pre)
        kv = make_kv_cache(model, 6, 9 + 10)
        kv.share_prefix(pre)
        return kv

    # the program and the modules walked one by one (other roundings of bf16)
    kv = caches()
    native = model(asks, kv_cache=kv)
    for layer in model.model.layers:
        layer.self_attn.use_fused_qkv = False
    walked = model(asks, kv_cache=caches())
    for layer in model.model.layers:
        layer.self_attn.use_fused_qkv = True
    whole = torch.cat([system.repeat_interleave(3, 0), asks], 1)
    logits, plain = model(asks, kv_cache=caches()), model(whole)[:, 70:]
    # two forms of the same forward: each within the path's own bar of the
    # oracle's logits (bf16 0.5, fp32 1e-3)
    bar = 0.5 if dtype == torch.bfloat16 else 1e-3
    for got in (logits, native, walked):
        assert (got.float() - plain.float()).abs().max() <= 2 * bar
    # one more token on the program
    tok = native[:, -1].argmax(-1, keepdim=True)
    step, plain = model(tok, kv_cache=kv), model(torch.cat([whole, tok], 1))[:, -1:]
    assert kv.seq_len == 10 and (step.float() - plain.float()).abs().max() <= 2 * bar
    if dtype == torch.float32:
        out = generate_greedy(model, asks, 10, kv=caches())
        assert torch.equal(out, generate_greedy(model, whole, 10)[:, 70:])


def test_an_end_token_under_a_shared_prefix():
    """generate_greedy's early stop behind prefixes: the same ids, the same end."""
    from minitp.generation import generate_greedy, make_kv_cache

    model, _ = _pair("tiny")
    g = torch.Generator().manual_seed(5)
    system = torch.randint(0, 1000, (2, 33), generator=g).to(DEV)
    asks = torch.randint(0, 1000, (4, 6), generator=g).to(DEV)
    whole = torch.cat([system.repeat_interleave(2, 0), asks], 1)
    free = generate_greedy(model, whole, 20)
    for eos in {int(free[0, 42]), int(free[3, 50])}:
        pre = make_kv_cache(model, 2, 33)
        model(system, kv_cache=pre)
        kv = make_kv_cache(model, 4, 26)
        kv.share_prefix(pre)
        out = generate_greedy(model, asks, 20, eos_token_id=eos, kv=kv)
        assert torch.equal(out, generate_greedy(model, whole, 20, eos_token_id=eos)[:, 33:])


def test_beam_search_module_by_module():
    """The modules walked one by one give the program's beams."""
    from minitp.generation import generate_beam

    model, _ = _pair("tiny")
    prompts = torch.randint(0, 1000, (3, 8), generator=torch.Generator().manual_seed(6)).to(DEV)
    ids, scores = generate_beam(model, prompts.int(), 7, 4)
    for layer in model.model.layers:
        layer.self_attn.use_fused_qkv = False
    walked, other = generate_beam(model, prompts, 7, 4)
    assert torch.equal(ids, walked) and (scores - other).abs().max() <= 7e-5


def test_a_step_behind_a_prefix_in_a_graph():
    """One captured step of a beam search, replayed for other tokens between the
    program's own eager work."""
    from minitp.generation import make_kv_cache

    model, _ = _pair("qwen2.5-0.5b", torch.bfloat16)
    g = torch.Generator().manual_seed(9)
    system = torch.randint(0, 151936, (2, 600), generator=g).to(DEV)
    pre = make_kv_cache(model, 2, 256)
    model(system[:, :200], kv_cache=pre)
    toks = [torch.randint(0, 151936, (6, 1), generator=g).to(DEV) for _ in range(4)]

    def behind():
        kv = make_kv_cache(model, 6, 8)
        kv.share_prefix(pre)
        model(toks[3], kv_cache=kv)
        return kv

    with torch.inference_mode():
        kv, tok = behind(), toks[0].clone()
        model(tok, kv_cache=kv)  # (workspaces of this shape are there)
        kv.seq_len = 1
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = model(tok, kv_cache=kv)
        for t in toks[:3]:
            want = model(t, kv_cache=behind())
            tok.copy_(t)
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want)
