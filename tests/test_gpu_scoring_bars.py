"""Scores of texts in bfloat16 against the oracle, within bars that a scorer
which ignores the model, or mixes its rows up, does not meet.

Bars. The exact scores are the oracle's in float32 over the same (bfloat16)
weights. Its own bfloat16 forward is off from them by e at most over all logits,
0.005; the device rounds at the same places or fewer, in other orders of sums,
and gets B = 4 e. A log-probability is a logit less a weighted mean's growth: at
most 2 B. The entropy moves by sum p (log p + H) d for logits that move by d: at
most B times the mean distance of log p from its mean, and for the second order
half of (1 + max |log p + H|) B^2, where that maximum is below 1.5.
"""

import pytest
import torch

from tests.test_gpu_scoring import LENS, build, texts_of

pytestmark = pytest.mark.gpu


def test_tiny_in_bf16_against_the_oracle():
    from minitp.scoring import score_tokens
    from oracle import qwen2_ref

    model = build("tiny", torch.bfloat16)
    shape = qwen2_ref.TINY
    state = qwen2_ref.synthetic_state(shape, 0, torch.bfloat16)
    rounded = qwen2_ref.OracleQwen2(shape, state)
    exact = qwen2_ref.OracleQwen2(shape, {name: w.float() for name, w in state.items()})
    texts = [t for t in texts_of(LENS, 1000) if len(t) > 1]
    logits = [exact.forward(t[None])[0, :-1].double() for t in texts]
    e = max((rounded.forward(t[None])[0, :-1].double() - x).abs().max().item() for t, x in zip(texts, logits))
    b = 4 * e
    wants, entropies, entropy_bars = [], [], []
    for text, x, r in zip(texts, logits, score_tokens(model, texts, top=3)):
        lp = torch.log_softmax(x, -1)
        p = lp.exp()
        entropy = -(p * lp).sum(-1)
        around = (lp + entropy[:, None]).abs()
        assert around.max() < 1.5
        want, entropy_bar = lp.gather(1, text[1:, None])[:, 0], b * (p * around).sum(-1) + 1.25 * b * b
        assert ((r.logprobs.double().cpu() - want).abs() <= 2 * b).all()
        assert ((r.entropy.double().cpu() - entropy).abs() <= entropy_bar).all()
        # the best three have their own scores, and no token is above them by more
        best = lp.gather(1, r.top_tokens.cpu()[:, :1])
        assert ((r.top_logprobs.double().cpu() - lp.gather(1, r.top_tokens.cpu())).abs() <= 2 * b).all()
        assert (best[:, 0] >= lp.amax(-1) - 2 * b).all()
        wants.append(want)
        entropies.append(entropy)
        entropy_bars.append(entropy_bar)
    want, entropy, entropy_bar = (torch.cat(x) for x in (wants, entropies, entropy_bars))
    # what the bars tell apart: even odds, and the scores of other places
    log_v = torch.tensor(1000.0, dtype=torch.float64).log()
    assert ((want + log_v).abs() > 2 * b).float().mean() > 0.5
    assert ((want - want.roll(1)).abs() > 2 * b).float().mean() > 0.5
    assert ((entropy - log_v).abs() > entropy_bar).float().mean() > 0.5


@pytest.mark.parametrize("name,layers", [("qwen2.5-0.5b", 2), ("qwen2.5-7b", 1)])
def test_packed_texts_in_bf16_against_prompts_on_their_own(name, layers):
    """Logits of the packed forward against the prompt's, within the suite's bar
    for two device paths (0.05 and 2 %), which another place's logits are outside."""
    model = build(name, torch.bfloat16, layers)
    texts = [t for t in texts_of(LENS, model.cfg.vocab_size) if len(t) > 0]
    ids = torch.cat(texts).to("cuda")
    packed = model.lm_head(model.forward_packed(ids, [len(t) for t in texts])).double()
    alone = torch.cat([model(t[None].to("cuda"))[0] for t in texts]).double()
    bar = 0.05 + 0.02 * alone.abs()
    assert ((packed - alone).abs() <= bar).all(), ((packed - alone).abs() / bar).max()
    assert ((alone.roll(1, 0) - alone).abs() > bar).any(-1).all()
