"""Log-probabilities of given texts (no counterpart in mini-tp, which generates).

``score_tokens`` runs token lists of any lengths through the model in packed
forwards (``TPQwen2ForCausalLM.forward_packed``: no padding, one pass for all)
and takes the log-probability, entropy, rank and alternatives of every token
from the logits of the one before it (``kernels.token_logprobs``): perplexity
of texts, the likelihoods of the answers to a question, log-probabilities of a
prompt. Only the rows that are scored go through the LM head.
"""

from __future__ import annotations

from collections.abc import Sequence

import torch

from minitp import _native as N
from minitp import kernels as K
from minitp.layer import TPQwen2ForCausalLM

LOGIT_ROWS = 4096  # rows that go through the LM head at a time (1.2 GB of bf16 logits at 152,064 tokens)


@torch.inference_mode()
def score_tokens(model: TPQwen2ForCausalLM, sequences: Sequence[Sequence[int] | torch.Tensor], top: int = 0,
                 starts: Sequence[int] | None = None, max_tokens: int = 16384) -> list[K.TokenLogprobs]:
    """What the model says of the tokens of each sequence: one TokenLogprobs a
    sequence, on the model's device (views of a forward's results: clone what is
    kept or saved by itself).

    A sequence is a list of ids or a 1-D tensor. Its entries are those of its
    tokens ``starts[i]`` (at least 1, the default: the first token has none
    before it) to the last, given all that come before each; none for a
    sequence that ends before. ``top`` asks for that many of the most likely
    tokens at each place. Forwards take whole sequences, up to ``max_tokens``
    tokens at a time (a longer one alone). An id outside the vocabulary gives
    NaN, for itself and for what comes after it."""
    if top < 0 or top > min(K.MAX_TOP, model.cfg.vocab_size):
        raise ValueError(f"score_tokens: top={top} of {model.cfg.vocab_size} tokens (0 to {K.MAX_TOP})")
    if max_tokens < 1:
        raise ValueError(f"score_tokens: max_tokens={max_tokens}")
    if starts is not None and (len(starts) != len(sequences) or any(s < 1 for s in starts)):
        raise ValueError(f"score_tokens: starts {list(starts)[:8]} for {len(sequences)} sequences, each at least 1")
    weight = model.model.embed_tokens.weight
    N.require_gpu(weight, what="score_tokens")
    if K._elsewhere(weight.get_device()):
        with torch.cuda.device(weight.device):
            return score_tokens(model, sequences, top, starts, max_tokens)
    if torch.cuda.is_current_stream_capturing():
        raise RuntimeError("score_tokens: texts come from the host, a captured graph would keep them")
    texts = []
    for s in sequences:
        t = s if isinstance(s, torch.Tensor) else torch.tensor(list(s), dtype=torch.long)
        if t.dim() != 1 or t.is_floating_point() or t.is_complex():
            raise ValueError(f"score_tokens: a sequence {tuple(t.shape)} {t.dtype}, expected whole numbers [T]")
        texts.append(t.long())
    longest, limit = max((t.numel() for t in texts), default=0), model.cfg.max_position_embeddings
    if longest > limit:
        raise IndexError(f"position {longest - 1} out of range for RoPE table of {limit} rows")
    results: list[K.TokenLogprobs] = []
    first = 0
    while first < len(texts):
        end, tokens = first, 0
        while end < len(texts) and (end == first or tokens + texts[end].numel() <= max_tokens):
            tokens += texts[end].numel()
            end += 1
        results += _score_batch(model, texts[first:end], [1] * (end - first) if starts is None else starts[first:end], top)
        first = end
    return results


def _score_batch(model: TPQwen2ForCausalLM, texts: list[torch.Tensor], starts: Sequence[int],
                 top: int) -> list[K.TokenLogprobs]:
    device = model.model.embed_tokens.weight.device
    lens = [t.numel() for t in texts]
    counts = [max(n - s, 0) for n, s in zip(lens, starts)]
    on_host = all(not t.is_cuda for t in texts)
    ids = torch.cat(texts).to(device) if on_host else torch.cat([t.to(device) for t in texts])
    total = sum(counts)
    if total == 0:
        rows = torch.empty(0, dtype=torch.long, device=device)
        return [_empty(rows, top) for _ in texts]
    # the rows that are scored, each by the logits of the row before it
    ends = torch.tensor(lens).cumsum(0)
    count = torch.tensor(counts)
    rows = torch.arange(total) + torch.repeat_interleave(ends - count - (count.cumsum(0) - count), count)
    rows = rows.to(device)
    hidden = model.forward_packed(ids, lens)
    wanted = K.embedding(rows - 1, hidden)
    given = ids[rows]
    parts = []
    for i in range(0, total, LOGIT_ROWS):
        logits = model.lm_head(wanted[i:i + LOGIT_ROWS])
        parts.append(K.token_logprobs(logits, given[i:i + LOGIT_ROWS], top=top))
    whole = parts[0] if len(parts) == 1 else K.TokenLogprobs(*(torch.cat(p) for p in zip(*parts)))
    return [K.TokenLogprobs(*p) for p in zip(*(x.split(counts) for x in whole))]


def _empty(like: torch.Tensor, top: int) -> K.TokenLogprobs:
    none = like.new_empty(0, dtype=torch.float32)
    return K.TokenLogprobs(none, none, like, like.new_empty((0, top)), none.new_empty((0, top)))
