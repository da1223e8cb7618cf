"""Performance cases of the operators that score texts.

Two operators, each called as a program calls it:

* ``attention``: causal attention over packed sequences of different lengths.
  The rows of all sequences follow each other in one stream of N tokens, with
  no padding between them; a query attends the rows of its own sequence up to
  itself. Rows behind the last sequence belong to none and come out as zeros.
* ``logprobs``: the log-probabilities of given tokens, one a row of logits,
  with the distribution's entropy, the tokens' ranks and the best tokens.

Head shapes and vocabularies are those of ``minitp.synthetic.SHAPES``. Queries
and keys are normal with the spread that gives peaked rather than flat
attention, logits are normal with that of an LM head's; the given tokens are
partly the likely ones of a text, partly any.
"""

from __future__ import annotations

import math
import os
import random
import sys

import torch

_PKG = os.path.join(os.getcwd(), "mini-tp_amd")
if _PKG not in sys.path:
    sys.path.insert(1, _PKG)

own = False

# query heads, KV heads, head dim, vocabulary
DIMS = {
    "tiny": (4, 2, 16, 1000),
    "qwen2.5-0.5b": (14, 2, 64, 151936),
    "qwen2.5-7b": (28, 4, 128, 152064),
}
DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
DEV = "cuda"
MAX_TOP = 32


def listed() -> list[dict]:
    return [
        # three short prompts: the smallest call, where latency counts
        _attention("few-short", "qwen2.5-0.5b", "bf16", sequences=3, longest=30),
        # the answers of some hundred multiple-choice questions, in the layout
        # of the projection's output (q, k and v of a token side by side)
        _attention("choices", "qwen2.5-0.5b", "bf16", sequences=400, longest=60, empty=3, together=True),
        # one prompt of the smaller model
        _attention("prompt-8191", "qwen2.5-0.5b", "bf16", sequences=1, longest=8191),
        # 16 prompts of unequal length, in a buffer that has room for more
        _attention("prompts-16", "qwen2.5-7b", "bf16", sequences=16, longest=1500, pad=77),
        # the large model's prompt workload, 4 x 4096
        _attention("prompts-4x4096", "qwen2.5-7b", "bf16", sequences=4, longest=4096, equal=True),
        # three documents: the largest
        _attention("documents-3", "qwen2.5-7b", "bf16", sequences=3, longest=20011),
        # a handful of prompts in fp32
        _attention("prompts-5-fp32", "qwen2.5-0.5b", "fp32", sequences=5, longest=700),
        # the token that a step of one sequence took, with its alternatives:
        # the smallest call
        _logprobs("step-1", "qwen2.5-0.5b", "bf16", rows=1, top=5),
        # a step of 32 sequences of the large model
        _logprobs("steps-32", "qwen2.5-7b", "bf16", rows=32, top=20),
        # the tokens of prompts with the best five
        _logprobs("prompt-1999", "qwen2.5-7b", "bf16", rows=1999, top=5),
        # perplexity over a long text: no alternatives, the largest
        _logprobs("text-8191", "qwen2.5-0.5b", "bf16", rows=8191, top=0),
        # prompts in fp32
        _logprobs("prompt-331-fp32", "qwen2.5-0.5b", "fp32", rows=331, top=10),
    ]


def _attention(name: str, shape: str, dtype: str, *, sequences: int, longest: int, equal: bool = False, empty: int = 0,
               pad: int = 0, together: bool = False) -> dict:
    return {"name": name, "op": "attention", "shape": shape, "dtype": dtype, "sequences": sequences, "longest": longest,
            "equal": equal, "empty": empty, "pad": pad, "together": together}


def _logprobs(name: str, shape: str, dtype: str, *, rows: int, top: int) -> dict:
    return {"name": name, "op": "logprobs", "shape": shape, "dtype": dtype, "rows": rows, "top": top}


def _log_int(rng: random.Random, lo: int, hi: int) -> int:
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng: random.Random) -> dict:
    """One more case of the same ranges, no dearer than the largest listed one
    of its operator."""
    op = rng.choice(["attention", "attention", "logprobs"])
    limit = max(_cost(c) for c in listed() if c["op"] == op)
    while True:
        shape = rng.choice(sorted(DIMS))
        dtype = rng.choice(["bf16", "bf16", "bf16", "fp32"])
        if op == "attention":
            case = _attention("", shape, dtype, sequences=_log_int(rng, 1, 1000), longest=_log_int(rng, 1, 32256),
                              equal=rng.random() < 0.25, empty=rng.choice([0, 0, rng.randint(1, 5)]),
                              pad=rng.choice([0, 0, _log_int(rng, 1, 300)]), together=rng.random() < 0.5)
        else:
            case = _logprobs("", shape, dtype, rows=_log_int(rng, 1, 8191),
                             top=rng.choice([0, 1, rng.randint(2, 20), MAX_TOP]))
        del case["name"]
        if _cost(case) <= limit:
            return case


def _cost(case: dict) -> float:
    """Seconds at 1 PFLOP/s bf16 (a sixteenth of that in fp32) plus 4 TB/s; for
    attention no less than the plain form's scores and launches take."""
    w = work(case)
    cost = w["flops"] / (1e15 if case["dtype"] == "bf16" else 6e13) + w["bytes"] / 4e12
    if case["op"] == "attention":
        pairs = sum(n * (n + 1) // 2 for n in _lens(case)) * DIMS[case["shape"]][0]
        cost = max(cost, pairs * 5e-13)
    return cost


# ---------------------------------------------------------------------------
# inputs


def _gen(seed: int, stream: int) -> torch.Generator:
    return torch.Generator(device=DEV).manual_seed(seed * 1013 + stream)


def _normal(g: torch.Generator, shape, dtype: torch.dtype, std: float) -> torch.Tensor:
    return torch.empty(shape, dtype=dtype, device=DEV).normal_(0.0, std, generator=g)


def _lens(case: dict) -> list[int]:
    """Lengths up to the longest, the same for every seed; the empty sequences
    lie between the others."""
    count, most = case["sequences"], case["longest"]
    lens = [most if case["equal"] else max(1, round(most * (1 - 0.9 * (i * 0.6180339887 % 1.0)))) for i in range(count)]
    for i in range(case["empty"]):
        lens.insert(i * 7 % (len(lens) + 1), 0)
    return lens


def prepare(case: dict, seed: int) -> dict:
    made = _prepare_attention(case, seed) if case["op"] == "attention" else _prepare_logprobs(case, seed)
    return {"case": dict(case), **made}


def _prepare_attention(case: dict, seed: int) -> dict:
    hq, hkv, d, _ = DIMS[case["shape"]]
    dt, lens = DTYPES[case["dtype"]], _lens(case)
    n = sum(lens) + case["pad"]
    g = _gen(seed, 1)
    if case["together"]:
        qkv = _normal(g, (n, hq + 2 * hkv, d), dt, 1.0)
        qkv[:, :hq] *= 1.5
        q, k, v = qkv.split([hq, hkv, hkv], 1)
    else:  # q by tokens, K and V by heads, as the model keeps them
        q = _normal(g, (n, hq, d), dt, 1.5)
        k, v = (_normal(g, (hkv, n, d), dt, 1.0).transpose(0, 1) for _ in range(2))
    offsets = torch.tensor([0] + lens).cumsum(0)
    return {"q": q, "k": k, "v": v, "lens": lens, "offsets": offsets.to(DEV)}


def _prepare_logprobs(case: dict, seed: int) -> dict:
    vocab, rows = DIMS[case["shape"]][3], case["rows"]
    g = _gen(seed, 2)
    logits = _normal(g, (rows, vocab), DTYPES[case["dtype"]], 2.5)
    tokens = torch.randint(0, vocab, (rows,), generator=g, device=DEV)
    kind = torch.randint(0, 3, (rows,), generator=g, device=DEV)
    tokens = torch.where(kind == 0, logits.argmax(-1), torch.where(kind == 1, logits[:, :500].argmax(-1), tokens))
    return {"logits": logits, "tokens": tokens}


# ---------------------------------------------------------------------------
# one pass


def run(state: dict):
    if own:
        return _run_own(state)
    return _plain_attention(state) if state["case"]["op"] == "attention" else _plain_logprobs(state)


def _run_own(s: dict):
    from minitp import kernels as K

    if s["case"]["op"] == "attention":
        return K.packed_attention(s["q"], s["k"], s["v"], s["offsets"])
    r = K.token_logprobs(s["logits"], s["tokens"], top=s["case"]["top"])
    return {"logprobs": r.logprobs, "entropy": r.entropy, "ranks": r.ranks, "top_tokens": r.top_tokens,
            "top_logprobs": r.top_logprobs}


PLAIN_SCORES = 1 << 28  # scores, and logits, that the plain forms hold at a time


def _plain_attention(s: dict) -> torch.Tensor:
    n, hq, d = s["q"].shape
    hkv = s["k"].shape[1]
    per = hq // hkv
    out = torch.zeros(n, hkv, per, d, device=DEV)
    at = 0
    for length in s["lens"]:
        if length == 0:
            continue
        # [Hkv, L, ...]; a KV head's query heads are more rows of one product
        q = s["q"][at:at + length].float().view(length, hkv, per, d).transpose(0, 1) * d ** -0.5
        k = s["k"][at:at + length].float().permute(1, 2, 0).contiguous()
        v = s["v"][at:at + length].float().transpose(0, 1).contiguous()
        step = max(1, PLAIN_SCORES // (hq * length))
        for lo in range(0, length, step):
            hi = min(lo + step, length)
            x = torch.bmm(q[:, lo:hi].reshape(hkv, -1, d), k[:, :, :hi].contiguous()).view(hkv, hi - lo, per, hi)
            later = torch.arange(hi, device=DEV) > torch.arange(lo, hi, device=DEV)[:, None]
            x.masked_fill_(later[None, :, None], -math.inf)
            x = x.sub_(x.amax(-1, keepdim=True)).exp_()
            o = torch.bmm(x.view(hkv, -1, hi), v[:, :hi].contiguous()).view(hkv, hi - lo, per, d)
            out[at + lo:at + hi] = (o / x.sum(-1, keepdim=True)).transpose(0, 1)
        at += length
    return out.view(n, hq * d).to(s["q"].dtype)


def _plain_logprobs(s: dict) -> dict:
    rows, vocab = s["logits"].shape
    top = s["case"]["top"]
    step = max(1, PLAIN_SCORES // vocab)
    parts = [_plain_rows(s["logits"][i:i + step], s["tokens"][i:i + step], top) for i in range(0, rows, step)]
    return {name: torch.cat([p[name] for p in parts]) for name in parts[0]}


def _plain_rows(logits: torch.Tensor, tokens: torch.Tensor, top: int) -> dict:
    vocab = logits.shape[1]
    x, ids = logits.float(), torch.arange(logits.shape[1], device=DEV)
    above = x - x.amax(-1, keepdim=True)
    e = above.exp()
    # sums over the vocabulary: in 64 bits
    total = e.sum(-1, dtype=torch.float64)
    log_total = total.log()
    entropy = log_total - (e * above).sum(-1, dtype=torch.float64) / total
    mine = x.gather(1, tokens[:, None])
    ranks = ((x > mine) | ((x == mine) & (ids < tokens[:, None]))).sum(-1)
    # the best tokens, ties to the lowest: value and token in one whole number
    bits = (x + 0.0).view(torch.int32).long()
    bits = torch.where(bits < 0, -(bits & 0x7FFFFFFF) - 1, bits)
    best = 0xFFFFFFFF - (((bits << 32) + (0xFFFFFFFF - ids)).topk(top, -1).values & 0xFFFFFFFF)
    return {"logprobs": (above.gather(1, tokens[:, None])[:, 0] - log_total).float(), "entropy": entropy.float(),
            "ranks": ranks, "top_tokens": best, "top_logprobs": (above.gather(1, best) - log_total[:, None]).float()}


# ---------------------------------------------------------------------------
# work, and the results in 64 bits


def work(case: dict) -> dict:
    hq, hkv, d, vocab = DIMS[case["shape"]]
    es = 2 if case["dtype"] == "bf16" else 4
    if case["op"] == "attention":
        lens = _lens(case)
        n = sum(lens)
        return {"bytes": es * d * (n * (2 * hq + 2 * hkv) + case["pad"] * hq),
                "flops": 4 * d * hq * sum(length * (length + 1) // 2 for length in lens)}
    return {"bytes": case["rows"] * (vocab * es + 24 + 12 * case["top"]), "flops": 5 * case["rows"] * vocab}


def exact(case: dict, seed: int):
    s = prepare(case, seed)
    return _exact_attention(s) if case["op"] == "attention" else _exact_logprobs(case, s)


def _exact_attention(s: dict) -> torch.Tensor:
    n, hq, d = s["q"].shape
    hkv = s["k"].shape[1]
    out = torch.zeros(n, hq, d, dtype=torch.float64, device=DEV)
    ends = s["offsets"].tolist()
    for lo, hi in zip(ends, ends[1:]):
        for kv in range(hkv):
            k, v = s["k"][lo:hi, kv].double(), s["v"][lo:hi, kv].double()
            kt = k.t().contiguous()
            for h in range(kv * hq // hkv, (kv + 1) * hq // hkv):
                for a in range(lo, hi, 4096):
                    b = min(a + 4096, hi)
                    x = s["q"][a:b, h].double() @ kt[:, :b - lo].contiguous() / math.sqrt(d)
                    hidden = torch.ones(b - a, b - lo, dtype=torch.bool, device=DEV).triu(a - lo + 1)
                    out[a:b, h] = torch.softmax(x.masked_fill_(hidden, -math.inf), -1) @ v[:b - lo]
    return out.view(n, hq * d)


def _exact_logprobs(case: dict, s: dict) -> dict:
    top = case["top"]
    res: dict = {"logprobs": [], "entropy": [], "ranks": [], "top_tokens": [], "top_logprobs": []}
    for x, t in zip(s["logits"].split(256), s["tokens"].split(256)):
        lp = torch.log_softmax(x.double(), -1)
        res["logprobs"].append(lp.gather(1, t[:, None])[:, 0])
        res["entropy"].append(-(lp.exp() * lp).sum(-1))
        # places in the order of the logits, equal ones by the lower token
        places = x.double().sort(dim=-1, descending=True, stable=True).indices
        res["ranks"].append((places == t[:, None]).int().argmax(-1))
        res["top_tokens"].append(places[:, :top])
        res["top_logprobs"].append(lp.gather(1, places[:, :top]))
    return {name: torch.cat(v) for name, v in res.items()}
