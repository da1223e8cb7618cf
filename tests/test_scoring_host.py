"""Refusals of the entry points that score texts: every invalid call is turned
down on the host, before any pointer is used (no GPU)."""

import ctypes

import pytest
import torch

from minitp import _native as N
from minitp import kernels as K

P = 4096  # a 16-byte aligned address that no refused call looks at


def attention(dtype=N.BF16, q=P, q_row=256, q_head=64, k=P, v=P, kv_row=128, kv_head=64, out=P, n=10, s=2, hq=4, hkv=2,
              d=64, offsets=P):
    return N.lib().minitp_packed_attention(None, dtype, q, q_row, q_head, k, v, kv_row, kv_head, out, n, s, hq, hkv, d,
                                           offsets)


@pytest.mark.parametrize("status,change", [
    (N.ERR_ARG, dict(dtype=2)), (N.ERR_ARG, dict(q=None)), (N.ERR_ARG, dict(k=None)), (N.ERR_ARG, dict(v=None)),
    (N.ERR_ARG, dict(out=None)), (N.ERR_ARG, dict(offsets=None)), (N.ERR_ARG, dict(n=-1)), (N.ERR_ARG, dict(s=-1)),
    (N.ERR_ARG, dict(hq=0)), (N.ERR_ARG, dict(hkv=0)), (N.ERR_ARG, dict(d=0)), (N.ERR_ARG, dict(d=12)),
    (N.ERR_ARG, dict(q=P + 8)), (N.ERR_ARG, dict(k=P + 2)), (N.ERR_ARG, dict(v=P + 4)), (N.ERR_ARG, dict(out=P + 8)),
    (N.ERR_ARG, dict(q_row=-256)), (N.ERR_ARG, dict(q_head=-64)), (N.ERR_ARG, dict(kv_row=-128)),
    (N.ERR_ARG, dict(kv_head=-64)), (N.ERR_ARG, dict(q_row=257)), (N.ERR_ARG, dict(q_head=4)),
    (N.ERR_ARG, dict(kv_row=130)), (N.ERR_ARG, dict(kv_head=63)), (N.ERR_DIVISIBLE, dict(hq=5)),
    (N.ERR_UNSUPPORTED, dict(d=256)), (N.ERR_UNSUPPORTED, dict(d=40)), (N.ERR_UNSUPPORTED, dict(n=1 << 31)),
    (N.ERR_UNSUPPORTED, dict(n=(1 << 62) + 1)), (N.ERR_UNSUPPORTED, dict(s=1 << 31)),
    (N.ERR_UNSUPPORTED, dict(n=1 << 27, hq=64, hkv=32)), (N.ERR_UNSUPPORTED, dict(hq=1 << 62, hkv=1 << 61)),
    (N.ERR_UNSUPPORTED, dict(kv_row=(1 << 24) + 8)), (N.ERR_UNSUPPORTED, dict(dtype=N.F32, kv_row=(1 << 23) + 4)),
])
def test_packed_attention_refuses(status, change):
    assert attention(**change) == status and N.last_error()


def test_packed_attention_of_nothing():
    assert attention(n=0) == N.OK
    assert attention(n=0, q=None, offsets=None) == N.OK


def logprobs(dtype=N.BF16, logits=P, ld=1000, b=4, v=1000, tokens=P, top=3, lp=P, entropy=P, ranks=P, top_tokens=P,
             top_lp=P, ws=P, nbytes=1 << 40):
    return N.lib().minitp_token_logprobs(None, dtype, logits, ld, b, v, tokens, top, lp, entropy, ranks, top_tokens, top_lp,
                                         ws, nbytes)


@pytest.mark.parametrize("change", [
    dict(dtype=3), dict(logits=None), dict(tokens=None), dict(lp=None), dict(entropy=None), dict(ranks=None),
    dict(top_tokens=None), dict(top_lp=None), dict(ld=-1), dict(b=-1), dict(v=0), dict(v=-5), dict(v=1 << 31),
    dict(top=-1), dict(top=33), dict(v=2, top=3),
])
def test_token_logprobs_refuses(change):
    assert logprobs(**change) == N.ERR_ARG and N.last_error()


def test_token_logprobs_too_large_and_of_nothing():
    assert logprobs(b=1 << 40) == N.ERR_UNSUPPORTED and "too many" in N.last_error()
    assert logprobs(b=1 << 62) == N.ERR_UNSUPPORTED
    assert logprobs(b=0) == N.OK and logprobs(b=0, logits=None) == N.OK
    size = N.lib().minitp_token_logprobs_workspace_bytes
    assert size(N.BF16, 0, 1000, 3) == 0
    for bad in ((4, 1, 1000, 3), (0, -1, 1000, 3), (0, 1, 0, 0), (0, 1, 1000, 33), (0, 1, 2, 3), (0, 1, 1 << 31, 3),
                (0, 1, 1000, -1), (1, 1 << 62, 1000, 0)):
        assert size(*bad) == -1, bad


def test_wrappers_check_their_arguments():
    q, k = torch.zeros(6, 4, 16), torch.zeros(6, 2, 16)
    offsets, tokens = torch.tensor([0, 6]), torch.zeros(3, dtype=torch.long)
    for call in (lambda: K.packed_attention(q, k, k, offsets), lambda: K.token_logprobs(torch.zeros(3, 5), tokens)):
        with pytest.raises(RuntimeError, match="no CPU path"):
            call()


def _program():
    """A native program whose pointers no refused call looks at."""
    cfg = N.Qwen2Config(N.BF16, 1, 64, 4, 2, 16, 128, 1000, 256, 1e-6)
    layers = (ctypes.c_void_p * N.W_PER_LAYER)(*([P] * N.W_PER_LAYER))
    weights = N.Qwen2Weights(P, P, P, P, P, ctypes.cast(layers, ctypes.POINTER(ctypes.c_void_p)))
    handle = ctypes.c_void_p()
    assert N.lib().minitp_qwen2_create(ctypes.byref(cfg), ctypes.byref(weights), ctypes.byref(handle)) == N.OK
    return handle


@pytest.mark.parametrize("status,change", [
    (N.ERR_ARG, dict(offsets=None)), (N.ERR_ARG, dict(hidden=None)), (N.ERR_ARG, dict(hidden=P + 8)),
    (N.ERR_ARG, dict(sequences=-1)), (N.ERR_ARG, dict(batch=2)), (N.ERR_ARG, dict(tokens=0)),
    (N.ERR_ARG, dict(cache_len=1)), (N.ERR_ARG, dict(next_tok=P)), (N.ERR_ARG, dict(ids=None)),
    (N.ERR_ARG, dict(positions=None)), (N.ERR_ARG, dict(k_cache=None)), (N.ERR_ARG, dict(v_cache=P + 2)),
    (N.ERR_ARG, dict(workspace=None)), (N.ERR_ARG, dict(workspace_bytes=100)), (N.ERR_ARG, dict(ids_ld=5)),
    (N.ERR_OVERFLOW, dict(max_seq=9)), (N.ERR_UNSUPPORTED, dict(sequences=1 << 31)),
])
def test_forward_packed_refuses(status, change):
    handle = _program()
    a = dict(ids=P, ids_ld=10, positions=P, batch=1, tokens=10, cache_len=0, k_cache=P, v_cache=P, max_seq=16, logits=None,
             logits_all=0, next_tok=None, next_tok_ld=0, workspace=P, workspace_bytes=1 << 40, offsets=P, sequences=2,
             hidden=P)
    a.update(change)
    offsets, sequences, hidden = a.pop("offsets"), a.pop("sequences"), a.pop("hidden")
    step = N.Qwen2Step(**a)
    assert N.lib().minitp_qwen2_forward_packed(handle, None, ctypes.byref(step), offsets, sequences, hidden) == status
    assert N.last_error()
    N.lib().minitp_qwen2_destroy(handle)


def test_forward_packed_without_arguments():
    assert N.lib().minitp_qwen2_forward_packed(None, None, None, None, 0, None) == N.ERR_ARG


def test_scoring_has_no_cpu_path():
    from minitp.config import ModelConfig
    from minitp.distributed.context import ParallelContext
    from minitp.layer import TPQwen2ForCausalLM
    from minitp.scoring import score_tokens

    cfg = ModelConfig(32, 48, 1, 2, 1, 16, 64, 1e-6, 1e6, 64)
    model = TPQwen2ForCausalLM(cfg, ParallelContext(0, 0, 1, 0, 1, torch.device("cpu"), None), init_weights=False)
    with pytest.raises(RuntimeError, match="no CPU path"):
        score_tokens(model, [[1, 2, 3]])
    with pytest.raises(RuntimeError, match="no CPU path"):
        model.forward_packed(torch.zeros(3, dtype=torch.long), [3])
    for kw in (dict(top=-1), dict(top=33), dict(starts=[1, 1]), dict(starts=[0]), dict(max_tokens=0)):
        with pytest.raises(ValueError):
            score_tokens(model, [[1, 2, 3]], **kw)
