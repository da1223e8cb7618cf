"""Refusals of the beam-search and shared-prefix entry points: every invalid
call is turned down on the host, before any pointer is used (no GPU)."""

import ctypes
import math

import pytest
import torch

from minitp import _native as N
from minitp import kernels as K

P = 4096  # a 16-byte aligned address that no refused call looks at


def attention(dtype=N.BF16, q=P, kp=P, vp=P, kc=P, vc=P, out=P, b=4, g=2, t=1, hq=4, hkv=2, d=64, sp=5000, p=5000, plens=None,
              s=16, c=10, clens=None, ws=P, nbytes=1 << 30):
    return N.lib().minitp_shared_prefix_attention(None, dtype, q, kp, vp, kc, vc, out, b, g, t, hq, hkv, d, sp, p, plens,
                                                  s, c, clens, ws, nbytes)


@pytest.mark.parametrize("status,change", [
    (N.ERR_ARG, dict(dtype=2)), (N.ERR_ARG, dict(q=None)), (N.ERR_ARG, dict(kp=None)), (N.ERR_ARG, dict(vc=None)),
    (N.ERR_ARG, dict(out=None)), (N.ERR_ARG, dict(g=0)), (N.ERR_ARG, dict(g=-2)), (N.ERR_ARG, dict(b=-4)),
    (N.ERR_ARG, dict(t=-1)), (N.ERR_ARG, dict(p=-1)), (N.ERR_ARG, dict(c=-1)), (N.ERR_ARG, dict(hkv=0)),
    (N.ERR_ARG, dict(d=12)), (N.ERR_ARG, dict(d=0)), (N.ERR_ARG, dict(q=P + 8)), (N.ERR_ARG, dict(kc=P + 2)),
    (N.ERR_ARG, dict(vp=P + 4)), (N.ERR_ARG, dict(ws=None)), (N.ERR_ARG, dict(nbytes=64)), (N.ERR_ARG, dict(ws=P + 4)),
    (N.ERR_DIVISIBLE, dict(hq=5)), (N.ERR_DIVISIBLE, dict(b=5)), (N.ERR_OVERFLOW, dict(c=16)),
    (N.ERR_OVERFLOW, dict(t=7)), (N.ERR_OVERFLOW, dict(p=5001)), (N.ERR_UNSUPPORTED, dict(d=256)),
    (N.ERR_UNSUPPORTED, dict(d=40)),
])
def test_shared_prefix_attention_refuses(status, change):
    assert attention(**change) == status and N.last_error()


def test_shared_prefix_attention_of_nothing():
    assert attention(b=0) == N.OK and attention(t=0) == N.OK
    size = N.lib().minitp_shared_prefix_attention_workspace_bytes
    assert size(N.F32, 0, 1, 1, 4, 2, 64, 10, 10) == 0
    assert size(N.F32, 4, 2, 1, 4, 2, 64, 0, 0) == 0  # (one block a row: nothing to join)
    assert size(N.F32, 4, 2, 1, 4, 2, 64, 5000, 0) > 0
    for bad in ((5, 4, 2, 1, 4, 2, 64, 1, 1), (0, 4, 3, 1, 4, 2, 64, 1, 1), (0, 4, 2, 1, 3, 2, 64, 1, 1),
                (0, 4, 0, 1, 4, 2, 64, 1, 1), (0, 4, 2, 1, 4, 2, 64, -1, 1)):
        assert size(*bad) == -1


def select(dtype=N.F32, logits=P, ldg=800, ldb=100, g=2, w=8, v=100, scores=P, finished=None, lengths=None, eos=-1,
           alpha=0.0, outs=(P,) * 5, ws=P, nbytes=1 << 30):
    return N.lib().minitp_beam_select(None, dtype, logits, ldg, ldb, g, w, v, scores, finished, lengths, eos, alpha, *outs,
                                      ws, nbytes)


@pytest.mark.parametrize("change", [
    dict(dtype=7), dict(logits=None), dict(scores=None), dict(outs=(P, P, None, P, P)), dict(w=0), dict(w=33), dict(g=-1),
    dict(v=0), dict(v=1 << 31), dict(ldg=-1), dict(ldb=-5), dict(eos=-2), dict(eos=100), dict(finished=P),
    dict(alpha=math.nan), dict(alpha=math.inf), dict(alpha=17.0), dict(alpha=-16.5), dict(ws=None), dict(nbytes=100), dict(ws=P + 8),
])
def test_beam_select_refuses(change):
    assert select(**change) == N.ERR_ARG and N.last_error()


def test_beam_select_of_nothing():
    assert select(g=0) == N.OK
    size = N.lib().minitp_beam_select_workspace_bytes
    assert size(1, 33, 10) == size(1, 0, 10) == size(-1, 4, 10) == size(1, 4, 0) == -1 and size(1, 4, 10) > 0


def reorder(dtype=N.BF16, k=P, v=P, layers=2, g=2, w=4, hkv=2, s=32, d=64, rows=10, parents=P):
    return N.lib().minitp_kv_reorder(None, dtype, k, v, layers, g, w, hkv, s, d, rows, parents)


@pytest.mark.parametrize("status,change", [
    (N.ERR_ARG, dict(dtype=-1)), (N.ERR_ARG, dict(k=None)), (N.ERR_ARG, dict(parents=None)), (N.ERR_ARG, dict(w=0)),
    (N.ERR_ARG, dict(w=33)), (N.ERR_ARG, dict(rows=-1)), (N.ERR_ARG, dict(layers=-1)), (N.ERR_ARG, dict(d=12)),
    (N.ERR_ARG, dict(v=P + 8)), (N.ERR_OVERFLOW, dict(rows=33)), (N.ERR_UNSUPPORTED, dict(layers=1 << 16)),
    (N.ERR_UNSUPPORTED, dict(g=1 << 16)), (N.ERR_UNSUPPORTED, dict(s=1 << 30, rows=1 << 29)),
])
def test_kv_reorder_refuses(status, change):
    assert reorder(**change) == status and N.last_error()


def test_kv_reorder_of_nothing():
    assert reorder(rows=0, k=None, v=None, parents=None) == N.OK
    assert reorder(layers=0) == N.OK and reorder(g=0) == N.OK


@pytest.mark.parametrize("change", [
    dict(t=1 << 40, s=1 << 41, c=0), dict(t=(1 << 31) - 70, s=1 << 32, c=0), dict(b=1 << 33), dict(b=1 << 62, t=4),
    dict(b=1 << 30, hq=1 << 30), dict(hq=1 << 40, hkv=1 << 40), dict(b=1 << 26, hq=2), dict(c=1 << 31, s=1 << 32),
    dict(p=(1 << 31) - 64, sp=1 << 31),
])
def test_shared_prefix_attention_too_large(change):
    """Past 32-bit rows, keys and launches: refused before any size is computed from it."""
    assert attention(**change) == N.ERR_UNSUPPORTED and "too many" in N.last_error()
    x = dict(b=4, g=2, t=1, hq=4, hkv=2, d=64, p=5000, c=10) | {k: v for k, v in change.items() if k not in ("s", "sp")}
    size = N.lib().minitp_shared_prefix_attention_workspace_bytes
    assert size(N.BF16, *(x[k] for k in ("b", "g", "t", "hq", "hkv", "d", "p", "c"))) == -1


def test_sizes_that_pass_64_bits_are_refused():
    top = (1 << 63) - 1
    assert attention(c=top) == attention(c=top - 3, t=4) == N.ERR_OVERFLOW
    assert select(g=1 << 60) == select(g=1 << 31) == N.ERR_ARG
    assert select(g=1 << 22) in (N.ERR_ARG, N.ERR_UNSUPPORTED) and select(g=1 << 22, nbytes=1 << 62) == N.ERR_UNSUPPORTED
    assert N.lib().minitp_beam_select_workspace_bytes(1 << 31, 4, 10) == -1
    assert reorder(d=1 << 62) == reorder(layers=1 << 62, hkv=4) == N.ERR_UNSUPPORTED


def test_forward_shared_refuses():
    lib = N.lib()
    cfg = N.Qwen2Config(N.BF16, 2, 64, 4, 2, 16, 128, 1000, 9000, 1e-6)
    fake = (ctypes.c_void_p * 14)(*([P] * 14))
    w = N.Qwen2Weights(P, P, P, P, P, ctypes.cast(fake, ctypes.POINTER(ctypes.c_void_p)))
    h = ctypes.c_void_p()
    assert lib.minitp_qwen2_create(ctypes.byref(cfg), ctypes.byref(w), ctypes.byref(h)) == N.OK
    try:
        step = N.Qwen2Step()
        step.batch, step.tokens, step.cache_len, step.max_seq, step.ids_ld = 6, 1, 20, 24, 1
        step.ids = step.positions = step.k_cache = step.v_cache = step.logits = step.workspace = P
        step.workspace_bytes = 1 << 40

        def call(cache_len=20, **change):
            step.cache_len = cache_len
            pre = N.SharedPrefix(P, P, 2, 5000, 8192, P, 1 << 40)
            for name, value in change.items():
                setattr(pre, name, value)
            return lib.minitp_qwen2_forward_shared(h, None, ctypes.byref(step), ctypes.byref(pre))

        assert lib.minitp_qwen2_forward_shared(h, None, ctypes.byref(step), None) == N.ERR_ARG
        assert call(groups=0) == call(len=-1) == call(k=None) == call(v=P + 4) == N.ERR_ARG
        assert call(workspace=None) == call(workspace_bytes=100) == call(workspace=P + 8) == N.ERR_ARG
        assert call(groups=4) == N.ERR_DIVISIBLE
        assert call(len=8193) == call(cache_len=24) == N.ERR_OVERFLOW
        assert call(len=(1 << 31) - 64, max_seq=1 << 31) == N.ERR_UNSUPPORTED
    finally:
        lib.minitp_qwen2_destroy(h)


def test_wrappers_have_no_cpu_path():
    x = torch.zeros(2, 1, 4, 16)
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        K.shared_prefix_attention(x, x, x, x, x, 1, 0)
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        K.beam_select(torch.zeros(1, 2, 8), torch.zeros(1, 2))
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        K.kv_reorder(torch.zeros(1, 2, 1, 4, 16), torch.zeros(1, 2, 1, 4, 16), torch.zeros(1, 2, dtype=torch.long), 1)


def test_share_prefix_checks_the_caches():
    from minitp.kv_cache import KVCache

    def cache(layers=2, batch=4, heads=2, d=16, dtype=torch.float32):
        return KVCache(layers, batch, heads, d, 8, dtype, torch.device("cpu"))

    kv = cache(batch=6)
    assert kv.prefix is None
    for bad in (cache(layers=1), cache(heads=1), cache(d=32), cache(dtype=torch.bfloat16), cache(batch=4), kv):
        with pytest.raises(ValueError):
            kv.share_prefix(bad)
    good = cache(batch=3)
    kv.share_prefix(good)
    assert kv.prefix is good
    with pytest.raises(ValueError):
        cache(batch=12).share_prefix(kv)
    with pytest.raises(ValueError):
        good.share_prefix(cache(batch=1))  # (it serves as a prefix itself)
    full = cache(batch=6)
    full.advance(2)
    with pytest.raises(ValueError, match="2 rows"):
        full.share_prefix(good)


def test_generation_state_keeps_to_its_prefix():
    """A prefix put in front of the cache, or grown, after the positions were
    laid out is refused, and so is the decode graph with one."""
    from minitp.config import ModelConfig
    from minitp.distributed.context import ParallelContext
    from minitp.generation import GenerationState, make_kv_cache
    from minitp.layer import TPQwen2ForCausalLM

    cfg = ModelConfig(32, 48, 1, 2, 1, 16, 64, 1e-6, 1e6, 64)
    model = TPQwen2ForCausalLM(cfg, ParallelContext(0, 0, 1, 0, 1, torch.device("cpu"), None), init_weights=False)
    ids = torch.zeros(2, 3, dtype=torch.long)
    pre = make_kv_cache(model, 1, 8)
    pre.advance(5)
    late = GenerationState(model, ids, 4)
    late.kv.share_prefix(pre)
    with pytest.raises(ValueError, match="prefix rows"):
        late.prefill()
    with pytest.raises(ValueError, match="shared prefix"):
        model.decode_native(ids[:, 0], torch.tensor(0), late.kv, torch.zeros(2, 1, 64), None)
    kv = make_kv_cache(model, 2, 8)
    kv.share_prefix(pre)
    state = GenerationState(model, ids, 4, kv=kv)
    assert state.positions_buf.tolist() == list(range(5, 12))
    pre.advance(1)
    with pytest.raises(ValueError, match="prefix rows"):
        state.prefill()
