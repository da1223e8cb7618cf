"""Caches behind a shared prefix on the host (no GPU): what each forward takes
as its prefix, and the calls that would attend other rows than those that the
cache's own rows were written behind."""

import pytest
import torch

from minitp.config import ModelConfig
from minitp.distributed.context import ParallelContext
from minitp.generation import GenerationState, make_kv_cache
from minitp.layer import TPQwen2ForCausalLM


def _model():
    cfg = ModelConfig(32, 48, 1, 2, 1, 16, 64, 1e-6, 1e6, 64)
    return TPQwen2ForCausalLM(cfg, ParallelContext(0, 0, 1, 0, 1, torch.device("cpu"), None), init_weights=False)


def _behind(model, rows=5, batch=2, prefixes=1):
    """(a cache behind a prefix of `rows` rows, the prefix)."""
    pre, kv = make_kv_cache(model, prefixes, 16), make_kv_cache(model, batch, 16)
    pre.advance(rows)
    kv.share_prefix(pre)
    return kv, pre


def _grow(pre):
    pre.advance(4)


def _cut(pre):
    pre.seq_len = 3


def _refill(pre):
    rows = pre.seq_len
    pre.seq_len = 0
    pre.advance(rows)


def _permute(pre, monkeypatch):
    from minitp import kernels as K

    monkeypatch.setattr(K, "kv_reorder", lambda *a: None)
    pre.reorder(torch.zeros(1, 1, dtype=torch.long))


@pytest.mark.parametrize("change", ["grow", "cut", "refill", "permute"])
def test_a_prefix_that_changes_under_written_rows_is_refused(change, monkeypatch):
    """Rows behind a prefix hold positions that go on from it: once there are
    some, a prefix of another length or with other rows is refused by every
    way to a forward, and nothing is written."""
    model = _model()
    seen = []
    monkeypatch.setattr("minitp._native.require_gpu", lambda *a, **k: None)
    monkeypatch.setattr(model, "_native", lambda ids, pos, kv, **k: seen.append(pos.tolist()) or kv.advance(ids.shape[1]))
    ids = torch.zeros(2, 3, dtype=torch.long)
    kv, pre = _behind(model)
    state = GenerationState(model, ids, 4, kv=kv)
    state.prefill()
    assert seen == [[5, 6, 7]] and kv.seq_len == 3
    pos = state.append(ids[:, 0])
    if change == "permute":
        _permute(pre, monkeypatch)
    else:
        {"grow": _grow, "cut": _cut, "refill": _refill}[change](pre)
    for call in (lambda: state.decode_step(ids[:, 0], pos), lambda: model(ids[:, :1], kv_cache=kv),
                 lambda: model(ids[:, :1], positions=torch.tensor([8]), kv_cache=kv),
                 lambda: GenerationState(model, ids, 4, kv=kv), kv.prefix_rows):
        with pytest.raises(ValueError, match="prefix"):
            call()
    model.use_rotary_cache = False  # (the modules one by one)
    with pytest.raises(ValueError, match="prefix"):
        model(ids[:, :1], kv_cache=kv)
    assert kv.seq_len == 3 and len(seen) == 1


def test_attention_alone_refuses_a_changed_prefix(monkeypatch):
    """The attention module is a way of its own to a prefix's rows."""
    from minitp import kernels as K

    model = _model()
    attn = model.model.layers[0].self_attn
    monkeypatch.setattr(attn.qkv_proj, "project", lambda x, fused: x)
    monkeypatch.setattr(K, "rope_kv_write", lambda *a: None)
    taken = []
    monkeypatch.setattr(K, "shared_prefix_attention", lambda *a: taken.append(a[5:]) or torch.zeros(2, 1, 32))
    monkeypatch.setattr(attn.o_proj, "forward", lambda x: x)
    kv, pre = _behind(model)
    x, pos = torch.zeros(2, 1, 32), torch.tensor([5])
    attn(x, pos, kv, 0)
    kv.advance(1)
    attn(x, pos, kv, 0)
    pre.advance(2)
    with pytest.raises(ValueError, match="prefix"):
        attn(x, pos, kv, 0)
    assert taken == [(5, 0), (5, 1)]


def test_an_empty_cache_takes_its_prefix_as_it_is():
    """Until a row is written the prefix may be filled, and after the cache is
    emptied it may be another one."""
    model = _model()
    pre, kv = make_kv_cache(model, 1, 16), make_kv_cache(model, 2, 16)
    kv.share_prefix(pre)
    assert kv.prefix_rows() == 0
    pre.advance(6)
    assert kv.prefix_rows() == 6
    kv.advance(2)
    assert kv.prefix_rows() == 6
    pre.advance(1)
    with pytest.raises(ValueError, match="6 prefix rows"):
        kv.prefix_rows()
    kv.seq_len = 0
    assert kv.prefix_rows() == 7
    kv.advance(1)
    assert kv.prefix_rows() == 7
    kv.seq_len = 2  # (more rows, or fewer, of its own: the prefix is the same)
    kv.seq_len = 1
    assert kv.prefix_rows() == 7
    assert make_kv_cache(model, 2, 8).prefix_rows() == 0


@pytest.mark.parametrize("prefixes,groups", [(2, 1), (2, 3), (3, 2), (3, 1), (6, 3)])
def test_reordering_over_several_prefixes_is_refused(prefixes, groups, monkeypatch):
    """Groups of beams that span rows of two prefixes: a row would go on behind
    a prefix that it was not computed behind."""
    from minitp import kernels as K

    moved = []
    monkeypatch.setattr(K, "kv_reorder", lambda *a: moved.append(a[2:]))
    model = _model()
    kv, _ = _behind(model, batch=6, prefixes=prefixes)
    kv.advance(2)
    with pytest.raises(ValueError, match="prefix"):
        kv.reorder(torch.zeros(groups, 6 // groups, dtype=torch.long))
    assert not moved
    for fits in (prefixes, 6):
        parents = torch.arange(6).view(fits, -1)
        kv.reorder(parents)
        assert moved.pop() == (parents, 2)
    free = make_kv_cache(model, 6, 8)
    free.reorder(torch.zeros(groups, 6 // groups, dtype=torch.long))  # (no prefix: any groups)
    assert moved


def test_forwards_have_a_workspace_a_stream_and_captured_ones_their_own(monkeypatch):
    """Forwards of one program on two streams may run at once. A captured one is
    replayed later, beside others: its workspace is memory of its graph (from
    the allocator, within the capture), not the one that the next larger
    forward replaces."""
    from minitp import _native as N
    from minitp.layer import _Program

    now = {"stream": 11, "capturing": False}
    monkeypatch.setattr(N, "stream", lambda: now["stream"])
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: now["capturing"])
    prog = _Program.__new__(_Program)
    prog.device, prog.fwd_ws, prog.decode_ws = torch.device("cpu"), {}, {}
    prog.workspace_bytes = lambda tokens, batch, max_seq: 40000 + tokens
    one = prog.forward_ws(4, 1, 8)
    assert (one == 0).all() and prog.forward_ws(3, 1, 8) is one
    now["stream"] = 22
    two = prog.forward_ws(4, 1, 8)
    assert two.data_ptr() != one.data_ptr() and prog.forward_ws(4, 1, 8) is two
    now["stream"] = 11
    more = prog.forward_ws(90, 1, 8)
    assert more.numel() >= 40090 and (more == 0).all() and prog.forward_ws(4, 1, 8) is more
    now["stream"] = 22
    assert prog.forward_ws(4, 1, 8) is two
    now["capturing"] = True
    kept = [x.data_ptr() for x in prog.fwd_ws.values()]
    first, second = prog.forward_ws(4, 1, 8), prog.forward_ws(4, 1, 8)
    assert len({first.data_ptr(), second.data_ptr(), *kept}) == 4
    assert (first[: N.QWEN2_STATE_BYTES] == 0).all() and first.numel() >= 40004
    now["capturing"] = False
    assert prog.forward_ws(4, 1, 8) is two and [x.data_ptr() for x in prog.fwd_ws.values()] == kept


def test_the_step_state_size_is_the_headers():
    import os
    import re

    from minitp import _native as N
    from tests.conftest import ROOT

    header = open(os.path.join(ROOT, "include", "minitp.h")).read()
    assert N.QWEN2_STATE_BYTES == int(re.search(r"#define MINITP_QWEN2_STATE_BYTES (\d+)", header).group(1))


@pytest.mark.parametrize("prefixed", [False, True])
def test_the_last_positions_logits_alone_on_every_path(prefixed, monkeypatch):
    """prefill_logits="last" is [B, 1, V] whatever runs the forward."""
    model = _model()
    every = torch.arange(2 * 3 * 64, dtype=torch.float32).view(2, 3, 64)
    monkeypatch.setattr(model, "forward", lambda ids, positions, kv_cache: every)
    ids = torch.zeros(2, 3, dtype=torch.long)
    for form, want in (("last", every[:, -1:]), ("all", every)):
        kv = _behind(model)[0] if prefixed else make_kv_cache(model, 2, 8)
        assert torch.equal(GenerationState(model, ids, 4, kv=kv, prefill_logits=form).prefill(), want)


def test_no_operator_keeps_scratch_between_calls(monkeypatch):
    """Scratch that calls share would be written by two streams at once, and
    replaced under a captured call when a larger one comes."""
    from minitp import _native as N
    from minitp import kernels as K

    class Lib:
        def __init__(self):
            self.took = []

        def __getattr__(self, name):
            if name.endswith("_workspace_bytes"):
                return lambda *a: 1000
            return lambda *a: self.took.append(a) or N.OK

    def kept(*a):
        raise AssertionError("scratch that is kept")

    lib = Lib()
    for sizes in ("_argmax_bytes", "_attention_bytes"):
        if hasattr(K, sizes):
            monkeypatch.setattr(K, sizes, lambda *a: 1000)
    monkeypatch.setattr(K, "_lib", lambda: lib)
    monkeypatch.setattr(N, "require_gpu", lambda *a, **k: None)
    monkeypatch.setattr(N, "stream", lambda: 0)
    monkeypatch.setattr(N, "scratch", kept, raising=False)
    K.argmax(torch.zeros(2, 50))
    K.attention(torch.zeros(2, 1, 4, 16), torch.zeros(2, 2, 8, 16), torch.zeros(2, 2, 8, 16), 3)
    assert [a[-1] for a in lib.took] == [1000, 1000] and all(a[-2] % 16 == 0 for a in lib.took)
