"""Steps behind a shared prefix that run beside other work of the same model:
on two streams at once, and captured, with larger forwards between replays."""

import pytest
import torch

from tests.test_gpu_beam_search import _pair

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _busy(streams):
    """Work in front of what is queued next, so that the streams' queues fill
    before either begins."""
    a = torch.randn(8192, 8192, device=DEV, dtype=torch.bfloat16)
    torch.cuda.synchronize()
    for s in streams:
        with torch.cuda.stream(s):
            for _ in range(30):
                a @ a
    return a


def _prefix(model, rows=200, seed=9):
    from minitp.generation import make_kv_cache

    ids = torch.randint(0, 151936, (2, rows), generator=torch.Generator().manual_seed(seed)).to(DEV)
    pre = make_kv_cache(model, 2, 256)
    model(ids, kv_cache=pre)
    return pre


def _behind(model, pre, first):
    """A cache of six rows behind `pre` that holds one row of its own."""
    from minitp.generation import make_kv_cache

    kv = make_kv_cache(model, 6, 8)
    kv.share_prefix(pre)
    model(first, kv_cache=kv)
    return kv


def _tokens(count, seed):
    g = torch.Generator().manual_seed(seed)
    return [torch.randint(0, 151936, (6, 1), generator=g).to(DEV) for _ in range(count)]


def test_two_beam_searches_at_once():
    from minitp.generation import generate_beam

    model, _ = _pair("qwen2.5-0.5b", torch.bfloat16)
    g = torch.Generator().manual_seed(4)
    prompts = [torch.randint(0, 151936, (2, t), generator=g).to(DEV) for t in (40, 57)]
    want = [generate_beam(model, p, 8, 4) for p in prompts]
    streams = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(2):
        held = _busy(streams)
        got = []
        for s, p in zip(streams, prompts):
            with torch.cuda.stream(s):
                got.append(generate_beam(model, p, 8, 4))
        torch.cuda.synchronize()
        del held
        for (ids, scores), (i, s) in zip(got, want):
            assert torch.equal(ids, i) and torch.equal(scores, s)


def test_a_captured_step_beside_larger_forwards():
    """The forwards between the replays outgrow every workspace, and memory
    that was given back is taken and filled."""
    model, _ = _pair("qwen2.5-0.5b", torch.bfloat16)
    pre, toks = _prefix(model), _tokens(4, 2)
    with torch.inference_mode():
        want = [model(t, kv_cache=_behind(model, pre, toks[3])) for t in toks[:3]]
        kv, tok = _behind(model, pre, toks[3]), toks[0].clone()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = model(tok, kv_cache=kv)
        for i in range(3):
            long = torch.randint(0, 151936, (8, 100 + 70 * i), device=DEV)
            model(long)
            taken = [torch.full((1 << 22,), float("nan"), device=DEV) for _ in range(16)]
            tok.copy_(toks[i])
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want[i])
            assert all(torch.isnan(x).all() for x in taken)


def test_two_captured_steps_at_once():
    """Each graph has its scratch; replays on two streams and an eager step on
    a third do not meet."""
    model, _ = _pair("qwen2.5-0.5b", torch.bfloat16)
    pre, toks = _prefix(model), _tokens(4, 6)
    with torch.inference_mode():
        want = [model(t, kv_cache=_behind(model, pre, toks[3])) for t in toks[:3]]
        graphs, outs = [], []
        caches = [_behind(model, pre, toks[3]) for _ in range(3)]
        for i in range(2):
            graphs.append(torch.cuda.CUDAGraph())
            with torch.cuda.graph(graphs[i]):
                outs.append(model(toks[i], kv_cache=caches[i]))
        streams = [torch.cuda.Stream() for _ in range(3)]
        for _ in range(3):
            held = _busy(streams)
            for i in range(2):
                with torch.cuda.stream(streams[i]):
                    for _ in range(4):
                        graphs[i].replay()
            with torch.cuda.stream(streams[2]):
                eager = []
                for _ in range(4):
                    caches[2].seq_len = 1
                    eager.append(model(toks[2], kv_cache=caches[2]))
            torch.cuda.synchronize()
            del held
            assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1])
            assert all(torch.equal(e, want[2]) for e in eager)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("t", [1, 9, 40])
def test_the_last_positions_logits_behind_a_prefix(t, dtype):
    """prefill_logits="last" gives [B, 1, V], the last row of the whole form,
    and never holds the others; greedy generation uses it."""
    from minitp.generation import GenerationState, generate_greedy, make_kv_cache

    model, _ = _pair("qwen2.5-0.5b", dtype)
    pre = _prefix(model, 70)
    asks = torch.randint(0, 151936, (6, t), generator=torch.Generator().manual_seed(t)).to(DEV)

    def behind():
        kv = make_kv_cache(model, 6, t + 4)
        kv.share_prefix(pre)
        return kv

    got, last_kv, all_kv = {}, behind(), behind()
    for form, kv in (("all", all_kv), ("last", last_kv)):
        st = GenerationState(model, asks, 4, kv=kv, prefill_logits=form)
        st.prefill()  # (workspaces are there)
        kv.seq_len = 0
        torch.cuda.synchronize()
        torch.cuda.reset_peak_memory_stats()
        start = torch.cuda.memory_allocated()
        got[form] = st.prefill()
        peak = torch.cuda.max_memory_allocated() - start
        assert got[form].shape == (6, t if form == "all" else 1, 151936) and kv.seq_len == t
    if t >= 9:
        assert peak < got["all"].numel() * got["all"].element_size() / 2
    # two forms of one forward, each within the path's own bar of the oracle's
    # logits (bf16 0.5, fp32 1e-3)
    bar = 0.5 if dtype == torch.bfloat16 else 1e-3
    assert (got["last"].float() - got["all"][:, -1:].float()).abs().max() <= 2 * bar
    assert torch.equal(last_kv.k_buf[:, :, :, :t], all_kv.k_buf[:, :, :, :t])
    ids = generate_greedy(model, asks, 4, kv=behind())
    assert torch.equal(ids[:, t].cpu(), got["last"][:, 0].float().cpu().argmax(-1))


def test_positions_past_the_table_behind_a_prefix():
    from minitp.generation import GenerationState, make_kv_cache

    model, _ = _pair("qwen2.5-0.5b", torch.bfloat16)
    pre = _prefix(model, 250)  # (of 256 positions)
    for form in ("all", "last"):
        kv = make_kv_cache(model, 2, 16)
        kv.share_prefix(pre)
        with pytest.raises(IndexError, match="position 256"):
            GenerationState(model, torch.zeros(2, 7, dtype=torch.long, device=DEV), 4, kv=kv, prefill_logits=form).prefill()
        assert kv.seq_len == 0


def _picks(seed):
    """An argmax over many slices and a one-token attention over many splits."""
    from minitp import kernels as K

    g = torch.Generator(device=DEV).manual_seed(seed)
    logits = torch.randn(6, 151936, generator=g, device=DEV)
    q = torch.randn(1, 1, 14, 64, generator=g, device=DEV).bfloat16()
    kc, vc = torch.randn(2, 1, 2, 4096, 64, generator=g, device=DEV).bfloat16().unbind(0)
    return lambda: (K.argmax(logits), K.attention(q, kc, vc, 4000))


def test_picks_and_attention_on_two_streams_and_in_graphs():
    """The calls of a greedy step module by module: scratch of their own, beside
    each other and beside larger calls between the replays."""
    from minitp import kernels as K

    calls = [_picks(1), _picks(2)]
    want = [c() for c in calls]
    streams = torch.cuda.Stream(), torch.cuda.Stream()
    held = _busy(streams)
    got = [[], []]
    for _ in range(6):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                got[i].append(calls[i]())
    torch.cuda.synchronize()
    graphs, outs = [], []
    for c in calls:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(c())
    for n in range(3):
        K.argmax(torch.randn(40 + 20 * n, 151936, device=DEV))
        taken = [torch.full((1 << 18,), float("nan"), device=DEV) for _ in range(16)]
        for s, g in zip(streams, graphs):
            with torch.cuda.stream(s):
                for _ in range(4):
                    g.replay()
        torch.cuda.synchronize()
        for i in range(2):
            got[i].append(tuple(x.clone() for x in outs[i]))
    del held, taken
    for i in range(2):
        assert all(torch.equal(a, b) for out in got[i] for a, b in zip(out, want[i]))


def test_greedy_generation_behind_a_prefix_on_two_streams():
    from minitp.generation import generate_greedy, make_kv_cache

    model, _ = _pair("qwen2.5-0.5b", torch.bfloat16)
    pre = _prefix(model, 120)
    g = torch.Generator().manual_seed(8)
    asks = [torch.randint(0, 151936, (6, t), generator=g).to(DEV) for t in (7, 12)]

    def run(ids):
        kv = make_kv_cache(model, 6, ids.shape[1] + 6)
        kv.share_prefix(pre)
        return generate_greedy(model, ids, 6, kv=kv)

    want = [run(a) for a in asks]
    streams = torch.cuda.Stream(), torch.cuda.Stream()
    held = _busy(streams)
    got = []
    for s, a in zip(streams, asks):
        with torch.cuda.stream(s):
            got.append(run(a))
    torch.cuda.synchronize()
    del held
    assert all(torch.equal(a, b) for a, b in zip(got, want))
