"""Greedy token loop over the KV cache (minitp/generation.py:36-171).

Same objects and methods as the reference. ``GenerationState`` is the one
hot path: ``prefill`` runs the native whole-model program, ``decode_step``
replays the program's decode hipGraph (one graph launch per token), and the
greedy token of every step is written by the LM-head kernel straight into
``out_ids[:, cursor]``, so ``select_next`` on the logits a step just
produced returns that column and ``append`` has nothing left to copy.
Fixed-length mode (``early_stop=False``) therefore issues no host sync and
no extra kernels per token.

Early stop on an EOS token keeps the reference's finished mask on the
device: one more kernel after each token selection applies
``tok = where(finished, eos, tok); finished |= tok == eos`` and, once every
row has finished, records the stop column and writes it to a pinned host
word. The host reads that word instead of a blocking ``finished.all()``
copy each step; it keeps at most ``EOS_LAG`` steps queued ahead of the GPU,
and the steps it queued past the stop write no KV rows, so the result, the
cursor and ``kv.seq_len`` are the reference's.

Each ``decode_step`` returns a new logits tensor [B, 1, V], as the
reference does. ``reuse_decode_logits=True`` (what ``generate_greedy`` and
the benchmark use, since they only read the token the step picked) writes
every step's logits into one buffer instead, so the logits a step returned
are overwritten by the next step.

``prefill`` returns every prompt position's logits [B, T, V], as the
reference does, unless the state was made with ``prefill_logits="last"``:
then [B, 1, V] of the last position, the only row a token is picked from.
``generate_greedy`` uses that form, which skips T - 1 of the T LM-head rows
of the prompt (the greedy ids are the same).
"""

from __future__ import annotations

import collections
import ctypes

import torch

from minitp import _native as N
from minitp.kv_cache import KVCache
from minitp.layer import TPQwen2ForCausalLM

EOS_LAG = 2  # decode steps the host may queue before it reads the stop word


def _kv_heads_local(model: TPQwen2ForCausalLM) -> int:
    return model.model.layers[0].self_attn.kv_heads_local


def make_kv_cache(model: TPQwen2ForCausalLM, batch_size: int, max_seq_len: int, init: str = "empty") -> KVCache:
    p = next(model.parameters())
    return KVCache(num_layers=model.cfg.num_hidden_layers, batch_size=batch_size,
                   kv_heads_local=_kv_heads_local(model), head_dim=model.cfg.head_dim, max_seq_len=max_seq_len,
                   dtype=p.dtype, device=p.device, init=init)


def select_token(model: TPQwen2ForCausalLM, logits: torch.Tensor, distributed_argmax: bool = True) -> torch.Tensor:
    """Greedy pick from the last position's logits (generation.py:54-67)."""
    if distributed_argmax:
        return model.lm_head.distributed_argmax(logits[:, -1]).squeeze(-1)
    if model.ctx.tp_size == 1:
        from minitp import kernels as K

        return K.argmax(logits[:, -1])
    raise NotImplementedError("tp_size > 1 is not built on MI355X")


class GenerationState:
    """KV cache + positions buffer + output buffer (generation.py:70-130)."""

    def __init__(self, model: TPQwen2ForCausalLM, input_ids: torch.Tensor, max_new_tokens: int,
                 kv: KVCache | None = None, distributed_argmax: bool = True, kv_init: str = "empty",
                 prefill_logits: str = "all", reuse_decode_logits: bool = False) -> None:
        if prefill_logits not in ("all", "last"):
            raise ValueError(f"prefill_logits must be 'all' or 'last', got {prefill_logits!r}")
        self.model = model
        self.prefill_logits = prefill_logits
        self.reuse_decode_logits = reuse_decode_logits
        self.distributed_argmax = distributed_argmax
        b, t = input_ids.shape
        self.prompt_len = t
        self.max_new_tokens = max_new_tokens
        self.total = t + max_new_tokens
        self.kv = kv if kv is not None else make_kv_cache(model, b, self.total, init=kv_init)
        device = input_ids.device
        self.out_ids = torch.empty(b, self.total, dtype=torch.long, device=device)
        self.out_ids[:, :t] = input_ids
        self._start = self.kv.prefix_rows()  # positions continue a shared prefix
        self.positions_buf = torch.arange(self._start, self._start + self.total, device=device)  # the only arange
        self.cursor = t
        self.finished: torch.Tensor | None = None
        self.eos = -1
        self._native = model.native_path() and device.type == "cuda" and self.kv.prefix is None
        self._last_logits: torch.Tensor | None = None
        self._last_tok: torch.Tensor | None = None
        self._decode_logits: torch.Tensor | None = None
        self._eos_dev: torch.Tensor | None = None  # [B + 2] finished flags, halted, stop column
        self._eos_host: torch.Tensor | None = None  # pinned stop column (0 = running)
        self._eos_host_dev: int | None = None

    def _check_prefix(self) -> None:
        """The positions in the buffer go on from the prefix that the cache had."""
        rows = self.kv.prefix_rows()
        if rows != self._start:
            raise ValueError(f"GenerationState: built for {self._start} prefix rows, the cache has {rows}")

    def _enable_device_eos(self, eos: int) -> None:
        """Keep generate_greedy's finished mask and stop test on the device."""
        b = self.out_ids.shape[0]
        self.eos = eos
        self._eos_dev = torch.zeros(b + 2, dtype=torch.long, device=self.out_ids.device)
        self._eos_host = torch.zeros(1, dtype=torch.long, pin_memory=True)
        dev = ctypes.c_void_p()
        N.check(N.lib().minitp_host_device_pointer(self._eos_host.data_ptr(), ctypes.byref(dev)), "host_device_pointer")
        self._eos_host_dev = dev.value

    def _eos_args(self) -> tuple | None:
        if self._eos_dev is None:
            return None
        return (self._eos_dev.data_ptr(), self.eos, self.cursor, self._eos_host_dev)

    def _eos_stop(self) -> int:
        """Stop column the device recorded (0 while some row is running)."""
        return int(self._eos_host[0])

    def _next_column(self) -> torch.Tensor | None:
        return self.out_ids[:, self.cursor] if self.cursor < self.total else None

    def _check_position(self, last: int) -> None:
        limit = self.model.cfg.max_position_embeddings
        if last >= limit:
            raise IndexError(f"position {last} out of range for RoPE table of {limit} rows")

    def prefill(self) -> torch.Tensor:
        """Prompt forward; positions come from the buffer (0..T-1, behind a
        shared prefix the T after it)."""
        self._check_prefix()
        positions = self.positions_buf[: self.prompt_len]
        ids = self.out_ids[:, : self.prompt_len]
        last_only = self.prefill_logits == "last"
        if not self._native:
            if last_only and self.kv.prefix is not None and self.model.native_path() and ids.is_cuda:
                self._check_position(self._start + self.prompt_len - 1)
                return self.model._native(ids, positions, self.kv, last_only=True)
            logits = self.model(ids, positions=positions, kv_cache=self.kv)
            return logits[:, -1:] if last_only else logits
        self._check_position(self.prompt_len - 1)
        col = self._next_column()
        logits = self.model._native(ids, positions, self.kv, next_tok=col, eos=self._eos_args(),
                                    last_only=last_only)
        self._last_logits, self._last_tok = logits, col
        return logits

    def select_next(self, logits: torch.Tensor) -> torch.Tensor:
        if logits is self._last_logits and self._last_tok is not None:
            return self._last_tok
        return select_token(self.model, logits, self.distributed_argmax)

    def append(self, tok: torch.Tensor) -> torch.Tensor:
        """Write the token at the cursor; return its absolute position tensor."""
        col = self.out_ids[:, self.cursor]
        if not (tok.data_ptr() == col.data_ptr() and tok.shape == col.shape and tok.stride() == col.stride()):
            self.out_ids[:, self.cursor] = tok
        pos = self.positions_buf[self.cursor]
        self.cursor += 1
        return pos

    def decode_step(self, tok: torch.Tensor, pos: torch.Tensor) -> torch.Tensor:
        if not self._native:
            self._check_prefix()
            return self.model(tok.unsqueeze(-1), positions=pos.unsqueeze(-1), kv_cache=self.kv)
        b = tok.shape[0]
        if pos.data_ptr() == self.positions_buf.data_ptr() + (self.cursor - 1) * 8:
            self._check_position(self.cursor - 1)  # pos is positions_buf[cursor - 1]: value known
        else:
            # any other position tensor: read its value (one host sync, off the
            # generate_greedy path) so that it indexes the RoPE table as the
            # reference's gather does: past the table raises IndexError, a
            # negative position wraps (rope.py:37-45)
            from minitp.rope import _check_positions

            limit = self.model.cfg.max_position_embeddings
            _check_positions(pos, limit)
            pos = torch.where(pos < 0, pos + limit, pos)
        if not self.reuse_decode_logits or self._decode_logits is None or self._decode_logits.shape[0] != b:
            self._decode_logits = torch.empty(b, 1, self.model.cfg.vocab_size, dtype=self.kv.k_buf.dtype,
                                              device=self.out_ids.device)
        if tok.dtype != torch.long:
            tok = tok.long()
        col = self._next_column()
        logits = self.model.decode_native(tok, pos.reshape(()), self.kv, self._decode_logits, col,
                                          eos=self._eos_args())
        self._last_logits, self._last_tok = logits, col
        return logits


@torch.inference_mode()
def generate_greedy(model: TPQwen2ForCausalLM, input_ids: torch.Tensor, max_new_tokens: int,
                    eos_token_id: int | None = None, distributed_argmax: bool = True, early_stop: bool = True,
                    kv: KVCache | None = None, kv_init: str = "empty") -> torch.Tensor:
    """Greedy decode through GenerationState (generation.py:133-171): trimmed at
    the first step where every row has produced EOS when ``early_stop``;
    exactly prompt + max_new_tokens columns otherwise."""
    state = GenerationState(model, input_ids, max_new_tokens, kv=kv, distributed_argmax=distributed_argmax,
                            kv_init=kv_init, prefill_logits="last", reuse_decode_logits=True)
    b = input_ids.shape[0]
    if early_stop and eos_token_id is not None and state._native and max_new_tokens > 0:
        return _generate_device_eos(state, eos_token_id, max_new_tokens)
    if early_stop and eos_token_id is not None:
        state.eos = eos_token_id
        state.finished = torch.zeros(b, dtype=torch.bool, device=input_ids.device)
    logits = state.prefill()
    eos_tok = torch.tensor(state.eos, device=input_ids.device)
    for step in range(max_new_tokens):
        tok = state.select_next(logits)
        if state.finished is not None:
            tok = torch.where(state.finished, eos_tok, tok)
            state.finished = state.finished | (tok == state.eos)
        pos = state.append(tok)
        if state.finished is not None and bool(state.finished.all()):
            break
        if step + 1 < max_new_tokens:
            logits = state.decode_step(tok, pos)
    return state.out_ids[:, : state.cursor] if early_stop else state.out_ids


EOS_BEAM_STEPS = 8  # steps between the host's looks at the finished flags of a beam search


@torch.inference_mode()
def generate_beam(model: TPQwen2ForCausalLM, input_ids: torch.Tensor, max_new_tokens: int, num_beams: int,
                  eos_token_id: int | None = None, length_penalty: float = 0.0,
                  early_stop: bool = True) -> tuple[torch.Tensor, torch.Tensor]:
    """Beam search from prompts [B, T] (no counterpart in the reference, which
    decodes greedily): (ids [B, num_beams, T + n], scores [B, num_beams]), best
    first by score / length ** length_penalty, n = max_new_tokens, or with
    ``early_stop`` the longest beam's tokens once every beam has finished.

    A prompt's K/V rows are computed and kept once; its beams share them
    (KVCache.share_prefix) and only their new rows follow the selection. A
    beam that has produced ``eos_token_id`` stays a candidate with its score
    and length and is padded with that token. scores are summed
    log-probabilities; a beam that does not exist (fewer continuations than
    beams) scores minus infinity."""
    from minitp import kernels as K

    b, t = input_ids.shape
    if not 1 <= num_beams <= K.MAX_BEAMS or max_new_tokens < 1:
        raise ValueError(f"generate_beam: num_beams={num_beams}, max_new_tokens={max_new_tokens}")
    limit = model.cfg.max_position_embeddings
    if t + max_new_tokens - 1 > limit:  # the last token is selected, not forwarded
        raise IndexError(f"position {t + max_new_tokens - 2} out of range for RoPE table of {limit} rows")
    device, beams = input_ids.device, b * num_beams
    prompt = make_kv_cache(model, b, t)
    if model.native_path() and device.type == "cuda":
        logits = model._native(input_ids, torch.arange(t, device=device), prompt, last_only=True)
    else:
        logits = model(input_ids, kv_cache=prompt)[:, -1:]
    kv = make_kv_cache(model, beams, max_new_tokens)
    kv.share_prefix(prompt)
    logits = logits.expand(b, num_beams, -1)  # one beam a prompt so far
    scores = torch.full((b, num_beams), float("-inf"), device=device)
    scores[:, 0] = 0.0
    lengths = torch.zeros(b, num_beams, dtype=torch.long, device=device)
    finished = None if eos_token_id is None else torch.zeros(b, num_beams, dtype=torch.bool, device=device)
    steps: list[K.BeamStep] = []
    for step in range(max_new_tokens):
        s = K.beam_select(logits, scores, finished, lengths, eos_token_id=eos_token_id, length_penalty=length_penalty)
        steps.append(s)
        scores, lengths = s.scores, s.lengths
        if eos_token_id is not None:
            finished = s.finished
            if early_stop and (step + 1) % EOS_BEAM_STEPS == 0 and bool(finished.all()):
                break
        if step + 1 < max_new_tokens:
            kv.reorder(s.parents)
            logits = model(s.tokens.view(-1, 1), kv_cache=kv).view(b, num_beams, -1)
    # the beams' tokens, from the last step back through the parents
    out = torch.empty(beams, t + len(steps), dtype=torch.long, device=device)
    row = torch.arange(beams, device=device)
    for i in reversed(range(len(steps))):
        out[:, t + i] = steps[i].tokens.view(-1)[row]
        row = steps[i].parents.view(-1)[row]
    out = out.view(b, num_beams, -1)
    out[:, :, :t] = input_ids[:, None]
    order = (scores.double() / lengths.clamp(min=1).double() ** length_penalty).sort(
        dim=1, descending=True, stable=True).indices
    if early_stop and eos_token_id is not None:
        out = out[:, :, :t + int(lengths.max())]
    return out.gather(1, order[:, :, None].expand_as(out)), scores.gather(1, order)


def _generate_device_eos(state: GenerationState, eos: int, max_new_tokens: int) -> torch.Tensor:
    """generate_greedy's early-stop loop with the finished mask on the device."""
    if eos < 0:
        raise ValueError(f"eos_token_id must be >= 0, got {eos}")
    state._enable_device_eos(eos)
    kv_start = state.kv.seq_len
    logits = state.prefill()
    inflight: collections.deque = collections.deque()
    for step in range(max_new_tokens):
        tok = state.select_next(logits)
        pos = state.append(tok)
        if step + 1 >= max_new_tokens:
            break
        while len(inflight) >= EOS_LAG:
            inflight.popleft().synchronize()
        if state._eos_stop():
            break
        logits = state.decode_step(tok, pos)
        ev = torch.cuda.Event()
        ev.record()
        inflight.append(ev)
    torch.cuda.current_stream().synchronize()
    stop = state._eos_stop()
    if stop:
        # every column after the stop was a step the device ran halted
        state.cursor = stop
        state.kv.seq_len = kv_start + stop - 1  # the prompt, then one decode per column before the stop
    state.finished = state._eos_dev[: state.out_ids.shape[0]].bool()
    return state.out_ids[:, : state.cursor]
