"""Contiguous KV cache (minitp/kv_cache.py:8-63).

One buffer each for K and V, laid out [layer, batch, kv_head, seq, head_dim]
so a whole forward's cache is one allocation the kernels index directly.
``k[i]`` / ``v[i]`` are the per-layer [B, Hkv, S, D] views of the reference
API. ``seq_len`` is the host-side fill cursor; only rows [0, seq_len) are
ever read (write-before-read, so ``init="empty"`` is safe).

The buffers hold ``capacity`` >= max_seq_len rows per (batch row, KV head):
max_seq_len rounded up to a power of two (a multiple of 8192 past 8192).
The kernels index the cache with that row stride, so the native program
records one decode graph per capacity rather than one per generation length
(a 128-token prompt with 200 or with 256 new tokens replays the same graph).
The views keep the reference's [B, Hkv, max_seq_len, D] shape, and every
bound (``update``, ``check_room``) is max_seq_len.
"""

from __future__ import annotations

import torch

from minitp import kernels as K


def cache_capacity(max_seq_len: int) -> int:
    """Rows the buffers hold for a cache of max_seq_len positions."""
    if max_seq_len <= 8192:
        return 1 << max(0, (max_seq_len - 1).bit_length())
    return -(-max_seq_len // 8192) * 8192


class KVCache:
    def __init__(self, num_layers: int, batch_size: int, kv_heads_local: int, head_dim: int, max_seq_len: int,
                 dtype: torch.dtype, device: torch.device, init: str = "empty") -> None:
        if init not in ("empty", "zeros"):
            raise ValueError(f"init must be 'empty' or 'zeros', got {init!r}")
        self.max_seq_len = max_seq_len
        self.capacity = cache_capacity(max_seq_len)
        self.prefix: KVCache | None = None  # rows that groups of this cache's batch rows share (share_prefix)
        self.is_prefix = False
        self._rewrites = 0  # times that rows [0, seq_len) may have become others
        self._behind: tuple[int, int] | None = None  # the prefix's rows and rewrites under the rows written here
        self._seq_len = 0
        self.num_layers = num_layers
        shape = (num_layers, batch_size, kv_heads_local, self.capacity, head_dim)
        self.k_buf = torch.empty(shape, dtype=dtype, device=device)
        self.v_buf = torch.empty(shape, dtype=dtype, device=device)
        if init == "zeros":
            self._fill(0.0)
        self.k = [t[:, :, :max_seq_len] for t in self.k_buf.unbind(0)]
        self.v = [t[:, :, :max_seq_len] for t in self.v_buf.unbind(0)]

    @property
    def seq_len(self) -> int:
        return self._seq_len

    @seq_len.setter
    def seq_len(self, rows: int) -> None:
        if rows < self._seq_len:
            self._rewrites += 1
        if self._seq_len == 0 and self.prefix is not None:
            self._behind = self.prefix._seq_len, self.prefix._rewrites
        self._seq_len = rows

    def _fill(self, value: float) -> None:
        for buf in (self.k_buf, self.v_buf):
            if buf.is_cuda:
                K.fill_(buf, value)
            else:
                buf.fill_(value)

    def update(self, layer_idx: int, k_new: torch.Tensor, v_new: torch.Tensor):
        """Write [B, H, T, D] at the cursor; return the valid [:, :, :end] views."""
        t = k_new.shape[2]
        end = self.seq_len + t
        if end > self.max_seq_len:
            raise ValueError(f"KV cache overflow: seq {self.seq_len}+{t} > max_seq_len={self.max_seq_len}")
        K.kv_write(k_new, v_new, self.k[layer_idx], self.v[layer_idx], self.seq_len)
        return self.k[layer_idx][:, :, :end], self.v[layer_idx][:, :, :end]

    def check_room(self, t: int) -> None:
        if self.seq_len + t > self.max_seq_len:
            raise ValueError(f"KV cache overflow: seq {self.seq_len}+{t} > max_seq_len={self.max_seq_len}")

    def share_prefix(self, prefix: "KVCache") -> None:
        """Put ``prefix`` in front of this cache: every run of batch / (prefix
        batch) consecutive rows here continues one row of ``prefix``, whose
        rows [0, prefix.seq_len) are kept once and attended by all of them (no
        counterpart in the reference, whose caches hold a prompt per row). This
        cache must be empty: its rows' positions go on from the prefix's, and
        once there are some the prefix has to stay as it is (prefix_rows)."""
        mine, shared = self.k_buf.shape, prefix.k_buf.shape
        if prefix.prefix is not None or prefix is self or self.is_prefix:
            raise ValueError("a shared prefix cannot have a prefix of its own")
        if self.seq_len != 0:
            raise ValueError(f"share_prefix: the cache holds {self.seq_len} rows already")
        if mine[0] != shared[0] or mine[2] != shared[2] or mine[4] != shared[4] or \
                prefix.k_buf.dtype != self.k_buf.dtype or prefix.k_buf.device != self.k_buf.device:
            raise ValueError(f"prefix cache {tuple(shared)} {prefix.k_buf.dtype} on {prefix.k_buf.device} does not fit "
                             f"{tuple(mine)} {self.k_buf.dtype} on {self.k_buf.device}")
        if shared[1] == 0 or mine[1] % shared[1] != 0:
            raise ValueError(f"batch {mine[1]} not divisible by the prefix cache's batch {shared[1]}")
        self.prefix = prefix
        prefix.is_prefix = True

    def prefix_rows(self) -> int:
        """Rows of the shared prefix in front of this cache, 0 without one. A
        prefix that was continued, cut, filled anew or reordered since the first
        row was written here is refused: this cache's rows have positions, and
        hold keys and values, that go on from the rows that it had then."""
        pre = self.prefix
        if pre is None:
            return 0
        if self._seq_len > 0 and self._behind != (pre._seq_len, pre._rewrites):
            raise ValueError(f"shared prefix: the cache's {self._seq_len} rows were written behind {self._behind[0]} prefix "
                             f"rows, and the prefix, now of {pre._seq_len} rows, has changed since")
        return pre._seq_len

    def reorder(self, parents: torch.Tensor) -> None:
        """The written rows follow their beams, in place: batch row b of every
        layer takes the rows of batch row parents[b] (``kernels.kv_reorder``;
        parents [G, W] int64, beams of a group). A shared prefix stays, so
        the beams of a group have to share one."""
        if self.prefix is not None and parents.dim() == 2 and parents.shape[1] > 0:
            rows = self.k_buf.shape[1] // self.prefix.k_buf.shape[1]
            if rows % parents.shape[1] != 0:
                raise ValueError(f"reorder: groups of {parents.shape[1]} beams span several prefixes, of {rows} rows each")
        K.kv_reorder(self.k_buf, self.v_buf, parents, self.seq_len)
        self._rewrites += 1

    def advance(self, tokens: int) -> None:
        self.seq_len += tokens

    def poison(self, value: float = float("nan")) -> None:
        """Test helper: fill every slot (written or not) with a sentinel."""
        self._fill(value)
