"""Cache of a batch whose sequences share a prefix (samples of one prompt, questions about one document): the prefix's
rows exist once, each sequence keeps only the rows behind it, and a decode step reads the prefix once for all of them."""

from __future__ import annotations

import math
from contextlib import nullcontext

import torch

from . import _lib
from ._lib import SkvError, SkvPrefix, check, dtype_code, elsewhere, lib, stream_ptr
from .qwen3 import KVCache

__all__ = ["PrefixKVCache", "PrefixAttentionGraph"]


class PrefixKVCache:
    """``prefix`` is a plain cache of one sequence (``model.prefill(prompt, cache.prefix)`` fills it); ``k[i], v[i] [B,
    H_kv, L, d]`` hold each sequence's own rows: position ``p`` of a sequence is own row ``p - first``."""

    plain = False

    def __init__(self, layers: int, batch: int, h_kv: int, prefix_len: int, own_len: int, d: int, dtype, device):
        self.prefix = KVCache(layers, 1, h_kv, prefix_len, d, dtype, device)
        self._own = KVCache(layers, batch, h_kv, own_len, d, dtype, device)
        self.k, self.v = self._own.k, self._own.v

    @property
    def first(self) -> int:
        """Position of the sequences' first own row: the prefix's length."""
        n = self.prefix.cur_len
        return n[0] if isinstance(n, list) else n          # (a list: prefilled as a ragged batch of one)

    @property
    def max_seq_len(self) -> int:
        return self.first + self._own.max_seq_len

    @property
    def cur_len(self):
        n = self._own.cur_len
        return [self.first + x for x in n] if isinstance(n, list) else self.first + n

    @cur_len.setter
    def cur_len(self, n) -> None:
        own = [x - self.first for x in n] if isinstance(n, (list, tuple)) else n - self.first
        if min(own) < 0 if isinstance(own, list) else own < 0:
            raise ValueError(f"the sequences begin behind the prefix's {self.first} rows")
        self._own.cur_len = own

    def prefix_rows(self, layer: int) -> tuple[torch.Tensor, torch.Tensor]:
        """``k, v [H_kv, first, d]`` of the shared rows."""
        return self.prefix.k[layer][0, :, :self.first], self.prefix.v[layer][0, :, :self.first]

    def sequence(self, b: int) -> "PrefixKVCache":
        """Sequence ``b`` alone behind the same prefix, on the same memory."""
        view = PrefixKVCache.__new__(PrefixKVCache)
        view.prefix, view._own = self.prefix, self._own.sequence(b)
        view.k, view.v = view._own.k, view._own.v
        return view

    def write(self, layer: int, k: torch.Tensor, v: torch.Tensor, start: int) -> None:
        if start < self.first:
            raise ValueError(f"the sequences begin behind the prefix's {self.first} rows")
        self._own.write(layer, k, v, start - self.first)

    def rows(self, layer: int, b: int, n: int, dtype: torch.dtype) -> tuple[torch.Tensor, torch.Tensor]:
        """Positions ``[0, n)`` of the first ``b`` sequences, the prefix repeated, for a prefill chunk's attention."""
        kp, vp = self.prefix_rows(layer)
        k, v = self._own.rows(layer, b, n - self.first, dtype)
        return torch.cat((kp.expand(b, -1, -1, -1), k), 2), torch.cat((vp.expand(b, -1, -1, -1), v), 2)


class PrefixAttentionGraph:
    """Exact decode attention of ``B`` sequences over a prefix they share and over their own rows ``[0, n)`` behind it,
    with ``n`` in device memory.  ``H, H_kv`` are per sequence.  The object owns the workspace and the output buffer,
    which the next call overwrites: calls of one object (and graphs captured from it) must not overlap on the GPU.  bf16:
    weights are rounded to bf16 in the product with the values, as in ``DenseAttentionGraph``; scores and sums are float32.
    ``check_status()`` tells of lengths beyond the own rows and of a wait that gave up."""

    def __init__(self, *, B: int, H: int, H_kv: int, d: int, dtype, device):
        if H % H_kv:
            raise ValueError("the query heads must divide into the KV heads")
        L = lib()
        self.B, self.H, self.H_kv, self.d, self.G = B, H, H_kv, d, H // H_kv
        self.n_group = 0                                   # KV heads per entry of the device-side lengths (0: one length)
        self.dtype = dtype
        self._code = dtype_code(dtype)
        with torch.cuda.device(device) if torch.device(device).type == "cuda" else nullcontext():
            self.num_splits = L.skv_prefix_splits(B, H_kv, self.G, self._code)
            size = L.skv_prefix_workspace_bytes(B, H_kv, self.G, d, self.num_splits) if self.num_splits > 0 \
                else self.num_splits
            if size < 0:
                raise SkvError(L.skv_error_string(int(size)).decode())
            self.ws = torch.zeros(size, dtype=torch.uint8, device=device)
            self.out = torch.empty(B * H, d, dtype=dtype, device=device)
            self.status = torch.zeros(B * H_kv, dtype=torch.int32, device=device)
        self.device = self.out.device                      # (with its index)
        self._shape, self._scale = self.out.shape, 1.0 / math.sqrt(d)
        self._layout = self._call = None                   # of the last call, and what it passed on
        self._second = None                                # launches of such a call beyond the first

    def check_status(self) -> int:
        """Bits of ``SKV_ST_*`` over all heads (a length beyond the own rows, a wait that gave up and left a wrong output);
        synchronises."""
        bits = 0
        for s in set(self.status.tolist()):
            bits |= s
        return bits

    def _plan(self, Kp, Vp, K, V) -> SkvPrefix:
        """What calls with caches of this layout pass on, checked once."""
        heads = self.B * self.H_kv
        if Kp.dim() != 3 or Kp.shape != Vp.shape or Kp.shape[0] != self.H_kv or Kp.shape[2] != self.d:
            raise ValueError(f"the prefix must be [{self.H_kv}, rows, {self.d}]")
        if K.dim() != 3 or K.shape != V.shape or K.shape[0] != heads or K.shape[2] != self.d:
            raise ValueError(f"the sequences' rows must be [{heads}, rows, {self.d}]")
        if any(t.shape[1] and t.stride(2) != 1 for t in (Kp, Vp, K, V)):
            raise ValueError("the caches must have a unit last stride")
        strides = [s for t in (Kp, Vp, K, V) for s in t.stride()[:2]]
        return SkvPrefix(0, 0, 0, 0, *strides, Kp.shape[1], K.shape[1], self.B, self.H_kv, self.G, self.d, self._code, 0)

    def __call__(self, q: torch.Tensor, Kp: torch.Tensor, Vp: torch.Tensor, K: torch.Tensor, V: torch.Tensor,
                 n_dev: torch.Tensor) -> torch.Tensor:
        """``q [B*H, d]``; ``Kp, Vp [H_kv, P, d]`` the shared rows; ``K, V [B*H_kv, L, d]`` the sequences' own rows;
        ``n_dev`` int32 on the device, own lengths: one, or one per ``n_group`` KV heads.  A row without keys gets zeros."""
        layout = (Kp.shape, Kp.stride(), Vp.shape, Vp.stride(), K.shape, K.stride(), V.shape, V.stride())
        if layout != self._layout:                         # (a decode step has the same layout again and again)
            self._call, self._layout, self._second = self._plan(Kp, Vp, K, V), layout, None
        dev, dtype = self.device, self.dtype
        if q.shape != self._shape or q.dtype is not dtype:
            raise ValueError(f"queries must be {tuple(self._shape)} {dtype}")
        if not (Kp.dtype is Vp.dtype is K.dtype is V.dtype is dtype and
                Kp.device == Vp.device == K.device == V.device == q.device == dev):
            raise ValueError("the caches must have the queries' type and device")
        if n_dev.dtype is not torch.int32 or n_dev.device != dev or not n_dev.is_contiguous() \
                or n_dev.numel() < (-(-self.B * self.H_kv // self.n_group) if self.n_group else 1):
            raise ValueError("lengths must be int32 on the queries' device: one, or one per n_group KV heads")
        if dev.type != "cuda":
            raise ValueError("a shared prefix is attended over on a CUDA device only")
        if not q.is_contiguous() or q.data_ptr() % 16 or q.data_ptr() == self.out.data_ptr():
            q = q.clone(memory_format=torch.contiguous_format)
        if elsewhere(dev):
            with torch.cuda.device(dev):
                return self(q, Kp, Vp, K, V, n_dev)
        c = self._call
        c.k_prefix, c.v_prefix, c.k, c.v = Kp.data_ptr(), Vp.data_ptr(), K.data_ptr(), V.data_ptr()
        c.n_group = self.n_group
        check(lib().skv_attend_prefix(c, q.data_ptr(), n_dev.data_ptr(), self.out.data_ptr(), self.ws.data_ptr(),
                                      self.num_splits, self.status.data_ptr(), self._scale, stream_ptr(dev)),
              "skv_attend_prefix")
        if self._second != 0:
            if self._second is None:
                self._second = lib().skv_prefix_launches(c, self.num_splits, self._scale) - 1
            _lib.launches += self._second
        return self.out
