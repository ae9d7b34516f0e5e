"""KV cache held in 8 or 4 bits: rows are quantised as they are written, read back for a prefill chunk, and attended over
in their quantised form by a decode step.

A row (one token of one KV head, 128 values) has one bf16 scale in 8 bits and one for each 32 values in 4 bits, so a cached
token takes 260 or 144 bytes per KV head where bf16 takes 512.  ``value = (stored - 128) * scale`` or
``(stored - 8) * scale``, within half a scale of what was written.  In 4 bits a row's 32 runs of four values are stored in
the order ``(run % 8, run // 8)``, the lower nibble of a byte first.  Values have no gradient: this is a serving cache.
"""

from __future__ import annotations

import math
import threading
from contextlib import nullcontext
from operator import index

import torch

from ._lib import SkvError, SkvQCache, SkvRows, check, dtype_code, elsewhere, lib, stream_ptr

__all__ = ["QuantKVCache", "QuantAttentionGraph"]

_empty_like, _CONTIGUOUS = torch.empty_like, torch.contiguous_format


class QuantKVCache:
    """Quantised cache of all layers, in place of ``KVCache``: ``k[i], v[i] [B, H_kv, L, 128 * bits / 8]`` uint8 and
    ``scale[i] [B, H_kv, L, 2, groups]`` bf16 (the key's scales, then the value's)."""

    plain = False
    first = 0                                              # position of the first row

    def __init__(self, layers: int, batch: int, h_kv: int, max_seq_len: int, d: int, bits: int, device):
        if bits not in (8, 4):
            raise ValueError("a quantised cache holds 8 or 4 bits per value")
        if d != 128:
            raise ValueError("the kernels are built for head_dim 128")
        groups, width = (1 if bits == 8 else 4), d * bits // 8
        # a code of 0 with a scale of 0: rows that were never written read as zeros
        self._set([torch.zeros(batch, h_kv, max_seq_len, width, dtype=torch.uint8, device=device) for _ in range(layers)],
                  [torch.zeros(batch, h_kv, max_seq_len, width, dtype=torch.uint8, device=device) for _ in range(layers)],
                  [torch.zeros(batch, h_kv, max_seq_len, 2, groups, dtype=torch.bfloat16, device=device)
                   for _ in range(layers)], bits, None)

    @classmethod
    def from_tensors(cls, k: list, v: list, scale: list, bits: int, status: torch.Tensor | None = None) -> "QuantKVCache":
        """A cache over tensors that the caller holds (per layer, contiguous, in the layout above)."""
        if bits not in (8, 4):
            raise ValueError("a quantised cache holds 8 or 4 bits per value")
        if not (len(k) == len(v) == len(scale) >= 1):
            raise ValueError("one tensor of codes of the keys, of the values and of scales is needed per layer")
        B, H, L, w = k[0].shape
        want = {"codes": ((B, H, L, 16 * bits), torch.uint8), "scales": ((B, H, L, 2, 1 if bits == 8 else 4), torch.bfloat16)}
        for name, ts in (("codes", k), ("codes", v), ("scales", scale)):
            for t in ts:
                if tuple(t.shape) != want[name][0] or t.dtype != want[name][1] or not t.is_contiguous() \
                        or t.device != k[0].device:
                    raise ValueError(f"{name} must be contiguous {want[name][0]} {want[name][1]} on one device")
        if status is not None and (status.shape != (B * H,) or status.dtype != torch.int32 or not status.is_contiguous()
                                   or status.device != k[0].device):
            raise ValueError(f"status must be contiguous ({B * H},) int32 on the cache's device")
        self = cls.__new__(cls)
        self._set(list(k), list(v), list(scale), bits, status)
        return self

    def _set(self, k, v, scale, bits, status) -> None:
        self._k, self._v, self._scale, self.bits = tuple(k), tuple(v), tuple(scale), bits
        self.batch, self.h_kv, self.max_seq_len, _ = k[0].shape
        self.d, self.device = 128, k[0].device
        self.cur_len = 0
        self._kept = threading.local()                     # plans of writes and reads (below), one set per thread
        self._status = torch.zeros(self.batch * self.h_kv, dtype=torch.int32, device=self.device) if status is None else status
        self._st = [SkvQCache(a.data_ptr(), b.data_ptr(), s.data_ptr(), self.status.data_ptr(), self.batch, self.h_kv,
                              self.max_seq_len, self.d, bits, 0) for a, b, s in zip(k, v, scale)]

    # (read-only: calls go by the addresses taken above)
    k = property(lambda self: self._k)
    v = property(lambda self: self._v)
    scale = property(lambda self: self._scale)
    status = property(lambda self: self._status)

    def _on_gpu(self) -> None:
        if self.device.type != "cuda":
            raise ValueError("a quantised cache is written, read and attended over on a CUDA device only")

    def sequence(self, b: int) -> "QuantKVCache":
        """Sequence ``b`` alone, on the same memory."""
        if not 0 <= b < self.batch:
            raise ValueError(f"the cache holds {self.batch} sequences")
        h = self.h_kv
        one = self.from_tensors([t[b:b + 1] for t in self.k], [t[b:b + 1] for t in self.v],
                                [t[b:b + 1] for t in self.scale], self.bits, self.status[b * h:(b + 1) * h])
        # (its own scales may begin off the 16-byte boundary that a call's buffers have to be on: the whole cache's, and b on)
        one._st = [SkvQCache(s.k, s.v, s.scale, s.status, 1, h, self.max_seq_len, self.d, self.bits, s.skip + b) for s in self._st]
        return one

    def check_status(self) -> int:
        """Bits of ``SKV_ST_*`` over all heads (a position outside the cache was skipped); synchronises."""
        bits = 0
        for s in set(self.status.tolist()):
            bits |= s
        return bits

    def _where(self, rows: SkvRows, pos, b: int, count: int) -> None:
        """Set the call's position, checked where the host knows it."""
        if torch.is_tensor(pos):
            if pos.dtype is not torch.long or pos.device != self.device or pos.dim() != 1 or not pos.is_contiguous() \
                    or pos.shape[0] not in (1, b):
                raise ValueError("positions are an int, or int64 [1] or [sequences] on the cache's device")
            rows.pos, rows.pos_per_seq = pos.data_ptr(), int(pos.shape[0] != 1)
            return
        at = index(pos)
        if not 0 <= at <= self.max_seq_len - count:
            raise ValueError(f"rows [{at}, {at + count}) lie outside the cache's {self.max_seq_len} positions")
        rows.pos, rows.pos_per_seq, rows.pos0 = None, 0, at

    def _plan(self, key, make):
        """What calls of one shape and type have in common, checked once (a decode step makes the same call again and
        again).  Per thread: the struct is filled in and read by the call."""
        kept = self._kept.__dict__
        plan = kept.get(key)
        if plan is None:
            if len(kept) >= 256:
                kept.clear()
            plan = kept[key] = make()
        return plan

    def _plan_write(self, k: torch.Tensor, v: torch.Tensor):
        """``(rows, straight)``; not straight: the rows have to be copied first (a last stride other than 1, rows off the
        16-byte boundaries)."""
        if k.dim() != 4 or k.shape != v.shape or k.shape[1] != self.h_kv or k.shape[3] != self.d or k.shape[0] > self.batch:
            raise ValueError(f"keys and values must be [sequences <= {self.batch}, {self.h_kv}, tokens, {self.d}]")
        if k.dtype != v.dtype:
            raise ValueError("keys and values must be of one type, on the cache's device")
        if k.shape[2] > self.max_seq_len:
            raise ValueError(f"{k.shape[2]} rows do not fit the cache's {self.max_seq_len} positions")
        strides = k.stride()[:3] + v.stride()[:3]
        straight = k.stride(3) == v.stride(3) == 1 and not any(s % (16 // k.element_size()) for s in strides)
        return SkvRows(0, 0, None, 0, *strides, 0, dtype_code(k.dtype), k.shape[0], k.shape[2]), straight

    def write(self, layer: int, k: torch.Tensor, v: torch.Tensor, pos) -> None:
        """Quantise ``k, v [b, H_kv, T, 128]`` (bf16 or float32, any strides) into the rows ``[pos, pos + T)`` of the
        first ``b`` sequences.  ``pos``: an int, or int64 in device memory, one for all or one per sequence; rows that a
        device position puts behind the cache's end (all rows, where it is negative) are left out and recorded in ``status``."""
        rows, straight = self._plan((k.shape, k.stride(), k.dtype, v.shape, v.stride(), v.dtype), lambda: self._plan_write(k, v))
        dev = self.device
        if k.device != dev or v.device != dev:
            raise ValueError("keys and values must be of one type, on the cache's device")
        if (k.requires_grad or v.requires_grad) and torch.is_grad_enabled():
            raise ValueError("a quantised cache has no gradient: write under torch.no_grad()")
        kp, vp = k.data_ptr(), v.data_ptr()
        if not straight or (kp | vp) % 16:
            return self.write(layer, k.clone(memory_format=torch.contiguous_format),
                              v.clone(memory_format=torch.contiguous_format), pos)
        self._where(rows, pos, rows.batch, rows.tokens)
        if rows.batch == 0 or rows.tokens == 0:
            return
        self._on_gpu()
        if elsewhere(dev):
            with torch.cuda.device(dev):
                return self.write(layer, k, v, pos)
        rows.k, rows.v = kp, vp
        check(lib().skv_quant_write(self._st[layer], rows, stream_ptr(dev)), "skv_quant_write")

    def _plan_read(self, b: int, count: int, dtype: torch.dtype):
        if not 0 <= b <= self.batch:
            raise ValueError(f"the cache holds {self.batch} sequences")
        if not 0 <= count <= self.max_seq_len:
            raise ValueError(f"{count} rows lie outside the cache's {self.max_seq_len} positions")
        hs = count * self.d
        # (a result made like a tensor at hand costs the host half of one made from a shape: 2.5 against 4.5 us for both; this
        # one is a single element, expanded)
        like = torch.empty(1, dtype=dtype, device=self.device).expand(b, self.h_kv, count, self.d)
        return like, SkvRows(0, 0, None, 0, self.h_kv * hs, hs, self.d, self.h_kv * hs, hs, self.d,
                                                         0, dtype_code(dtype), b, count)

    def read(self, layer: int, pos, count: int, *, dtype: torch.dtype = torch.bfloat16,
             batch: int | None = None) -> tuple[torch.Tensor, torch.Tensor]:
        """The rows ``[pos, pos + count)`` of the first ``batch`` (all) sequences as ``k, v [b, H_kv, count, 128]`` of
        ``dtype``; ``pos`` as in ``write`` (rows outside the cache come back as zeros and are recorded)."""
        b, dev = self.batch if batch is None else batch, self.device
        like, rows = self._plan((b, count, dtype), lambda: self._plan_read(b, count, dtype))
        self._where(rows, pos, b, count)
        k, v = _empty_like(like, memory_format=_CONTIGUOUS), _empty_like(like, memory_format=_CONTIGUOUS)
        if b == 0 or count == 0:
            return k, v
        self._on_gpu()
        if elsewhere(dev):
            with torch.cuda.device(dev):
                return self.read(layer, pos, count, dtype=dtype, batch=batch)
        rows.k, rows.v = k.data_ptr(), v.data_ptr()
        check(lib().skv_quant_read(self._st[layer], rows, stream_ptr(dev)), "skv_quant_read")
        return k, v

    def rows(self, layer: int, b: int, n: int, dtype: torch.dtype) -> tuple[torch.Tensor, torch.Tensor]:
        """Rows ``[0, n)`` of the first ``b`` sequences, for a prefill chunk's attention."""
        return self.read(layer, 0, n, dtype=dtype, batch=b)


class QuantAttentionGraph:
    """Exact decode attention over the quantised rows ``[0, n)``, with ``n`` in device memory: ``DenseAttentionGraph``
    for a ``QuantKVCache``.  The object owns the workspace and the output buffer, which the next call overwrites: calls
    of one object (and graphs captured from it) must not overlap on the GPU.  bf16: a weight times a value's scale is a half
    float (11 bits) in the product with the codes; scores and sums are float32."""

    def __init__(self, *, H: int, H_kv: int, d: int, dtype, device):
        if H % H_kv:
            raise ValueError("the query heads must divide into the KV heads")
        L = lib()
        self.H, self.H_kv, self.d, self.G = H, H_kv, d, H // H_kv
        self.n_group = 0                                   # heads per entry of the device-side lengths (0: one length)
        self.dtype = dtype
        self._code = dtype_code(dtype)
        with torch.cuda.device(device) if torch.device(device).type == "cuda" else nullcontext():
            self.ctas = L.skv_quant_ctas()
            size = L.skv_quant_workspace_bytes(H_kv, self.G, d, self.ctas)
            if size < 0:
                raise SkvError(L.skv_error_string(int(size)).decode())
            self.ws = torch.zeros(size, dtype=torch.uint8, device=device)
            self.out = torch.empty(H, d, dtype=dtype, device=device)
        self.device = self.out.device                      # (with its index)
        self._shape, self._scale = self.out.shape, 1.0 / math.sqrt(d)

    def __call__(self, q: torch.Tensor, cache: QuantKVCache, layer: int, n_dev: torch.Tensor) -> torch.Tensor:
        """``q [H, d]`` (all sequences' query heads), ``n_dev`` int32 on the device: one length, or one per ``n_group``
        heads.  A head without rows gets zeros."""
        if q.shape != self._shape or q.dtype is not self.dtype:
            raise ValueError(f"queries must be {tuple(self._shape)} {self.dtype}")
        dev = self.device
        if cache.batch * cache.h_kv != self.H_kv or cache.device != dev or q.device != dev:
            raise ValueError(f"the cache must hold {self.H_kv} KV heads, on the queries' device")
        if n_dev.dtype is not torch.int32 or n_dev.device != dev or not n_dev.is_contiguous() \
                or n_dev.numel() < (-(-self.H_kv // self.n_group) if self.n_group else 1):
            raise ValueError("lengths must be int32 on the queries' device: one, or one per n_group heads")
        cache._on_gpu()
        if not q.is_contiguous() or q.data_ptr() % 16 or q.data_ptr() == self.out.data_ptr():
            q = q.clone(memory_format=torch.contiguous_format)
        if elsewhere(dev):
            with torch.cuda.device(dev):
                return self(q, cache, layer, n_dev)
        check(lib().skv_attend_quant(cache._st[layer], q.data_ptr(), self._code, self.G, n_dev.data_ptr(), self.n_group,
                                     self.out.data_ptr(), self.ws.data_ptr(), self.ctas, self._scale, stream_ptr(dev)),
              "skv_attend_quant")
        return self.out
