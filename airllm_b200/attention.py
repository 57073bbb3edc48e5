"""Attention over a paged key-value cache on torch CUDA tensors (the amoe_rope_*, amoe_kv_*
and amoe_attn_* entry points of include/amoe.h).

The operators of the GPT-OSS layer's attention half between its two projections
(internal/model/gptoss/layer.go:40-92, internal/backend/cpuref/attention.go:11-171,
rope.go:10-86).  A serving loop holds one ``KVCache`` a layer, all over one page table:

    rope = Rope.yarn(64, 150000.0)
    cache = KVCache(pages, 64, kv_heads=8, head_dim=64, dtype=torch.float8_e4m3fn)
    # a prompt: packed rows of all sequences, cu their starts
    q = cache.append(k, v, table, past, cu, q=q, rope=rope, k_out=kr)   # kr: the rotated keys
    out = prefill(q, kr, v, cu, window=128, sinks=sinks)
    # a later chunk of the prompt reads what came before it back
    k_all, v_all = cache.read(table, cu_k, total, dtype=torch.bfloat16)
    # then one token a sequence and step
    q = cache.append(k, v, table, length, cu, q=q, rope=rope)
    out = cache.decode(q, table, length + 1, window=128, sinks=sinks)

Work is enqueued on ``stream`` (default: torch's current stream on the tensors' device) and
nothing waits for it.  Inputs, outputs and the cache must be ready on that stream, and not
be freed before it has run them (``Tensor.record_stream``), as with any torch operation.  Rows may be strided views with adjacent elements whose strides and
address are multiples of 16 bytes (a fused projection's slices are).  Arguments that cannot
be served raise ``AmoeError``; wrong page ids and lengths, which only the device sees, are
skipped there and reported by ``KVCache.check``.  Rows that a call writes must not lie in its inputs'
memory.  The operators serve; they have no backward pass, and their results carry no gradient.
"""
from __future__ import annotations

import ctypes
import struct

import torch

from .moe import (AMOE_ERR_INVALID, AMOE_OK, GGUF_BF16, GGUF_F16, GGUF_F32, KV_BAD_LENGTHS, KV_BAD_PAGE, KV_E4M3,
                  KV_PAST_TABLE, AmoeError, AmoeKvCache, AmoeRope, load_library)

_TYPES = {torch.float32: GGUF_F32, torch.float16: GGUF_F16, torch.bfloat16: GGUF_BF16}
_LEAST, _MOST = 2.0 ** -149, torch.finfo(torch.float32).max
_CACHE_TYPES = {torch.float16: GGUF_F16, torch.bfloat16: GGUF_BF16, torch.float8_e4m3fn: KV_E4M3}


def _invalid(message: str):
    raise AmoeError(AMOE_ERR_INVALID, message)


def _check(lib, rc: int):
    if rc != AMOE_OK:
        raise AmoeError(rc, lib.amoe_last_error(None).decode())


# The C structures of include/amoe.h, packed: a bytes object is a pointer to ctypes, and packing
# one costs a fraction of building a ctypes.Structure.
_pack_rows = struct.Struct("Pqqii").pack  # amoe_rows
_pack_seqs = struct.Struct("Pii").pack    # amoe_kv_seqs
_pack_attn = struct.Struct("fiP").pack    # amoe_attn


def _rows(t, name: str, tokens: int, head_dim: int, device: int) -> bytes:
    """A [tokens, heads, head_dim] tensor as the C ABI's rows."""
    shape = t.shape
    if len(shape) != 3 or shape[0] != tokens or shape[2] != head_dim:
        _invalid(f"{name} must be [{tokens}, heads, {head_dim}], got {list(shape)}")
    if t.get_device() != device:
        _invalid(f"{name} is on {t.device}, want cuda:{device}")
    kind = _TYPES.get(t.dtype)
    if kind is None:
        _invalid(f"{name} has type {t.dtype}")
    st, sh, sd = t.stride()
    if sd != 1:
        _invalid(f"{name}: the elements of a row must be adjacent")
    # a call without rows has no address to give
    return _pack_rows(t.data_ptr() or 16, st, sh, shape[1], kind)


def _written(t, name: str):
    """Rows that a call writes must not share memory with one another."""
    if t.dim() != 3:
        _invalid(f"{name} must be [tokens, heads, head_dim], got {list(t.shape)}")
    n, h, d = t.shape
    st, sh, _ = t.stride()
    if (n > 1 and st < d) or (h > 1 and sh < d) or (n > 1 and h > 1 and min(st, sh) * ((h if sh <= st else n) - 1) + d
                                                   > max(st, sh)):
        _invalid(f"{name}: its rows overlap")


def _ints(t, name: str, n: int, device: int) -> int:
    if t.dtype != torch.int32 or t.dim() != 1 or t.shape[0] != n or not t.is_contiguous():
        _invalid(f"{name} must be {n} adjacent int32 values")
    if t.get_device() != device:
        _invalid(f"{name} is on {t.device}, want cuda:{device}")
    return t.data_ptr()


def _stream(stream, device: int):
    """(the raw stream, a torch stream to allocate under or None for the current one)."""
    if stream is None:
        return torch._C._cuda_getCurrentRawStream(device), None
    if not hasattr(stream, "cuda_stream"):
        stream = torch.cuda.ExternalStream(int(stream), device=device)
    if stream.device.index != device:
        _invalid(f"stream is on {stream.device}, want cuda:{device}")
    return stream.cuda_stream, stream


def _like(t, dtype, stream):
    """A new contiguous tensor of t's shape (empty_like: half the host time of empty)."""
    if stream is None:
        return torch.empty_like(t, dtype=dtype, memory_format=torch.contiguous_format)
    with torch.cuda.stream(stream):
        return torch.empty_like(t, dtype=dtype, memory_format=torch.contiguous_format)


def _empty(like, shape, dtype, stream):
    """A new tensor on like's device."""
    if stream is None:
        return like.new_empty(shape, dtype=dtype)
    with torch.cuda.stream(stream):
        return like.new_empty(shape, dtype=dtype)


def _attn(scale, window: int, sinks, heads: int, device: int) -> bytes:
    if scale is None:
        scale = 0.0
    elif not _LEAST <= scale <= _MOST:  # float32 would make it 0, the default, or an infinity
        _invalid("scale must be positive, finite and a float32")
    at = 0
    if sinks is not None:
        if sinks.dtype != torch.float32 or sinks.dim() != 1 or sinks.shape[0] != heads or not sinks.is_contiguous():
            _invalid(f"sinks must be {heads} adjacent float32 values")
        if sinks.get_device() != device:
            _invalid(f"sinks is on {sinks.device}, want cuda:{device}")
        at = sinks.data_ptr()
    if not -(1 << 31) <= window < 1 << 31:
        _invalid("window must fit 32 bits")
    return _pack_attn(scale, window, at)


class Rope:
    """Rotary frequencies, equal to the reference's: RoPE (yarn=False) or its YaRN table (rope.go:10-44).

    The reference's YaRN table is not the published one: it divides the fast pairs by the factor instead of
    the slow ones.  It is for results that have to equal the reference's; ``Rope.yarn`` makes the
    frequencies that GPT-OSS and other models were trained with."""

    def __init__(self, head_dim: int, theta: float = 150000.0, yarn: bool = True):
        lib = self._new()
        _check(lib, lib.amoe_rope_init(head_dim, theta, 1 if yarn else 0, self._at))

    @classmethod
    def yarn(cls, head_dim: int, theta: float = 150000.0, factor: float = 32.0, original_context: float = 4096.0,
             beta_fast: float = 32.0, beta_slow: float = 1.0, truncate: bool = False,
             concentration: float | None = None) -> "Rope":
        """YaRN as published (amoe_rope_init_yarn); the defaults are GPT-OSS's.  ``truncate`` rounds the
        ramp's corners, as some models' configurations ask; concentration None: 1 + 0.1 ln(factor)."""
        self = cls.__new__(cls)
        lib = self._new()
        _check(lib, lib.amoe_rope_init_yarn(head_dim, theta, factor, original_context, beta_fast, beta_slow,
                                            1 if truncate else 0, self._at))
        if concentration is not None:
            self._c.concentration = concentration
        return self

    def _new(self):
        self._c = AmoeRope()
        return load_library()

    @property
    def _at(self) -> int:  # not kept: a copied Rope has a table of its own
        return ctypes.addressof(self._c)

    @property
    def frequencies(self) -> list:
        return list(self._c.freq)[:self._c.head_dim // 2]

    @property
    def concentration(self) -> float:
        return self._c.concentration


class KVCache:
    """One layer's paged cache: ``k`` and ``v`` [pages, kv_heads, page_size, head_dim] in float16,
    bfloat16 or float8_e4m3fn, the last with one E8M0 byte for each token and head in
    ``k_scale`` and ``v_scale`` [pages, kv_heads, page_size].  Calls take the page table
    [seqs, n] (int32; row s lists sequence s's pages in order)."""

    def __init__(self, pages: int, page_size: int, kv_heads: int, head_dim: int, dtype=torch.bfloat16,
                 device="cuda"):
        shape = (pages, kv_heads, page_size, head_dim)
        if min(shape) < 1:
            _invalid(f"a cache of shape {shape}")
        k, v = (torch.zeros(shape, dtype=dtype, device=device) for _ in range(2))
        ks = vs = None
        if dtype == torch.float8_e4m3fn:
            ks, vs = (torch.full(shape[:3], 127, dtype=torch.uint8, device=device) for _ in range(2))
        self._set(k, v, ks, vs)

    @classmethod
    def from_tensors(cls, k, v, k_scale=None, v_scale=None) -> "KVCache":
        """A cache over pages that the caller holds."""
        self = cls.__new__(cls)
        self._set(k, v, k_scale, v_scale)
        return self

    def _set(self, k, v, k_scale, v_scale):
        kind = _CACHE_TYPES.get(k.dtype)
        if kind is None or v.dtype != k.dtype:
            _invalid(f"a cache of {k.dtype} and {v.dtype}: float16, bfloat16 or float8_e4m3fn")
        if k.dim() != 4 or v.shape != k.shape or not k.is_contiguous() or not v.is_contiguous():
            _invalid("cache pages must be [pages, kv_heads, page_size, head_dim], contiguous, alike for k and v")
        if not k.is_cuda or v.device != k.device:
            _invalid("cache pages must be on one CUDA device")
        if any((s is not None) != (kind == KV_E4M3) for s in (k_scale, v_scale)):
            _invalid("k_scale and v_scale go with an E4M3 cache, and with no other")
        for s in (k_scale, v_scale):
            if s is not None and (s.dtype != torch.uint8 or s.shape != k.shape[:3] or not s.is_contiguous()
                                  or s.device != k.device):
                _invalid("scales must be uint8 [pages, kv_heads, page_size] beside the pages")
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self.device = k.device
        self.pages, self.kv_heads, self.page_size, self.head_dim = k.shape
        self.status = torch.zeros(1, dtype=torch.int32, device=k.device)
        self._lib = load_library()
        self._workspace = {}
        self._c = AmoeKvCache(k.data_ptr(), v.data_ptr(), None if k_scale is None else k_scale.data_ptr(),
                              None if v_scale is None else v_scale.data_ptr(), self.status.data_ptr(), self.pages,
                              self.page_size, self.kv_heads, self.head_dim, kind, k.device.index)
        self._at, self._index = ctypes.addressof(self._c), k.device.index

    def _seqs(self, page_table):
        """(the C ABI's sequences, how many)."""
        t = page_table
        shape = t.shape
        if t.dtype != torch.int32 or len(shape) != 2 or not t.is_contiguous() or min(shape) < 1:
            _invalid("page_table must be int32 [seqs, pages], contiguous and not empty")
        if t.get_device() != self._index:
            _invalid(f"page_table is on {t.device}, want {self.device}")
        return _pack_seqs(t.data_ptr(), shape[1], shape[0]), shape[0]

    def append(self, k, v, page_table, past, cu, q=None, rope: Rope | None = None, q_type=None, q_out=None,
               k_out=None, v_out=None, stream=None):
        """Rotates and writes packed new rows (amoe_kv_append): rows cu[s]..cu[s+1] of k and v
        [tokens, kv_heads, head_dim] become sequence s's tokens past[s], past[s] + 1, ...
        Returns the rotated q [tokens, q_heads, head_dim] (``q_out``, or a new tensor of
        ``q_type``, by default q's own), None without q."""
        n, d, dev = k.shape[0], self.head_dim, self._index
        seqs, count = self._seqs(page_table)
        raw, st = _stream(stream, dev)
        cq = cqo = cko = cvo = None
        if q is not None:
            cq = _rows(q, "q", n, d, dev)
            if q_out is None:
                q_out = _like(q, q_type, st)
            else:
                if q_type is not None and q_out.dtype != q_type:
                    _invalid(f"q_out is {q_out.dtype}, q_type {q_type}")
                _written(q_out, "q_out")
            cqo = _rows(q_out, "q_out", n, d, dev)
        elif q_out is not None:
            _invalid("q_out without q")
        if k_out is not None:
            _written(k_out, "k_out")
            cko = _rows(k_out, "k_out", n, d, dev)
        if v_out is not None:
            _written(v_out, "v_out")
            cvo = _rows(v_out, "v_out", n, d, dev)
        rc = self._lib.amoe_kv_append(
            self._at, seqs, _ints(cu, "cu", count + 1, dev), _ints(past, "past", count, dev), n,
            None if rope is None else rope._at, cq, _rows(k, "k", n, d, dev), _rows(v, "v", n, d, dev), cqo, cko, cvo,
            raw)
        if rc:
            _check(self._lib, rc)
        return q_out

    def read(self, page_table, cu, total: int, dtype=None, first=None, k_out=None, v_out=None, stream=None):
        """Sequence s's keys and values from position first[s] (default 0) on as packed rows
        cu[s]..cu[s+1] (amoe_kv_read).  Returns (k, v) [total, kv_heads, head_dim]: k_out and v_out,
        or new tensors of ``dtype`` (default: the cache's own type, bfloat16 for E4M3)."""
        if total < 0:
            _invalid("total must not be negative")
        d, dev = self.head_dim, self._index
        seqs, count = self._seqs(page_table)
        raw, st = _stream(stream, dev)
        if dtype is None:
            dtype = torch.bfloat16 if self.k_scale is not None else self.k.dtype
        shape = (total, self.kv_heads, d)
        if k_out is None:
            k_out = _empty(self.k, shape, dtype, st)
        else:
            _written(k_out, "k_out")
        if v_out is None:
            v_out = _empty(self.k, shape, dtype, st)
        else:
            _written(v_out, "v_out")
        rc = self._lib.amoe_kv_read(
            self._at, seqs, _ints(cu, "cu", count + 1, dev),
            None if first is None else _ints(first, "first", count, dev), total, _rows(k_out, "k_out", total, d, dev),
            _rows(v_out, "v_out", total, d, dev), raw)
        if rc:
            _check(self._lib, rc)
        return k_out, v_out

    def decode(self, q, page_table, kv_len, scale: float | None = None, window: int = 0, sinks=None,
               max_len: int = 0, out=None, stream=None):
        """Attention of one new token a sequence (amoe_attn_decode): q [seqs, q_heads, head_dim] at
        position kv_len[s] - 1.  Returns out, like q."""
        d, dev = self.head_dim, self._index
        seqs, count = self._seqs(page_table)
        raw, st = _stream(stream, dev)
        cq = _rows(q, "q", count, d, dev)
        heads = q.shape[1]
        if out is None:
            out = _like(q, None, st)
        else:
            _written(out, "out")
        shape = (count, page_table.shape[1], heads, window, max_len)
        size = self._workspace.get(shape)
        if size is None:  # the library's answer for these shapes
            size = self._lib.amoe_attn_decode_workspace(self._at, seqs, heads, window, max_len)
            _check(self._lib, min(size, AMOE_OK))
            if len(self._workspace) > 1000:
                self._workspace.clear()
            self._workspace[shape] = size
        work = _empty(self.k, size, torch.uint8, st) if size else None
        rc = self._lib.amoe_attn_decode(
            self._at, seqs, _attn(scale, window, sinks, heads, dev), cq, _rows(out, "out", count, d, dev),
            _ints(kv_len, "kv_len", count, dev), max_len, None if work is None else work.data_ptr(), size, raw)
        if rc:
            _check(self._lib, rc)
        return out

    def check(self):
        """Waits for the device and raises if a call met a wrong page id or length since the last check."""
        torch.cuda.synchronize(self.device)  # calls on every stream
        bits = int(self.status.item())
        if not bits:
            return
        self.status.zero_()
        torch.cuda.synchronize(self.device)  # before a call on another stream reports anew
        said = [m for b, m in ((KV_BAD_PAGE, "a page id outside the cache"),
                               (KV_PAST_TABLE, "a position beyond the page table"),
                               (KV_BAD_LENGTHS, "negative or decreasing lengths")) if bits & b]
        _invalid("kv cache: " + ", ".join(said))


_prefill_workspace: dict = {}


def prefill(q, k, v, cu_q, cu_k=None, scale: float | None = None, window: int = 0, sinks=None, out=None,
            stream=None):
    """Causal attention of packed prompts (amoe_attn_prefill): rows cu_q[s]..cu_q[s+1] of q
    [tokens, q_heads, head_dim] are the last of the positions that rows cu_k[s]..cu_k[s+1] of
    k and v [keys, kv_heads, head_dim] hold (cu_k None: cu_q).  Returns out, like q."""
    lib = load_library()
    dev = q.get_device()
    if dev < 0 or q.dim() != 3:
        _invalid("q must be a CUDA tensor [tokens, q_heads, head_dim]")
    if cu_k is None:
        cu_k = cu_q
    seqs = cu_q.shape[0] - 1
    raw, st = _stream(stream, dev)
    n, heads, d = q.shape
    m = k.shape[0]
    if out is None:
        out = _like(q, None, st)
    else:
        _written(out, "out")
    cq, ck = _rows(q, "q", n, d, dev), _rows(k, "k", m, d, dev)
    shape = (d, window, heads, k.shape[1], n, m, seqs)
    size = _prefill_workspace.get(shape)
    if size is None:  # the library's answer for these shapes; what it refuses, the call below refuses too
        size = max(lib.amoe_attn_prefill_workspace(*shape), 0)
        if len(_prefill_workspace) > 1000:
            _prefill_workspace.clear()
        _prefill_workspace[shape] = size
    work = _empty(q, size, torch.uint8, st) if size else None
    rc = lib.amoe_attn_prefill(
        dev, d, _attn(scale, window, sinks, heads, dev), cq, ck, _rows(v, "v", m, d, dev),
        _rows(out, "out", n, d, dev), n, m, _ints(cu_q, "cu_q", seqs + 1, dev), _ints(cu_k, "cu_k", seqs + 1, dev),
        seqs, None if work is None else work.data_ptr(), size, raw)
    if rc:
        _check(lib, rc)
    return out
