"""Paged key/value cache in fp16 or 4 bits, and the attention over it.

The reference keeps one fp16 / fp32 array per sequence (attention.py:99-104).
:class:`PagedKVCache` keeps the keys and values of many sequences in a pool of
fixed-size pages, so that sequences of any length share the memory, stored as
fp16 or as 4-bit blocks with the values of GGUF ``Q4_0`` (gguf_dequant.py:25-46;
72 bytes instead of 256 per key or value of a 128-wide head).

All calls name the new tokens the same way.  ``cu_seqlens`` (int32 [B + 1]) gives
the rows of each sequence (None: one new token per sequence, row b is sequence
b), ``kv_lens`` (int32 [B]) the tokens of each sequence *with* its new ones, and
``block_table`` (int32 [B, W]) the pages of each sequence in order; everything
lives on the device, so that a step can be captured into a CUDA graph.  Rows
behind ``cu_seqlens[-1]`` are left alone; a row before position 0 is not stored
and yields zeros; a position without a page does too (as a key it is left out of
the attention) and shows up in ``_lib.check_device``.  Entries of pages that no
row sees, behind a window, may be anything: those pages can go back to the pool.

There is no CPU fallback; calls run on the current stream of the pool's device.
"""

from __future__ import annotations

import functools

import torch

from ._lib import DT_BF16, DT_F16, DT_F32, KV, call_on, check, lib

__all__ = ["PagedKVCache", "rope_table"]

_DT = {torch.float32: DT_F32, torch.bfloat16: DT_BF16, torch.float16: DT_F16}


def rope_table(positions: int, head_dim: int, theta: float = 1e4, device=None) -> torch.Tensor:
    """(cos, sin) of pos / theta^(2i / head_dim), fp32 [positions, head_dim / 2, 2], from angles in 64 bits."""
    if positions < 1 or head_dim < 2 or head_dim % 2:
        raise ValueError(f"rope_table: {positions} positions, head_dim {head_dim}")
    dev = torch.device(device) if device is not None else torch.device("cuda", torch.cuda.current_device())
    i = torch.arange(0, head_dim, 2, dtype=torch.float64, device=dev)
    ang = torch.arange(positions, dtype=torch.float64, device=dev)[:, None] / float(theta) ** (i / head_dim)
    return torch.stack((ang.cos(), ang.sin()), -1).float()


def _ints(t, what, dim, dev):
    if not isinstance(t, torch.Tensor) or t.dtype != torch.int32 or t.dim() != dim:
        raise ValueError(f"{what} must be a {dim}-D int32 tensor")
    if t.device != dev:
        raise ValueError(f"{what} is on {t.device}, the cache on {dev}")
    if t.stride(-1) != 1 and t.shape[-1] > 1:
        raise ValueError(f"{what} must have unit stride in its last dimension")


@functools.lru_cache(maxsize=1024)
def _workspace_size(*sizes) -> int:
    return lib.xm_kv_attention_workspace_size(*sizes)


class PagedKVCache:
    """A pool of ``num_pages`` pages of ``page_size`` tokens for ``num_kv_heads`` heads.

    ``kv_type``: ``"F16"`` or ``"Q4_0"``; ``head_dim``: 64 or 128; ``page_size``: a power of two, 16 to 1024.
    ``pool``: an existing uint8 tensor [num_pages, num_kv_heads, bytes of a head of a page] to use.
    """

    def __init__(self, num_pages: int, num_kv_heads: int, head_dim: int = 128, page_size: int = 64,
                 kv_type: str = "F16", device=None, pool: torch.Tensor | None = None):
        if kv_type not in KV:
            raise NotImplementedError(f"PagedKVCache: unknown cache type {kv_type!r} (one of {sorted(KV)})")
        if head_dim not in (64, 128):
            raise NotImplementedError(f"PagedKVCache: head_dim {head_dim} (64 or 128)")
        if page_size < 16 or page_size > 1024 or page_size & (page_size - 1):
            raise ValueError(f"PagedKVCache: page size {page_size} (a power of two from 16 to 1024)")
        if num_pages < 1 or num_kv_heads < 1:
            raise ValueError(f"PagedKVCache: {num_pages} pages, {num_kv_heads} heads")
        self.num_pages, self.num_kv_heads, self.head_dim = int(num_pages), int(num_kv_heads), int(head_dim)
        self.page_size, self.kv_type, self._kv = int(page_size), kv_type, KV[kv_type]
        head_bytes = lib.xm_kv_page_bytes(self._kv, self.num_kv_heads, self.head_dim, self.page_size) // self.num_kv_heads
        shape = (self.num_pages, self.num_kv_heads, head_bytes)
        if pool is None:
            dev = torch.device(device) if device is not None else torch.device("cuda", torch.cuda.current_device())
            pool = torch.zeros(shape, dtype=torch.uint8, device=dev)
        elif pool.dtype != torch.uint8 or tuple(pool.shape) != shape or not pool.is_contiguous():
            raise ValueError(f"PagedKVCache: the pool must be a contiguous uint8 tensor of shape {shape}, got "
                             f"{pool.dtype} {tuple(pool.shape)}")
        if not pool.is_cuda:
            raise ValueError("PagedKVCache: the pool must live on a CUDA device")
        self.pool = pool
        self.device = pool.device

    # -- helpers ------------------------------------------------------------
    def _rows(self, block_table, kv_lens, cu_seqlens, rows):
        """Checks the arguments that name the tokens; the C ABI's (table, stride, width, cu, lens, B)."""
        dev = self.device
        _ints(block_table, "block_table", 2, dev)
        _ints(kv_lens, "kv_lens", 1, dev)
        b = kv_lens.shape[0]
        n, width = block_table.shape
        if n != b or b < 1 or width < 1:
            raise ValueError(f"block_table {tuple(block_table.shape)} does not fit {b} sequences")
        cu = None
        if cu_seqlens is not None:
            _ints(cu_seqlens, "cu_seqlens", 1, dev)
            if cu_seqlens.shape[0] != b + 1:
                raise ValueError(f"cu_seqlens has {cu_seqlens.shape[0]} entries, {b} sequences need {b + 1}")
            cu = cu_seqlens.data_ptr()
        elif rows != b:
            raise ValueError(f"{rows} rows for {b} sequences: give cu_seqlens")
        return block_table.data_ptr(), block_table.stride(0), width, cu, kv_lens.data_ptr(), b

    def _out(self, out, rows, heads, dtype):
        """(out, its row pitch): a new tensor [rows, heads, head_dim], or the caller's, checked."""
        if out is None:
            return self.pool.new_empty((rows, heads, self.head_dim), dtype=dtype), heads * self.head_dim
        if tuple(out.shape) != (rows, heads, self.head_dim) or out.dtype != dtype or out.device != self.device:
            raise ValueError(f"out must be {dtype} {(rows, heads, self.head_dim)} on {self.device}, got {out.dtype} "
                             f"{tuple(out.shape)} on {out.device}")
        return out, self._pitch(out, "out")

    def _pitch(self, t, what):
        """The row pitch of t [T, heads, head_dim], whose heads must lie one after another."""
        rows, heads, d = t.shape
        pitch, head, one = t.stride()
        if one != 1 or (heads > 1 and head != d):
            raise ValueError(f"{what}: the heads of a row must be contiguous")
        return pitch if rows > 1 else max(pitch, heads * d)

    # -- operators ------------------------------------------------------------
    def append(self, qkv: torch.Tensor, num_heads: int, block_table: torch.Tensor, kv_lens: torch.Tensor,
               cu_seqlens: torch.Tensor | None = None, rope: torch.Tensor | None = None,
               q_norm: torch.Tensor | None = None, k_norm: torch.Tensor | None = None, eps: float = 1e-5,
               out: torch.Tensor | None = None, out_dtype: torch.dtype | None = None) -> torch.Tensor:
        """Normalise (``q_norm`` / ``k_norm``: fp32 [head_dim], per head), rotate (``rope``: see
        :func:`rope_table`) and store the rows of a QKV projection.

        ``qkv`` [T, (num_heads + 2 kv heads) * head_dim], fp32, fp16 or bf16.  Returns the queries
        [T, num_heads, head_dim] in ``out_dtype`` (fp16 or bf16; default: qkv's type, fp16 for fp32)."""
        d, dev, hk = self.head_dim, self.device, self.num_kv_heads
        dt = _DT.get(qkv.dtype) if isinstance(qkv, torch.Tensor) else None
        if dt is None or qkv.dim() != 2 or qkv.device != dev:
            raise ValueError(f"append: qkv must be a 2-D fp32, fp16 or bf16 tensor on {dev}")
        rows, width = qkv.shape
        if num_heads < 1 or num_heads % hk or width != (num_heads + 2 * hk) * d:
            raise ValueError(f"append: qkv rows of {width} values for {num_heads} query and {hk} KV heads of {d}")
        pitch, one = qkv.stride()
        if one != 1:
            raise ValueError("append: qkv must have unit stride in its last dimension")
        where = self._rows(block_table, kv_lens, cu_seqlens, rows)
        angles, positions = None, 0
        if rope is not None:
            if (rope.dtype != torch.float32 or rope.dim() != 3 or rope.shape[0] < 1 or rope.shape[1] != d // 2
                    or rope.shape[2] != 2 or not rope.is_contiguous() or rope.device != dev):
                raise ValueError(f"append: rope must be a contiguous fp32 tensor [positions, {d // 2}, 2] on {dev}")
            angles, positions = rope.data_ptr(), rope.shape[0]
        norms = [None, None]
        for i, w in enumerate((q_norm, k_norm)):
            if w is not None:
                if (w.dtype != torch.float32 or w.dim() != 1 or w.shape[0] != d or not w.is_contiguous()
                        or w.device != dev):
                    raise ValueError(f"append: {'qk'[i]}_norm must be a contiguous fp32 tensor [{d}] on {dev}")
                norms[i] = w.data_ptr()
        if out_dtype is None:
            out_dtype = out.dtype if out is not None else torch.float16 if dt == DT_F32 else qkv.dtype
        if out_dtype is not torch.float16 and out_dtype is not torch.bfloat16:
            raise ValueError(f"append: queries are fp16 or bf16, not {out_dtype}")
        q, q_pitch = self._out(out, rows, num_heads, out_dtype)
        check(call_on(dev, lib.xm_kv_append, qkv.data_ptr(), dt, rows, pitch if rows > 1 else max(pitch, width),
                      num_heads, hk, d, angles, positions, *norms, eps, self.pool.data_ptr(), self.num_pages, self._kv,
                      self.page_size, *where, q.data_ptr(), _DT[out_dtype], q_pitch), "kv append")
        return q

    def read(self, block_table: torch.Tensor, kv_lens: torch.Tensor, cu_seqlens: torch.Tensor | None = None,
             num_tokens: int | None = None):
        """The cached keys and values of the rows (the last tokens of each sequence) as fp16
        [num_tokens, num_kv_heads, head_dim] each."""
        rows = kv_lens.shape[0] if num_tokens is None and cu_seqlens is None else num_tokens
        if rows is None or rows < 0:
            raise ValueError("read: num_tokens (the number of rows) is needed with cu_seqlens")
        where = self._rows(block_table, kv_lens, cu_seqlens, rows)
        # rows behind the last sequence stay zeros
        make = self.pool.new_empty if cu_seqlens is None else self.pool.new_zeros
        k, v = make((2, rows, self.num_kv_heads, self.head_dim), dtype=torch.float16).unbind(0)
        check(call_on(self.device, lib.xm_kv_read, self.pool.data_ptr(), self.num_pages, self._kv, self.num_kv_heads,
                      self.head_dim, self.page_size, *where, rows, k.data_ptr(), v.data_ptr()), "kv read")
        return k, v

    def attend(self, q: torch.Tensor, block_table: torch.Tensor, kv_lens: torch.Tensor,
               cu_seqlens: torch.Tensor | None = None, scale: float | None = None, window: int = 0, sinks: int = 0,
               out: torch.Tensor | None = None) -> torch.Tensor:
        """Causal attention of the rows ``q`` [T, heads, head_dim] (fp16 or bf16, as :meth:`append` returns
        them) over their sequences' cached positions up to their own; ``window`` > 0 restricts a row at
        position p to positions above p - window and the first ``sinks`` ones.  Query head h reads KV head
        h // (heads / kv heads).  ``scale`` defaults to 1 / sqrt(head_dim).  A row that sees no key is zeros.
        Without ``out``, rows behind the last sequence are not initialised."""
        d, dev, hk = self.head_dim, self.device, self.num_kv_heads
        if (not isinstance(q, torch.Tensor) or q.dim() != 3 or q.dtype not in (torch.float16, torch.bfloat16)
                or q.device != dev):
            raise ValueError(f"attend: q must be a 3-D fp16 or bf16 tensor on {dev}")
        rows, heads, width = q.shape
        if width != d or heads < 1 or heads % hk:
            raise ValueError(f"attend: q {tuple(q.shape)} for {hk} KV heads of {d}")
        if window < 0 or sinks < 0:
            raise ValueError("attend: window and sinks must not be negative")
        window, sinks = min(window, 1 << 31), min(sinks, 1 << 31)      # (longer than any context; numbers that C can hold)
        pitch = self._pitch(q, "attend: q")
        where = self._rows(block_table, kv_lens, cu_seqlens, rows)
        if out is None and q.is_contiguous():
            o, o_pitch = torch.empty_like(q), heads * d
        else:
            o, o_pitch = self._out(out, rows, heads, q.dtype)
        need = _workspace_size(rows, where[5], heads, hk, d, where[2] * self.page_size)
        # a workspace for each call: two captured graphs, or two streams, never share one
        ws = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
        check(call_on(dev, lib.xm_kv_attention, q.data_ptr(), _DT[q.dtype], rows, pitch, heads, hk, d,
                      d ** -0.5 if scale is None else scale, window, sinks, self.pool.data_ptr(), self.num_pages,
                      self._kv, self.page_size, *where, o.data_ptr(), o_pitch, None if ws is None else ws.data_ptr(),
                      need), "kv attention")
        return o

    def __repr__(self):
        return (f"<PagedKVCache {self.kv_type} {self.num_pages} pages of {self.page_size}, {self.num_kv_heads} heads "
                f"of {self.head_dim} on {self.device}>")
