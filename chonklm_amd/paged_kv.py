"""Paged K/V cache operators on torch tensors (chonk_kv_*, include/chonk.h).

For programs that drive a decoder's layers themselves: K and V of many
sequences live in pages of 64 positions, as fp16 or as 8- or 4-bit codes with an
fp16 scale per 32 dims (about a half and a quarter of fp16's bytes):

    pages = torch.empty(n_pages, page_bytes("q8", kv_heads, head_dim), dtype=torch.uint8, device="cuda")
    kv = PagedKv(pages, table, kv_heads, head_dim, "q8")        # table: int32 [n_seqs, max_pages]
    q = kv.append(q, k, v, seqs, positions, q_norm=wq, k_norm=wk, eps=1e-6, rope=rope_table(4096, 128, 1e6))
    o = kv.attend(q, seqs, positions + 1)

Calls enqueue on torch's current stream of the pages' device and do not wait;
they can be captured into a graph. Results and workspace come from torch's
allocator. Import this module (or torch) before the first engine is loaded:
libchonk.so then runs on torch's HIP runtime, whose pointers and streams it is given.
"""
from __future__ import annotations

import ctypes as C
import sys
from typing import Optional

_OWN_RUNTIME = "torch" not in sys.modules and "chonklm_amd._lib" in sys.modules and \
    sys.modules["chonklm_amd._lib"]._LIB is not None

import torch  # noqa: E402

from . import _lib  # noqa: E402
from ._lib import CHONK_EINVAL, ChonkError, check, lib  # noqa: E402

PAGE = 64
KV_TYPES = {"f16": _lib.KV_F16, "q8": _lib.KV_Q8, "q4": _lib.KV_Q4}
_ACT = {torch.float32: _lib.F32, torch.float16: _lib.F16}
_FAULTS = ((1, "a sequence outside the table"), (2, "a position outside its tables"), (4, "a page outside the pool"))


def _refuse(message: str):
    raise ChonkError(CHONK_EINVAL, "paged K/V cache: " + message)


def page_bytes(kv_dtype: str, kv_heads: int, head_dim: int) -> int:
    """Bytes of one page (64 positions of K and V of every kv head)."""
    if kv_dtype not in KV_TYPES:
        _refuse(f"unsupported kv type {kv_dtype!r}")
    n = lib().chonk_kv_page_bytes(KV_TYPES[kv_dtype], int(kv_heads), int(head_dim))
    if n < 0:
        check(n)
    return n


def rope_table(positions: int, rope_dim: int, theta: float, device="cuda") -> torch.Tensor:
    """(cos, sin) [positions, rope_dim / 2, 2] of the angles p * theta^(-2 i / rope_dim),
    taken in 64 bits: at far positions an fp32 angle has lost the turn's fraction."""
    i = torch.arange(0, rope_dim, 2, dtype=torch.float64, device=device)
    angle = torch.arange(positions, dtype=torch.float64, device=device)[:, None] * float(theta) ** (-i / rope_dim)
    return torch.stack([angle.cos(), angle.sin()], dim=-1).float()


class PagedKv:
    """One layer's paged cache over memory that the caller holds.

    pages  uint8 [n_pages, page_bytes(...)], contiguous
    table  int32 [n_seqs, max_pages], contiguous: the page of each 64 positions
    fault  int32 [1] (optional): set by rows that name no place (see check())
    """

    def __init__(self, pages: torch.Tensor, table: torch.Tensor, kv_heads: int, head_dim: int, kv_dtype: str = "q8",
                 fault: Optional[torch.Tensor] = None):
        if _OWN_RUNTIME:
            _refuse("libchonk.so was loaded before torch and uses another HIP runtime: import torch first")
        size = page_bytes(kv_dtype, kv_heads, head_dim)
        if pages.dtype != torch.uint8 or pages.dim() != 2 or pages.shape[1] != size or not pages.is_contiguous():
            _refuse(f"pages must be contiguous uint8 [n_pages, {size}]")
        if table.dtype != torch.int32 or table.dim() != 2 or not table.is_contiguous():
            _refuse("table must be contiguous int32 [n_seqs, max_pages]")
        if not pages.is_cuda:
            _refuse("pages must be on a GPU")
        if table.device != pages.device or (fault is not None and fault.device != pages.device):
            _refuse("table and fault must be on the pages' device")
        if fault is not None and (fault.dtype != torch.int32 or fault.numel() != 1):
            _refuse("fault must be int32 [1]")
        self.pages, self.table, self.fault = pages, table, fault
        self.kv_heads, self.head_dim, self.device = kv_heads, head_dim, pages.device
        self._c = _lib.KvCacheC(KV_TYPES[kv_dtype], kv_heads, head_dim, pages.shape[0], pages.data_ptr(),
                                table.shape[0], table.shape[1], table.data_ptr(),
                                fault.data_ptr() if fault is not None else None, pages.device.index)

    # -- arguments ------------------------------------------------------------------
    def _stream(self) -> int:
        return torch.cuda.current_stream(self.device).cuda_stream

    def _index(self, x: torch.Tensor, n: int, name: str) -> torch.Tensor:
        if x.dtype != torch.int32 or x.dim() != 1 or x.shape[0] != n or x.device != self.device:
            _refuse(f"{name} must be int32 [{n}] on {self.device}")
        return x if x.is_contiguous() else x.contiguous()

    def _rows(self, x: torch.Tensor, heads: Optional[int], dtype: Optional[torch.dtype], name: str) -> int:
        """Checks rows [n, heads, head_dim] and returns the elements from row to row."""
        if x.dim() != 3 or x.shape[2] != self.head_dim or (heads is not None and x.shape[1] != heads):
            _refuse(f"{name} must be [n, {heads if heads is not None else 'heads'}, {self.head_dim}]")
        if x.dtype not in _ACT or (dtype is not None and x.dtype != dtype):
            _refuse(f"{name} must be {dtype or 'float32 or float16'}")
        if x.device != self.device:
            _refuse(f"{name} must be on {self.device}")
        if (x.stride(2) != 1 or (x.shape[1] > 1 and x.stride(1) != self.head_dim)) and x.numel():
            _refuse(f"a row of {name} must be contiguous")
        return x.stride(0) if x.shape[0] > 1 else x.shape[1] * self.head_dim

    def _weights(self, x: Optional[torch.Tensor], name: str) -> Optional[int]:
        if x is None:
            return None
        if x.dtype != torch.float32 or x.shape != (self.head_dim,) or x.device != self.device or not x.is_contiguous():
            _refuse(f"{name} must be contiguous float32 [{self.head_dim}] on {self.device}")
        return x.data_ptr()

    # -- operators ------------------------------------------------------------------
    def append(self, q: Optional[torch.Tensor], k: torch.Tensor, v: torch.Tensor, seqs: torch.Tensor,
               positions: torch.Tensor, *, q_norm: Optional[torch.Tensor] = None,
               k_norm: Optional[torch.Tensor] = None, eps: float = 1e-6, rope: Optional[torch.Tensor] = None,
               interleaved: bool = False, out: Optional[torch.Tensor] = None) -> Optional[torch.Tensor]:
        """Writes rows k, v [n, kv_heads, head_dim] to (seqs[i], positions[i]) and returns q
        [n, heads, head_dim] (None without q), q and k normalised per head and rotated where the
        weights and the table [positions, rope_dim / 2, 2] are given. `out` may be q.
        Rows with a negative sequence are left out."""
        n = k.shape[0]
        k_ld = self._rows(k, self.kv_heads, None, "k")
        v_ld = self._rows(v, self.kv_heads, k.dtype, "v")
        if v.shape[0] != n:
            _refuse("k and v differ in rows")
        q_ld = o_ld = heads = 0
        if q is not None:
            q_ld, heads = self._rows(q, None, k.dtype, "q"), q.shape[1]
            if out is None:
                out = torch.empty(q.shape, dtype=q.dtype, device=self.device)
            o_ld = self._rows(out, heads, k.dtype, "out")
            if q.shape[0] != n or out.shape[0] != n:
                _refuse("q, k and out differ in rows")
        elif out is not None:
            _refuse("out without q")
        if rope is not None and (rope.dtype != torch.float32 or rope.dim() != 3 or rope.shape[2] != 2 or
                                 not rope.is_contiguous() or rope.device != self.device):
            _refuse(f"rope must be contiguous float32 [positions, rope_dim / 2, 2] on {self.device}")
        seqs, positions = self._index(seqs, n, "seqs"), self._index(positions, n, "positions")
        rows = _lib.KvRowsC(n, seqs.data_ptr(), positions.data_ptr())
        a = _lib.KvAppendArgsC(
            _ACT[k.dtype], heads, q.data_ptr() if q is not None else None, k.data_ptr(), v.data_ptr(),
            out.data_ptr() if out is not None else None, q_ld, k_ld, v_ld, o_ld, self._weights(q_norm, "q_norm"),
            self._weights(k_norm, "k_norm"), eps, rope.data_ptr() if rope is not None else None,
            2 * rope.shape[1] if rope is not None else 0, rope.shape[0] if rope is not None else 0, bool(interleaved))
        check(lib().chonk_kv_append(C.byref(self._c), C.byref(rows), C.byref(a), self._stream()))
        return out

    def read(self, seqs: torch.Tensor, positions: torch.Tensor, dtype: torch.dtype = torch.float16):
        """The values stored at (seqs[i], positions[i]): k, v [n, kv_heads, head_dim]."""
        if dtype not in _ACT:
            _refuse("dtype must be float32 or float16")
        n = seqs.shape[0]
        seqs, positions = self._index(seqs, n, "seqs"), self._index(positions, n, "positions")
        k, v = (torch.empty((n, self.kv_heads, self.head_dim), dtype=dtype, device=self.device) for _ in range(2))
        rows = _lib.KvRowsC(n, seqs.data_ptr(), positions.data_ptr())
        check(lib().chonk_kv_read(C.byref(self._c), C.byref(rows), _ACT[dtype], k.data_ptr(), v.data_ptr(),
                                  self.kv_heads * self.head_dim, self.head_dim, self._stream()))
        return k, v

    def attend(self, q: torch.Tensor, seqs: torch.Tensor, lengths: torch.Tensor, *, scale: Optional[float] = None,
               window: int = 0, out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """Attention of rows q [n, heads, head_dim] over the first lengths[i] positions of
        sequence seqs[i] (the last `window` of them where given). Length 0 gives zeros; rows
        with a negative sequence are left out."""
        n, heads = q.shape[0], q.shape[1] if q.dim() == 3 else 0
        q_ld = self._rows(q, None, None, "q")
        if out is None:
            out = torch.empty(q.shape, dtype=q.dtype, device=self.device)
        o_ld = self._rows(out, heads, q.dtype, "out")
        if out.shape[0] != n:
            _refuse("q and out differ in rows")
        seqs, lengths = self._index(seqs, n, "seqs"), self._index(lengths, n, "lengths")
        L = lib()
        need = L.chonk_kv_attend_workspace(C.byref(self._c), n, heads)
        if need < 0:
            check(need)
        work = torch.empty(need, dtype=torch.uint8, device=self.device) if need else None
        a = _lib.KvAttendArgsC(_ACT[q.dtype], heads, n, seqs.data_ptr(), lengths.data_ptr(), q.data_ptr(),
                               out.data_ptr(), q_ld, o_ld, self.head_dim ** -0.5 if scale is None else scale, window,
                               work.data_ptr() if work is not None else None, need)
        check(L.chonk_kv_attend(C.byref(self._c), C.byref(a), self._stream()))
        return out

    def check(self) -> None:
        """Waits for the stream and raises if a row since the last check named no place."""
        if self.fault is None:
            _refuse("check() needs a fault word")
        bits = int(self.fault.item())
        if bits:
            self.fault.zero_()
            _refuse("rows named " + ", ".join(text for bit, text in _FAULTS if bits & bit))
