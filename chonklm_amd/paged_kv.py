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
import functools
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


# torch's current stream of a device, as a hipStream_t (what torch.cuda.current_stream().cuda_stream says)
_stream = torch._C._cuda_getCurrentRawStream if hasattr(torch._C, "_cuda_getCurrentRawStream") else \
    lambda at: torch.cuda.current_stream(at).cuda_stream


@functools.lru_cache(maxsize=None)
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
        shape, tshape = pages.shape, table.shape
        if pages.dtype != torch.uint8 or len(shape) != 2 or shape[1] != size or not pages.is_contiguous():
            _refuse(f"pages must be contiguous uint8 [n_pages, {size}]")
        if table.dtype != torch.int32 or len(tshape) != 2 or not table.is_contiguous():
            _refuse("table must be contiguous int32 [n_seqs, max_pages]")
        if not pages.is_cuda:
            _refuse("pages must be on a GPU")
        at = pages.get_device()
        if table.get_device() != at or (fault is not None and fault.get_device() != at):
            _refuse("table and fault must be on the pages' device")
        if fault is not None and (fault.dtype != torch.int32 or fault.numel() != 1):
            _refuse("fault must be int32 [1]")
        self.pages, self.table, self.fault = pages, table, fault
        self.kv_heads, self.head_dim, self._at = kv_heads, head_dim, at
        self._c = C.byref(_lib.KvCacheC(KV_TYPES[kv_dtype], kv_heads, head_dim, shape[0], pages.data_ptr(), tshape[0],
                                        tshape[1], table.data_ptr(), fault.data_ptr() if fault is not None else None, at))

    @property
    def device(self) -> torch.device:
        return self.pages.device

    # -- arguments ------------------------------------------------------------------
    def _index(self, x: torch.Tensor, n: int, name: str) -> int:
        if x.dtype != torch.int32 or x.shape != (n,) or x.get_device() != self._at or not x.is_contiguous():
            _refuse(f"{name} must be contiguous int32 [{n}] on {self.device}")
        return x.data_ptr()

    def _rows(self, x: torch.Tensor, n: int, heads: int, dtype: torch.dtype, name: str) -> int:
        """Checks rows [n, heads, head_dim] and returns the elements from row to row."""
        if x.shape != (n, heads, self.head_dim):
            _refuse(f"{name} must be [{n}, {heads}, {self.head_dim}]")
        if x.dtype != dtype:
            _refuse(f"{name} must be {dtype}")
        if x.get_device() != self._at:
            _refuse(f"{name} must be on {self.device}")
        row, head, one = x.stride()
        if n == 0:
            return heads * self.head_dim
        if one != 1 or (heads > 1 and head != self.head_dim):
            _refuse(f"a row of {name} must be contiguous")
        return row if n > 1 else heads * self.head_dim

    def _weights(self, x: Optional[torch.Tensor], name: str) -> Optional[int]:
        if x is None:
            return None
        if x.dtype != torch.float32 or x.shape != (self.head_dim,) or x.get_device() != self._at or not x.is_contiguous():
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
        dtype, n = k.dtype, len(k)
        if dtype not in _ACT:
            _refuse("k must be float32 or float16")
        k_ld = self._rows(k, n, self.kv_heads, dtype, "k")
        v_ld = self._rows(v, n, self.kv_heads, dtype, "v")
        q_at = out_at = rope_at = None
        q_ld = o_ld = heads = rope_dim = rope_n = 0
        if q is not None:
            if q.dim() != 3:
                _refuse("q must be [n, heads, head_dim]")
            heads = q.shape[1]
            q_ld = self._rows(q, n, heads, dtype, "q")
            if out is None:
                out, o_ld = torch.empty_like(q, memory_format=torch.contiguous_format), heads * self.head_dim
            else:
                o_ld = self._rows(out, n, heads, dtype, "out")
            q_at, out_at = q.data_ptr(), out.data_ptr()
        elif out is not None:
            _refuse("out without q")
        if rope is not None:
            if (rope.dtype != torch.float32 or rope.dim() != 3 or rope.shape[2] != 2 or not rope.is_contiguous() or
                    rope.get_device() != self._at):
                _refuse(f"rope must be contiguous float32 [positions, rope_dim / 2, 2] on {self.device}")
            rope_at, rope_n, rope_dim = rope.data_ptr(), rope.shape[0], 2 * rope.shape[1]
        rows = _lib.KvRowsC(n, self._index(seqs, n, "seqs"), self._index(positions, n, "positions"))
        a = _lib.KvAppendArgsC(_ACT[dtype], heads, q_at, k.data_ptr(), v.data_ptr(), out_at, q_ld, k_ld, v_ld, o_ld,
                               self._weights(q_norm, "q_norm"), self._weights(k_norm, "k_norm"), eps, rope_at, rope_dim,
                               rope_n, bool(interleaved))
        status = lib().chonk_kv_append(self._c, C.byref(rows), C.byref(a), _stream(self._at))
        if status:
            check(status)
        return out

    def read(self, seqs: torch.Tensor, positions: torch.Tensor, dtype: torch.dtype = torch.float16):
        """The values stored at (seqs[i], positions[i]): k, v [n, kv_heads, head_dim]."""
        if dtype not in _ACT:
            _refuse("dtype must be float32 or float16")
        n, heads, hd = len(seqs), self.kv_heads, self.head_dim
        rows = _lib.KvRowsC(n, self._index(seqs, n, "seqs"), self._index(positions, n, "positions"))
        k = torch.empty((n, heads, hd), dtype=dtype, device=self.pages.device)
        v = torch.empty_like(k)
        status = lib().chonk_kv_read(self._c, C.byref(rows), _ACT[dtype], k.data_ptr(), v.data_ptr(), heads * hd, hd,
                                     _stream(self._at))
        if status:
            check(status)
        return k, v

    def attend(self, q: torch.Tensor, seqs: torch.Tensor, lengths: torch.Tensor, *, scale: Optional[float] = None,
               window: int = 0, out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """Attention of rows q [n, heads, head_dim] over the first lengths[i] positions of
        sequence seqs[i] (the last `window` of them where given). Length 0 gives zeros; rows
        with a negative sequence are left out."""
        if q.dim() != 3 or q.dtype not in _ACT:
            _refuse("q must be float32 or float16 [n, heads, head_dim]")
        dtype, (n, heads, hd) = q.dtype, q.shape
        q_ld = self._rows(q, n, heads, dtype, "q")
        if out is None:
            out, o_ld = torch.empty_like(q, memory_format=torch.contiguous_format), heads * hd
        else:
            o_ld = self._rows(out, n, heads, dtype, "out")
        L = lib()
        need, work, work_at = L.chonk_kv_attend_workspace(self._c, n, heads), None, None
        if need > 0:
            work = torch.empty(need, dtype=torch.uint8, device=self.pages.device)
            work_at = work.data_ptr()
        elif need < 0:
            check(need)
        a = _lib.KvAttendArgsC(_ACT[dtype], heads, n, self._index(seqs, n, "seqs"), self._index(lengths, n, "lengths"),
                               q.data_ptr(), out.data_ptr(), q_ld, o_ld, hd ** -0.5 if scale is None else scale, window,
                               work_at, need)
        status = L.chonk_kv_attend(self._c, C.byref(a), _stream(self._at))
        if status:
            check(status)
        return out

    def check(self) -> None:
        """Waits for the stream and raises if a row since the last check named no place."""
        if self.fault is None:
            _refuse("check() needs a fault word")
        bits = int(self.fault.item())
        if bits:
            self.fault.zero_()
            _refuse("rows named " + ", ".join(text for bit, text in _FAULTS if bits & bit))
