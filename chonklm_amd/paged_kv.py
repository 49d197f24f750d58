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

import functools
import importlib.util
import sys
from typing import Optional

_OWN_RUNTIME = "torch" not in sys.modules and "chonklm_amd._lib" in sys.modules and \
    sys.modules["chonklm_amd._lib"]._LIB is not None

import torch  # noqa: E402

from . import _lib  # noqa: E402
from ._lib import CHONK_EINVAL, ChonkError, check, lib  # noqa: E402

PAGE = 64
KV_TYPES = {"f16": _lib.KV_F16, "q8": _lib.KV_Q8, "q4": _lib.KV_Q4}
_FAULTS = ((1, "a sequence outside the table"), (2, "a position outside its tables"), (4, "a page outside the pool"))


def _refuse(message: str):
    raise ChonkError(CHONK_EINVAL, "paged K/V cache: " + message)


def _load():
    """The native calls (csrc/torch_kv/paged_kv_ext.cpp); fails loudly where they are not built."""
    lib()
    path = _lib.LIB_PATH.with_name("_paged_kv.so")
    if not path.exists():
        raise RuntimeError(f"{path} is missing: build it with `python -m chonklm_amd.build` (torch's headers are needed)")
    spec = importlib.util.spec_from_file_location("chonklm_amd._paged_kv", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    module.bind(ChonkError, torch._C._cuda_getCurrentRawStream, torch.float32, torch.float16)
    return module


_native = _load()


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


class PagedKv(_native.Cache):
    """One layer's paged cache over memory that the caller holds.

    pages  uint8 [n_pages, page_bytes(...)], contiguous
    table  int32 [n_seqs, max_pages], contiguous: the page of each 64 positions
    fault  int32 [1] (optional): set by rows that name no place (see check())

    append(q, k, v, seqs, positions, *, q_norm=None, k_norm=None, eps=1e-6, rope=None,
           interleaved=False, out=None) -> q
        Writes rows k, v [n, kv_heads, head_dim] to (seqs[i], positions[i]) and returns q
        [n, heads, head_dim] (None without q), q and k normalised per head and rotated where the
        weights [head_dim] and the table [positions, rope_dim / 2, 2] are given. `out` may be q.
    read(seqs, positions, dtype=torch.float16) -> k, v
        The values stored at (seqs[i], positions[i]), [n, kv_heads, head_dim].
    attend(q, seqs, lengths, *, scale=head_dim ** -0.5, window=0, out=None) -> out
        Attention of rows q [n, heads, head_dim] over the first lengths[i] positions of
        sequence seqs[i] (the last `window` of them where given). Length 0 gives zeros.
        `out` may be q.

    Rows are float32 or float16 and may be strided (a row's heads and dims together);
    seqs, positions and lengths are contiguous int32 [n]. Rows with a negative sequence
    are left out: their results stay as they were (without `out`, as new memory is).
    The operators have no gradient.
    """

    def __init__(self, pages: torch.Tensor, table: torch.Tensor, kv_heads: int, head_dim: int, kv_dtype: str = "q8",
                 fault: Optional[torch.Tensor] = None):
        if _OWN_RUNTIME:
            _refuse("libchonk.so was loaded before torch and uses another HIP runtime: import torch first")
        if kv_dtype not in KV_TYPES:
            _refuse(f"unsupported kv type {kv_dtype!r}")
        super().__init__(pages, table, kv_heads, head_dim, KV_TYPES[kv_dtype], fault)

    @property
    def device(self) -> torch.device:
        return self.pages.device

    def check(self) -> None:
        """Waits for the stream and raises if a row since the last check named no place."""
        if self.fault is None:
            _refuse("check() needs a fault word")
        bits = int(self.fault.item())
        if bits:
            self.fault.zero_()
            _refuse("rows named " + ", ".join(text for bit, text in _FAULTS if bits & bit))
