"""The paged K/V cache's entry points without a GPU: sizes, refusals of bad arguments
(all of them made before any device call), and the reference's page format."""
from __future__ import annotations

import ctypes as C
import subprocess
import sys
from pathlib import Path

import numpy as np
import pytest

from chonklm_amd import _lib
from chonklm_amd._lib import lib
from tests import paged_ref as ref

KINDS = {"f16": _lib.KV_F16, "q8": _lib.KV_Q8, "q4": _lib.KV_Q4}


@pytest.mark.parametrize("kv", ref.TYPES)
@pytest.mark.parametrize("hd", [32, 64, 128, 256])
def test_every_byte_of_a_page_has_one_owner(kv, hd):
    assert lib().chonk_kv_page_bytes(KINDS[kv], 3, hd) == 3 * 2 * ref.part_bytes(kv, hd)
    owned = sum(ref.owned_bytes(kv, hd, j).astype(int) for j in range(64))
    assert (owned == 1).all()


@pytest.mark.parametrize("args", [(1, 2, 64), (7, 2, 64), (2, 0, 64), (2, 2, 96), (2, 2, 0), (3, -1, 128)])
def test_page_bytes_refuses(args):
    assert lib().chonk_kv_page_bytes(*args) == _lib.CHONK_EINVAL
    assert b"paged K/V cache" in lib().chonk_last_error()


def cache(**kw):
    # (addresses that are never followed: every call below is refused before it)
    d = dict(kv_type=_lib.KV_Q8, kv_heads=2, head_dim=64, n_pages=4, pages=0x1000, n_seqs=2, max_pages=2, table=0x2000,
             fault=None, device=0)
    d.update(kw)
    return _lib.KvCacheC(**d)


def append(**kw):
    d = dict(type=0, heads=4, q=0x10, k=0x10, v=0x10, q_out=0x10, q_stride=256, k_stride=128, v_stride=128,
             q_out_stride=256, eps=1e-6)
    d.update(kw)
    return _lib.KvAppendArgsC(**d)


def attend(**kw):
    d = dict(type=0, heads=4, n=1, seq=0x10, lengths=0x10, q=0x10, out=0x10, q_stride=256, out_stride=256, scale=1.0,
             window=0, workspace=0x1000, workspace_bytes=1 << 30)
    d.update(kw)
    return _lib.KvAttendArgsC(**d)


BAD_CACHE = [dict(kv_type=_lib.KV_F32), dict(kv_heads=0), dict(head_dim=48), dict(n_pages=0), dict(pages=None),
             dict(pages=0x1008), dict(table=None), dict(n_seqs=0), dict(max_pages=0)]


@pytest.mark.parametrize("kw", BAD_CACHE)
def test_bad_caches_are_refused_everywhere(kw):
    c, rows = cache(**kw), _lib.KvRowsC(1, 0x10, 0x10)
    L = lib()
    assert L.chonk_kv_append(C.byref(c), C.byref(rows), C.byref(append()), None) == _lib.CHONK_EINVAL
    assert L.chonk_kv_read(C.byref(c), C.byref(rows), 0, 0x10, 0x10, 128, 64, None) == _lib.CHONK_EINVAL
    assert L.chonk_kv_attend(C.byref(c), C.byref(attend()), None) == _lib.CHONK_EINVAL
    assert L.chonk_kv_attend_workspace(C.byref(c), 1, 4) == _lib.CHONK_EINVAL
    assert b"paged K/V cache" in L.chonk_last_error() or b"null argument" in L.chonk_last_error()


@pytest.mark.parametrize("kw", [dict(type=2), dict(heads=3), dict(heads=0), dict(k=None), dict(v=None), dict(q_out=None),
                                dict(q_stride=255), dict(k_stride=127), dict(v_stride=-128), dict(q_out_stride=0),
                                dict(rope=0x10, rope_dim=66, rope_positions=4),
                                dict(rope=0x10, rope_dim=63, rope_positions=4),
                                dict(rope=0x10, rope_dim=64, rope_positions=0),
                                dict(k_norm=0x10, eps=-1e-9), dict(k_norm=0x10, eps=float("nan"))])
def test_append_refuses(kw):
    c, rows = cache(), _lib.KvRowsC(1, 0x10, 0x10)
    assert lib().chonk_kv_append(C.byref(c), C.byref(rows), C.byref(append(**kw)), None) == _lib.CHONK_EINVAL


@pytest.mark.parametrize("n,seq,pos", [(-1, 0x10, 0x10), (1 << 23, 0x10, 0x10), (1, None, 0x10), (1, 0x10, None)])
def test_rows_are_checked(n, seq, pos):
    c, rows = cache(), _lib.KvRowsC(n, seq, pos)
    assert lib().chonk_kv_append(C.byref(c), C.byref(rows), C.byref(append()), None) == _lib.CHONK_EINVAL
    assert lib().chonk_kv_read(C.byref(c), C.byref(rows), 0, 0x10, 0x10, 128, 64, None) == _lib.CHONK_EINVAL


@pytest.mark.parametrize("args", [(2, 0x10, 0x10, 128, 64), (0, None, None, 128, 64), (0, 0x10, 0x10, 127, 64),
                                  (0, 0x10, 0x10, 128, 63), (0, 0x10, None, 64, 128), (0, 0x10, 0x10, -128, 64)])
def test_read_refuses(args):
    c, rows = cache(), _lib.KvRowsC(3, 0x10, 0x10)
    assert lib().chonk_kv_read(C.byref(c), C.byref(rows), *args, None) == _lib.CHONK_EINVAL


@pytest.mark.parametrize("kw", [dict(type=-1), dict(heads=5), dict(n=-1), dict(seq=None), dict(lengths=None), dict(q=None),
                                dict(out=None), dict(q_stride=100), dict(out_stride=255), dict(window=-1),
                                dict(n=1 << 22, heads=4096, q_stride=1 << 18, out_stride=1 << 18)])
def test_attend_refuses(kw):
    c = cache()
    assert lib().chonk_kv_attend(C.byref(c), C.byref(attend(**kw)), None) == _lib.CHONK_EINVAL


def test_attend_wants_its_workspace():
    c = cache(max_pages=64)
    need = lib().chonk_kv_attend_workspace(C.byref(c), 1, 4)
    assert need > 0
    for kw in (dict(workspace=None), dict(workspace_bytes=need - 1), dict(workspace=0x1004)):
        assert lib().chonk_kv_attend(C.byref(c), C.byref(attend(**kw)), None) == _lib.CHONK_EINVAL
        assert b"workspace" in lib().chonk_last_error()
    assert lib().chonk_kv_attend_workspace(C.byref(c), 0, 4) == 0
    assert lib().chonk_kv_attend_workspace(C.byref(c), 1, 5) == _lib.CHONK_EINVAL


def test_reference_quantiser_is_within_half_a_unit():
    x = np.random.default_rng(0).standard_normal((50, 64))
    for kv in ("q8", "q4"):
        d = ref.scales(kv, x)
        c = np.clip(np.rint(x / d), -127 if kv == "q8" else -8, 127 if kv == "q8" else 7)
        ok = np.abs(x / d) <= (127 if kv == "q8" else 7.5)
        assert (np.abs(c * d - x) <= np.abs(d) * 0.5 * (1 + 1e-9) + 1e-12)[ok].all()


def test_torch_after_the_library_is_refused():
    """libchonk.so loaded before torch runs on another HIP runtime than torch's tensors and streams."""
    code = ("from chonklm_amd._lib import lib\nlib()\nfrom chonklm_amd.paged_kv import ChonkError, PagedKv\n"
            "try:\n    PagedKv(None, None, 2, 64)\nexcept ChonkError as e:\n    print('refused:', e)\n")
    root = Path(__file__).resolve().parents[1]
    out = subprocess.run([sys.executable, "-c", code], cwd=root, stdout=subprocess.PIPE, stderr=subprocess.PIPE, text=True)
    assert "refused: paged K/V cache: libchonk.so was loaded before torch" in out.stdout, out.stdout + out.stderr


def test_tensors_off_the_gpu_are_refused():
    import torch

    from chonklm_amd.paged_kv import ChonkError, PagedKv, page_bytes

    pages = torch.zeros((2, page_bytes("q4", 2, 64)), dtype=torch.uint8)
    table = torch.zeros((1, 2), dtype=torch.int32)
    for f, text in ((lambda: PagedKv(pages, table, 2, 64, "q4"), "must be on a GPU"),
                    (lambda: PagedKv(pages, table, 2, 64, "q8"), "pages must be contiguous uint8"),
                    (lambda: PagedKv(pages, table, 2, 64, "q5"), "unsupported kv type"),
                    (lambda: PagedKv(pages, table, 2, 72, "q4"), "head_dim must be"),
                    (lambda: PagedKv(pages, table.long(), 2, 64, "q4"), "table must be contiguous int32"),
                    (lambda: page_bytes("f32", 2, 64), "unsupported kv type")):
        with pytest.raises(ChonkError, match=text) as e:
            f()
        assert e.value.status_name == "EINVAL"
    with pytest.raises(TypeError):
        PagedKv(pages)
