"""The paged K/V cache operators on the GPU against tests/paged_ref.py (64 bits):
writing with norm and rotation, reading back, attention over the pages.

Tolerances. A product or sum rounded to fp32 is off by 2^-24 of itself. A stored
code is off by half a unit of its scale, more only where a 4-bit block's largest
element has an opposite of the same size (code 8 does not exist). Attention: a
score is a sum of hd products, each with q held in two fp16 halves (2^-22), so
it is off by (2^-22 + (hd + 8) 2^-24) sum |q k| scale; a weight by that and the
exponential's 2^-21; the weighted sum of n terms adds n 2^-24.
"""
from __future__ import annotations

import functools

import numpy as np
import pytest
import torch

from chonklm_amd.paged_kv import ChonkError, PagedKv, page_bytes, rope_table
from tests import paged_ref as ref

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
DEV = "cuda:0"


def host(x):
    return x.detach().cpu().numpy()


def dev(x, dtype=None):
    t = torch.from_numpy(np.ascontiguousarray(x)).to(DEV)
    return t if dtype is None else t.to(dtype)


class Cache:
    """A pool of random bytes (finite scales) with pages in random order."""

    def __init__(self, kv, kv_heads, hd, n_seqs, max_pages, seed=0, fill=None, spare=3):
        rng = np.random.default_rng(seed)
        n_pages = n_seqs * max_pages + spare
        self.kv_dtype, self.kv_heads, self.hd = kv, kv_heads, hd
        data = rng.integers(0, 256, (n_pages, page_bytes(kv, kv_heads, hd)), dtype=np.uint8)
        if fill is not None:
            data[:] = fill
        else:
            parts = data.reshape(n_pages, kv_heads, 2, -1)
            if kv == "f16":
                parts[:] = rng.standard_normal((n_pages, kv_heads, 2, 64 * hd)).astype(np.float16).view(np.uint8)
            else:
                n = 64 * hd // 32
                s = np.exp(rng.normal(-4, 1, (n_pages, kv_heads, 2, n))).astype(np.float16)
                if kv == "q4":
                    s *= rng.choice([-1, 1], s.shape).astype(np.float16)
                parts[..., ref.code_bytes(kv, hd):] = s.view(np.uint8).reshape(n_pages, kv_heads, 2, -1)
        self.table_np = rng.permutation(n_pages)[: n_seqs * max_pages].reshape(n_seqs, max_pages).astype(np.int32)
        self.pages, self.table = dev(data), dev(self.table_np)
        self.fault = torch.zeros(1, dtype=torch.int32, device=DEV)
        self.op = PagedKv(self.pages, self.table, kv_heads, hd, kv, fault=self.fault)
        self.rng = rng

    def stored(self, seq, positions):
        return ref.gather(self.kv_dtype, host(self.pages), self.table_np, self.kv_heads, self.hd, seq, positions)


def check_codes(kv, got, want, slack):
    """got: read-back fp32 values; want: exact values before quantisation, from which those
    that were quantised are off by at most `slack` (fp32 rounding of norm and rotation).
    Near zero a rotation's two products cancel: their roundings stay, U |product| each,
    so the slack is a number and no share of the value."""
    if kv == "f16":
        # two roundings: to fp32 arithmetic's result, then to fp16
        assert np.all(np.abs(got - want) <= (np.abs(want) + slack) * 2.0 ** -11 + slack + 2.0 ** -25)
        return
    d = np.abs(ref.scales(kv, want)) * (1 + 2.0 ** -10) + 2.0 ** -24  # a scale may round the other way
    err = np.abs(got - want)
    room = 0.5 * d + slack + 127 * 2.0 ** -11 * d
    if kv == "q4":  # codes end at 7 on the side away from the largest element
        room = np.where(want / ref.scales(kv, want) > 7.4, 1.01 * d, room)
    assert np.all(err <= room), float((err / room).max())


GEOMETRIES = [(3, 3, 32), (6, 2, 64), (16, 8, 128), (4, 1, 256), (18, 1, 64)]


@pytest.mark.parametrize("kv", ref.TYPES)
@pytest.mark.parametrize("heads,kv_heads,hd", GEOMETRIES)
@pytest.mark.parametrize("norm,rope,interleaved", [(False, 0, False), (True, 1, False), (True, 1, True), (False, 2, True),
                                                   (True, 2, False)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_append_and_read(kv, heads, kv_heads, hd, norm, rope, interleaved, dtype):
    c = Cache(kv, kv_heads, hd, n_seqs=3, max_pages=3, seed=heads + hd)
    rng, n = c.rng, 37
    places = rng.permutation(3 * 192)[:n]
    seqs, pos = (places // 192).astype(np.int32), (places % 192).astype(np.int32)
    q, k, v = (dev(rng.standard_normal((n, h, hd)), dtype) for h in (heads, kv_heads, kv_heads))
    wq, wk = ((dev(1 + 0.2 * rng.standard_normal(hd), torch.float32) for _ in range(2)) if norm else (None, None))
    dim = hd if rope == 1 else hd // 2
    table = rope_table(192, dim, 1e4, DEV) if rope else None
    cs = host(table)[pos] if rope else None
    out = c.op.append(q, k, v, dev(seqs), dev(pos), q_norm=wq, k_norm=wk, eps=1e-5, rope=table, interleaved=interleaved)
    c.op.check()
    want_q = ref.turn(host(q), host(wq) if norm else None, 1e-5, cs, interleaved)
    want_k = ref.turn(host(k), host(wk) if norm else None, 1e-5, cs, interleaved)
    # norm: 3 roundings; a rotation: two products, a sum of two terms of up to the pair's length
    pair = np.sqrt(2.0)
    big = np.abs(ref.turn(host(q), host(wq) if norm else None, 1e-5, None, False)).max()
    eps_out = 2.0 ** -11 if dtype == torch.float16 else 0.0
    assert np.all(np.abs(host(out) - want_q) <= 8 * U * pair * big + (eps_out + U) * np.abs(want_q) + 2.0 ** -25)
    got_k, got_v = (host(x).astype(np.float64) for x in c.op.read(dev(seqs), dev(pos), torch.float32))
    bigk = np.abs(ref.turn(host(k), host(wk) if norm else None, 1e-5, None, False)).max()
    check_codes(kv, got_k, want_k, 8 * U * pair * bigk)
    check_codes(kv, got_v, host(v).astype(np.float64), 0.0)
    if kv == "f16" and not rope and not norm:
        assert np.array_equal(got_k, host(k).astype(np.float16).astype(np.float64))
    # where the bytes lie, and what an fp16 read rounds
    for s in range(3):
        mine = np.flatnonzero(seqs == s)
        stored = c.stored(s, pos[mine])
        assert np.array_equal(stored[0].astype(np.float32), got_k[mine].astype(np.float32))
        assert np.array_equal(stored[1].astype(np.float32), got_v[mine].astype(np.float32))
    half_k, half_v = c.op.read(dev(seqs), dev(pos))
    assert np.array_equal(host(half_k), got_k.astype(np.float16)) and np.array_equal(host(half_v), got_v.astype(np.float16))


@pytest.mark.parametrize("kv", ref.TYPES)
@pytest.mark.parametrize("hd", [32, 64, 128, 256])
def test_append_leaves_every_other_byte(kv, hd):
    c = Cache(kv, 2, hd, n_seqs=2, max_pages=2, seed=hd)
    before = host(c.pages).copy()
    rng = c.rng
    seqs = np.array([0, 1, -1, 1, 0], dtype=np.int32)
    pos = np.array([0, 63, 5, 64, 97], dtype=np.int32)
    q, k, v = (dev(rng.standard_normal((5, h, hd)), torch.float32) for h in (4, 2, 2))
    out = torch.full_like(q, 7.0)
    c.op.append(q, k, v, dev(seqs), dev(pos), out=out)
    after = host(c.pages)
    mask = np.zeros(after.shape, dtype=bool).reshape(len(after), 2, 2, -1)
    for s, p in zip(seqs, pos):
        if s >= 0:
            mask[c.table_np[s, p // 64]] |= ref.owned_bytes(kv, hd, p % 64)[None]
    mask = mask.reshape(after.shape)
    assert np.array_equal(after[~mask], before[~mask])
    assert np.all(host(out)[2] == 7.0) and np.array_equal(host(out)[[0, 1, 3, 4]], host(q)[[0, 1, 3, 4]])
    k2, v2 = c.op.read(dev(seqs), dev(pos))
    for i in (0, 1, 3, 4):
        assert np.array_equal(host(k2)[i], c.stored(seqs[i], [pos[i]])[0][0].astype(np.float16))


@pytest.mark.parametrize("kv", ["q8", "q4"])
def test_blocks_at_the_formats_ends(kv):
    """Zeros, fp16's smallest and largest scales, ties, NaN and infinities."""
    c = Cache(kv, 1, 64, n_seqs=1, max_pages=1)
    x = np.zeros((8, 1, 64), dtype=np.float32)
    x[1, 0, :32] = np.linspace(-1, 1, 32)           # both ends of one size: the first is the largest
    x[2, 0, :32] = np.linspace(1, -1, 32)
    x[3, 0, 5] = 1e30                                # the scale saturates
    x[4, 0, 3] = 1e-9                                # ... or vanishes
    x[5, 0, 40] = np.nan
    x[6, 0, 33] = -np.inf
    x[7, 0] = 3.0
    seqs, pos = dev(np.zeros(8, np.int32)), dev(np.arange(8, dtype=np.int32))
    c.op.append(None, dev(x), dev(x[:, :, ::-1].copy()), seqs, pos)
    k, v = (host(t)[:, 0].astype(np.float64) for t in c.op.read(seqs, pos, torch.float32))
    for got, src in ((k, x[:, 0]), (v, x[:, 0, ::-1])):
        for r in (0, 4):
            assert np.all(got[r] == 0)
        assert np.isfinite(got[3]).all() and got[3].max() == 65504.0 * (127 if kv == "q8" else 7) or \
            (kv == "q4" and got[3].max() == 65504.0 * 8)
        for r in (5, 6):
            block = np.isfinite(src[r].reshape(2, 32)).all(-1)
            assert np.array_equal(np.isnan(got[r].reshape(2, 32)).all(-1), ~block)
            assert np.all(got[r].reshape(2, 32)[block] == 0)
        for r in (1, 2, 7):
            check_codes(kv, got[r], src[r].astype(np.float64), 0.0)


def attend_tolerance(mass, reach, n, hd, out_eps):
    s = (2.0 ** -22 + (hd + 8) * U) * reach[:, None]
    return mass * (2 * s + 2.0 ** -20 + n * U) + out_eps * mass + 2.0 ** -25


LENGTHS = [0, 1, 2, 31, 32, 33, 63, 64, 65, 127, 128, 130, 300, 449]


@pytest.mark.parametrize("kv", ref.TYPES)
@pytest.mark.parametrize("heads,kv_heads,hd", GEOMETRIES + [(2, 2, 256), (40, 2, 128), (17, 1, 32)])
@pytest.mark.parametrize("window", [0, 1, 70])
def test_attend(kv, heads, kv_heads, hd, window):
    c = Cache(kv, kv_heads, hd, n_seqs=4, max_pages=8, seed=hd + heads)
    n = len(LENGTHS)
    seqs = np.arange(n, dtype=np.int32) % 4
    q = c.rng.standard_normal((n, heads, hd)).astype(np.float32)
    q[:, :, 1::7] *= 3
    if kv != "f16":
        q *= 4  # (the pool's values are small)
    out = host(c.op.attend(dev(q), dev(seqs), dev(np.array(LENGTHS, np.int32)), window=window))
    c.op.check()
    for r, length in enumerate(LENGTHS):
        at = np.arange(max(0, length - window) if window else 0, length)
        k, v = c.stored(seqs[r], at) if len(at) else (np.zeros((0, kv_heads, hd)),) * 2
        want, mass, reach = ref.attend(q[r].astype(np.float64), k, v, hd ** -0.5)
        tol = attend_tolerance(mass, reach, length, hd, 0.0)
        assert np.all(np.abs(out[r] - want) <= tol), (length, float((np.abs(out[r] - want) / tol).max()))


@pytest.mark.parametrize("kv", ref.TYPES)
def test_attend_does_not_see_what_lies_elsewhere(kv):
    """NaN bytes in every place that no row sees, and rows behind the batch's end."""
    c = Cache(kv, 2, 64, n_seqs=2, max_pages=4, seed=3)
    rng = c.rng
    clean = host(c.pages).copy()
    dirty = np.full_like(clean, 0xFF)
    lengths, window = np.array([130, 70, 9], np.int32), 50
    seqs = np.array([0, 1, -1], np.int32)
    for s, n in ((0, 130), (1, 70)):
        for p in range(n - window, n):
            m = np.broadcast_to(ref.owned_bytes(kv, 64, p % 64), (2,) + ref.owned_bytes(kv, 64, 0).shape).reshape(-1)
            page = c.table_np[s, p // 64]
            dirty[page][m] = clean[page][m]
    q = dev(rng.standard_normal((3, 4, 64)).astype(np.float32))
    a = torch.full_like(q, 5.0)
    b = torch.full_like(q, 5.0)
    c.op.attend(q, dev(seqs), dev(lengths), window=window, out=a)
    c.pages.copy_(dev(dirty))
    c.op.attend(q, dev(seqs), dev(lengths), window=window, out=b)
    assert torch.equal(a, b) and torch.isfinite(a).all() and (a[2] == 5.0).all()


@pytest.mark.parametrize("kv", ref.TYPES)
@pytest.mark.parametrize("rows,length", [(1, 9000), (3, 4097), (300, 65)])
def test_attend_split_over_the_length(kv, rows, length):
    c = Cache(kv, 2, 128, n_seqs=1, max_pages=(length + 63) // 64, seed=rows)
    heads = 6
    q = c.rng.standard_normal((rows, heads, 128)).astype(np.float32) * (1 if kv == "f16" else 6)
    seqs, lengths = np.zeros(rows, np.int32), np.full(rows, length, np.int32)
    lengths[rows // 2:] -= np.arange(rows - rows // 2, dtype=np.int32) % 60
    out = host(c.op.attend(dev(q), dev(seqs), dev(lengths)))
    k, v = c.stored(0, np.arange(length))
    for r in {0, rows // 2, rows - 1}:
        n = lengths[r]
        want, mass, reach = ref.attend(q[r].astype(np.float64), k[:n], v[:n], 128 ** -0.5)
        tol = attend_tolerance(mass, reach, n, 128, 0.0)
        assert np.all(np.abs(out[r] - want) <= tol), float((np.abs(out[r] - want) / tol).max())


@pytest.mark.parametrize("kv", ref.TYPES)
def test_sizes_of_values_and_half_precision_rows(kv):
    """Queries and values far from 1, one weight that outweighs the others, strided fp16 rows."""
    c = Cache(kv, 1, 64, n_seqs=1, max_pages=2, seed=9)
    rng, n = c.rng, 100
    for size_k, size_v, size_q in ((1.0, 1.0, 1.0), (100.0, 3000.0, 0.02), (0.01, 1e-3, 200.0), (8.0, 1.0, 30.0)):
        k = (rng.standard_normal((n, 1, 64)) * size_k).astype(np.float32)
        v = (rng.standard_normal((n, 1, 64)) * size_v).astype(np.float32)
        v[::7] *= 9
        seqs, pos = dev(np.zeros(n, np.int32)), dev(np.arange(n, dtype=np.int32))
        c.op.append(None, dev(k), dev(v), seqs, pos)
        stored = c.stored(0, np.arange(n))
        for dtype in (torch.float32, torch.float16):
            wide = dev((rng.standard_normal((3, 5, 64)) * size_q), dtype)
            q = wide[:, 1:4]
            o = torch.zeros((3, 7, 64), dtype=dtype, device=DEV)
            lengths = dev(np.array([n, 50, 1], np.int32))
            c.op.attend(q, seqs[:3], lengths, scale=0.3, out=o[:, 2:5])
            assert (o[:, :2] == 0).all() and (o[:, 5:] == 0).all()
            for r, m in enumerate((n, 50, 1)):
                want, mass, reach = ref.attend(host(q)[r].astype(np.float64), stored[0][:m], stored[1][:m], 0.3)
                tol = attend_tolerance(mass, reach, m, 64, 2.0 ** -11 if dtype == torch.float16 else 0.0)
                got = host(o)[r, 2:5].astype(np.float64)
                # (values over 65504 are infinite in an fp16 cache, and so are their dims of the
                # result or NaN; an fp16 result over 65504 is infinite too)
                fine = np.isfinite(stored[1][:m, 0]).all(0)[None] & (np.abs(want) < (65504 if dtype == torch.float16 else 1e30))
                assert not np.isfinite(got[~fine]).any()
                assert np.all((np.abs(got - want) <= tol)[fine]), float((np.abs(got - want) / tol)[fine].max())


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("max_pages", [3, 70])
def test_attend_over_q_itself(dtype, max_pages):
    """Results that take q's place, whole rows and cut ones, one left out."""
    c = Cache("q8", 2, 64, n_seqs=3, max_pages=max_pages, seed=max_pages)
    n = 40
    q = dev(c.rng.standard_normal((n, 36, 64)), dtype)
    seqs = c.rng.integers(0, 3, n).astype(np.int32)
    seqs[5] = -1
    lengths = dev(c.rng.integers(0, 64 * max_pages + 1, n).astype(np.int32))
    apart = c.op.attend(q, dev(seqs), lengths, out=q.clone())
    assert c.op.attend(q, dev(seqs), lengths, out=q) is q
    c.op.check()
    assert torch.equal(q, apart)


@pytest.mark.parametrize("kv", ref.TYPES)
@pytest.mark.parametrize("heads,kv_heads,hd", [(16, 1, 256), (9, 1, 256), (5, 1, 128), (8, 8, 32), (32, 2, 64)])
@pytest.mark.parametrize("max_pages", [1, 70])
def test_attend_wide_groups_whole_and_split(kv, heads, kv_heads, hd, max_pages):
    """Five to sixteen heads over one kv head, rows walked whole by eight waves and cut."""
    c = Cache(kv, kv_heads, hd, n_seqs=2, max_pages=max_pages, seed=heads)
    lengths = [1, 40, 64] if max_pages == 1 else [4480, 0, 2013]
    seqs = np.array([0, 1, 1], np.int32)
    q = c.rng.standard_normal((3, heads, hd)).astype(np.float32) * (1 if kv == "f16" else 4)
    out = host(c.op.attend(dev(q), dev(seqs), dev(np.array(lengths, np.int32))))
    c.op.check()
    for r, n in enumerate(lengths):
        k, v = c.stored(seqs[r], np.arange(n)) if n else (np.zeros((0, kv_heads, hd)),) * 2
        want, mass, reach = ref.attend(q[r].astype(np.float64), k, v, hd ** -0.5)
        tol = attend_tolerance(mass, reach, n, hd, 0.0)
        assert np.all(np.abs(out[r] - want) <= tol), (n, float((np.abs(out[r] - want) / tol).max()))


@pytest.mark.parametrize("rows", [255, 256, 257, 600])
def test_many_rows_share_few_sequences(rows):
    """Around the number of rows up to which they are cut; every row its own length, one of
    16 empty and one of 16 left out, results equal to those of a call a row."""
    c = Cache("q8", 1, 64, n_seqs=3, max_pages=40, seed=rows)
    rng = c.rng
    q = dev(rng.standard_normal((rows, 2, 64)).astype(np.float32))
    seqs = rng.integers(0, 3, rows).astype(np.int32)
    lengths = rng.integers(1, 2561, rows).astype(np.int32)
    lengths[::16] = 0
    seqs[5::16] = -1
    out = torch.full_like(q, 9.0)
    c.op.attend(q, dev(seqs), dev(lengths), out=out)
    c.op.check()
    out = host(out)
    assert (out[5::16] == 9.0).all() and (out[::16] == 0.0).all()
    k, v = zip(*(c.stored(s, np.arange(2560)) for s in range(3)))
    for r in list(range(0, rows, 41)) + [rows - 1]:
        if seqs[r] < 0 or lengths[r] == 0:
            continue
        n = lengths[r]
        want, mass, reach = ref.attend(host(q)[r].astype(np.float64), k[seqs[r]][:n], v[seqs[r]][:n], 0.125)
        tol = attend_tolerance(mass, reach, n, 64, 0.0)
        assert np.all(np.abs(out[r] - want) <= tol), (r, float((np.abs(out[r] - want) / tol).max()))


@functools.lru_cache(maxsize=1)
def _long_tables(kv, kv_heads, hd):
    """A cache of two sequences of 4480 positions, and what they hold."""
    c = Cache(kv, kv_heads, hd, n_seqs=2, max_pages=70, seed=hd)
    return (c,) + tuple(zip(*(c.stored(s, np.arange(4480)) for s in range(2))))


@pytest.mark.parametrize("lengths", ["ragged", "like", "short", "one long"])
@pytest.mark.parametrize("window", [0, 4200])
@pytest.mark.parametrize("kv,rows,heads,kv_heads,hd", [("q8", 64, 12, 12, 64), ("q4", 64, 32, 8, 128), ("q4", 96, 8, 8, 128),
                                                      ("q8", 97, 8, 8, 128), ("f16", 200, 4, 2, 256)])
def test_many_rows_of_long_tables(kv, rows, heads, kv_heads, hd, lengths, window):
    """Enough (row, head)s to fill half of the device: cut where the lengths differ, whole
    where they are alike or short, or where there are more than the device holds at once."""
    c, k, v = _long_tables(kv, kv_heads, hd)
    rng = np.random.default_rng(rows)
    q = dev(rng.standard_normal((rows, heads, hd)).astype(np.float32) * (1 if kv == "f16" else 4))
    seqs = rng.integers(0, 2, rows).astype(np.int32)
    n = {"ragged": rng.integers(1, 4481, rows), "like": rng.integers(4300, 4481, rows),
         "short": rng.integers(1, 4097, rows), "one long": np.full(rows, 33)}[lengths].astype(np.int32)
    n[rows // 2] = 4096 if lengths == "short" else 4480
    n[3], seqs[7] = 0, -1
    out = torch.full_like(q, 9.0)
    c.op.attend(q, dev(seqs), dev(n), window=window, out=out)
    c.op.check()
    out = host(out)
    assert np.isfinite(out).all() and (out[7] == 9.0).all() and (out[3] == 0.0).all()
    for r in (0, rows // 2, int(n.argmax()), rows - 1):
        at = slice(max(0, n[r] - window) if window else 0, n[r])
        want, mass, reach = ref.attend(host(q)[r].astype(np.float64), k[seqs[r]][at], v[seqs[r]][at], hd ** -0.5)
        tol = attend_tolerance(mass, reach, n[r], hd, 0.0)
        assert np.all(np.abs(out[r] - want) <= tol), (r, float((np.abs(out[r] - want) / tol).max()))


def test_two_streams_and_two_graphs_of_one_cache():
    """Split calls of one cache on two streams at once, and two captured calls replayed together:
    each has a workspace of its own."""
    c = Cache("q4", 2, 128, n_seqs=1, max_pages=100, seed=8)
    rng = c.rng
    qs = [dev(rng.standard_normal((1, 32, 128)).astype(np.float32)) for _ in range(2)]
    seqs, lengths = dev(np.zeros(1, np.int32)), [dev(np.array([n], np.int32)) for n in (6400, 5003)]
    want = [c.op.attend(q, seqs, n).clone() for q, n in zip(qs, lengths)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(c.op.attend(qs[i], seqs, lengths[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(x, want[i]) for x in got[i])
    graphs, outs = [], []
    for i, s in enumerate(streams):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            outs.append(c.op.attend(qs[i], seqs, lengths[i]))
        graphs.append(g)
    for k in range(4):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                graphs[i].replay()
        torch.cuda.synchronize()
        assert all(torch.equal(outs[i], want[i]) for i in range(2)), k
        (qs[0] * 2).sum().item()


@pytest.mark.parametrize("kv", ref.TYPES)
def test_read_rows_in_any_order(kv):
    """Whole half pages, ragged ends, rows out of order, the same row twice, another sequence's
    rows between, rows left out: values do not depend on the company."""
    c = Cache(kv, 3, 64, n_seqs=3, max_pages=4, seed=77)
    runs = [(0, 0, 64), (1, 5, 100), (2, 40, 41), (0, 250, 256), (1, 31, 33), (2, 96, 160)]
    seqs = np.concatenate([np.full(b - a, s) for s, a, b in runs] + [[0, 0, 2, 1], np.full(9, -1)]).astype(np.int32)
    pos = np.concatenate([np.arange(a, b) for _, a, b in runs] + [[7, 7, 255, 0], np.arange(9)]).astype(np.int32)
    for cut in (0, 1, 17, 70):  # where the first half page starts
        s, p = seqs[cut:], pos[cut:]
        for dtype in (torch.float16, torch.float32):
            k, v = (host(x) for x in c.op.read(dev(s), dev(p), dtype))
            for i in range(len(s) - 9):
                want = c.stored(s[i], [p[i]])
                kind = np.float16 if dtype == torch.float16 else np.float32
                assert np.array_equal(k[i], want[0][0].astype(kind)) and np.array_equal(v[i], want[1][0].astype(kind)), (cut, i)
    c.op.check()


def test_rows_that_name_no_place():
    c = Cache("q8", 2, 64, n_seqs=2, max_pages=2)
    before = host(c.pages).copy()
    rng = c.rng
    q, k, v = (dev(rng.standard_normal((4, h, 64)), torch.float32) for h in (4, 2, 2))
    seqs, pos = dev(np.array([2, 0, 1, 0], np.int32)), dev(np.array([0, 128, -1, 127], np.int32))
    c.op.append(q, k, v, seqs, pos)
    with pytest.raises(ChonkError, match="a sequence outside the table, a position outside"):
        c.op.check()
    c.op.check()  # reported once
    changed = np.flatnonzero((host(c.pages) != before).any(-1))
    assert list(changed) == [c.table_np[0, 1]]
    c.op.append(q, k, v, dev(np.zeros(4, np.int32)), dev(np.arange(60, 64, dtype=np.int32)), rope=rope_table(62, 64, 1e4, DEV))
    with pytest.raises(ChonkError, match="a position outside"):
        c.op.check()
    out = c.op.attend(q, dev(np.array([0, 5, 0, 0], np.int32)), dev(np.array([128, 3, 129, 7], np.int32)))
    with pytest.raises(ChonkError, match="a sequence outside the table, a position outside"):
        c.op.check()
    nan = torch.isnan(out).all(-1).all(-1)
    assert nan.tolist() == [False, True, True, False]
    c.table[0, 1] = len(before)
    out = c.op.attend(q, dev(np.zeros(4, np.int32)), dev(np.array([128, 64, 65, 1], np.int32)))
    k2, _ = c.op.read(dev(np.zeros(4, np.int32)), dev(np.array([0, 63, 63, 0], np.int32)))
    with pytest.raises(ChonkError, match="a page outside the pool"):
        c.op.check()
    assert torch.isnan(out).all(-1).all(-1).tolist() == [True, False, True, False]
    assert torch.isfinite(k2).all()


@pytest.mark.parametrize("kv", ["q8", "q4"])
def test_prompt_rows_and_single_tokens_store_the_same_bytes(kv):
    """The same rows written in one call, or one by one, give the same pages."""
    a, b = (Cache(kv, 2, 128, n_seqs=1, max_pages=2, seed=5) for _ in range(2))
    rng = np.random.default_rng(1)
    q, k, v = (dev(rng.standard_normal((100, h, 128)), torch.float32) for h in (4, 2, 2))
    w, table = dev(1 + 0.1 * rng.standard_normal(128), torch.float32), rope_table(128, 128, 1e6, DEV)
    seqs, pos = dev(np.zeros(100, np.int32)), dev(np.arange(100, dtype=np.int32) + 3)
    qa = a.op.append(q, k, v, seqs, pos, q_norm=w, k_norm=w, rope=table)
    qb = [b.op.append(q[i:i + 1], k[i:i + 1], v[i:i + 1], seqs[:1], pos[i:i + 1], q_norm=w, k_norm=w, rope=table)
          for i in range(100)]
    assert torch.equal(a.pages, b.pages) and torch.equal(qa, torch.cat(qb))


@pytest.mark.parametrize("kv", ref.TYPES)
def test_steps_together_eager_and_captured(kv):
    """append then attend, step after step: a captured step replayed with other inputs,
    on a stream of its own, gives what eager calls give."""
    heads, kvh, hd, n = 8, 2, 64, 5
    a, b = (Cache(kv, kvh, hd, n_seqs=n, max_pages=3, seed=2) for _ in range(2))
    rng = np.random.default_rng(4)
    table = rope_table(192, hd, 1e4, DEV)
    seqs = dev(np.arange(n, dtype=np.int32))
    start = np.array([0, 60, 63, 100, 126], np.int32)
    steps = [[dev(rng.standard_normal((n, h, hd)), torch.float32) for h in (heads, kvh, kvh)] for _ in range(6)]

    def step(c, q, k, v, pos):
        q = c.op.append(q, k, v, seqs, pos, rope=table)
        return c.op.attend(q, seqs, pos + 1)

    eager = [step(a, *x, dev(start + i)) for i, x in enumerate(steps)]
    torch.cuda.synchronize()
    held = [torch.empty_like(x) for x in steps[0]]
    pos = dev(start)
    side = torch.cuda.Stream()
    before = b.pages.clone()
    with torch.cuda.stream(side):
        step(b, *steps[0], pos)
        side.synchronize()
        b.pages.copy_(before)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            got = step(b, *held, pos)
    torch.cuda.synchronize()
    for i, x in enumerate(steps):
        for h, y in zip(held, x):
            h.copy_(y)
        pos.copy_(dev(start + i))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, eager[i]), i
        (torch.randn(1000, device=DEV) * 2).sum()  # the program's other work
    assert torch.equal(a.pages, b.pages)
    a.op.check(), b.op.check()


@pytest.mark.parametrize("kv", ref.TYPES)
def test_pools_past_four_gigabytes(kv):
    """Pages whose bytes lie past 2^32 of the pool (and past 2^31 before it)."""
    size = page_bytes(kv, 8, 128)
    n_pages = (9 << 29) // size + 3
    pages = torch.empty((n_pages, size), dtype=torch.uint8, device=DEV)
    ids = np.array([[n_pages - 1, (5 << 29) // size, 0]], np.int32)
    op = PagedKv(pages, dev(ids), 8, 128, kv)
    rng = np.random.default_rng(6)
    k, v = (dev(rng.standard_normal((150, 8, 128)), torch.float32) for _ in range(2))
    seqs, pos = dev(np.zeros(150, np.int32)), dev(np.arange(150, dtype=np.int32))
    op.append(None, k, v, seqs, pos)
    got_k, got_v = op.read(seqs, pos, torch.float32)
    stored = ref.gather(kv, host(pages[dev(ids[0]).long()]), np.array([[0, 1, 2]]), 8, 128, 0, range(150))
    assert np.array_equal(host(got_k), stored[0].astype(np.float32)) and np.array_equal(host(got_v), stored[1].astype(np.float32))
    check_codes(kv, host(got_k).astype(np.float64), host(k).astype(np.float64), 0.0)
    q = dev(rng.standard_normal((1, 16, 128)), torch.float32)
    out = host(op.attend(q, seqs[:1], dev(np.array([150], np.int32))))
    want, mass, reach = ref.attend(host(q)[0].astype(np.float64), *stored, 128 ** -0.5)
    assert np.all(np.abs(out[0] - want) <= attend_tolerance(mass, reach, 150, 128, 0.0))


def test_rows_that_want_a_gradient_are_refused():
    c = Cache("q8", 2, 64, n_seqs=1, max_pages=1)
    q, k = torch.ones((1, 4, 64), device=DEV, requires_grad=True), torch.ones((1, 2, 64), device=DEV)
    i = torch.zeros(1, dtype=torch.int32, device=DEV)
    for f in (lambda: c.op.attend(q, i, i + 1), lambda: c.op.append(q, k, k, i, i)):
        with pytest.raises(ChonkError, match="requires a gradient"):
            f()
        with torch.no_grad():
            f()


def test_refusals_of_tensors():
    c = Cache("q8", 2, 64, n_seqs=2, max_pages=2)
    q, k = torch.zeros((3, 4, 64), device=DEV), torch.zeros((3, 2, 64), device=DEV)
    i = torch.zeros(3, dtype=torch.int32, device=DEV)
    bad = [
        lambda: c.op.append(q, k, k.half(), i, i),
        lambda: c.op.append(q.half(), k, k, i, i),
        lambda: c.op.append(q, k, k, i.long(), i),
        lambda: c.op.append(q, k, k, i[:2], i),
        lambda: c.op.append(q, k, k[:2], i, i),
        lambda: c.op.append(q[:, :3].contiguous(), k, k, i, i),
        lambda: c.op.append(q, k.cpu(), k, i, i),
        lambda: c.op.append(q, k, k, i, i, q_norm=torch.zeros(32, device=DEV)),
        lambda: c.op.append(q, k, k, i, i, rope=torch.zeros((8, 33, 2), device=DEV)),
        lambda: c.op.append(None, k, k, i, i, out=q),
        lambda: c.op.append(q, k, k, i, i, eps=-1.0, k_norm=torch.ones(64, device=DEV)),
        lambda: c.op.read(i, i, torch.float64),
        lambda: c.op.read(i, i[:1]),
        lambda: c.op.attend(q[..., :32], i, i),
        lambda: c.op.attend(q.transpose(0, 1), i, i),
        lambda: c.op.attend(q, i, i, window=-1),
        lambda: c.op.attend(q[:, :3], i, i),
        lambda: c.op.attend(q, i, i, out=q.half()),
        lambda: PagedKv(c.pages[:, :-2], c.table, 2, 64, "q8"),
        lambda: PagedKv(c.pages, c.table.long(), 2, 64, "q8"),
        lambda: PagedKv(c.pages, c.table, 2, 80, "q8"),
        lambda: PagedKv(c.pages, c.table, 2, 64, "q5"),
    ]
    for f in bad:
        with pytest.raises(ChonkError):
            f()
    empty = c.op.attend(q[:0], i[:0], i[:0])
    assert empty.shape == (0, 4, 64) and c.op.append(q[:0], k[:0], k[:0], i[:0], i[:0]).shape == (0, 4, 64)
