"""The quantised, paged K/V cache and its operators, as measurable cases.

A serving program keeps K and V of many sequences in pages of 64 positions (a
pool of pages and a table [sequence][page]), as fp16 or as 8- or 4-bit codes
with one fp16 scale for 32 dims of a position. Per layer and step it

  store    normalises and rotates the new rows' q and k, writes k and v into
           their pages (quantised), and for a prompt reads them back
  read     fetches a sequence's history from its pages as values
  attend   attends with one new token a sequence over the pages
  step     does all of it for one token of every sequence

The head geometries are those of the package's registry. ``run`` computes a
pass in elementary torch operations, or with ``own`` through
chonklm_amd.paged_kv. ``exact`` is the same from the definitions in 64 bits,
with every stored value found by its address.

Format of a page, for every kv head: K codes, K scales, V codes, V scales.
Codes are in units of 32 positions (half u) x 32 dims (block b), [u][b], a unit
in the order in which the matrix instructions take it (n = 16 g + i names a
lane, 0 <= i < 16):
  K: of position 16 t + i, dims 8 g .. 8 g + 7      [n][t] (fp16: [t][n])
  V: of dim 16 h + i, positions 4 g + (e % 4) + 16 (e / 4), e = 0 .. 7
                                                    [n][h] (fp16: [h][n])
as 8 halves, or 8 bytes (code + 128), or nibbles (code + 8): for K 4 bytes with
dims m | m + 4 << 4, for V [n] 8 bytes with dim i | dim 16 + i << 4.
Scales are [u][b][32], place 8 g + e holding position 4 g + (e % 4) + 16 (e / 4).
"""
from __future__ import annotations

import math

import torch

own = False

PAGE = 64
# heads, kv heads, head_dim, norms of q and k, rotary (0 none, 1 halves, 2 neighbours)
SHAPES = {
    "smollm2": (9, 3, 64, False, 2),
    "qwen3": (16, 8, 128, True, 1),
    "gemma3": (4, 1, 256, True, 1),
    "gpt2": (12, 12, 64, False, 0),
    "openelm": (20, 5, 64, True, 1),
    "lfm2": (16, 8, 64, True, 1),
    "granite": (12, 4, 64, False, 0),
    "tiny-lfm2": (6, 2, 32, True, 1),
}
THETA = {"smollm2": 1e5, "openelm": 1e4}


# ---- the cases ------------------------------------------------------------------


def _case(kind, shape, kv, rows, tokens, seqs=1, window=0, dtype="f32", ragged=False, name=None):
    c = dict(kind=kind, shape=shape, kv=kv, rows=rows, tokens=tokens, seqs=seqs, window=window, dtype=dtype,
             ragged=ragged)
    return dict(c, name=name) if name else c


def listed():
    return [
        # one token of one conversation into the cache (launches and latency)
        _case("store", "smollm2", "q8", 1, 301, name="store_token_smollm2_q8"),
        # one token of each of 64 sequences at different positions
        _case("store", "qwen3", "q4", 64, 640, seqs=64, ragged=True, name="store_batch_qwen3_q4"),
        # a prompt of odd length
        _case("store", "qwen3", "q8", 2047, 2047, name="store_prompt_qwen3_q8"),
        # a document's history, for a prompt's attention or for moving a sequence
        _case("read", "qwen3", "q8", 11003, 11003, name="read_document_qwen3_q8"),
        # several sequences' histories, 256-wide heads
        _case("read", "gemma3", "q4", 8192, 1152, seqs=8, name="read_batch_gemma3_q4"),
        # a short chat turn: one sequence, latency
        _case("attend", "smollm2", "q8", 1, 301, name="attend_short_smollm2_q8"),
        # one conversation at the model's full context: split over its length
        _case("attend", "qwen3", "q8", 1, 40960, name="attend_one_qwen3_41k_q8"),
        # a serving batch of ragged requests, fp16 activations
        _case("attend", "qwen3", "q8", 64, 640, seqs=64, ragged=True, dtype="f16", name="attend_batch_qwen3_q8"),
        # long ragged requests in 4 bits (the largest)
        _case("attend", "qwen3", "q4", 32, 16384, seqs=32, ragged=True, name="attend_long_qwen3_q4"),
        # sliding windows and 256-wide heads over fp16 pages
        _case("attend", "gemma3", "f16", 48, 8192, seqs=48, window=512, ragged=True, name="attend_window_gemma3_f16"),
        # a layer's whole step for a batch, every head its own kv head
        _case("step", "gpt2", "q8", 24, 1024, seqs=24, ragged=True, name="step_gpt2_q8"),
        # the same in 4 bits with groups of query heads and norms, two tokens short of a page
        _case("step", "lfm2", "q4", 5, 4094, seqs=5, name="step_lfm2_q4"),
    ]


def draw(rng):
    """One more case of the same ranges."""
    def log_int(lo, hi):
        return int(round(lo * (hi / lo) ** rng.random()))

    kind = rng.choice(["store", "read", "attend", "attend", "step"])
    shape = rng.choice(sorted(SHAPES))
    heads, kvh, hd, _, _ = SHAPES[shape]
    kv = rng.choice(["f16", "q8", "q8", "q4", "q4"])
    dtype = rng.choice(["f32", "f32", "f16"])
    seqs = log_int(1, 64)
    if kind == "read":
        seqs, tokens = min(seqs, 8), log_int(1, 16384)
        rows = log_int(1, min(16384, seqs * tokens))
        return _case(kind, shape, kv, rows, tokens, seqs=seqs, dtype=dtype)
    if kind == "store" and rng.random() < 0.5:
        rows = log_int(2, 2048)  # a prompt, or the rest of one
        return _case(kind, shape, kv, rows, rows + rng.randrange(0, 500), dtype=dtype)
    most = int(2.5e8 / (seqs * 2 * kvh * hd * {"f16": 2.0, "q8": 1.07, "q4": 0.57}[kv]))  # as the largest listed
    tokens = log_int(1, 8192 if kind == "store" else min(most, 16384 if seqs > 1 else 40960))
    window = rng.choice([0, 0, 0, log_int(1, 4096)])
    return _case(kind, shape, kv, seqs, tokens, seqs=seqs, window=window if kind != "store" else 0, dtype=dtype,
                 ragged=rng.random() < 0.7)


def work(case):
    heads, kvh, hd, _, _ = SHAPES[case["shape"]]
    el = 4 if case["dtype"] == "f32" else 2
    per = {"f16": 2.0, "q8": 34 / 32, "q4": 18 / 32}[case["kv"]]
    rows, new = case["rows"], 2.0 * kvh * hd * per
    lens = _lengths(case)
    seen = sum(min(n, case["window"] or n) for n in lens)
    bytes_ = flops = 0.0
    if case["kind"] in ("store", "step"):
        bytes_ += rows * hd * el * (2 * heads + 2 * kvh) + rows * new + 2.0 * rows * kvh * hd * 2
        flops += 12.0 * rows * hd * (heads + 2 * kvh)
    if case["kind"] == "read":
        bytes_ += rows * new + 2.0 * rows * kvh * hd * el
        flops += 2.0 * rows * kvh * hd
    if case["kind"] in ("attend", "step"):
        bytes_ += seen * new + 2.0 * rows * heads * hd * el
        flops += 4.0 * heads * hd * seen
    return {"bytes": bytes_, "flops": flops}


# ---- what a program has in hand -----------------------------------------------------


def _lengths(case):
    """Positions that each sequence holds; of 16 ragged ones at most one is empty."""
    n, top = case["seqs"], case["tokens"]
    if not case["ragged"]:
        return [top] * n
    lens = [max(1, int(round(top * ((i * 0.6180339887) % 1.0)))) for i in range(1, n + 1)]
    lens[0] = top
    if case["kind"] == "attend" and n >= 16:
        lens[5] = 0  # a sequence that has been taken off the batch
    return lens


def _places(case, gen, device):
    """Sequence and position of every row that is stored, read or attends."""
    lens = torch.tensor(_lengths(case), device=device)
    rows = case["rows"]
    if case["kind"] in ("attend", "step") or (case["kind"] == "store" and case["seqs"] > 1):
        seqs = torch.arange(rows, device=device)
        return seqs, lens - 1
    if case["kind"] == "store":
        return torch.zeros(rows, dtype=torch.long, device=device), torch.arange(rows, device=device) + case["tokens"] - rows
    at = torch.arange(rows, device=device)  # read: history by history, over again where they are shorter
    return (at // case["tokens"]) % case["seqs"], at % case["tokens"]


def _rows_like(shape, gen, device, dtype):
    """Projections as a trained model's: unit variance, a few channels that stand out."""
    x = torch.randn(shape, generator=gen, device=device)
    x[..., 3::29] *= 4.0
    return x.to(dtype)


def prepare(case, seed):
    device = torch.device("cuda")
    gen = torch.Generator(device=device).manual_seed(int(seed))
    heads, kvh, hd, norm, rope = SHAPES[case["shape"]]
    dtype = torch.float32 if case["dtype"] == "f32" else torch.float16
    max_pages = max(1, -(-case["tokens"] // PAGE))
    need = torch.tensor([-(-n // PAGE) for n in _lengths(case)], device=device)
    n_pages = max(1, int(need.sum()))
    ids = torch.randperm(n_pages, generator=gen, device=device).to(torch.int32)
    used = torch.arange(max_pages, device=device)[None, :] < need[:, None]
    table = torch.zeros((case["seqs"], max_pages), dtype=torch.int32, device=device)
    table[used] = ids[: int(used.sum())]
    pages = torch.empty((n_pages, kvh, _head_bytes(case["kv"], hd)), dtype=torch.uint8, device=device)
    for a in range(0, n_pages, 1024):  # what earlier steps have stored
        n = min(1024, n_pages - a)
        k, v = (_rows_like((n, kvh, PAGE, hd), gen, device, torch.float32) for _ in range(2))
        pages[a:a + n] = _packed(case["kv"], k, v)
    seqs, pos = _places(case, gen, device)
    state = dict(case=case, pages=pages.view(n_pages, -1), table=table, seqs=seqs.to(torch.int32),
                 pos=pos.to(torch.int32), lens=torch.tensor(_lengths(case), dtype=torch.int32, device=device))
    rows = case["rows"]
    if case["kind"] != "read":
        state["q"] = _rows_like((rows, heads, hd), gen, device, dtype)
    if case["kind"] in ("store", "step"):
        state["k"] = _rows_like((rows, kvh, hd), gen, device, dtype)
        state["v"] = _rows_like((rows, kvh, hd), gen, device, dtype)
        state["qn"] = 1 + 0.1 * torch.randn(hd, generator=gen, device=device) if norm else None
        state["kn"] = 1 + 0.1 * torch.randn(hd, generator=gen, device=device) if norm else None
        state["rope"] = _rope(case, device) if rope else None
    return state


def _rope(case, device):
    """(cos, sin) of every position's angles: the table that a program makes once."""
    hd = SHAPES[case["shape"]][2]
    inv = THETA.get(case["shape"], 1e6) ** (-torch.arange(0, hd, 2, dtype=torch.float64, device=device) / hd)
    ang = torch.arange(case["tokens"], dtype=torch.float64, device=device)[:, None] * inv
    return torch.stack([ang.cos(), ang.sin()], dim=-1).float()


# ---- the calls, and their plain form ------------------------------------------------


def run(state):
    case = state["case"]
    kind = case["kind"]
    heads, kvh, hd, _, rope = SHAPES[case["shape"]]
    if own:
        from chonklm_amd.paged_kv import PagedKv

        kv = PagedKv(state["pages"], state["table"], kvh, hd, case["kv"])
        if kind == "read":
            return kv.read(state["seqs"], state["pos"], dtype=torch.float32 if case["dtype"] == "f32" else torch.float16)
        if kind == "attend":
            return kv.attend(state["q"], state["seqs"], state["lens"], window=case["window"])
        q = kv.append(state["q"], state["k"], state["v"], state["seqs"], state["pos"], q_norm=state["qn"],
                      k_norm=state["kn"], eps=1e-6, rope=state["rope"], interleaved=rope == 2)
        out = {"q": q} if kind == "store" else {
            "o": kv.attend(q, state["seqs"], state["lens"], window=case["window"])}
        out["k"], out["v"] = kv.read(state["seqs"], state["pos"])
        return out
    if kind == "read":
        return _plain_read(state, torch.float32 if case["dtype"] == "f32" else torch.float16)
    if kind == "attend":
        return _plain_attend(state, state["q"])
    q = _turned(state["q"].float(), state["qn"], state).to(state["q"].dtype)
    k, v = _turned(state["k"].float(), state["kn"], state), state["v"].float()
    _plain_write(state, k, v)
    out = {"q": q} if kind == "store" else {"o": _plain_attend(state, q)}
    out["k"], out["v"] = _plain_read(state, torch.float16)
    return out


def _turned(x, weight, state):
    """Norm of every head and rotation of its pairs, fp32 products one by one."""
    if weight is not None:
        # the sum of squares in 64 bits: codes must not hang on the order of a sum
        inv = (x.double().square().mean(-1, keepdim=True) + 1e-6).rsqrt().float()
        x = x * inv * weight
    if state["rope"] is None:
        return x
    cs = state["rope"][state["pos"].long()][:, None]
    c, s = cs[..., 0], cs[..., 1]
    if SHAPES[state["case"]["shape"]][4] == 2:
        a, b = x[..., 0::2], x[..., 1::2]
        return torch.stack([a * c - b * s, a * s + b * c], dim=-1).flatten(-2)
    a, b = x.chunk(2, dim=-1)
    return torch.cat([a * c - b * s, a * s + b * c], dim=-1)


def _codes(kv, x):
    """Codes (whole numbers) and fp16 scales of blocks of 32 along the last axis."""
    x = x.unflatten(-1, (-1, 32))
    big = x.abs().max(-1, keepdim=True)
    top = 127 if kv == "q8" else 7
    if kv == "q8":
        d = big.values / torch.full_like(big.values, 127.0)  # (by a number it is a product with 1 / 127)
    else:
        d = x.gather(-1, big.indices) / -8
    d = d.clamp(-65504, 65504).half()
    c = (x / d.float()).round().clamp(-127 if kv == "q8" else -8, top).nan_to_num(0.0)
    d = torch.where(big.values.isfinite(), d, torch.full_like(d, float("nan")))
    return c, d[..., 0]


def _head_bytes(kv, hd):
    """Bytes of one kv head's K and V in a page."""
    return 2 * PAGE * {"f16": 2 * hd, "q8": hd + hd // 16, "q4": hd // 2 + hd // 16}[kv]


def _operand_k(x):
    """[.., 64, hd] -> [.., u, b, g, i, t, 8] of K."""
    x = x.unflatten(-1, (-1, 4, 8)).unflatten(-4, (2, 2, 16))  # u t i b g 8
    return x.movedim((-6, -3, -2, -4, -5), (-6, -5, -4, -3, -2))


def _operand_v(x):
    """[.., 64, hd] -> [.., u, b, g, i, h, 8] of V."""
    x = x.unflatten(-1, (-1, 2, 16)).unflatten(-4, (2, 2, 4, 4))  # u e4 g e b h i
    x = x.movedim((-7, -3, -5, -1, -2, -6, -4), (-7, -6, -5, -4, -3, -2, -1))  # u b g i h e4 e
    return x.flatten(-2)


def _scale_order(d):
    """[.., 64, blocks] -> [.., u, b, 32] in the order of the positions' places."""
    return d.unflatten(-2, (2, 2, 4, 4)).movedim((-5, -1, -3, -4, -2), (-5, -4, -3, -2, -1)).flatten(-3)


def _as_bytes(x):
    return x.contiguous().view(torch.uint8)


def _packed(kv, k, v):
    """[.., 64, hd] values of K and V -> the bytes of the head's page."""
    parts = []
    for x, operand in ((k, _operand_k), (v, _operand_v)):
        if kv == "f16":
            parts.append(_as_bytes(operand(x.half()).movedim(-2, -4)).flatten(-6))
            continue
        c, d = _codes(kv, x)
        c = operand(c.flatten(-2) + (128 if kv == "q8" else 8)).to(torch.uint8)
        if kv == "q4" and operand is _operand_k:
            c = c[..., :4] | (c[..., 4:] << 4)
        elif kv == "q4":
            c = c[..., 0, :] | (c[..., 1, :] << 4)
            c = c.unsqueeze(-2)
        parts += [c.flatten(-6), _as_bytes(_scale_order(d)).flatten(-3)]
    return torch.cat(parts, dim=-1)


def _unpacked(kv, data, hd):
    """The bytes of heads' pages [.., bytes] -> fp32 values of K and V [.., 64, hd]."""
    out = []
    nb = hd // 32
    for which, x in enumerate(data.chunk(2, dim=-1)):
        if kv == "f16":
            c = x.contiguous().view(torch.float16).float().unflatten(-1, (2, nb, 2, 4, 16, 8)).movedim(-4, -2)
        else:
            size = 64 * hd if kv == "q8" else 32 * hd
            d = x[..., size:].contiguous().view(torch.float16).float().unflatten(-1, (2, nb, 4, 2, 4))
            d = d.movedim((-5, -2, -3, -1, -4), (-5, -4, -3, -2, -1)).flatten(-5, -2)  # positions, blocks
            x = x[..., :size]
            if kv == "q8":
                c = x.unflatten(-1, (2, nb, 4, 16, 2, 8)).float() - 128
            elif which == 0:
                x = x.unflatten(-1, (2, nb, 4, 16, 2, 4))
                c = torch.cat([x & 15, x >> 4], dim=-1).float() - 8
            else:
                x = x.unflatten(-1, (2, nb, 4, 16, 8))
                c = torch.stack([x & 15, x >> 4], dim=-2).float() - 8
        if which == 0:  # u b g i t 8 -> u t i, b g 8
            c = c.movedim((-6, -2, -3, -5, -4), (-6, -5, -4, -3, -2))
        else:  # u b g i h (e4 e) -> u e4 g e, b h i
            c = c.unflatten(-1, (2, 4)).movedim((-7, -2, -5, -1, -6, -3, -4), (-7, -6, -5, -4, -3, -2, -1))
        c = c.flatten(-3)  # dims
        c = c.flatten(-4 if which == 0 else -5, -2)  # positions
        out.append(c if kv == "f16" else (c.unflatten(-1, (nb, 32)) * d[..., None]).flatten(-2))
    return out


def _plain_write(state, k, v):
    """Stores rows k and v [rows, kv_heads, hd] at their places: touched pages are
    taken apart, changed and put together again with the codes of the new rows."""
    case = state["case"]
    kv, hd = case["kv"], k.shape[-1]
    pos = state["pos"].long()
    page = state["table"][state["seqs"].long(), pos // PAGE].long()
    at = pos % PAGE
    touched, where = page.unique(return_inverse=True)
    # bytes of the new rows in pages of their own, and which bytes those are
    pages = state["pages"].view(len(state["pages"]), k.shape[1], -1)
    fresh = [torch.zeros((len(touched), PAGE) + x.shape[1:], device=x.device) for x in (k, v)]
    for x, y in zip((k, v), fresh):
        x = x.half().float() if kv == "f16" else x
        y[where, at] = x
    data = _packed(kv, *(y.transpose(1, 2) for y in fresh))
    mark = torch.zeros((len(touched), PAGE), dtype=torch.bool, device=k.device)
    mark[where, at] = True
    pages[touched] = torch.where(_byte_mask(kv, mark, hd), data, pages[touched])


def _byte_mask(kv, mark, hd):
    """Which bytes of a head's page belong to the marked positions [n, 64] -> [n, 1, bytes]."""
    m = mark[:, :, None].expand(-1, -1, hd)
    parts = []
    for operand in (_operand_k, _operand_v):
        c = operand(m)
        if kv == "f16":
            parts.append(c.movedim(-2, -4)[..., None].expand(*c.movedim(-2, -4).shape, 2).flatten(1))
            continue
        if kv == "q4":
            c = c[..., :4] if operand is _operand_k else c[..., 0, :]
        s = _scale_order(m[:, :, :: 32])
        parts += [c.flatten(1), s[..., None].expand(*s.shape, 2).flatten(1)]
    return torch.cat(parts, dim=-1)[:, None]


def _plain_read(state, dtype):
    case = state["case"]
    heads, kvh, hd, _, _ = SHAPES[case["shape"]]
    pages = state["pages"].view(len(state["pages"]), kvh, -1)
    table, pos = state["table"].long(), state["pos"].long()
    page = table[state["seqs"].long(), pos // PAGE]
    touched, where = page.unique(return_inverse=True)
    k, v = _unpacked(case["kv"], pages[touched], hd)
    return tuple(x[where, :, pos % PAGE].to(dtype) for x in (k, v))


def _plain_attend(state, q):
    case = state["case"]
    heads, kvh, hd, _, _ = SHAPES[case["shape"]]
    rows = len(q)
    pages = state["pages"].view(len(state["pages"]), kvh, -1)
    table, lens = state["table"].long()[state["seqs"].long()], state["lens"].long()
    k, v = _unpacked(case["kv"], pages[table], hd)  # [rows, max_pages, kv_heads, 64, hd]
    k, v = (x.transpose(1, 2).flatten(2, 3) for x in (k, v))
    s = torch.matmul(q.float().view(rows, kvh, heads // kvh, hd) / math.sqrt(hd), k.transpose(-1, -2))
    at = torch.arange(k.shape[2], device=q.device)
    seen = at[None, :] < lens[:, None]
    if case["window"]:
        seen &= at[None, :] >= lens[:, None] - case["window"]
    seen = seen[:, None, None]
    s = s.masked_fill(~seen, float("-inf"))
    top = s.amax(-1, keepdim=True)
    e = torch.where(seen, (s - top).exp(), torch.zeros_like(s))
    o = torch.matmul(e / e.sum(-1, keepdim=True).clamp_min(1e-30), v)
    return o.reshape(rows, heads, hd).to(q.dtype)


# ---- from the definitions, in 64 bits -----------------------------------------------


def exact(case, seed):
    state = prepare(case, seed)
    kind = case["kind"]
    heads, kvh, hd, _, rope = SHAPES[case["shape"]]
    seqs, pos = state["seqs"].long(), state["pos"].long()
    if kind == "read":
        return tuple(_stored(state, seqs, pos, which) for which in (0, 1))
    if kind == "attend":
        return _exact_attend(state, state["q"].double(), None)
    q = _exact_turn(state, state["q"].double(), state["qn"], rope)
    k = _exact_block(case["kv"], _exact_turn(state, state["k"].double(), state["kn"], rope))
    v = _exact_block(case["kv"], state["v"].double())
    if kind == "store":
        return {"q": q, "k": k, "v": v}
    return {"o": _exact_attend(state, q, (k, v)), "k": k, "v": v}


def _exact_turn(state, x, weight, rope):
    if weight is not None:
        x = x / torch.sqrt((x * x).sum(-1, keepdim=True) / x.shape[-1] + 1e-6) * weight.double()
    if not rope:
        return x
    half = x.shape[-1] // 2
    i = torch.arange(half, device=x.device)
    first, second = (2 * i, 2 * i + 1) if rope == 2 else (i, i + half)
    turn = state["rope"].double()[state["pos"].long()][:, None]
    z = torch.complex(x[..., first], x[..., second]) * torch.complex(turn[..., 0].contiguous(), turn[..., 1].contiguous())
    y = torch.empty_like(x)
    y[..., first], y[..., second] = z.real, z.imag
    return y


def _exact_block(kv, x):
    """The values that stored rows stand for."""
    if kv == "f16":
        return x.half().double()
    y = x.reshape(*x.shape[:-1], -1, 32)
    low, high = y.min(-1, keepdim=True).values, y.max(-1, keepdim=True).values
    if kv == "q8":
        d = torch.maximum(-low, high) / 127
        most, least = 127.0, -127.0
    else:
        # the largest magnitude, the lower index where both signs have it
        first_low, first_high = ((y == m).float().argmax(-1, keepdim=True) for m in (low, high))
        down = (-low > high) | ((-low == high) & (first_low < first_high))
        d = torch.where(down, -low, -high) / 8
        most, least = 7.0, -8.0
    d = d.half().double()
    c = torch.where(d == 0, torch.zeros_like(y), (y / torch.where(d == 0, torch.ones_like(d), d)).round())
    return (c.clamp(least, most) * d).reshape(x.shape)


def _stored(state, seqs, pos, which):
    """Values [n, kv_heads, hd] of K (which = 0) or V stored at these places, each found by its address."""
    case = state["case"]
    kv, (_, kvh, hd, _, _) = case["kv"], SHAPES[case["shape"]]
    data = state["pages"].reshape(-1)
    head_bytes = _head_bytes(kv, hd)
    page = state["table"].long()[seqs, pos // PAGE]
    base = ((page[:, None] * kvh + torch.arange(kvh, device=pos.device)) * head_bytes + which * (head_bytes // 2))[..., None]
    j, d = (pos % PAGE)[:, None, None], torch.arange(hd, device=pos.device)[None, None]
    unit = (j // 32) * (hd // 32) + d // 32
    i, p = d % 32, j % 32
    if which == 0:
        lane, piece, e = (i // 8) * 16 + p % 16, p // 16, i % 8
    else:
        lane, piece, e = (p % 16) // 4 * 16 + i % 16, i // 16, p % 4 + 4 * (p // 16)

    def half_at(at):
        return (data[at].int() | (data[at + 1].int() << 8)).to(torch.int16).view(torch.float16).double()

    if kv == "f16":
        return half_at(base + 2 * (unit * 1024 + piece * 512 + lane * 8 + e))
    if kv == "q8":
        c = data[base + unit * 1024 + lane * 16 + piece * 8 + e].double() - 128
        scales = 64 * hd
    else:
        if which == 0:
            byte, high = unit * 512 + lane * 8 + piece * 4 + e % 4, e // 4
        else:
            byte, high = unit * 512 + lane * 8 + e, piece
        c = ((data[base + byte].int() >> (4 * high)) & 15).double() - 8
        scales = 32 * hd
    place = (p % 16) // 4 * 8 + p % 4 + 4 * (p // 16)
    return c * half_at(base + scales + 2 * (unit * 32 + place))


def _exact_attend(state, q, new):
    """Row by row; `new`: (k, v) just stored at the rows' positions."""
    case = state["case"]
    heads, kvh, hd, _, _ = SHAPES[case["shape"]]
    out = torch.zeros_like(q)
    for r, (s, n) in enumerate(zip(state["seqs"].tolist(), state["lens"].tolist())):
        if n == 0:
            continue
        first = max(0, n - case["window"]) if case["window"] else 0
        at = torch.arange(first, n, device=q.device)
        k, v = (_stored(state, torch.full_like(at, s), at, which) for which in (0, 1))
        if new is not None:
            k[-1], v[-1] = new[0][r], new[1][r]
        for h in range(heads):
            w = torch.softmax(k[:, h // (heads // kvh)] @ q[r, h] / math.sqrt(hd), 0)
            out[r, h] = w @ v[:, h // (heads // kvh)]
    return out
