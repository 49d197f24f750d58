"""Batched decoding over 8- and 4-bit K/V pages: against a float64 decoder whose cache
holds the same codes' values, across prompts of several passes, windows, and
any subset of sequences a step.

The float64 decoder rounds each K and V row to the values its codes stand for; a prompt's
rows read them back in fp16, a step's as they are. The engine's row differs from it by fp32 rounding (about 1e-6 of the row), so a share of about
1e-6 * 127 (8 bits; 8 for 4) of the codes lands on the other side of a rounding border and is off by
one unit, 1/127 (1/8) of its block's largest element. fp16 rows (bar 1e-3 of the largest
logit in test_gpu_batch.py) do the same at 1e-6 * 2^11 of the values by 2^-11: in the root
of the summed squares, sqrt(share) * unit, 8 bits are 4 times that and 4 bits 16 times.
"""
from __future__ import annotations

import numpy as np
import pytest

from chonklm_amd import WORKLOADS, ChonkError, load_llama_wgsl_model
from chonklm_amd.runtime import LlamaWgslBatch
from tests import paged_ref as ref
from tests.conftest import rel_err
from tests.numpy_ref import NumpyDecoder

pytestmark = pytest.mark.gpu

BAR = {"q8": 4e-3, "q4": 1.6e-2}


class _Coded(np.ndarray):
    """[layer, kv head, position, hd] that keeps what a row's codes stand for."""

    kv, prompt = "q8", True

    def __getitem__(self, at):
        x = np.asarray(self)[at]
        return x.astype(np.float16).astype(np.float64) if self.prompt else x

    def __setitem__(self, at, rows):
        d = ref.scales(self.kv, rows)
        low, high = (-127, 127) if self.kv == "q8" else (-8, 7)
        c = np.clip(np.rint(np.divide(rows, d, out=np.zeros_like(rows), where=d != 0)), low, high)
        np.asarray(self)[at] = c * d


def _decoder(path, w, context, kv):
    d = NumpyDecoder(path, w.spec.vocab, context)

    def reset():
        d.pos = 0
        for name in ("K", "V"):
            x = np.zeros((d.L, d.nkv, d.ctx, d.hd)).view(_Coded)
            x.kv = kv
            setattr(d, name, x)

    def feed(token, prompt):
        d.K.prompt = d.V.prompt = prompt
        return d.step(token)

    d.reset, d.feed = reset, feed
    reset()
    return d


def _check(got_id, logits, want, bar, what):
    assert rel_err(logits, want) <= bar, f"{what}: {rel_err(logits, want):.2e}"
    assert got_id == int(np.argmax(logits)), what


@pytest.mark.parametrize("kv", ["q8", "q4"])
@pytest.mark.parametrize("name", ["tiny-qwen3", "tiny-llama", "tiny-gemma3", "tiny-qwen3-hd128"])
def test_coded_batch_matches_a_float64_decoder(name, kv, synth):
    w, path = WORKLOADS[name], synth(name)
    loaded = load_llama_wgsl_model(w.model_def(path))
    batch = LlamaWgslBatch(loaded.engine, 3, 90, kv_dtype=kv)
    refs = [_decoder(path, w, 96, kv) for _ in range(3)]
    rng = np.random.default_rng(43)
    for s, n in enumerate((11, 66, 1)):
        p = rng.integers(0, w.spec.vocab, n).tolist()
        got = batch.prefill(s, p)
        for t in p:
            want = refs[s].feed(t, True)
        _check(got, batch.read_logits(0), want, BAR[kv], f"seq {s} prefill")
    for step, seqs in enumerate([[0, 1, 2], [2, 0], [1], [2, 1, 0], [0, 2]]):
        tokens = rng.integers(0, w.spec.vocab, len(seqs)).tolist()
        got = batch.step(seqs, tokens)
        for row, s in enumerate(seqs):
            _check(got[row], batch.read_logits(row), refs[s].feed(tokens[row], False), BAR[kv], f"step {step} seq {s}")
    # a sequence started over forgets its earlier tokens
    refs[1].reset()
    got = batch.prefill(1, [5, 6, 7])
    for t in (5, 6, 7):
        want = refs[1].feed(t, True)
    _check(got, batch.read_logits(0), want, BAR[kv], "started over")
    batch.close()
    loaded.engine.dispose()


@pytest.mark.parametrize("kv", ["q8", "q4"])
@pytest.mark.parametrize("name,prompt", [("tiny-gemma3-hd256", 2300), ("tiny-gemma3-hd64", 5000), ("tiny-gemma3-hd64", 600)])
def test_long_prompts_and_split_steps(name, prompt, kv, synth):
    """Several passes of a prompt (its attention reads earlier passes back from the pages),
    windows of 512 and steps whose pages are split: a sequence's logits do not depend on the others,
    and stay as near the fp16 pages' as the codes allow."""
    w = WORKLOADS[name]
    loaded = load_llama_wgsl_model(w.model_def(synth(name)))
    p = w.prompt(5, prompt)
    rng = np.random.default_rng(2)
    forced = rng.integers(0, w.spec.vocab, 4).tolist()
    logits = {}
    for kind in ("f16", kv):
        batch = LlamaWgslBatch(loaded.engine, 2, 5200, kv_dtype=kind)
        batch.prefill(0, p)
        logits[kind] = [batch.read_logits(0)]
        for t in forced:
            batch.step([0], [t])
            logits[kind].append(batch.read_logits(0))
        if kind == kv:
            # again beside another sequence: other rows, other cuts of the pages
            batch.prefill(1, p[:77])
            batch.prefill(0, p)
            assert rel_err(batch.read_logits(0), logits[kv][0]) <= 1e-6
            for i, t in enumerate(forced):
                batch.step([1, 0], [3, t])
                # (fp32 sums in another order flip a few codes of later layers)
                assert rel_err(batch.read_logits(1), logits[kv][i + 1]) <= BAR[kv] / 4
        batch.close()
    for a, b in zip(logits[kv], logits["f16"]):
        # a unit is 1/127 (1/8) of a block's largest element: values are off by a share of
        # 0.3 / 60 (0.3 / 4) of their size at most, and so is what the layers make of them
        assert rel_err(a, b) <= (0.02 if kv == "q8" else 0.3), rel_err(a, b)
    loaded.engine.dispose()


def test_coded_batch_refusals(synth):
    w = WORKLOADS["tiny-qwen3"]
    loaded = load_llama_wgsl_model(w.model_def(synth("tiny-qwen3")))
    with pytest.raises(ChonkError, match="unsupported kv_dtype"):
        LlamaWgslBatch(loaded.engine, 2, 20, kv_dtype="q5")
    with pytest.raises(ChonkError, match="needs 1..1024 sequences"):
        LlamaWgslBatch(loaded.engine, 0, 20, kv_dtype="q8")
    batch = LlamaWgslBatch(loaded.engine, 2, 20, kv_dtype="q8")
    with pytest.raises(ChonkError) as ei:
        batch.prefill(0, list(range(21)))
    assert ei.value.status_name == "ECONTEXT"
    with pytest.raises(ChonkError):
        batch.step([0, 0], [1, 2])
    t = batch.prefill(0, list(range(1, 20)))
    t = batch.step([0], [t])[0]
    with pytest.raises(ChonkError) as ei:
        batch.step([0], [t])
    assert ei.value.status_name == "ECONTEXT"
    batch.close()
    loaded.engine.dispose()
