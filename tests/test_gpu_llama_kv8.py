"""The Llama runner on 8-bit KV states, against the CPU restatement of the
graph with the same states: the reference's tiny F32 models, decoded token by
token. The bound: both sides' projections differ
in their last bits, so a K or V value that lies next to half a step may be
rounded the other way. Rounding every value (up to half a step each) moves
these logits by 2.6e-3 to 1.4e-2 of the largest, as the CPU test below sees;
a few values off by a whole step move them by less than 2e-3."""
from __future__ import annotations

import numpy as np
import pytest

import llama_host
from kv8_util import attend64, values
from synapse_amd.llama import DeviceLlama
from test_llama_golden import MODELS, _load


class _States:
    """binding's cache calls, on rows as an 8-bit state holds them."""

    def new_cache(self, max_ctx, n_kv, hd):
        return [], (n_kv, hd)

    def attention_rows(self, q, k, v, pos, rows, shape, n_heads, scale):
        assert len(rows) == pos
        rows.append([values(x.reshape(shape)) for x in (k, v)])
        ks, vs = (np.stack(x) for x in zip(*rows))
        return attend64(q, ks, vs, n_heads, scale, np.ones((1, pos + 1), bool))[0].astype(np.float32)

    def __getattr__(self, name):
        return getattr(self.real, name)


def _host_logits(monkeypatch, model, tokens):
    states = _States()
    states.real = llama_host.orc
    monkeypatch.setattr(llama_host, "orc", states)
    return llama_host.decode_logits(model, tokens)


@pytest.mark.parametrize("name", MODELS)
def test_cpu_states_in_eight_bits_stay_near_the_golden_logits(monkeypatch, name):
    """What 8-bit states cost these models (heads of 16: a step is up to a
    127th of the largest of 16 values): a few percent, and not nothing."""
    model, tokens, ref = _load(name)
    got = _host_logits(monkeypatch, model, tokens)
    off = np.linalg.norm(got - ref, axis=1) / np.linalg.norm(ref, axis=1)
    assert off[0] < 0.05 and 1e-4 < off.max() < 0.05


@pytest.mark.gpu
@pytest.mark.parametrize("name", MODELS)
def test_gpu_decode(monkeypatch, name):
    model, tokens, _ = _load(name)
    want = _host_logits(monkeypatch, model, tokens)
    llama = DeviceLlama(model, 32, kv8=True)
    try:
        for _ in range(2):  # twice: reset() starts a new sequence
            got = np.stack([llama.step(t, pos) for pos, t in enumerate(tokens)])
            assert max(e for e, _ in llama_host.compare(got, want)) < 2e-3
            llama.reset()
    finally:
        llama.close()
