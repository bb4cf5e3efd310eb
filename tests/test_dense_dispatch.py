"""Which path the layer body gives a request to and what it keeps between calls, without a device: the layer's own
bookkeeping runs, the operators behind it are replaced by recorders."""
from __future__ import annotations

from types import SimpleNamespace

import pytest
import torch

DIM, HQ, HKV = 64, 4, 2


def _config(**kw):
    from semblo_b200.config import SembloVllmConfig
    return SembloVllmConfig(**{**dict(token_capacity=2048, target_tokens=256, flat_unit_tokens=32, index_dim=DIM,
                                      engage_above_tokens=100, dense_cache_bits=8), **kw})


def _state(max_model_len=512):
    from semblo_b200.state import SembloRuntimeState
    return SembloRuntimeState(max_model_len=max_model_len)


def _layer(state, index, *, source=None, sparse=True, config=None):
    from semblo_b200.model import SembloAttention

    class Layer(SembloAttention):
        def __init__(self):
            super().__init__()
            self.num_heads, self.num_kv_heads, self.head_dim = HQ, HKV, DIM
            self.scaling = DIM ** -0.5
            self.is_kv_shared_layer = source is not None
            self._init_semblo_runtime(runtime_config=config or _config(), runtime_state=state, layer_idx=index,
                                      source_layer_idx=index if source is None else source, uses_sparse_attention=sparse,
                                      builds_product_index=sparse and source is None)

    return Layer()


@pytest.mark.parametrize("source", [None, 0])
def test_a_recorded_step_and_dense_requests_exclude_each_other(monkeypatch, source):
    """Under the recorded decode step every request has to engage the index: a short request's prompt would go to the
    8-bit cache and its generated tokens to the arena, which never saw it."""
    monkeypatch.setenv("SEMBLO_FULL_GRAPH_DECODE", "1")
    state = _state()
    with pytest.raises(RuntimeError, match="engage_above_tokens"):
        _layer(state, 3, source=source)
    _layer(state, 3, source=source, config=_config(engage_above_tokens=0))      # every request engages the index
    _layer(state, 3, source=source, config=_config(dense_cache_bits=0))         # short requests raise as they did
    _layer(state, 3, source=source, sparse=False)                               # a dense layer has no other path


def test_the_variable_set_after_the_layer_was_made(monkeypatch):
    monkeypatch.delenv("SEMBLO_FULL_GRAPH_DECODE", raising=False)
    layer = _layer(_state(), 0)
    taken = []
    monkeypatch.setattr(layer, "_dense_attention", lambda *a: taken.append("dense"))
    monkeypatch.setattr(layer, "_full_graph_decode_step", lambda *a, **k: taken.append("arena"))
    prompt, token = torch.arange(40), torch.tensor([40])
    q = torch.zeros(40, HQ * DIM)
    layer.attention_forward(prompt, None, q, None, None, None, None, q)
    layer.attention_forward(token, None, q[:1], None, None, None, None, q[:1])
    assert taken == ["dense", "dense"]
    monkeypatch.setenv("SEMBLO_FULL_GRAPH_DECODE", "1")
    for positions in (prompt, token):
        with pytest.raises(RuntimeError, match="engage_above_tokens"):
            layer.attention_forward(positions, None, q, None, None, None, None, q)
    assert taken == ["dense", "dense"]
