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


@pytest.fixture
def operators(monkeypatch):
    """The operators replaced: what each call was given, in order."""
    from semblo_b200 import model
    calls = []
    monkeypatch.delenv("SEMBLO_FULL_GRAPH_DECODE", raising=False)
    monkeypatch.setattr(model, "kv8_append", lambda cache, k, v, table, cu, start: calls.append(("append", k)))
    monkeypatch.setattr(model, "dense_prefill_attention", lambda q, k, v, **kw: calls.append(("prompt", k)))
    monkeypatch.setattr(model, "kv8_decode_attention", lambda q, cache, *a, **kw: calls.append(("decode", cache)))
    monkeypatch.setattr(model._lib, "status_for", lambda device: SimpleNamespace(poll=lambda: None))
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    monkeypatch.setattr(model.SembloAttention, "_windows_ahead_enabled", lambda *a: True)
    monkeypatch.setattr(model.SembloAttention, "_prompt_with_windows_ahead", lambda *a: calls.append(("sparse", None)))
    return calls


def _run(layer, positions):
    n = positions.numel()
    q = torch.zeros(n, HQ * DIM)
    kv = None if layer.is_kv_shared_layer else torch.zeros(n, HKV * DIM)
    layer.attention_forward(positions, None, q, kv, kv, None, None, q)


def test_a_prompt_that_no_layer_shares_is_not_kept(operators):
    state = _state()
    dense, sparse = _layer(state, 0, sparse=False), _layer(state, 1)
    for layer in (dense, sparse):
        _run(layer, torch.arange(40))
    assert [c[0] for c in operators] == ["append", "prompt"] * 2 and not state.dense_prompt_kv


def test_a_shared_prompt_is_kept_until_its_last_reader(operators):
    """Layer 0 runs before the layer that begins the prompt, layer 1 begins it."""
    state = _state()
    layers = [_layer(state, 0, sparse=False), _layer(state, 1), _layer(state, 2, source=0, sparse=False),
              _layer(state, 3, source=1), _layer(state, 4, source=1)]
    for _ in range(2):
        held = []
        for layer in layers:
            _run(layer, torch.arange(40))
            held.append(sorted(state.dense_prompt_kv))
        assert held == [[0], [0, 1], [1], [1], []]
        assert operators[4][1] is operators[1][1] and operators[5][1] is operators[3][1] and operators[6][1] is operators[3][1]
        operators.clear()


@pytest.mark.parametrize("sparse", [True, False])
def test_a_shared_prompt_does_not_outlive_its_request(operators, sparse):
    """A request that ends before the reader ran, then one whose source layer takes the sparse path."""
    state = _state()
    source, reader = _layer(state, 1), _layer(state, 2, source=1, sparse=sparse)
    _run(source, torch.arange(40))
    _run(source, torch.arange(200))
    assert operators[-1][0] == "sparse" and not state.dense_prompt_kv
    if not sparse:
        operators.clear()
        with pytest.raises(RuntimeError):
            _run(reader, torch.arange(200))
        assert not operators


def test_a_dense_layer_does_not_read_what_its_sparse_source_did_not_write(operators):
    """A request on the sparse path leaves nothing in its source layer's 8-bit cache: what is there is another's."""
    state = _state()
    source, reader = _layer(state, 1), _layer(state, 2, source=1, sparse=False)
    for layer in (source, reader):                                             # a short request fills the cache
        _run(layer, torch.arange(40))
    for layer in (source, reader):
        _run(layer, torch.tensor([40]))
    assert [c[0] for c in operators] == ["append", "prompt", "prompt", "append", "decode", "decode"]
    _run(source, torch.arange(200))
    operators.clear()
    for positions in (torch.arange(200), torch.tensor([200])):
        with pytest.raises(RuntimeError, match="sparse path"):
            _run(reader, positions)
    assert not operators


def test_a_refused_piece_of_a_prompt_writes_nothing(operators):
    layer = _layer(_state(), 0, sparse=False)
    with pytest.raises(RuntimeError, match="one call"):
        _run(layer, torch.arange(8, 48))
    assert not operators


def test_a_reader_without_its_source_writes_nothing(operators):
    layer = _layer(_state(), 2, source=1, sparse=False)
    with pytest.raises(RuntimeError, match="has not seen"):
        _run(layer, torch.arange(40))
    assert not operators


def test_the_cache_is_not_made_while_a_step_is_recorded(operators, monkeypatch):
    """Its memory and its first fill would become part of the recording: every replay would empty it."""
    state = _state()
    layer = _layer(state, 0, sparse=False)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    with pytest.raises(RuntimeError, match="before"):
        _run(layer, torch.tensor([3]))
    assert not operators and not state.index_buffers
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    _run(layer, torch.arange(40))
    operators.clear()
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    _run(layer, torch.tensor([40]))
    assert [c[0] for c in operators] == ["append", "decode"]
