"""Dense requests and dense layers through the operator boundary: rotary positions, attention of the prompt, the
8-bit cache and the attention of generated tokens over it, run together as a layer runs them."""
from __future__ import annotations

from types import SimpleNamespace

import pytest
import torch

import test_gpu_dense_prefill as prompt_ref
import test_gpu_kv8_append as append_ref
import test_gpu_kv8_decode as decode_ref
import test_gpu_rotary as rotary_ref

pytestmark = pytest.mark.gpu

DIM, HQ, HKV, LENGTH, STEPS = 128, 8, 2, 700, 6


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    from semblo_b200 import _lib
    _lib.lib()
    return torch.device("cuda:0")


def _config(**kw):
    from semblo_b200.config import SembloVllmConfig
    return SembloVllmConfig(token_capacity=2048, target_tokens=256, flat_unit_tokens=32, index_dim=DIM,
                            engage_above_tokens=1024, query_chunk_size=1024, **{"dense_cache_bits": 8, **kw})


def _layer(data, state, cfg, index, name, *, source=None, sparse=True, cap=None, window=0, rotary=None):
    from semblo_b200.model import SembloAttention

    class Layer(SembloAttention):
        def __init__(self):
            super().__init__()
            self.num_heads, self.num_kv_heads, self.head_dim = HQ, HKV, DIM
            self.scaling = DIM ** -0.5
            self.is_kv_shared_layer = source is not None
            self.attn = SimpleNamespace(layer_name=name)
            self._init_semblo_runtime(runtime_config=cfg, runtime_state=state, layer_idx=index,
                                      source_layer_idx=index if source is None else source, uses_sparse_attention=sparse,
                                      builds_product_index=sparse and source is None, attention_logits_soft_cap=cap,
                                      attention_window=window, rotary=rotary)

        def _project_qkv(self, positions, hidden_states):
            idx = positions.long()
            q_pre, k_pre, v = (data[n][index, idx] for n in ("q", "k", "v"))
            n = idx.numel()
            q_post, k_post = self._rotate(positions, q_pre.reshape(n, HQ * DIM), k_pre.reshape(n, HKV * DIM))
            if source is not None:
                return q_post, None, None, q_pre, None, None
            return q_post, k_post, v.reshape(n, HKV * DIM), q_pre, k_pre, None

        def _finish_output(self, attn_output, gate):
            return attn_output

    return Layer()


def _data(dev, layers, total):
    gen = torch.Generator(device=dev).manual_seed(77)
    mk = lambda heads, s: (torch.randn(layers, total, heads, DIM, device=dev, generator=gen) * s).to(torch.bfloat16)
    return {"q": mk(HQ, 2.0), "k": mk(HKV, 1.0), "v": mk(HKV, 1.0)}


def _rotated(data, index, freq, total, dev):
    from semblo_b200.rotary import apply_rotary
    pos = torch.arange(total, device=dev)
    q, k = apply_rotary(data["q"][index], data["k"][index], pos, freq)
    want, mag = rotary_ref._turned(data["q"][index], pos, freq, False, False)
    rotary_ref._check(q, want, mag)
    return q, k


def test_dense_request_through_the_layers(dev):
    """Layer 0 is dense (capped, windowed), layer 1 sparse but the request is short, layer 2 shares layer 1's K/V."""
    from semblo_b200 import _lib
    from semblo_b200.rotary import rotary_frequencies
    from semblo_b200.state import SembloRuntimeState
    total = LENGTH + STEPS
    data = _data(dev, 3, total)
    freq = rotary_frequencies(DIM, 500000.0, scaling={"type": "yarn", "factor": 4.0, "original_max_position": 4096},
                              device=dev)
    state = SembloRuntimeState(max_model_len=1500)
    kinds = [dict(cap=5.0, window=200), dict(cap=0.0, window=0), dict(cap=0.0, window=0)]
    layers = [_layer(data, state, _config(), 0, "dense.0", sparse=False, cap=5.0, window=200, rotary=freq),
              _layer(data, state, _config(), 1, "dense.1", rotary=freq),
              _layer(data, state, _config(), 2, "dense.2", source=1, rotary=freq)]
    hidden = torch.zeros(total, 8, dtype=torch.bfloat16, device=dev)
    for request in range(2):                                   # the second request writes the same blocks anew
        positions = torch.arange(LENGTH, device=dev)
        outs = [layer._sparse_layer_forward(positions, hidden[:LENGTH]) for layer in layers]
        assert state.dense_request
        for i, out in enumerate(outs):
            q, _ = _rotated(data, i, freq, total, dev)
            src = min(i, 1)
            _, k = _rotated(data, src, freq, total, dev)
            kw = dict(sm_scale=DIM ** -0.5, softcap=kinds[i]["cap"], window=kinds[i]["window"])
            want = prompt_ref._formula(q[:LENGTH], k[:LENGTH], data["v"][src, :LENGTH], [LENGTH], [LENGTH], **kw)
            prompt_ref._check(SimpleNamespace(output=out.view(LENGTH, HQ, DIM), logsumexp=None), want, LENGTH)
        for s in range(STEPS):
            at = LENGTH + s
            step = [layer._sparse_layer_forward(torch.tensor([at], device=dev), hidden[:1]) for layer in layers]
            for i, out in enumerate(step):
                src = min(i, 1)
                cache, table = state.dense_cache(src, num_kv_heads=HKV, head_dim=DIM, device=dev)
                q, _ = _rotated(data, i, freq, total, dev)
                _, k = _rotated(data, src, freq, total, dev)
                want = decode_ref._formula(q[at].view(1, 1, HQ, DIM), cache, table, [at + 1], DIM ** -0.5, kinds[i]["cap"],
                                           kinds[i]["window"], None, None)
                got = SimpleNamespace(output=out.view(1, 1, HQ, DIM), logsumexp=want[1].float())
                decode_ref._check(got, want, at + 1)
                if i == 1 and s == STEPS - 1:
                    # the stored codes are those of the definition: the prompt at once, then token by token
                    d64 = torch.zeros(2, cache.num_blocks, HKV, 256, DIM, dtype=torch.float64, device=dev)
                    s64 = torch.ones(2, cache.num_blocks, HKV, dtype=torch.float64, device=dev)
                    rows = table.cpu().tolist()
                    append_ref._append_64(d64, s64, k[:LENGTH], data["v"][src, :LENGTH], rows, [0, LENGTH], [0], 256)
                    for t in range(LENGTH, at + 1):
                        append_ref._append_64(d64, s64, k[t:t + 1], data["v"][src, t:t + 1], rows, [0, 1], [t], 256)
                    assert torch.equal(cache.scales[:, :3].double(), s64[:, :3])
                    used = cache.data.double().transpose(2, 3)[:, :3].flatten(1, 2)[:, :at + 1]
                    assert torch.equal(used, d64.transpose(2, 3)[:, :3].flatten(1, 2)[:, :at + 1])
        _lib.status_for(dev).raise_if_set()


def test_long_request_takes_the_sparse_path(dev):
    """Above engage_above_tokens the same layer builds its index, with and without dense_cache_bits the same bytes."""
    from semblo_b200.rotary import rotary_frequencies
    from semblo_b200.state import SembloRuntimeState
    n = 1400
    data = _data(dev, 1, n)
    freq = rotary_frequencies(DIM, device=dev)
    hidden = torch.zeros(n, 8, dtype=torch.bfloat16, device=dev)
    outs = []
    for bits in (0, 8):
        state = SembloRuntimeState(max_model_len=4096)
        layer = _layer(data, state, _config(dense_cache_bits=bits, kmeans_sample_size=1024, flat_min_clusters_log2=5),
                       0, f"sparse.{bits}", rotary=freq)
        outs.append(layer._sparse_layer_forward(torch.arange(n, device=dev), hidden).clone())
        assert not state.dense_request and 0 in state.source_indexes
    assert torch.equal(outs[0], outs[1])


def test_decode_step_of_a_dense_layer_is_capturable(dev):
    from semblo_b200.rotary import rotary_frequencies
    from semblo_b200.state import SembloRuntimeState
    total = LENGTH + STEPS
    data = _data(dev, 1, total)
    freq = rotary_frequencies(DIM, device=dev)
    hidden = torch.zeros(total, 8, dtype=torch.bfloat16, device=dev)

    def fresh(name):
        state = SembloRuntimeState(max_model_len=1024)
        layer = _layer(data, state, _config(), 0, name, sparse=False, rotary=freq)
        layer._sparse_layer_forward(torch.arange(LENGTH, device=dev), hidden[:LENGTH])
        return layer

    eager, recorded = fresh("eager"), fresh("recorded")
    want = [eager._sparse_layer_forward(torch.tensor([LENGTH + s], device=dev), hidden[:1]).clone() for s in range(STEPS)]
    position = torch.tensor([LENGTH], device=dev)
    q, k = _rotated(data, 0, freq, total, dev)
    bufs = [x.clone() for x in (q[:1].view(1, -1), k[:1].view(1, -1), data["v"][0, :1].view(1, -1))]
    out = torch.empty_like(bufs[0])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        recorded.attention_forward(position, hidden[:1], bufs[0], bufs[1], bufs[2], None, None, out)
    for s in range(STEPS):
        at = LENGTH + s
        position.fill_(at)
        for b, x in zip(bufs, (q[at], k[at], data["v"][0, at])):
            b.copy_(x.reshape(1, -1))
        graph.replay()
        assert torch.equal(out, want[s].view(1, -1)), s


def test_refusals_of_the_layer(dev):
    from semblo_b200.rotary import rotary_frequencies
    from semblo_b200.state import SembloRuntimeState
    data = _data(dev, 3, 64)
    freq = rotary_frequencies(DIM, device=dev)
    hidden = torch.zeros(64, 8, dtype=torch.bfloat16, device=dev)
    state = SembloRuntimeState(max_model_len=256)
    for kw in (dict(cap=5.0), dict(window=64), dict(cap=5.0, sparse=False), dict(window=64, sparse=False)):
        bits = 0 if "sparse" in kw else 8
        with pytest.raises(RuntimeError):
            _layer(data, state, _config(dense_cache_bits=bits), 0, "no", rotary=freq, **kw)
    with pytest.raises(ValueError):
        _config(dense_cache_bits=4).validate()
    without = _layer(data, state, _config(dense_cache_bits=0), 0, "without", rotary=freq)
    with pytest.raises(RuntimeError, match="sparse path only"):
        without._sparse_layer_forward(torch.arange(60, device=dev), hidden[:60])
    state = SembloRuntimeState(max_model_len=256)
    layer = _layer(data, state, _config(), 0, "with", sparse=False, rotary=freq)
    with pytest.raises(RuntimeError, match="one call"):
        layer._sparse_layer_forward(torch.arange(8, 60, device=dev), hidden[:52])
    shared = _layer(data, state, _config(), 2, "shared", source=1, sparse=False, rotary=freq)
    with pytest.raises(RuntimeError, match="has not seen"):
        shared._sparse_layer_forward(torch.arange(60, device=dev), hidden[:60])
    bare = _layer(data, state, _config(), 1, "bare", sparse=False)
    with pytest.raises(RuntimeError, match="rotary"):
        bare._sparse_layer_forward(torch.arange(60, device=dev), hidden[:60])
