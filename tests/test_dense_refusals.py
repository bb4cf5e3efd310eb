"""What the dense-request operators refuse, checked without a device: the Python checks with the device test
taken out, and the C entries' own validation (which returns before any CUDA call)."""
from __future__ import annotations

import ctypes
import math

import pytest
import torch

LIB_CODES = (-1,)


def _lib():
    from semblo_b200 import _lib
    if not _lib.library_path().exists():
        pytest.skip("library not built")
    return _lib.lib()


@pytest.fixture
def hostside(monkeypatch):
    """The operators' modules with the CUDA check removed and the library replaced: reaching it is a failure."""
    from semblo_b200 import dense_prefill, kv8_cache, rotary

    def reached(*_):
        raise AssertionError("the call was not refused")

    for m in (rotary, kv8_cache, dense_prefill):
        monkeypatch.setattr(m, "require_cuda", lambda *_: None)
        monkeypatch.setattr(m, "lib", reached)
    return rotary, kv8_cache


def test_cpu_tensors_are_refused():
    from semblo_b200.rotary import apply_rotary, rotary_frequencies
    from semblo_b200.kv8_cache import Kv8Cache, kv8_append
    freq = rotary_frequencies(64, device="cpu")
    with pytest.raises(RuntimeError, match="CUDA"):
        apply_rotary(torch.zeros(2, 1, 64), None, torch.zeros(2, dtype=torch.int64), freq)
    cache = Kv8Cache.allocate(2, 16, 1, 64, "cpu")
    x = torch.zeros(1, 1, 64, dtype=torch.bfloat16)
    one = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="CUDA"):
        kv8_append(cache, x, x, torch.zeros(1, 1, dtype=torch.int32), torch.tensor([0, 1]), one)


def test_rotary_frequencies_values():
    from semblo_b200.rotary import rotary_frequencies
    f = rotary_frequencies(8, 10000.0, device="cpu")
    want = torch.tensor([10000.0 ** (-2 * i / 8) for i in range(4)], dtype=torch.float64)
    assert torch.allclose(f.inv_freq, want, rtol=1e-15, atol=0) and f.attention_scale == 1.0
    assert torch.allclose(rotary_frequencies(8, scaling={"type": "linear", "factor": 4.0}, device="cpu").inv_freq,
                          want / 4, rtol=1e-15, atol=0)
    ntk = rotary_frequencies(8, scaling={"type": "ntk", "factor": 4.0}, device="cpu").inv_freq
    assert float(ntk[0]) == 1.0 and math.isclose(float(ntk[3]), float(want[3]) / 4, rel_tol=1e-14)
    # turns within 1024 positions at base 100, R = 8: 163, 51.5, 16.3, 5.15
    w = rotary_frequencies(8, 100.0, scaling={"type": "wavelength", "factor": 2.0, "original_max_position": 1024,
                                              "low_freq_factor": 10.0, "high_freq_factor": 100.0}, device="cpu").inv_freq
    base = [100.0 ** (-2 * i / 8) for i in range(4)]
    for i, b in enumerate(base):
        turns = 1024 * b / (2 * math.pi)
        keep = min(1.0, max(0.0, (turns - 10.0) / 90.0))
        assert math.isclose(float(w[i]), b * (keep + (1 - keep) / 2), rel_tol=1e-14)
    assert float(w[0]) == base[0] and math.isclose(float(w[3]), base[3] / 2, rel_tol=1e-14)
    y = rotary_frequencies(64, 10000.0, scaling={"type": "yarn", "factor": 8.0, "original_max_position": 4096},
                           device="cpu")
    plain = [10000.0 ** (-2 * i / 64) for i in range(32)]
    lo = math.floor(64 * math.log(4096 / (32 * 2 * math.pi)) / (2 * math.log(10000.0)))
    hi = math.ceil(64 * math.log(4096 / (2 * math.pi)) / (2 * math.log(10000.0)))
    assert (lo, hi) == (10, 23)
    for i, b in enumerate(plain):
        r = min(1.0, max(0.0, (i - lo) / (hi - lo)))
        assert math.isclose(float(y.inv_freq[i]), b * (1 - r) + b / 8 * r, rel_tol=1e-14)
    assert math.isclose(y.attention_scale, 0.1 * math.log(8.0) + 1.0)


@pytest.mark.parametrize("args,kwargs", [
    ((7,), {}), ((0,), {}), ((8, 1.0), {}), ((8,), {"scaling": {"type": "spiral", "factor": 2.0}}),
    ((8,), {"scaling": {"factor": 2.0}}), ((8,), {"scaling": {"type": "linear"}}),
    ((8,), {"scaling": {"type": "linear", "factor": 0.5}}), ((8,), {"scaling": {"type": "ntk", "factor": 2.0, "turns": 1}}),
    ((8,), {"scaling": {"type": "yarn", "factor": 2.0}}),
    ((8,), {"scaling": {"type": "yarn", "factor": 2.0, "original_max_position": 64, "beta_fast": 1.0, "beta_slow": 2.0}}),
    ((8,), {"scaling": {"type": "wavelength", "factor": 2.0, "original_max_position": 64, "low_freq_factor": 4.0,
                        "high_freq_factor": 1.0}}),
])
def test_rotary_frequencies_refusals(args, kwargs):
    from semblo_b200.rotary import rotary_frequencies
    with pytest.raises(ValueError):
        rotary_frequencies(*args, device="cpu", **kwargs)


def test_rotary_refusals(hostside):
    rotary, _ = hostside
    freq = rotary.rotary_frequencies(64, device="cpu")
    q, k, pos = torch.zeros(4, 2, 64), torch.zeros(4, 1, 64), torch.arange(4)

    def no(exc, *a, **kw):
        with pytest.raises(exc):
            rotary.apply_rotary(*a, **kw)

    no(ValueError, q[0], k, pos, freq)
    no(ValueError, q, k[:3], pos, freq)
    no(ValueError, q, torch.zeros(4, 1, 32), pos, freq)
    no(ValueError, q, k.double(), pos, freq)
    no(ValueError, q.double(), k.double(), pos, freq)
    no(ValueError, q, k, pos[:3], freq)
    no(ValueError, q, k, pos.float(), freq)
    no(ValueError, q, k, pos[:, None], freq)
    no(ValueError, q, k, pos, rotary.rotary_frequencies(66, device="cpu"))
    no(ValueError, torch.zeros(4, 64, 2).transpose(1, 2), k, pos, freq)
    no(ValueError, q, k, pos, freq, q_out=torch.zeros(4, 2, 32))
    no(ValueError, q, k, pos, freq, q_out=q.bfloat16())
    no(ValueError, q, None, pos, freq, k_out=k)
    buf = torch.zeros(5, 2, 64)
    no(ValueError, buf[:4], None, pos, freq, q_out=buf[1:])
    no(ValueError, q, None, pos, freq, q_out=torch.zeros(1, 2, 64).expand(4, 2, 64))
    no(RuntimeError, q.clone().requires_grad_(), k, pos, freq)
    with pytest.raises(ValueError):
        rotary.RotaryFrequencies(torch.zeros(4))
    no(ValueError, q, k, pos, rotary.RotaryFrequencies(torch.zeros(4, dtype=torch.float64, device="meta")))


def test_kv8_cache_and_append_refusals(hostside):
    _, kv8 = hostside
    for bad in ((2, 24, 1, 64), (2, 8, 1, 64), (2, 512, 1, 64), (2, 16, 1, 96)):
        with pytest.raises(ValueError):
            kv8.Kv8Cache.allocate(*bad, "cpu")
    good = kv8.Kv8Cache.allocate(4, 16, 2, 64, "cpu")
    with pytest.raises(ValueError):
        kv8.Kv8Cache(good.data.view(torch.uint8), good.scales)
    with pytest.raises(ValueError):
        kv8.Kv8Cache(good.data, good.scales[:, :3])
    with pytest.raises(ValueError):
        kv8.Kv8Cache(good.data, good.scales.double())
    with pytest.raises(ValueError):
        kv8.Kv8Cache(good.data.transpose(1, 2), good.scales)
    x = torch.zeros(3, 2, 64, dtype=torch.bfloat16)
    table, cu, start = torch.zeros(1, 2, dtype=torch.int32), torch.tensor([0, 3]), torch.tensor([0])

    def no(exc, *a):
        with pytest.raises(exc):
            kv8.kv8_append(good, *a)

    no(ValueError, x[:, :1], x[:, :1], table, cu, start)
    no(ValueError, x, x[:2], table, cu, start)
    no(ValueError, x, x.half(), table, cu, start)
    no(ValueError, x.float(), x.float(), table, cu, start)
    no(ValueError, x, x, table[0], cu, start)
    no(ValueError, x, x, table.expand(2, 2), cu, start)
    no(ValueError, x, x, table, cu[None], start)
    no(ValueError, x, x, table, cu.float(), start)
    no(ValueError, x, x, table, cu, torch.tensor([0, 1]))
    no(ValueError, x, x, table, torch.empty(0, dtype=torch.int32), start)
    no(RuntimeError, x.clone().requires_grad_(), x, table, cu, start)
    no(ValueError, x, x, table.to("meta"), cu, start)


def test_decode_refusals(hostside):
    _, kv8 = hostside
    cache = kv8.Kv8Cache.allocate(4, 16, 2, 64, "cpu")
    q = torch.zeros(3, 1, 4, 64, dtype=torch.bfloat16)
    table, lens = torch.zeros(3, 2, dtype=torch.int32), torch.ones(3, dtype=torch.int32)

    def no(exc, q=q, table=table, lens=lens, **kw):
        with pytest.raises(exc):
            kv8.kv8_decode_attention(q, cache, table, lens, **{"sm_scale": 0.1, **kw})

    no(ValueError, q=q[0])
    no(ValueError, q=q.float())
    no(ValueError, q=torch.zeros(3, 1, 4, 128, dtype=torch.bfloat16))
    no(ValueError, q=torch.zeros(3, 1, 3, 64, dtype=torch.bfloat16))
    no(ValueError, q=torch.zeros(3, 1, 0, 64, dtype=torch.bfloat16))
    no(ValueError, q=torch.zeros(3, 17, 4, 64, dtype=torch.bfloat16))
    no(ValueError, q=torch.zeros(3, 0, 4, 64, dtype=torch.bfloat16))
    no(ValueError, table=table[:2])
    no(ValueError, table=table[0])
    no(ValueError, lens=lens[:2])
    no(ValueError, lens=lens.float())
    no(ValueError, lens=lens.to("meta"))
    no(ValueError, window=-1)
    no(ValueError, softcap=-1.0)
    no(ValueError, softcap=math.inf)
    no(ValueError, softcap=math.nan)
    no(ValueError, prefix_lens=lens[:2])
    no(ValueError, prefix_lens=lens.to("meta"))
    no(ValueError, alibi_slopes=torch.zeros(3))
    no(ValueError, alibi_slopes=torch.zeros(4, dtype=torch.float64))
    no(ValueError, out=torch.zeros(3, 1, 4, 64))
    no(ValueError, out=torch.zeros(3, 1, 64, 4, dtype=torch.bfloat16).transpose(2, 3))
    no(ValueError, out=q)
    no(ValueError, out=torch.zeros(769, dtype=torch.bfloat16)[1:].view(3, 1, 4, 64))
    no(ValueError, out=cache.data.view(torch.bfloat16).view(-1)[:768].view(3, 1, 4, 64))
    no(RuntimeError, out=torch.zeros_like(q).requires_grad_())
    no(RuntimeError, q=q.clone().requires_grad_())


def test_dense_prefill_refusals(hostside):
    from semblo_b200 import dense_prefill
    q, k = torch.zeros(5, 4, 64, dtype=torch.float16), torch.zeros(7, 2, 64, dtype=torch.float16)
    cu = torch.tensor([0, 5], dtype=torch.int32)

    def no(exc, q=q, k=k, v=None, **kw):
        with pytest.raises(exc):
            dense_prefill.dense_prefill_attention(q, k, k if v is None else v,
                                                  **{"cu_seqlens_q": cu, "sm_scale": 0.1, **kw})

    no(ValueError, q=q[0])
    no(ValueError, v=k[:6])
    no(ValueError, q=q.float())
    no(ValueError, k=k.bfloat16())
    no(ValueError, v=k.bfloat16())
    no(ValueError, q=torch.zeros(5, 4, 128, dtype=torch.float16))
    no(ValueError, q=torch.zeros(5, 4, 96, dtype=torch.float16), k=torch.zeros(7, 2, 96, dtype=torch.float16))
    no(ValueError, q=torch.zeros(5, 3, 64, dtype=torch.float16))
    no(ValueError, q=torch.zeros(5, 258, 64, dtype=torch.float16))
    no(ValueError, cu_seqlens_q=cu[None])
    no(ValueError, cu_seqlens_q=cu.float())
    no(ValueError, cu_seqlens_q=cu[:0])
    no(ValueError, cu_seqlens_q=cu.to("meta"))
    no(ValueError, cu_seqlens_k=torch.tensor([0, 5, 7]))
    no(ValueError, cu_seqlens_k=cu.to("meta"))
    no(ValueError, sm_scale=0.0)
    no(ValueError, sm_scale=-1.0)
    no(ValueError, sm_scale=math.nan)
    no(ValueError, window=-2)
    no(ValueError, softcap=-2.0)
    no(ValueError, causal=False, window=3)
    no(ValueError, causal=False, prefix_lens=torch.tensor([1]))
    no(ValueError, prefix_lens=torch.tensor([1, 2]))
    no(ValueError, alibi_slopes=torch.zeros(2))
    no(ValueError, out=torch.zeros(5, 4, 64))
    no(ValueError, out=torch.zeros(6, 4, 64, dtype=torch.float16)[:5, :, ::1].transpose(0, 1))
    no(ValueError, out=q)
    big = torch.zeros(20, 2, 64, dtype=torch.float16)
    no(ValueError, k=big[:7], v=big[12:19], out=big[2:12].view(5, 4, 64))
    no(ValueError, k=big[:7], v=big[12:19], out=big[9:19].view(5, 4, 64))
    no(RuntimeError, out=torch.zeros_like(q).requires_grad_())
    no(RuntimeError, k=k.clone().requires_grad_())


def test_token_rows_are_copied_where_a_kernel_cannot_read_them():
    from semblo_b200.kv8_cache import _token_rows
    x = torch.zeros(6, 4, 64, dtype=torch.bfloat16)
    assert _token_rows(x) is x and _token_rows(x[:, 1:3]).data_ptr() == x[:, 1:3].data_ptr()
    for y in (torch.zeros(6, 4, 65, dtype=torch.bfloat16)[..., 1:], x.transpose(1, 2).contiguous().transpose(1, 2),
              x[:1].expand(6, 4, 64), x[:, :1].expand(6, 4, 64)):
        z = _token_rows(y)
        assert z.is_contiguous() and z.shape == y.shape and z.data_ptr() != y.data_ptr()


def test_c_entries_refuse():
    lib = _lib()
    p = ctypes.c_void_p(256)

    def rotary(tokens=1, heads=1, rot=64, dim=64, code=0, k=None, k_out=None, q=p, pos=p, freq=p):
        return lib.semblo_rotary(q, 64, 64, p, 64, 64, heads, k, 0, 0, k_out, 0, 0, 0, tokens, dim, rot, code, pos, 1, freq,
                                 1.0, 0, 0, None)

    assert rotary(tokens=0) == 0
    assert rotary(rot=65) == -1 and rotary(rot=66) == -1 and rotary(heads=0) == -1 and rotary(tokens=-1) == -1
    assert rotary(k=p) == -1 and rotary(q=None) == -1 and rotary(pos=None) == -1 and rotary(freq=None) == -1
    assert rotary(code=9) == -1 and b"dtype" in lib.semblo_last_error()

    def append(tokens=1, code=0, block=16, dim=64, heads=1, k=p, cache=p, stride=64, table=p, batch=1, status=p):
        return lib.semblo_kv8_append(k, stride, 64, p, 64, 64, tokens, code, cache, p, 4, block, heads, dim, table, 1, 1, p, p,
                                     batch, status, None)

    assert append(tokens=0) == 0 and append(batch=0) == 0
    for kw in (dict(block=24), dict(block=8), dict(block=512), dict(dim=96), dict(heads=0), dict(k=None), dict(cache=None),
               dict(k=ctypes.c_void_p(264)), dict(stride=60), dict(table=None), dict(status=None), dict(code=1),
               dict(tokens=-1)):
        assert append(**kw) == -1, kw

    def decode(dtype=0, batch=1, queries=1, hq=2, hkv=1, dim=64, block=16, width=4, q=p, cache=p, softcap=0.0, window=0,
               ws=None, nbytes=0):
        return lib.semblo_kv8_decode(q, dtype, batch, queries, hq, hkv, dim, cache, p, 4, block, p, width, width, p, None,
                                     window, 0.1, softcap, None, p, None, ws, nbytes, p, None)

    assert decode(batch=0) == 0
    for kw in (dict(dtype=1), dict(queries=0), dict(queries=17), dict(hq=3, hkv=2), dict(hq=0), dict(dim=96), dict(block=8),
               dict(q=None), dict(cache=None), dict(q=ctypes.c_void_p(264)), dict(softcap=-1.0), dict(window=-1),
               dict(batch=5000), dict(batch=-1), dict(batch=4096, hkv=8, hq=8, width=1 << 20)):
        assert decode(**kw) == -1, kw
    long_table = dict(width=4096)                                # a workspace is needed, and none is given
    assert lib.semblo_kv8_decode_workspace_bytes(1, 1, 2, 1, 64, 16, 4096, 0, 0) > 0
    assert decode(**long_table) == -3
    assert lib.semblo_kv8_decode_workspace_bytes(1, 1, 2, 1, 64, 16, 4, 0, 0) == 0
    assert lib.semblo_kv8_decode_workspace_bytes(1, 1, 2, 1, 64, 16, 4096, 100, 0) == 0       # a window bounds the work
    assert lib.semblo_kv8_decode_workspace_bytes(1, 1, 3, 2, 64, 16, 4096, 0, 0) == -1

    def prefill(q=p, k=p, v=p, tq=4, tk=4, hq=2, hkv=1, dim=64, dtype=0, cu=p, docs=1, causal=1, window=0, prefix=None,
                sm=0.1, cap=0.0, out=p, stride=64, status=p, room=0):
        return lib.semblo_dense_prefill(q, stride, 64, k, 64, 64, v, 64, 64, tq, tk, hq, hkv, dim, dtype, cu, cu, docs, causal,
                                        window, prefix, sm, cap, None, out, 0, None, p, room, status, None)

    assert prefill(tq=0) == 0 and prefill(docs=0) == 0
    sizes = lib.semblo_dense_prefill_workspace_bytes
    assert sizes(4, 4, 2, 1, 64, 1, 1, 0, 0) == 0 and sizes(100000, 100000, 32, 8, 64, 1, 1, 0, 0) == 0
    need = sizes(4, 4096, 2, 1, 64, 1, 1, 0, 0)                  # a few queries over many keys
    assert need > 0 and sizes(4, 4096, 2, 1, 64, 1, 1, 100, 0) == 0
    assert prefill(tk=4096, room=need - 1) == -3
    assert sizes(4, 4096, 3, 2, 64, 1, 1, 0, 0) == -1
    for kw in (dict(dim=80), dict(hq=3, hkv=2), dict(hq=129), dict(dtype=1), dict(tq=-1), dict(window=-1), dict(cap=-1.0),
               dict(sm=0.0), dict(causal=0, window=4), dict(causal=0, prefix=p), dict(q=None), dict(k=None), dict(out=None),
               dict(cu=None), dict(status=None), dict(q=ctypes.c_void_p(264)), dict(stride=60)):
        assert prefill(**kw) == -1, kw
