"""Arguments whose 32-bit form would be another value, without a device: caps, and 64-bit lengths, positions and table
entries as the kernels are handed them."""
from __future__ import annotations

import contextlib
import ctypes
from types import SimpleNamespace

import pytest
import torch

from test_dense_refusals import _lib, hostside                       # noqa: F401 (the fixture)


def _decode(kv8, **kw):
    cache = kv8.Kv8Cache.allocate(4, 16, 2, 64, "cpu")
    q = torch.zeros(3, 1, 4, 64, dtype=torch.bfloat16)
    return kv8.kv8_decode_attention(q, cache, torch.zeros(3, 2, dtype=torch.int32), torch.ones(3, dtype=torch.int32),
                                    sm_scale=0.1, **kw)


@pytest.mark.parametrize("cap", [1e39, 1e300, 3e38, 1e-39, 1e-46, 1e-320])
def test_caps_beyond_32_bits(hostside, cap):                         # noqa: F811
    """A cap that rounds to 0 would be none, one that rounds to infinity gives NaN."""
    from semblo_b200 import dense_prefill
    _, kv8 = hostside
    with pytest.raises(ValueError, match="soft cap"):
        _decode(kv8, softcap=cap)
    q, k = torch.zeros(5, 4, 64, dtype=torch.float16), torch.zeros(5, 2, 64, dtype=torch.float16)
    with pytest.raises(ValueError, match="soft cap"):
        dense_prefill.dense_prefill_attention(q, k, k, cu_seqlens_q=torch.tensor([0, 5]), sm_scale=0.1, softcap=cap)


@pytest.mark.parametrize("cap", [3e38, 1e-39])
def test_caps_beyond_the_kernels_range(cap):
    lib, p = _lib(), ctypes.c_void_p(256)
    assert lib.semblo_kv8_decode(p, 0, 1, 1, 2, 1, 64, p, p, 4, 16, p, 4, 4, p, None, 0, 0.1, cap, None, p, None, None, 0, p,
                                 None) == -1 and b"cap" in lib.semblo_last_error()
    assert lib.semblo_dense_prefill(p, 64, 64, p, 64, 64, p, 64, 64, 4, 4, 2, 1, 64, 0, p, p, 1, 1, 0, None, 0.1, cap, None, p,
                                    0, None, p, 0, p, None) == -1 and b"cap" in lib.semblo_last_error()


FAR = [(1 << 32) + 1, 1 << 40, -(1 << 33) + 2, (1 << 31), -(1 << 31) - 1]


def _clamped(x):
    return [max(-(1 << 31), min((1 << 31) - 1, v)) for v in x]


def test_64_bit_values_stay_out_of_range(hostside):                  # noqa: F811
    """A table entry, length or position that does not fit 32 bits must not become another one that does."""
    _, kv8 = hostside
    x = torch.tensor(FAR + [0, 7, -1])
    assert kv8._per_request("lengths", x, len(x)).tolist() == _clamped(x.tolist())
    table = kv8._block_table(x[None], 1)
    assert table.dtype == torch.int32 and table[0].tolist() == _clamped(x.tolist())
    kept = torch.zeros(3, dtype=torch.int32)
    assert kv8._per_request("lengths", kept, 3) is kept


def test_tables_of_other_types(hostside):                            # noqa: F811
    _, kv8 = hostside
    for dtype in (torch.float32, torch.bool, torch.bfloat16):
        with pytest.raises(ValueError, match="block table"):
            kv8._block_table(torch.zeros(1, 2, dtype=dtype), 1)
    assert kv8._block_table(torch.tensor([[3, -1]], dtype=torch.int16), 1).tolist() == [[3, -1]]
