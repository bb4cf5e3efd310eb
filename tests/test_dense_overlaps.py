"""Outputs that share memory with an input or with each other: refused unless no element is shared, as in the slices of
one fused buffer.  Without a device, against the elements counted one by one."""
from __future__ import annotations

import contextlib
import ctypes
import itertools
import random
from types import SimpleNamespace

import pytest
import torch

from test_dense_refusals import _lib, hostside                       # noqa: F401 (the fixture)


def _elements(x):
    at = x.data_ptr()
    size = x.element_size()
    return {at + sum(i * s for i, s in zip(idx, x.stride())) * size
            for idx in itertools.product(*(range(n) for n in x.shape))}


def _views(rng):
    """Two views [T, heads, D] of one buffer as layers make them: head slices, token ranges, heads first, every other head
    or token."""
    t, h, d = rng.choice([1, 2, 5]), rng.choice([4, 6]), rng.choice([2, 3])
    flat = torch.zeros(2 * t * h * d + 7, dtype=torch.bfloat16)
    out = []
    for _ in range(2):
        off = rng.choice([0, 0, d, 1, h * d, t * h * d])
        x = flat[off:off + t * h * d].view(t, h, d)
        kind = rng.randrange(5)
        if kind == 0:
            a = rng.randrange(h)
            x = x[:, a:a + rng.randint(1, h - a)]
        elif kind == 1:
            x = x[rng.randrange(t):]
        elif kind == 2:
            x = flat[off:off + t * h * d].view(h, t, d).transpose(0, 1)
        elif kind == 3:
            x = x[:, rng.randrange(2)::2]
        else:
            x = x[rng.randrange(min(t, 2))::2]
        out.append(x)
    tokens = min(len(x) for x in out)
    return [x[:tokens] for x in out]


NO_TYPE = 9            # looked at after the overlaps and refused, so that nothing is ever launched


def _rotary(q, q_out, k, k_out):
    """The C entry's answer: b"dtype" where it found nothing to say about the memory."""
    lib, far = _lib(), ctypes.c_void_p(1 << 50)
    rows = lambda x: (x.data_ptr(), x.stride(0), x.stride(1))
    keys = (None, 0, 0, None, 0, 0, 0) if k is None else (*rows(k), *rows(k_out), k.shape[1])
    assert lib.semblo_rotary(*rows(q), *rows(q_out), q.shape[1], *keys, q.shape[0], q.shape[2], 2, NO_TYPE, far, 1, far, 1.0, 0,
                             0, None) == -1
    return lib.semblo_last_error()


def _fresh(x):
    return torch.zeros_like(x, memory_format=torch.contiguous_format)


def _shares(a, b):
    """a as the queries' output, b as the keys' input; and the other way round."""
    said = [b"overlap" in _rotary(_fresh(a), a, b, _fresh(b)), b"overlap" in _rotary(_fresh(b), b, a, _fresh(a)),
            b"overlap" in _rotary(a, _fresh(a), _fresh(b), b), b"overlap" in _rotary(_fresh(a), a, _fresh(b), b)]
    assert len(set(said)) == 1
    return said[0]


def test_shared_elements():
    rng, told = random.Random(1), 0
    for _ in range(1500):
        a, b = _views(rng)
        shared = bool(_elements(a) & _elements(b))
        found = _shares(a, b)
        assert found or not shared
        told += not shared and not found
    assert told > 200                                                # and disjoint views are told apart
    # the layouts that layers have, told apart exactly
    qkv = torch.zeros(7, 12, 16, dtype=torch.bfloat16)
    assert not _shares(qkv[:, :8], qkv[:, 8:10]) and not _shares(qkv[:, 8:10], qkv[:, 10:]) and _shares(qkv[:, :8], qkv[:, 7:9])
    grouped = torch.zeros(7, 2, 6, 16, dtype=torch.bfloat16)         # per KV head: its queries, K and V
    assert not _shares(grouped[:, :, 4], grouped[:, :, 5]) and not _shares(grouped[:, :, 0], grouped[:, :, 5])
    first = torch.zeros(12, 7, 16, dtype=torch.bfloat16).transpose(0, 1)                   # heads first
    assert not _shares(first[:, :8], first[:, 8:10]) and _shares(first[:, :8], first[:, 7:])
    assert not _shares(qkv[:3], qkv[3:6]) and _shares(qkv[:4], qkv[3:7])


def test_outputs_in_place_over_their_input_and_over_themselves():
    qkv, pool = torch.zeros(4, 12, 64, dtype=torch.bfloat16), torch.zeros(4000, dtype=torch.bfloat16)
    q, k = qkv[:, :8], qkv[:, 8:10]
    assert b"dtype" in _rotary(q, q, k, k) and b"dtype" in _rotary(q, q, None, None)
    assert b"dtype" in _rotary(q, q, k, _fresh(k)) and b"dtype" in _rotary(q, _fresh(q), k, k)
    assert b"overlap" in _rotary(q, qkv[:, 1:9], None, None) and b"overlap" in _rotary(k, qkv[:, 9:11], None, None)
    assert b"overlap" in _rotary(q, q, k, qkv[:, 7:9]) and b"overlap" in _rotary(q, qkv[:, 2:10], k, k)
    for strides in ((64, 64, 1), (512, 32, 1), (0, 64, 1), (256, 64, 1)):
        said = _rotary(_fresh(q), pool.as_strided((4, 8, 64), strides), None, None)
        assert b"repeat" in said, strides
    lib, p = _lib(), ctypes.c_void_p(1 << 40)
    assert lib.semblo_rotary(p, -64, 64, p, 64, 64, 2, None, 0, 0, None, 0, 0, 0, 4, 64, 2, NO_TYPE, p, 1, p, 1.0, 0, 0, None) == -1
    assert b"negative" in lib.semblo_last_error()


def test_rotary_outputs(hostside, monkeypatch):                      # noqa: F811
    """The same through the Python entry, which hands the library a type that it refuses."""
    rotary, _ = hostside
    freq, pos = rotary.rotary_frequencies(64, device="cpu"), torch.arange(4)
    monkeypatch.setattr(rotary, "device_scope", lambda device: contextlib.nullcontext())
    monkeypatch.setattr(rotary, "raw_stream", lambda index: None)
    monkeypatch.setattr(rotary, "dtype_code", lambda *_: NO_TYPE)
    monkeypatch.setattr(rotary, "lib", _lib)
    qkv = torch.zeros(4, 12, 64, dtype=torch.bfloat16)
    q, k = qkv[:, :8], qkv[:, 8:10]
    other = torch.zeros(4, 12, 64, dtype=torch.bfloat16)

    def says(what, **kw):
        with pytest.raises(ValueError, match=what):
            rotary.apply_rotary(q, k, pos, freq, **kw)

    says("overlap", q_out=qkv[:, 2:10])                              # over the keys
    says("overlap", k_out=q[:, :2])
    says("overlap", q_out=other[:, :8], k_out=other[:, 7:9])         # over each other
    says("overlap", q_out=other[:, :8], k_out=other[:, :2])
    says("repeat", q_out=torch.zeros(4000, dtype=torch.bfloat16).as_strided((4, 8, 64), (64, 64, 1)))
    for kw in (dict(q_out=q, k_out=k), dict(q_out=q), dict(k_out=k), dict(q_out=other[:, :8], k_out=other[:, 8:10]), {}):
        says("dtype", **kw)


def test_append_over_its_cache():
    """k and v apart from the codes and the scales, by addresses (nothing is read: the calls are refused)."""
    lib = _lib()
    blocks, block, heads, dim, tokens = 4, 16, 2, 64, 3
    cache, scales, codes = 1 << 20, 1 << 24, 2 * blocks * block * heads * dim
    rows = ((tokens - 1) * heads * dim + (heads - 1) * dim + dim) * 2

    def append(k=1 << 28, v=1 << 29, cache=cache, scales=scales, dtype=0):
        p = ctypes.c_void_p
        return lib.semblo_kv8_append(p(k), heads * dim, dim, p(v), heads * dim, dim, tokens, dtype, p(cache), p(scales), blocks,
                                     block, heads, dim, p(1 << 30), 1, 1, p(1 << 31), p(1 << 32), 1, p(1 << 33), None)

    for kw in (dict(k=cache), dict(v=cache + codes - 16), dict(k=cache - rows + 16), dict(v=scales),
               dict(k=scales + 2 * blocks * heads * 4 - 16), dict(v=scales - rows + 16)):
        assert append(**kw) == -1 and b"overlap" in lib.semblo_last_error(), kw
    # apart by nothing: the type is looked at next, and one is refused there, so that nothing is launched
    for kw in (dict(k=cache + codes), dict(v=cache - rows), dict(k=scales - rows), dict(v=scales + 2 * blocks * heads * 4)):
        assert append(**kw, dtype=1) == -1 and b"dtype" in lib.semblo_last_error(), kw


def test_append_to_a_cache_made_of_its_input(hostside, monkeypatch):   # noqa: F811
    """The same through the Python entry: a pool that was cut from the buffer of the keys."""
    _, kv8 = hostside
    buf = torch.zeros(4, 16, 2, 64, dtype=torch.bfloat16)
    cache = kv8.Kv8Cache(buf.view(torch.uint8).view(torch.float8_e4m3fn).view(-1)[:2 * 4 * 2 * 16 * 64].view(2, 4, 2, 16, 64),
                         torch.ones(2, 4, 2))
    x = buf[0, :3]
    monkeypatch.setattr(kv8, "device_scope", lambda device: contextlib.nullcontext())
    monkeypatch.setattr(kv8, "raw_stream", lambda index: None)
    monkeypatch.setattr(kv8._lib, "status_for", lambda device: SimpleNamespace(word=torch.zeros(1, dtype=torch.int32)))
    monkeypatch.setattr(kv8, "lib", _lib)
    with pytest.raises(ValueError, match="overlap"):
        kv8.kv8_append(cache, x, x, torch.zeros(1, 2, dtype=torch.int32), torch.tensor([0, 3]), torch.tensor([0]))
