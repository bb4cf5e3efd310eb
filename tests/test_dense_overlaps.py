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
    """Views of one buffer as layers make them: head slices, token ranges, heads first, every other head or token."""
    t, h, d = rng.choice([1, 2, 5]), rng.choice([4, 6]), rng.choice([2, 3])
    flat = torch.zeros(2 * t * h * d + 7)
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
    return out


def test_shared_elements():
    from semblo_b200._lib import shares_elements
    rng, told = random.Random(1), 0
    for _ in range(3000):
        a, b = _views(rng)
        shared = bool(_elements(a) & _elements(b))
        assert shares_elements(a, b) or not shared
        assert shares_elements(a, b) == shares_elements(b, a)
        told += not shared and not shares_elements(a, b)
    assert told > 500                                                # and disjoint views are told apart
    # the layouts that layers have, told apart exactly
    qkv = torch.zeros(7, 12, 16)
    q, k, v = qkv[:, :8], qkv[:, 8:10], qkv[:, 10:]
    assert not shares_elements(q, k) and not shares_elements(k, v) and shares_elements(q, qkv[:, 7:9])
    grouped = torch.zeros(7, 2, 6, 16)                               # per KV head: its queries, K and V
    assert not shares_elements(grouped[:, :, 4], grouped[:, :, 5]) and not shares_elements(grouped[:, :, 0], grouped[:, :, 5])
    first = torch.zeros(12, 7, 16).transpose(0, 1)                   # heads first
    assert not shares_elements(first[:, :8], first[:, 8:10]) and shares_elements(first[:, :8], first[:, 7:])
    assert not shares_elements(qkv[:0], qkv) and shares_elements(qkv[:1].expand(7, 12, 16), qkv[:1])
    assert not shares_elements(qkv[:3], qkv[3:]) and shares_elements(qkv[:4], qkv[3:])


def test_rotary_outputs(hostside, monkeypatch):                      # noqa: F811
    rotary, _ = hostside
    monkeypatch.setattr(rotary, "device_scope", lambda device: contextlib.nullcontext())
    freq, pos = rotary.rotary_frequencies(64, device="cpu"), torch.arange(4)
    qkv = torch.zeros(4, 12, 64)
    q, k = qkv[:, :8], qkv[:, 8:10]
    other = torch.zeros(4, 12, 64)

    def no(**kw):
        with pytest.raises(ValueError, match="overlap|repeat"):
            rotary.apply_rotary(q, k, pos, freq, **kw)

    def reaches(**kw):                                               # accepted: the library is asked for
        with pytest.raises(AssertionError, match="not refused"):
            rotary.apply_rotary(q, k, pos, freq, **kw)

    no(q_out=qkv[:, 2:10])                                           # over the keys
    no(q_out=qkv[:, 1:9])
    no(k_out=q[:, :2])
    no(k_out=qkv[:, 7:9])
    no(q_out=other[:, :8], k_out=other[:, 7:9])                      # over each other
    no(q_out=other[:, :8], k_out=other[:, :2])
    no(q_out=torch.zeros(4000).as_strided((4, 8, 64), (64, 64, 1)))  # rows over rows of their own
    no(q_out=torch.zeros(4000).as_strided((4, 8, 64), (512, 32, 1)))
    reaches(q_out=q, k_out=k)                                        # in place, in the fused buffer
    reaches(q_out=q)
    reaches(k_out=k)
    reaches(q_out=other[:, :8], k_out=other[:, 8:10])
    reaches(q_out=other[:, :8], k_out=qkv[:, 10:])                   # the value heads' place
    reaches()


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
