"""Outputs that share memory with an input or with each other: refused unless no element is shared, as in the slices of
one fused buffer.  Without a device, against the elements counted one by one."""
from __future__ import annotations

import contextlib
import itertools
import random

import pytest
import torch

from test_dense_refusals import hostside                             # noqa: F401 (the fixture)


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
