"""Rotary positions on the device against the formula in 64 bits."""
from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    from semblo_b200 import _lib
    _lib.lib()
    return torch.device("cuda:0")


def _turned(x, positions, freq, interleaved, inverse):
    """The formula in 64 bits, and for every element the magnitude that 32-bit rounding acts on."""
    y, mag = x.double().clone(), torch.zeros_like(x, dtype=torch.float64)
    inv = freq.inv_freq.to(x.device)
    r = 2 * inv.numel()
    ang = positions.double()[:, None] * inv
    c, s = ang.cos()[:, None] * freq.attention_scale, ang.sin()[:, None] * freq.attention_scale
    if inverse:
        s = -s
    a, b = (slice(0, r, 2), slice(1, r, 2)) if interleaved else (slice(0, r // 2), slice(r // 2, r))
    x1, x2 = x[..., a].double(), x[..., b].double()
    y[..., a], y[..., b] = x1 * c - x2 * s, x2 * c + x1 * s
    m = (x1.abs() + x2.abs()) * freq.attention_scale
    mag[..., a], mag[..., b] = m, m
    return y, mag


def _check(got, want, mag):
    # one rounding to the output type, at most eps / 2 of the value (or half the smallest subnormal); before it in
    # 32 bits: cos and sin off by 2 ulp (2^-22) each, the angle's fraction rounded to 24 bits (2 pi 2^-25 < 2^-22),
    # the scale, two products and a sum (4 * 2^-24): below 2^-20 of |x1| + |x2|
    eps = torch.finfo(got.dtype).eps
    tiny = torch.finfo(got.dtype).smallest_normal * eps / 2
    bound = want.abs() * eps / 2 + mag * 2.0 ** -20 * (1 + eps) + tiny
    err = (got.double() - want).abs()
    assert bool((err <= bound).all()), float((err - bound).max())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dim,rotary", [(128, 128), (256, 64), (256, 256), (80, 40), (64, 16), (66, 6), (33, 2), (128, 8)])
@pytest.mark.parametrize("tokens,hq,hkv,first", [(1, 16, 4, 524288), (5, 3, 1, 0), (301, 8, 2, 1048000)])
def test_formula(dev, dtype, interleaved, dim, rotary, tokens, hq, hkv, first):
    from semblo_b200.rotary import apply_rotary, rotary_frequencies
    gen = torch.Generator(device=dev).manual_seed(dim + rotary + tokens)
    q = torch.randn(tokens, hq, dim, device=dev, generator=gen).to(dtype)
    k = torch.randn(tokens, hkv, dim, device=dev, generator=gen).to(dtype)
    pos = torch.arange(first, first + tokens, device=dev)
    if tokens == 5:
        pos = torch.tensor([7, 0, 7, -3, 123456], device=dev, dtype=torch.int32)     # any order, twice, negative
    freq = rotary_frequencies(rotary, 500000.0, device=dev)
    for inverse in (False, True):
        qo, ko = apply_rotary(q, k, pos, freq, interleaved=interleaved, inverse=inverse)
        for x, y in ((q, qo), (k, ko)):
            want, mag = _turned(x, pos, freq, interleaved, inverse)
            _check(y, want, mag)
            assert torch.equal(y[..., rotary:], x[..., rotary:])


def test_views_in_place_and_no_keys(dev):
    from semblo_b200.rotary import apply_rotary, rotary_frequencies
    gen = torch.Generator(device=dev).manual_seed(3)
    qkv = torch.randn(77, 8 + 2 + 2, 128, device=dev, generator=gen).to(torch.bfloat16)
    held = qkv.clone()
    q, k = qkv[:, :8], qkv[:, 8:10]
    pos = torch.arange(77, device=dev)
    freq = rotary_frequencies(128, device=dev)
    qo, ko = apply_rotary(q, k, pos, freq)
    assert torch.equal(qkv, held)                                    # the inputs keep their pre-rotation values
    only, none = apply_rotary(q, None, pos, freq)
    assert none is None and torch.equal(only, qo)
    apply_rotary(q, k, pos, freq, q_out=q, k_out=k)
    assert torch.equal(q, qo) and torch.equal(k, ko)
    assert torch.equal(qkv[:, 10:], held[:, 10:])                    # the value heads between are untouched
    # rows that start off 16 bytes take the narrow form
    odd = torch.randn(9, 3, 131, device=dev, generator=gen)[:, :, 1:129].to(torch.bfloat16)
    raw = torch.empty(9 * 3 * 131 + 1, dtype=torch.bfloat16, device=dev)[1:].view(9, 3, 131)[:, :, :128]
    raw.copy_(odd)
    a, _ = apply_rotary(raw, None, pos[:9], freq)
    b, _ = apply_rotary(odd.contiguous(), None, pos[:9], freq)
    assert torch.equal(a, b)
    heads_first = torch.randn(4, 50, 128, device=dev, generator=gen).to(torch.bfloat16).transpose(0, 1)
    c, _ = apply_rotary(heads_first, None, pos[:50], freq)
    d, _ = apply_rotary(heads_first.contiguous(), None, pos[:50], freq)
    assert torch.equal(c, d)


def test_back_and_forth(dev):
    """The inverse is the transpose: <R x, y> = <x, R' y>, and R' R x = x for a scale of one."""
    from semblo_b200.rotary import apply_rotary, rotary_frequencies
    gen = torch.Generator(device=dev).manual_seed(4)
    x = torch.randn(64, 4, 96, device=dev, generator=gen)
    y = torch.randn(64, 4, 96, device=dev, generator=gen)
    pos = torch.arange(1000, 1064, device=dev)
    freq = rotary_frequencies(64, scaling={"type": "yarn", "factor": 4.0, "original_max_position": 4096}, device=dev)
    rx, _ = apply_rotary(x, None, pos, freq)
    ry, _ = apply_rotary(y, None, pos, freq, inverse=True)
    # 24576 products of size ~1, each off by a few 2^-23: the sums differ by at most n * 2^-20
    assert abs(float((rx.double() * y).sum() - (x.double() * ry).sum())) < 24576 * 2.0 ** -20
    plain = rotary_frequencies(64, device=dev)
    there, _ = apply_rotary(x, None, pos, plain)
    back, _ = apply_rotary(there, None, pos, plain, inverse=True)
    assert float((back - x).abs().max()) < 2 * 2.0 ** -20 * 2 * float(x.abs().max())


def test_empty_streams_and_graph(dev):
    from semblo_b200.rotary import apply_rotary, rotary_frequencies
    freq = rotary_frequencies(32, device=dev)
    e, _ = apply_rotary(torch.empty(0, 4, 64, device=dev), None, torch.empty(0, dtype=torch.int64, device=dev), freq)
    assert e.shape == (0, 4, 64)
    x = torch.randn(33, 2, 64, device=dev)
    pos = torch.arange(33, device=dev)
    want, _ = apply_rotary(x, None, pos, freq)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got, _ = apply_rotary(x, None, pos, freq)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, _ = apply_rotary(x, None, pos, freq)
    pos += 5
    x.mul_(0.5)
    want, _ = apply_rotary(x, None, pos, freq)
    graph.replay()
    assert torch.equal(out, want)


def test_many_tokens_and_heads(dev):
    """More rows than one wave, element offsets past 2^31 (the output's last rows against the formula)."""
    from semblo_b200.rotary import apply_rotary, rotary_frequencies
    tokens, heads, dim = 70000, 128, 256
    x = torch.empty(tokens, heads, dim, device=dev, dtype=torch.bfloat16).normal_()
    assert x.numel() > 1 << 31
    freq = rotary_frequencies(dim, device=dev)
    pos = torch.arange(tokens, device=dev)
    y, _ = apply_rotary(x, None, pos, freq)
    for sl in (slice(0, 2), slice(tokens - 2, tokens), slice(65534, 65538)):
        want, mag = _turned(x[sl], pos[sl], freq, False, False)
        _check(y[sl], want, mag)
