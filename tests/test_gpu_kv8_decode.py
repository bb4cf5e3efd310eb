"""Attention over the 8-bit paged cache against the formula in 64 bits on the stored values."""
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


def _pool(dev, seed, lens, block, heads, dim, width=None, k_scale=0.0, v_spread=2):
    from semblo_b200.kv8_cache import Kv8Cache
    gen = torch.Generator(device=dev).manual_seed(seed)
    need = [-(-n // block) for n in lens]
    blocks = sum(need) + 3
    cache = Kv8Cache.allocate(blocks, block, heads, dim, dev)
    codes = torch.randn(2, blocks, heads, block, dim, device=dev, generator=gen) * 64
    cache.data.copy_(codes.clamp(-448, 448).to(torch.float8_e4m3fn))
    cache.scales[0] = 2.0 ** -6 * torch.exp2(k_scale * torch.randn(blocks, heads, device=dev, generator=gen))
    cache.scales[1] = 2.0 ** -6 * torch.exp2(torch.randint(-v_spread, v_spread + 1, (blocks, heads), device=dev,
                                                           generator=gen).float())
    table = torch.full((len(lens), width or max(max(need), 1)), -1, dtype=torch.int32, device=dev)
    order = torch.randperm(blocks, device=dev, generator=gen).to(torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    return cache, table, gen


def _formula(q, cache, table, lens, sm_scale, softcap, window, prefix, slopes):
    """Output, log-sum-exp, sum of |p v| and a bound on what a score is off by, all in 64 bits."""
    bsz, n, hq, d = q.shape
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    mag = torch.zeros_like(out)
    lse = torch.full(q.shape[:3], -math.inf, dtype=torch.float64, device=q.device)
    off = torch.zeros(q.shape[:3], dtype=torch.float64, device=q.device)
    for b, length in enumerate(lens):
        if length == 0:
            continue
        k, v = (x[:length].double().repeat_interleave(hq // cache.num_kv_heads, 1)
                for x in cache.gather(table[b, :-(-length // cache.block_size)]))
        s = torch.einsum("nhd,jhd->nhj", q[b].double(), k) * sm_scale
        sabs = torch.einsum("nhd,jhd->nhj", q[b].double().abs(), k.abs()) * sm_scale
        if softcap:
            s = softcap * torch.tanh(s / softcap)
        p = torch.arange(length - n, length, device=q.device)[:, None]
        j = torch.arange(length, device=q.device)[None]
        bias = torch.zeros(n, hq, length, dtype=torch.float64, device=q.device)
        if slopes is not None:
            bias = slopes.double()[None, :, None] * (p - j).abs()[:, None]
        s = s - bias
        see = (j <= p) & ((p - j < window) if window else (j <= p))
        if prefix is not None:
            see = see | (j < int(prefix[b]))
        see = see[:, None].expand(n, hq, length)
        s = s.masked_fill(~see, -math.inf)
        lse[b] = torch.logsumexp(s, -1)
        w = torch.exp(s - lse[b].masked_fill(lse[b] == -math.inf, 0.0)[..., None])
        out[b] = torch.einsum("nhj,jhd->nhd", w, v)
        mag[b] = torch.einsum("nhj,jhd->nhd", w, v.abs())
        # 32-bit sums of D products (one rounding of 2^-23 each at most), the scalings, the cap's exponential and
        # division (2^-20 of the cap), the distance's product and difference
        err = sabs * (d + 16) * 2.0 ** -23 + (softcap or 0.0) * 2.0 ** -20 + (bias + s.abs().nan_to_num(posinf=0)) * 2.0 ** -22
        off[b] = torch.where(see, err, 0.0).amax(-1)
    return out, lse, mag, off


def _check(result, want, keys):
    got, lse = result.output, result.logsumexp
    out, wlse, mag, off = want
    eps = torch.finfo(got.dtype).eps
    # P is rounded to fp16 (half a step: 2^-11); the weights are off by e^(score error) in numerator and denominator,
    # two exponentials by 2^-21, the sum of up to `keys` 32-bit terms by keys 2^-24; then one rounding to the type
    rel = 2.0 ** -11 + 4 * off[..., None] + 2.0 ** -20 + keys * 2.0 ** -24
    tiny = torch.finfo(got.dtype).smallest_normal * eps
    bound = mag * rel * (1 + eps) + out.abs() * eps / 2 + tiny
    err = (got.double() - out).abs()
    assert bool(got.isfinite().all())
    assert bool((err <= bound).all()), float((err / bound).max())
    empty = wlse == -math.inf
    assert torch.equal(lse == -math.inf, empty)
    assert bool((got[empty] == 0).all())
    lerr = (lse.double() - wlse)[~empty].abs()
    lbound = (2 * off + 2.0 ** -20 + keys * 2.0 ** -24 + wlse.abs() * 2.0 ** -22)[~empty]
    assert bool((lerr <= lbound).all()), float((lerr / lbound).max())


def _call(q, cache, table, lens, **kw):
    from semblo_b200.kv8_cache import kv8_decode_attention
    lengths = torch.tensor(lens, dtype=torch.int32, device=q.device)
    return kv8_decode_attention(q, cache, table, lengths, return_logsumexp=True, **kw)


LENS = [1, 0, 15, 16, 17, 513, 1500, 33, 2]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("heads,group,queries", [(2, 4, 1), (1, 1, 1), (2, 8, 1), (1, 5, 2), (1, 16, 1), (2, 7, 5), (1, 2, 16)])
@pytest.mark.parametrize("options", ["plain", "cap", "window", "all"])
def test_formula(dev, dtype, dim, heads, group, queries, options):
    block = {64: 16, 128: 64, 256: 256}[dim]
    cache, table, gen = _pool(dev, dim + group, LENS, block, heads, dim)
    q = (torch.randn(len(LENS), queries, heads * group, dim, device=dev, generator=gen) * 2).to(dtype)
    kw = dict(sm_scale=dim ** -0.5, softcap=0.0, window=0, prefix_lens=None, alibi_slopes=None)
    if options in ("cap", "all"):
        kw["softcap"] = 5.0
    if options in ("window", "all"):
        kw["window"] = 100
        kw["prefix_lens"] = torch.tensor([3, 0, 20, 1, 0, 40, 257, 0, 1], device=dev)
    if options == "all":
        kw["alibi_slopes"] = torch.rand(heads * group, device=dev, generator=gen)
    want = _formula(q, cache, table, LENS, kw["sm_scale"], kw["softcap"], kw["window"], kw["prefix_lens"], kw["alibi_slopes"])
    _check(_call(q, cache, table, LENS, **kw), want, max(LENS))
    short = [min(n, 40) for n in LENS]                                       # a table one block's share long
    narrow = table[:, :-(-40 // block)]
    want = _formula(q, cache, narrow, short, kw["sm_scale"], kw["softcap"], kw["window"],
                    kw["prefix_lens"], kw["alibi_slopes"])
    _check(_call(q, cache, narrow, short, **kw), want, 40)


@pytest.mark.parametrize("window", [1, 16, 17, 999])
def test_windows_without_prefix(dev, window):
    cache, table, gen = _pool(dev, window, LENS, 32, 2, 128)
    q = torch.randn(len(LENS), 3, 8, 128, device=dev, generator=gen).to(torch.bfloat16)
    want = _formula(q, cache, table, LENS, 0.1, 0.0, window, None, None)
    _check(_call(q, cache, table, LENS, sm_scale=0.1, window=window), want, max(LENS))


def test_many_requests_and_long_rows(dev):
    lens = [(i * 131) % 700 for i in range(300)] + [40000]
    cache, table, gen = _pool(dev, 1, lens, 16, 1, 64)
    q = torch.randn(len(lens), 1, 4, 64, device=dev, generator=gen).to(torch.bfloat16)
    want = _formula(q, cache, table, lens, 0.125, 0.0, 0, None, None)
    first = _call(q, cache, table, lens, sm_scale=0.125)
    _check(first, want, 40000)
    again = _call(q, cache, table, lens, sm_scale=0.125)
    assert torch.equal(first.output, again.output) and torch.equal(first.logsumexp, again.logsumexp)


@pytest.mark.parametrize("long", [40, 300, 1100, 5000])
@pytest.mark.parametrize("queries,group", [(1, 4), (3, 8), (4, 8)])
def test_short_requests_in_a_wide_table(dev, long, queries, group):
    # a table for 6400 keys; what is in it decides whether blocks take whole segments or even pieces
    lens = [3, 0, 17, long, 1, 64, 5]
    for dim in (64, 128):
        cache, table, gen = _pool(dev, 31, lens, 64, 2, dim, width=100)
        q = torch.randn(len(lens), queries, 2 * group, dim, device=dev, generator=gen).to(torch.bfloat16)
        want = _formula(q, cache, table, lens, dim ** -0.5, None, 0, None, None)
        _check(_call(q, cache, table, lens, sm_scale=dim ** -0.5), want, max(lens))


def test_the_most_requests_in_a_wide_table(dev):
    lens = [i % 3 for i in range(4096)]
    lens[17], lens[4000] = 1500, 700
    cache, table, gen = _pool(dev, 32, lens, 16, 1, 64, width=100)
    q = torch.randn(len(lens), 1, 2, 64, device=dev, generator=gen).to(torch.float16)
    some = [0, 1, 2, 17, 18, 3999, 4000, 4095]
    want = _formula(q[some], cache, table[some], [lens[i] for i in some], 0.125, 30.0, 0, None, None)
    got = _call(q, cache, table, lens, sm_scale=0.125, softcap=30.0)
    _check(type(got)(got.output[some], got.logsumexp[some]), want, max(lens))


@pytest.mark.parametrize("dim", [128, 256])
def test_scales_of_every_size(dev, dim):
    """V in blocks of very different magnitude, K scales that are not powers of two, peaked scores."""
    lens = [900, 77]
    cache, table, gen = _pool(dev, 4, lens, 16, 2, dim, k_scale=1.0, v_spread=40)
    q = (torch.randn(2, 1, 8, dim, device=dev, generator=gen) * 8).to(torch.bfloat16)
    want = _formula(q, cache, table, lens, dim ** -0.5, 0.0, 0, None, None)
    _check(_call(q, cache, table, lens, sm_scale=dim ** -0.5), want, 900)
    cache.scales[1][::2] = 0.0                                               # blocks whose values are all zero
    want = _formula(q, cache, table, lens, dim ** -0.5, 0.0, 0, None, None)
    _check(_call(q, cache, table, lens, sm_scale=dim ** -0.5), want, 900)
    tiny = (q.float() * 2.0 ** -90).to(torch.bfloat16)                       # queries far below fp16's range
    cache.scales[0] *= 2.0 ** 90
    want = _formula(tiny, cache, table, lens, dim ** -0.5, 0.0, 0, None, None)
    _check(_call(tiny, cache, table, lens, sm_scale=dim ** -0.5), want, 900)


def test_nan_where_nothing_is_seen(dev):
    """Rows behind the last token, unread blocks and keys below the window may hold anything."""
    lens = [37, 300, 5]
    cache, table, gen = _pool(dev, 5, lens, 32, 2, 128)
    q = torch.randn(3, 1, 8, 128, device=dev, generator=gen).to(torch.bfloat16)
    args = dict(sm_scale=0.1, window=50, prefix_lens=torch.tensor([0, 3, 2], device=dev))
    clean = _call(q, cache, table, lens, **args)
    raw = cache.data.view(torch.uint8)
    used = torch.zeros(cache.num_blocks, 32, dtype=torch.bool, device=dev)
    for b, n in enumerate(lens):
        for j in range(n):
            if n - 1 - j < 50 or j < int(args["prefix_lens"][b]):
                used[int(table[b, j // 32]), j % 32] = True
    raw.masked_fill_(~used[None, :, None, :, None], 0x7f)
    dirty = _call(q, cache, table, lens, **args)
    assert torch.equal(clean.output, dirty.output) and torch.equal(clean.logsumexp, dirty.logsumexp)


@pytest.mark.parametrize("width", [1, 200])
def test_bad_pages_are_absent(dev, width):
    from semblo_b200 import _lib
    lens = [40, 20]
    cache, table, gen = _pool(dev, 6, lens, 64, 1, 128, width=width)
    q = torch.randn(2, 1, 4, 128, device=dev, generator=gen).to(torch.bfloat16)
    good = _call(q, cache, table, lens, sm_scale=0.1)
    for wrong in (-1, cache.num_blocks):
        bad = table.clone()
        bad[1, 0] = wrong
        got = _call(q, cache, bad, lens, sm_scale=0.1)
        with pytest.raises(RuntimeError, match="201"):
            _lib.status_for(dev).raise_if_set()
        assert torch.equal(got.output[0], good.output[0])
        assert bool((got.output[1] == 0).all()) and bool((got.logsumexp[1] == -math.inf).all())


def test_length_beyond_the_table(dev):
    from semblo_b200 import _lib
    cache, table, gen = _pool(dev, 7, [64], 64, 1, 64)
    q = torch.randn(1, 1, 4, 64, device=dev, generator=gen).to(torch.bfloat16)
    got = _call(q, cache, table, [65], sm_scale=0.1)
    with pytest.raises(RuntimeError, match="201"):
        _lib.status_for(dev).raise_if_set()
    assert torch.equal(got.output, _call(q, cache, table, [64], sm_scale=0.1).output)
    _lib.status_for(dev).raise_if_set()


def test_streams_and_graphs(dev):
    from semblo_b200.kv8_cache import kv8_decode_attention
    lens = [3000, 1, 4000]
    cache, table, gen = _pool(dev, 8, lens, 128, 2, 128)
    q = torch.randn(3, 1, 8, 128, device=dev, generator=gen).to(torch.bfloat16)
    other = torch.randn(3, 1, 8, 128, device=dev, generator=gen).to(torch.bfloat16)
    lengths = torch.tensor(lens, dtype=torch.int32, device=dev)
    side = [torch.cuda.Stream() for _ in range(2)]
    want = [_call(x, cache, table, lens, sm_scale=0.1).output for x in (q, other)]
    torch.cuda.synchronize()
    got = []
    for _ in range(5):                                                        # two calls at once
        for x, st in zip((q, other), side):
            with torch.cuda.stream(st):
                got.append(kv8_decode_attention(x, cache, table, lengths, sm_scale=0.1).output)
    torch.cuda.synchronize()
    for i, o in enumerate(got):
        assert torch.equal(o, want[i % 2])
    graphs, outs = [], []
    for x in (q, other):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(kv8_decode_attention(x, cache, table, lengths, sm_scale=0.1).output)
        graphs.append(g)
    lengths.copy_(torch.tensor([100, 4000, 17]))                              # a replay reads the lengths of its time
    table[1] = table[2]
    want = [_call(x, cache, table, [100, 4000, 17], sm_scale=0.1).output for x in (q, other)]
    for st, g in zip(side, graphs):
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st):
            g.replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1])


def test_views_out_and_empty_batch(dev):
    from semblo_b200.kv8_cache import kv8_decode_attention
    cache, table, gen = _pool(dev, 9, [70, 30], 32, 1, 64)
    lengths = torch.tensor([70, 30], device=dev)
    wide = torch.randn(2, 1, 12, 64, device=dev, generator=gen).to(torch.bfloat16)
    want = kv8_decode_attention(wide[:, :, 4:8].contiguous(), cache, table, lengths, sm_scale=0.1).output
    out = torch.empty_like(want)
    r = kv8_decode_attention(wide[:, :, 4:8], cache, table.long(), lengths.int(), sm_scale=0.1, out=out)
    assert r.output is out and r.logsumexp is None and torch.equal(out, want)
    none = kv8_decode_attention(wide[:0], cache, table[:0], lengths[:0], sm_scale=0.1)
    assert none.output.shape == (0, 1, 12, 64)


def test_cache_past_32_bits(dev):
    """Codes whose byte offset in the pool exceeds 2^31, read at the end of a long context."""
    from semblo_b200.kv8_cache import Kv8Cache
    block, heads, dim = 256, 4, 256
    blocks = (1 << 31) // (block * heads * dim) + 8
    cache = Kv8Cache.allocate(blocks, block, heads, dim, dev)
    table = torch.arange(blocks - 8, blocks, dtype=torch.int32, device=dev)[None]
    gen = torch.Generator(device=dev).manual_seed(10)
    codes = (torch.randn(2, 8, heads, block, dim, device=dev, generator=gen) * 64).clamp(-448, 448).to(torch.float8_e4m3fn)
    cache.data[:, blocks - 8:] = codes
    cache.scales.fill_(2.0 ** -6)
    q = torch.randn(1, 1, 16, dim, device=dev, generator=gen).to(torch.bfloat16)
    want = _formula(q, cache, table, [2000], 0.0625, 0.0, 0, None, None)
    _check(_call(q, cache, table, [2000], sm_scale=0.0625), want, 2000)
