"""Writing the 8-bit paged cache: the definition, followed block by block in 64 bits, equal code for code."""
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


def _codes(x64):
    """Round to e4m3 by arithmetic: three mantissa bits, exponents from -6, ties to even, saturating at 448."""
    mag = x64.abs().clamp(max=448.0)
    e = torch.floor(torch.log2(mag.clamp_min(2.0 ** -30))).clamp_min(-6)
    e = torch.where(mag >= torch.exp2(e + 1), e + 1, torch.where(mag < torch.exp2(e), (e - 1).clamp_min(-6), e))
    step = torch.exp2(e - 3)
    return torch.copysign((mag / step).round() * step, x64).clamp(-448.0, 448.0)


def _append_64(data, scales, k, v, table, cu, start, block):
    """data [2, blocks, H, block, D] and scales [2, blocks, H] in 64 bits, changed in place."""
    for part, x in enumerate((k.double(), v.double())):
        for b in range(len(start)):
            n, pos = cu[b + 1] - cu[b], start[b]
            row = cu[b]
            while n > 0:
                page, off = int(table[b][pos // block]), pos % block
                m = min(block - off, n)
                for h in range(x.shape[1]):
                    rows = x[row:row + m, h]
                    finite = rows[rows.isfinite()].abs()
                    top = float(finite.max()) if finite.numel() else 0.0
                    s = 2.0 ** -100
                    while top > 448.0 * s and s < 2.0 ** 120:
                        s *= 2
                    if off:
                        old = float(scales[part, page, h])
                        if old >= s:
                            s = old
                        else:
                            data[part, page, h, :off] = _codes(data[part, page, h, :off] * (old / s))
                    data[part, page, h, off:off + m] = _codes((rows / s).float().double())
                    scales[part, page, h] = s
                row, pos, n = row + m, pos + m, n - m


def _case(dev, seed, block, heads, dim, dtype, new, past, lift=True):
    from semblo_b200.kv8_cache import Kv8Cache
    gen = torch.Generator(device=dev).manual_seed(seed)
    need = [-(-(n + p) // block) + 1 for n, p in zip(new, past)]
    blocks = sum(need) + 2
    order = torch.randperm(blocks, device=dev, generator=gen).to(torch.int32)
    table = torch.full((len(new), max(need)), -1, dtype=torch.int32, device=dev)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    cache = Kv8Cache.allocate(blocks, block, heads, dim, dev)
    codes = torch.randn(2, blocks, heads, block, dim, device=dev, generator=gen) * 60
    cache.data.copy_(codes.clamp(-448, 448).to(torch.float8_e4m3fn))
    cache.scales.copy_(torch.exp2(torch.randint(-9, -4, cache.scales.shape, device=dev, generator=gen).float()))
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    t = cu[-1]
    scale = torch.exp2(torch.randint(-3, 5, (t, heads, 1), device=dev, generator=gen).float() / 2) if lift else 1.0
    k = (torch.randn(t, heads, dim, device=dev, generator=gen) * scale).to(dtype)
    v = (torch.randn(t, heads, dim, device=dev, generator=gen) * scale).to(dtype)
    return cache, k, v, table, cu, past


def _run_and_compare(cache, k, v, table, cu, past, block):
    from semblo_b200 import _lib
    from semblo_b200.kv8_cache import kv8_append
    dev = k.device
    data, scales = cache.data.double(), cache.scales.double()
    kv8_append(cache, k, v, table, torch.tensor(cu, dtype=torch.int32, device=dev),
               torch.tensor(past, dtype=torch.int32, device=dev))
    _append_64(data, scales, k, v, table.cpu().tolist(), cu, past, block)
    assert torch.equal(cache.scales.double(), scales)
    same = (cache.data.double() == data) | (cache.data.double().isnan() & data.isnan())
    assert bool(same.all()), int((~same).sum())
    _lib.status_for(dev).raise_if_set()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("block,dim", [(16, 64), (16, 128), (32, 256), (64, 64), (128, 128), (256, 256), (256, 64)])
@pytest.mark.parametrize("new,past", [([1], [0]), ([1, 1, 1, 1], [0, 15, 16, 700]), ([300, 1, 17, 0, 64], [0, 255, 9, 3, 64]),
                                      ([0, 0, 5], [1, 2, 3])])
def test_definition(dev, dtype, block, dim, new, past):
    _run_and_compare(*_case(dev, block + dim + len(new), block, 2, dim, dtype, new, past), block)


def test_many_requests(dev):
    new = [1 + (i * 37) % 40 for i in range(70)]
    past = [(i * 53) % 97 for i in range(70)]
    _run_and_compare(*_case(dev, 5, 32, 1, 64, torch.bfloat16, new, past), 32)


@pytest.mark.parametrize("block,dim,tokens", [(16, 64, 60000), (16, 128, 40000), (32, 128, 40000), (64, 128, 40000),
                                              (128, 128, 60000), (128, 256, 90000), (256, 256, 90000)])
def test_a_prompt_as_a_stream(dev, block, dim, tokens):
    """Enough blocks that every group of threads takes several: odd ends, continued blocks, special values, bad pages."""
    from semblo_b200 import _lib
    from semblo_b200.kv8_cache import Kv8Cache, kv8_append
    heads = 4
    new, past = [tokens - 777 - 40, 0, 777, 40], [3, 0, block - 1, 1]
    gen = torch.Generator(device=dev).manual_seed(block + dim)
    need = [-(-(n + p) // block) for n, p in zip(new, past)]
    blocks = sum(need) + 5
    order = torch.randperm(blocks, device=dev, generator=gen).to(torch.int32)
    table = torch.full((4, max(need)), -1, dtype=torch.int32, device=dev)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    table[0, 7] = blocks                                       # one block of the long request is not in the pool
    k = torch.randn(tokens, heads, dim, device=dev, generator=gen).to(torch.bfloat16)
    v = (k.float() * 3).to(torch.bfloat16)
    k[100, 1, 3], v[5000, 2, 7] = math.inf, math.nan
    cu = torch.tensor([0, new[0], new[0], new[0] + new[2], tokens], device=dev, dtype=torch.int32)
    start = torch.tensor(past, device=dev, dtype=torch.int32)
    base = Kv8Cache.allocate(blocks, block, heads, dim, dev)
    base.data.view(torch.uint8).random_(0, 120, generator=gen)
    base.scales.fill_(2.0 ** -9)
    whole = Kv8Cache(base.data.clone(), base.scales.clone())
    kv8_append(whole, k, v, table, cu, start)
    with pytest.raises(RuntimeError, match="201"):
        _lib.status_for(dev).raise_if_set()
    # in pieces of one block, a call each: the few-tokens kernel, which the definition test covers
    pieces = Kv8Cache(base.data.clone(), base.scales.clone())
    rows = [[0, new[0]], [new[0], new[0]], [new[0], new[0] + new[2]], [new[0] + new[2], tokens]]
    starts, cus, tables = [], [0], []
    ks, vs = [], []
    for b in range(4):
        pos, r = past[b], rows[b][0]
        while r < rows[b][1]:
            m = min(block - pos % block, rows[b][1] - r)
            starts.append(pos % block)
            tables.append(int(table[b, pos // block]) if (b, pos // block) != (0, 7) else -1)
            cus.append(m)
            pos, r = pos + m, r + m
    cum = torch.tensor(cus).cumsum(0).to(torch.int32)
    per_call = 8
    tab = torch.tensor(tables, dtype=torch.int32, device=dev)[:, None]
    st = torch.tensor(starts, dtype=torch.int32, device=dev)
    for i in range(0, len(starts), per_call):
        e = min(i + per_call, len(starts))
        a, z = int(cum[i]), int(cum[e])
        kv8_append(pieces, k[a:z], v[a:z], tab[i:e], (cum[i:e + 1] - a).to(dev), st[i:e])
    with pytest.raises(RuntimeError, match="201"):
        _lib.status_for(dev).raise_if_set()
    assert torch.equal(whole.scales, pieces.scales)
    assert torch.equal(whole.data.view(torch.uint8), pieces.data.view(torch.uint8))


def test_negative_starts_of_late_requests_are_reported(dev):
    from semblo_b200 import _lib
    cache, k, v, table, cu, past = _case(dev, 13, 16, 1, 64, torch.bfloat16, [2] * 80, [0] * 80)
    from semblo_b200.kv8_cache import kv8_append
    past[70] = -5
    kv8_append(cache, k, v, table, torch.tensor(cu, dtype=torch.int32, device=dev),
               torch.tensor(past, dtype=torch.int32, device=dev))
    with pytest.raises(RuntimeError, match="201"):
        _lib.status_for(dev).raise_if_set()


def test_token_by_token_grows_the_scale(dev):
    """One block filled token by token with rising magnitudes; a scale set by the caller (not a power of two) holds
    until a value needs more."""
    cache, k, v, table, _, _ = _case(dev, 9, 16, 2, 64, torch.bfloat16, [16], [0])
    k *= torch.exp2(torch.arange(16, device=dev) - 6.0)[:, None, None].to(k.dtype)
    for i in range(16):
        _run_and_compare(cache, k[i:i + 1], v[i:i + 1], table, [0, 1], [i], 16)
        if i == 3:
            cache.scales.mul_(1.3)


def test_special_values(dev):
    cache, k, v, table, cu, past = _case(dev, 10, 16, 2, 64, torch.bfloat16, [40], [5])
    k[3, 0, 5], k[4, 1, 6] = math.inf, -math.inf
    k[20:36] = 0.0                                           # a block of zeros
    v[30:32] = 2.0 ** -130                                   # far below the smallest scale's codes
    v[0, 0, 0] = 3.3e38
    k[37:40] = math.inf                                      # nothing finite in the last block's rows
    _run_and_compare(cache, k, v, table, cu, past, 16)
    from semblo_b200.kv8_cache import kv8_append
    k[1, 1, 1] = math.nan
    kv8_append(cache, k, v, table, torch.tensor(cu, dtype=torch.int32, device=dev),
               torch.tensor(past, dtype=torch.int32, device=dev))
    code = cache.data.float()
    assert int(code.isnan().sum()) == 1
    assert bool(code[0, int(table[0, 0]), 1, 6].isnan()[1])


def test_views_padding_streams_and_repeat(dev):
    from semblo_b200.kv8_cache import Kv8Cache, kv8_append
    cache, k, v, table, cu, past = _case(dev, 11, 64, 4, 128, torch.bfloat16, [50, 90], [10, 0])
    qkv = torch.randn(160, 16 + 8, 128, device=dev).to(torch.bfloat16)
    qkv[:140, 16:20], qkv[:140, 20:24] = k, v
    first = Kv8Cache(cache.data.clone(), cache.scales.clone())
    cu_t, st_t = torch.tensor(cu, device=dev), torch.tensor(past, device=dev)
    kv8_append(first, k, v, table, cu_t, st_t)
    for _ in range(2):
        other = Kv8Cache(cache.data.clone(), cache.scales.clone())
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):                        # 20 rows behind the last request: not read
            kv8_append(other, qkv[:, 16:20], qkv[:, 20:24], table.long(), cu_t.int(), st_t.int())
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(other.data.view(torch.uint8), first.data.view(torch.uint8))
        assert torch.equal(other.scales, first.scales)
    graph = torch.cuda.CUDAGraph()
    cu_i, st_i = cu_t.int(), st_t.int()
    held = Kv8Cache(cache.data.clone(), cache.scales.clone())
    with torch.cuda.graph(graph):
        kv8_append(held, k, v, table, cu_i, st_i)
    graph.replay()
    graph.replay()                                           # the same call twice writes the same bytes
    assert torch.equal(held.data.view(torch.uint8), first.data.view(torch.uint8))


@pytest.mark.parametrize("fault", ["page_high", "page_negative", "table_short", "start_negative"])
def test_bad_pages_are_skipped(dev, fault):
    from semblo_b200 import _lib
    from semblo_b200.kv8_cache import Kv8Cache, kv8_append
    cache, k, v, table, cu, past = _case(dev, 12, 16, 2, 64, torch.bfloat16, [20, 20], [0, 4])
    good = Kv8Cache(cache.data.clone(), cache.scales.clone())
    cu_t, st_t = torch.tensor(cu, dtype=torch.int32, device=dev), torch.tensor(past, dtype=torch.int32, device=dev)
    kv8_append(good, k, v, table, cu_t, st_t)
    bad = table.clone()
    if fault == "page_high":
        bad[1, 1] = cache.num_blocks
    elif fault == "page_negative":
        bad[1, 1] = -1
    elif fault == "table_short":
        bad = bad[:, :1]
    else:
        st_t[1] = -1
    before = cache.data.clone()
    kv8_append(cache, k, v, bad, cu_t, st_t)
    with pytest.raises(RuntimeError, match="201"):
        _lib.status_for(dev).raise_if_set()
    skipped = {"page_high": [(1, 1)], "page_negative": [(1, 1)], "table_short": [(0, 1), (1, 1)],
               "start_negative": [(1, 0), (1, 1)]}[fault]
    want = good.data.view(torch.uint8).clone()
    for b, i in skipped:
        want[:, int(table[b, i])] = before.view(torch.uint8)[:, int(table[b, i])]
    assert torch.equal(cache.data.view(torch.uint8), want)


def test_cache_past_32_bits(dev):
    """Blocks whose byte offset in the pool exceeds 2^31."""
    from semblo_b200.kv8_cache import Kv8Cache, kv8_append
    blocks = (1 << 31) // (256 * 4 * 256) + 8
    cache = Kv8Cache.allocate(blocks, 256, 4, 256, dev)
    k = torch.randn(300, 4, 256, device=dev).to(torch.bfloat16)
    table = torch.tensor([[blocks - 1, blocks - 3]], dtype=torch.int32, device=dev)
    kv8_append(cache, k, k, table, torch.tensor([0, 300], device=dev), torch.tensor([0], device=dev))
    small = Kv8Cache.allocate(2, 256, 4, 256, dev)
    kv8_append(small, k, k, torch.tensor([[0, 1]], dtype=torch.int32, device=dev), torch.tensor([0, 300], device=dev),
               torch.tensor([0], device=dev))
    got = cache.data.view(torch.uint8)[:, [blocks - 1, blocks - 3]]
    assert torch.equal(got, small.data.view(torch.uint8))
    assert torch.equal(cache.scales[:, [blocks - 1, blocks - 3]], small.scales)


def test_a_large_batch_of_single_tokens(dev):
    """More requests than threads in a block, some of them without a token."""
    new = [(i % 7 != 3) + 0 for i in range(700)]
    past = [(i * 29) % 64 for i in range(700)]
    _run_and_compare(*_case(dev, 14, 32, 1, 64, torch.bfloat16, new, past), 32)
