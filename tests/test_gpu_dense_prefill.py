"""Attention of packed prompts against the formula in 64 bits."""
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


def _starts(lens):
    out = [0]
    for n in lens:
        out.append(out[-1] + n)
    return out


def _formula(q, k, v, q_lens, k_lens, *, sm_scale, causal=True, window=0, prefix=None, softcap=0.0, slopes=None):
    """Output, log-sum-exp, sum of |p v| and a bound on what a score is off by, in 64 bits, document by document."""
    hq, hkv, d = q.shape[1], k.shape[1], q.shape[2]
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    mag = torch.zeros_like(out)
    lse = torch.full(q.shape[:2], -math.inf, dtype=torch.float64, device=q.device)
    off = torch.zeros(q.shape[:2], dtype=torch.float64, device=q.device)
    cq, ck = _starts(q_lens), _starts(k_lens)
    for b, (lq, lk) in enumerate(zip(q_lens, k_lens)):
        if lq == 0 or lk == 0:
            continue
        r = slice(cq[b], cq[b + 1])
        kk = k[ck[b]:ck[b + 1]].double().repeat_interleave(hq // hkv, 1)
        vv = v[ck[b]:ck[b + 1]].double().repeat_interleave(hq // hkv, 1)
        s = torch.einsum("ihd,jhd->hij", q[r].double(), kk) * sm_scale
        sabs = torch.einsum("ihd,jhd->hij", q[r].double().abs(), kk.abs()) * sm_scale
        if softcap:
            s = softcap * torch.tanh(s / softcap)
        p = torch.arange(lk - lq, lk, device=q.device)[:, None]
        j = torch.arange(lk, device=q.device)[None]
        bias = torch.zeros_like(s)
        if slopes is not None:
            bias = slopes.double()[:, None, None] * (p - j).abs()
        s = s - bias
        see = torch.ones(lq, lk, dtype=torch.bool, device=q.device)
        if causal:
            see = j <= p
            if window:
                see = see & (p - j < window)
            if prefix is not None:
                see = see | (j < int(prefix[b]))
        s = s.masked_fill(~see, -math.inf)
        ls = torch.logsumexp(s, -1)
        w = torch.exp(s - ls.masked_fill(ls == -math.inf, 0.0)[..., None])
        out[r] = torch.einsum("hij,jhd->ihd", w, vv)
        mag[r] = torch.einsum("hij,jhd->ihd", w, vv.abs())
        lse[r] = ls.T
        # 32-bit sums of D products (one rounding of 2^-23 each at most), the scalings, the cap's exponential and
        # division (2^-20 of the cap), the distance's product and difference
        err = sabs * (d + 16) * 2.0 ** -23 + softcap * 2.0 ** -20 + (bias + s.abs().nan_to_num(posinf=0)) * 2.0 ** -22
        off[r] = torch.where(see, err, 0.0).amax(-1).T
    return out, lse, mag, off


def _check(result, want, keys):
    got, lse = result.output, result.logsumexp
    out, wlse, mag, off = want
    eps = torch.finfo(got.dtype).eps
    # P is rounded to the type (half a step: eps / 2); the weights are off by e^(score error) in numerator and
    # denominator, two exponentials by 2^-21, the 32-bit sum of up to `keys` terms by keys 2^-24; then one rounding
    rel = eps / 2 + 4 * off[..., None] + 2.0 ** -20 + keys * 2.0 ** -24
    tiny = torch.finfo(got.dtype).smallest_normal * eps
    bound = mag * rel * (1 + eps) + out.abs() * eps / 2 + tiny
    assert bool(got.isfinite().all())
    err = (got.double() - out).abs()
    assert bool((err <= bound).all()), float((err / bound).max())
    empty = wlse == -math.inf
    assert bool((got[empty] == 0).all())
    if lse is not None:
        assert torch.equal(lse == -math.inf, empty)
        lerr = (lse.double() - wlse)[~empty].abs()
        lbound = (2 * off + 2.0 ** -20 + keys * 2.0 ** -24 + wlse.abs() * 2.0 ** -22)[~empty]
        assert bool((lerr <= lbound).all()), float((lerr / lbound).max())


def _inputs(dev, seed, q_lens, k_lens, hq, hkv, dim, dtype, scale=2.0):
    gen = torch.Generator(device=dev).manual_seed(seed)
    q = (torch.randn(sum(q_lens), hq, dim, device=dev, generator=gen) * scale).to(dtype)
    k, v = (torch.randn(sum(k_lens), hkv, dim, device=dev, generator=gen).to(dtype) for _ in range(2))
    return q, k, v, gen


def _call(q, k, v, q_lens, k_lens, prefix=None, slopes=None, **kw):
    from semblo_b200.dense_prefill import dense_prefill_attention
    cu = [torch.tensor(_starts(x), dtype=torch.int32, device=q.device) for x in (q_lens, k_lens)]
    return dense_prefill_attention(q, k, v, cu_seqlens_q=cu[0], cu_seqlens_k=cu[1], prefix_lens=prefix, alibi_slopes=slopes,
                                   return_logsumexp=True, **kw)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("options", ["plain", "full", "cap", "window", "all"])
def test_few_queries_over_many_keys(dev, dim, dtype, options):
    # enough keys per document for several pieces; documents of one piece and of none among them
    q_lens, k_lens = [5, 0, 33, 200, 1], [4100, 900, 1537, 1800, 3]
    q, k, v, gen = _inputs(dev, dim, q_lens, k_lens, 6, 2, dim, dtype)
    kw = {"sm_scale": dim ** -0.5}
    if options == "full":
        kw["causal"] = False
    if options in ("cap", "all"):
        kw["softcap"] = 20.0
    if options in ("window", "all"):
        kw["window"] = 1500
        kw["prefix"] = torch.tensor([700, 3, 0, 40, 2], device=dev)
    if options == "all":
        kw["slopes"] = torch.rand(6, device=dev, generator=gen) * 0.1
    want = _formula(q, k, v, q_lens, k_lens, **kw)
    got = _call(q, k, v, q_lens, k_lens, **kw)
    _check(got, want, max(k_lens))
    again = _call(q, k, v, q_lens, k_lens, **kw)
    assert torch.equal(got.output, again.output) and torch.equal(got.logsumexp, again.logsumexp)


@pytest.mark.parametrize("dim", [64, 256])
def test_pieces_of_many_documents(dev, dim):
    # more documents than a warp looks over, each with a few queries over many keys
    q_lens, k_lens = [i % 3 for i in range(70)], [1100 + 37 * (i % 20) for i in range(70)]
    q, k, v, _ = _inputs(dev, 4, q_lens, k_lens, 1, 1, dim, torch.bfloat16)
    want = _formula(q, k, v, q_lens, k_lens, sm_scale=dim ** -0.5)
    _check(_call(q, k, v, q_lens, k_lens, sm_scale=dim ** -0.5), want, max(k_lens))


def test_pieces_on_two_streams_and_in_graphs(dev):
    from semblo_b200.dense_prefill import dense_prefill_attention
    inputs = [_inputs(dev, 40 + i, [20], [4000], 8, 2, 128, torch.float16)[:3] for i in range(2)]
    cu_q, cu_k = torch.tensor([0, 20], dtype=torch.int32, device=dev), torch.tensor([0, 4000], dtype=torch.int32, device=dev)

    def call(i):
        q, k, v = inputs[i]
        return dense_prefill_attention(q, k, v, cu_seqlens_q=cu_q, cu_seqlens_k=cu_k, sm_scale=0.1).output

    want = [call(0), call(1)]
    streams, graphs, outs = [torch.cuda.Stream(), torch.cuda.Stream()], [], [None, None]
    torch.cuda.synchronize()
    for i, stream in enumerate(streams):
        with torch.cuda.stream(stream):
            for _ in range(5):
                outs[i] = call(i)
    torch.cuda.synchronize()
    assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1])
    for i in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[i]):
            outs[i] = call(i)
    for i, stream in enumerate(streams):                       # replayed side by side: each graph has its own workspace
        with torch.cuda.stream(stream):
            for _ in range(5):
                graphs[i].replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1])


def test_pieces_leave_the_tail_alone(dev):
    from semblo_b200.dense_prefill import dense_prefill_attention
    q, k, v, _ = _inputs(dev, 3, [50], [3000], 2, 1, 128, torch.bfloat16)
    cu_q, cu_k = torch.tensor([0, 7], device=dev), torch.tensor([0, 2500], device=dev)
    k[2500:], v[2500:] = math.nan, math.inf
    out = torch.full_like(q, 9.0)
    got = dense_prefill_attention(q, k, v, cu_seqlens_q=cu_q, cu_seqlens_k=cu_k, sm_scale=0.1, out=out, return_logsumexp=True)
    want = _formula(q[:7], k[:2500], v[:2500], [7], [2500], sm_scale=0.1)
    _check(type(got)(out[:7], got.logsumexp[:7]), want, 2500)
    assert bool((out[7:] == 9).all()) and bool((got.logsumexp[7:] == -math.inf).all())
    fresh = dense_prefill_attention(q, k, v, cu_seqlens_q=cu_q, cu_seqlens_k=cu_k, sm_scale=0.1, return_logsumexp=True)
    assert torch.equal(fresh.output[:7], out[:7]) and bool((fresh.output[7:] == 0).all())


Q_LENS = [1, 0, 63, 64, 65, 300, 17, 5, 130]
K_LENS = [1, 7, 63, 200, 65, 300, 529, 3, 0]          # more keys than queries, fewer, and none


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("hq,hkv", [(4, 1), (2, 2), (8, 1), (14, 2), (5, 1), (16, 1)])
@pytest.mark.parametrize("options", ["causal", "full", "cap", "window", "all"])
def test_formula(dev, dtype, dim, hq, hkv, options):
    q, k, v, gen = _inputs(dev, dim + hq, Q_LENS, K_LENS, hq, hkv, dim, dtype)
    kw = dict(sm_scale=dim ** -0.5)
    if options == "full":
        kw["causal"] = False
    if options in ("cap", "all"):
        kw["softcap"] = 4.0
    if options in ("window", "all"):
        kw["window"] = 70
        kw["prefix"] = torch.tensor([0, 2, 5, 66, 0, 129, 100, 3, 4], dtype=torch.int32, device=dev)
    if options == "all":
        kw["slopes"] = torch.rand(hq, device=dev, generator=gen)
    want = _formula(q, k, v, Q_LENS, K_LENS, **kw)
    _check(_call(q, k, v, Q_LENS, K_LENS, **kw), want, max(K_LENS))


@pytest.mark.parametrize("window", [1, 64, 65, 1000])
@pytest.mark.parametrize("dim", [64, 256])
def test_long_documents(dev, window, dim):
    lens = [1500, 1, 700]
    q, k, v, _ = _inputs(dev, window, lens, lens, 4, 2, dim, torch.bfloat16)
    for kw in (dict(), dict(window=window), dict(window=window, prefix=torch.tensor([300, 0, 1], device=dev))):
        want = _formula(q, k, v, lens, lens, sm_scale=0.1, **kw)
        _check(_call(q, k, v, lens, lens, sm_scale=0.1, **kw), want, 1500)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("softcap", [0.0, 20.0, 50.0, 80.0])
def test_a_row_that_sees_one_key_gives_its_value(dev, dim, dtype, softcap):
    # its weight is p / p with p a 16-bit number: p v is exact in 32 bits (22 bits at most), the reciprocal and the product
    # are off by 2^-23 together, and the rounding to 16 bits returns v.  In fp16 p is the power of two that the reference
    # stands for, and the sum as computed differs from it by the score's rounding, |s| 2^-23 < 2^-14 at most
    lens = [1] * 40
    q, k, v, _ = _inputs(dev, dim, lens, lens, 6, 2, dim, dtype, scale=6.0)
    got = _call(q, k, v, lens, lens, sm_scale=dim ** -0.5, softcap=softcap)
    assert torch.equal(got.output, v.repeat_interleave(3, 1))
    long = [300]
    q, k, v, _ = _inputs(dev, dim + 1, long, long, 6, 2, dim, dtype, scale=6.0)
    got = _call(q, k, v, long, long, sm_scale=dim ** -0.5, softcap=softcap, window=1)
    assert torch.equal(got.output, v.repeat_interleave(3, 1))


def test_rising_scores_rescale(dev):
    """Scores that climb along the keys by far more than the range of a lazy rescale, and large caps."""
    lens = [640]
    for dim, dtype in ((64, torch.float16), (128, torch.bfloat16), (256, torch.float16)):
        q, k, v, _ = _inputs(dev, 3, lens, lens, 2, 1, dim, dtype, scale=1.0)
        q[..., 0] = 8.0
        k[..., 0] = (torch.arange(640, device=dev) / 8).to(dtype)[:, None]
        for cap in (0.0, 50.0, 60.0):            # 60 and fp16: a running maximum, 50 in bf16: a fixed reference
            kw = dict(sm_scale=1.0, softcap=cap)
            _check(_call(q, k, v, lens, lens, **kw), _formula(q, k, v, lens, lens, **kw), 640)


def test_many_short_documents(dev):
    lens = [(i * 7) % 5 for i in range(400)]
    q, k, v, _ = _inputs(dev, 4, lens, lens, 8, 2, 128, torch.bfloat16)
    _check(_call(q, k, v, lens, lens, sm_scale=0.1), _formula(q, k, v, lens, lens, sm_scale=0.1), 5)


def test_garbage_behind_documents(dev):
    """Keys of other documents, and rows behind the last one, may be NaN or infinite."""
    q_lens, k_lens = [40, 30, 9], [50, 100, 9]
    for dim in (64, 128, 256):
        q, k, v, _ = _inputs(dev, 5, q_lens, k_lens, 4, 1, dim, torch.bfloat16)
        want = _call(q, k, v, q_lens, k_lens, sm_scale=0.1)
        k2, v2 = k.clone(), v.clone()
        for x in (k2, v2):
            x[50:150] = math.nan
            x[150:] = math.inf
        got = _call(q, k2, v2, q_lens, k_lens, sm_scale=0.1)
        assert torch.equal(got.output[:40], want.output[:40]) and torch.equal(got.logsumexp[:40], want.logsumexp[:40])
        # a store with room behind the last document
        pad = torch.full((77, 1, dim), math.nan, dtype=torch.bfloat16, device=dev)
        got = _call(q, torch.cat([k, pad]), torch.cat([v, pad]), q_lens, k_lens, sm_scale=0.1)
        assert torch.equal(got.output, want.output)


def test_rows_behind_the_last_document(dev):
    from semblo_b200.dense_prefill import dense_prefill_attention
    lens = [100, 30]
    q, k, v, _ = _inputs(dev, 6, [100, 30, 500], [100, 30, 500], 6, 2, 128, torch.float16)
    cu = torch.tensor([0, 100, 130], dtype=torch.int32, device=dev)
    want = _call(q[:130], k[:130], v[:130], lens, lens, sm_scale=0.1)
    got = dense_prefill_attention(q, k, v, cu_seqlens_q=cu, sm_scale=0.1, return_logsumexp=True)
    assert torch.equal(got.output[:130], want.output) and bool((got.output[130:] == 0).all())
    assert torch.equal(got.logsumexp[:130], want.logsumexp) and bool((got.logsumexp[130:] == -math.inf).all())
    out = torch.full_like(q, 7.0)
    got = dense_prefill_attention(q, k, v, cu_seqlens_q=cu, sm_scale=0.1, out=out, return_logsumexp=True)
    assert got.output is out and torch.equal(out[:130], want.output) and bool((out[130:] == 7.0).all())
    assert bool((got.logsumexp[130:] == -math.inf).all())
    none = dense_prefill_attention(q, k, v, cu_seqlens_q=cu[:1], sm_scale=0.1)
    assert bool((none.output == 0).all())


def test_views_of_a_fused_projection(dev):
    lens = [90, 200]
    hq, hkv, dim = 8, 2, 128
    gen = torch.Generator(device=dev).manual_seed(7)
    qkv = torch.randn(290, hq + 2 * hkv, dim, device=dev, generator=gen).to(torch.bfloat16)
    q, k, v = qkv[:, :hq], qkv[:, hq:hq + hkv], qkv[:, hq + hkv:]
    want = _call(q.contiguous(), k.contiguous(), v.contiguous(), lens, lens, sm_scale=0.1)
    got = _call(q, k, v, lens, lens, sm_scale=0.1)
    assert torch.equal(got.output, want.output)
    heads_first = k.transpose(0, 1).contiguous().transpose(0, 1)
    odd = torch.empty(290 * (hkv * dim + 1) + 1, dtype=torch.bfloat16, device=dev)[1:].view(290, hkv * dim + 1)[:, :-1]
    odd = odd.unflatten(1, (hkv, dim))
    odd.copy_(v)
    got = _call(q, heads_first, odd, lens, lens, sm_scale=0.1)
    assert torch.equal(got.output, want.output)


def test_streams_graph_and_repeat(dev):
    from semblo_b200.dense_prefill import dense_prefill_attention
    lens = [333, 500]
    q, k, v, _ = _inputs(dev, 8, lens, lens, 8, 2, 128, torch.bfloat16)
    cu = torch.tensor([0, 333, 833], dtype=torch.int32, device=dev)
    want = dense_prefill_attention(q, k, v, cu_seqlens_q=cu, sm_scale=0.1).output
    sides = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    torch.cuda.synchronize()
    for st in sides:
        with torch.cuda.stream(st):
            outs.append(dense_prefill_attention(q, k, v, cu_seqlens_q=cu, sm_scale=0.1).output)
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = dense_prefill_attention(q, k, v, cu_seqlens_q=cu, sm_scale=0.1).output
    cu.copy_(torch.tensor([0, 10, 600]))
    g.replay()
    want = dense_prefill_attention(q, k, v, cu_seqlens_q=cu, sm_scale=0.1).output
    assert torch.equal(out, want) and bool((out[600:] == 0).all())


def test_window_matches_the_chunk_kernel(dev):
    """The same attended set as the sparse path's window launch: two kernels, one result within their roundings."""
    from semblo_b200 import _lib
    from semblo_b200._lib import check, lib, ptr, stream_ptr
    n, hq, hkv, dim = 400, 8, 2, 128
    q, k, v, _ = _inputs(dev, 9, [n], [n], hq, hkv, dim, torch.bfloat16)
    out, lse = torch.empty_like(q), torch.empty(n, hq, device=dev)
    pos = torch.arange(n, dtype=torch.int32, device=dev)
    check(lib().semblo_window_prefill(ptr(q), n, hq, hkv, dim, ptr(pos), ptr(k), ptr(v), n, 0, 0, 0.1, ptr(out), None,
                                      ptr(lse), None, ptr(_lib.status_for(dev).word), stream_ptr()))
    want = _formula(q, k, v, [n], [n], sm_scale=0.1)
    got = _call(q, k, v, [n], [n], sm_scale=0.1)
    _check(got, want, n)
    # both are within eps of sum |p v| (P) and eps / 2 of the value (output) of the formula
    eps = 2.0 ** -7
    assert bool(((got.output.double() - out.double()).abs() <= (2 * want[2] + want[0].abs()) * eps).all())


@pytest.mark.parametrize("dim", [128, 256])
def test_very_many_documents_and_huge_windows(dev, dim):
    """More documents than threads in a block, empty ones among them, and a window beyond every position."""
    lens = [(i * 5) % 4 for i in range(1500)]
    q, k, v, _ = _inputs(dev, 11, lens, lens, 4, 1, dim, torch.bfloat16)
    pad = torch.randn(100, 4, dim, device=dev).to(torch.bfloat16)
    kw = dict(sm_scale=0.1, window=(1 << 40) + 3)
    got = _call(torch.cat([q, pad]), k, v, lens, lens, **kw)
    assert bool((got.output[len(q):] == 0).all()) and bool((got.logsumexp[len(q):] == -math.inf).all())
    plain = _call(q, k, v, lens, lens, sm_scale=0.1)
    assert torch.equal(got.output[:len(q)], plain.output)
    _check(plain, _formula(q, k, v, lens, lens, sm_scale=0.1), 3)


def test_scores_at_the_lower_end_of_the_cap(dev):
    """Every score of a row close to -cap, small values: the fixed reference must not run out of range."""
    for cap in (50.0, 52.0):
        lens = [300]
        q, k, v, _ = _inputs(dev, 12, lens, lens, 2, 1, 128, torch.bfloat16)
        q[...], k[...] = 4.0, -4.0
        q[::2] *= -1                                             # and every other row close to +cap
        v *= 2.0 ** -20
        kw = dict(sm_scale=1.0, softcap=cap)
        _check(_call(q, k, v, lens, lens, **kw), _formula(q, k, v, lens, lens, **kw), 300)
