"""The dense-request operators where their range ends: calls from two threads, scales that lie far apart, the ends of a
16-bit type's exponent, caps far above the scores, the angle's last bits."""
from __future__ import annotations

import math
import threading

import pytest
import torch

import test_gpu_dense_prefill as prompt_ref
import test_gpu_kv8_append as append_ref
import test_gpu_kv8_decode as decode_ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    from semblo_b200 import _lib
    _lib.lib()
    return torch.device("cuda:0")


# ---- calls from two threads

def test_decode_of_two_batch_sizes_from_several_threads(dev):
    """The launch's shared memory grows with the batch: one thread's small call must not take the limit away from
    another's large one.  The C entry, which a thread is in without the interpreter's lock most of the time."""
    from semblo_b200 import _lib
    lib, status = _lib.lib(), _lib.status_for(dev).word
    cache, table, gen = decode_ref._pool(dev, 1, [900, 40], 16, 1, 64, width=100)
    jobs = []
    for lens in ([900], [(i * 7) % 40 for i in range(4095)] + [900]):
        n = len(lens)
        q = torch.randn(n, 1, 2, 64, device=dev, generator=gen).to(torch.bfloat16)
        rows = table[torch.tensor([1] * (n - 1) + [0], device=dev)].contiguous()
        lengths = torch.tensor(lens, dtype=torch.int32, device=dev)
        nbytes = lib.semblo_kv8_decode_workspace_bytes(n, 1, 2, 1, 64, 16, 100, 0, 0)
        assert nbytes > 0
        want = decode_ref._call(q, cache, rows, lens, sm_scale=0.125).output
        for _ in range(3):
            out, stream = torch.empty_like(q), torch.cuda.Stream()
            room = torch.empty(nbytes, dtype=torch.uint8, device=dev)
            args = (q.data_ptr(), 0, n, 1, 2, 1, 64, cache.data.data_ptr(), cache.scales.data_ptr(), cache.num_blocks, 16,
                    rows.data_ptr(), 100, 100, lengths.data_ptr(), None, 0, 0.125, 0.0, None, out.data_ptr(), None,
                    room.data_ptr(), nbytes, status.data_ptr(), stream.cuda_stream)
            jobs.append((args, out, want, (q, rows, lengths, room, stream)))
    torch.cuda.synchronize()
    codes, start = [], threading.Barrier(len(jobs))

    def loop(args):
        start.wait()
        codes.append([lib.semblo_kv8_decode(*args) for _ in range(1000)])

    threads = [threading.Thread(target=loop, args=(job[0],)) for job in jobs]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert len(codes) == len(jobs) and sum(c != 0 for run in codes for c in run) == 0
    for _, out, want, _held in jobs:
        assert torch.equal(out, want)


# ---- the append's scales

@pytest.mark.parametrize("stored", [2.0 ** -100, 0.0])
@pytest.mark.parametrize("new", [[1, 1, 1, 1], [16, 1, 0, 30]])
def test_a_scale_that_grows_beyond_what_a_ratio_holds(dev, stored, new):
    """Rows stored near 2^-94, then tokens near 2^60: the ratio of the scales is 0 in 32 bits, and so are the earlier rows
    under the new scale.  One token per request, and whole blocks; more heads than a block has warps."""
    cache, k, v, table, cu, past = append_ref._case(dev, 21, 16, 12, 64, torch.bfloat16, new, [5, 15, 16, 7])
    cache.scales.fill_(stored)
    k, v = ((x.float() * 2.0 ** 60).to(torch.bfloat16) for x in (k, v))
    append_ref._run_and_compare(cache, k, v, table, cu, past, 16)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_special_values_in_single_tokens(dev, dtype):
    """Infinities, NaN and zeros in calls of one token per request, in blocks that start and that are continued."""
    cache, k, v, table, cu, past = append_ref._case(dev, 22, 32, 10, 128, dtype, [1] * 6, [0, 5, 31, 32, 64, 9])
    k[0, 0, 3], k[1, 9, 0], v[2, 4, 127], v[3, 8, 64] = math.inf, -math.inf, math.nan, math.inf
    k[4], v[5] = 0.0, math.inf                                      # nothing but zeros, nothing finite
    v[1, 2] = math.nan
    append_ref._run_and_compare(cache, k, v, table, cu, past, 32)


# ---- queries at the ends of bf16

@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("exponent", [125, 124, -113, -118, -122])
@pytest.mark.parametrize("softcap", [0.0, 5.0])
def test_queries_of_every_exponent(dev, dim, exponent, softcap):
    """Queries up to 2^128 and down to 2^-125 over K scales that bring the scores back to a few units."""
    lens = [200, 33, 1]
    cache, table, gen = decode_ref._pool(dev, 41 + dim, lens, 32, 2, dim)
    if exponent > 0:                                                # codes of a few units: scales below 2^-126 are not needed
        cache.data.copy_((cache.data.float() / 32).to(torch.float8_e4m3fn))
        cache.scales[0] = 2.0 ** (-exponent - 1)
    else:
        cache.scales[0] = 2.0 ** (-exponent - 6)
    q = torch.randn(3, 1, 8, dim, device=dev, generator=gen).clamp(-3.9, 3.9)
    q = (q.double() * 2.0 ** exponent).to(torch.bfloat16)
    q[0, 0, 0, 0], q[1, 0, 3, 5] = 3.9 * 2.0 ** exponent, -3.0 * 2.0 ** exponent
    assert bool(q.isfinite().all()) and float(q.double().abs().max()) > 1.9 * 2.0 ** (exponent + 1)
    kw = dict(sm_scale=dim ** -0.5, softcap=softcap)
    want = decode_ref._formula(q, cache, table, lens, kw["sm_scale"], softcap, 0, None, None)
    decode_ref._check(decode_ref._call(q, cache, table, lens, **kw), want, 200)


# ---- caps far above the scores

def _uncapped(want, cap, scores=40.0):
    """What is allowed where |score| stays below ``scores``: cap tanh(s / cap) is s but for s^3 / (3 cap^2), and its error
    is relative to the score (2^-17), not to the cap."""
    out, lse, mag, off = want
    assert scores < cap
    return out, lse, mag, off + scores ** 3 / (3 * cap * cap) + scores * 2.0 ** -17


@pytest.mark.parametrize("cap", [3.0e3, 1.0e5, 1.0e7, 1.0e30])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_decode_under_a_cap_far_above_its_scores(dev, dim, cap):
    lens = [700, 45]
    cache, table, gen = decode_ref._pool(dev, 51 + dim, lens, 64, 2, dim)
    q = torch.randn(2, 2, 8, dim, device=dev, generator=gen).to(torch.bfloat16)
    want = decode_ref._formula(q, cache, table, lens, dim ** -0.5, 0.0, 0, None, None)
    decode_ref._check(decode_ref._call(q, cache, table, lens, sm_scale=dim ** -0.5, softcap=cap), _uncapped(want, cap), 700)


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_decode_of_a_capped_head_beside_heads_far_below_the_cap(dev, dim):
    """One head's scores reach the cap; the others' are as accurate as without that head."""
    cap, sm, lens = 1.0e6, dim ** -0.5, [300]
    cache, table, gen = decode_ref._pool(dev, 61 + dim, lens, 64, 1, dim)
    q = torch.randn(1, 1, 8, dim, device=dev, generator=gen).to(torch.bfloat16)
    want = decode_ref._formula(q[:, :, 1:], cache, table, lens, sm, 0.0, 0, None, None)
    q[:, :, 0] *= 2.0 ** 21
    got = decode_ref._call(q, cache, table, lens, sm_scale=sm, softcap=cap)
    decode_ref._check(type(got)(got.output[:, :, 1:], got.logsumexp[:, :, 1:]), _uncapped(want, cap), 300)


# ---- what decides a tanh's form

@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("dtype,softcap,biased", [(torch.bfloat16, 20.0, False), (torch.float16, 20.0, False),
                                                  (torch.bfloat16, 80.0, False), (torch.bfloat16, 20.0, True)])
def test_a_document_keeps_its_bits_whatever_is_beside_it(dev, dim, dtype, softcap, biased):
    """The rows and keys that share a document's tiles without being its own: the next document's, of any size, NaN, none
    at all, and what an earlier launch left."""
    heads, lens = 6, [50, 75]
    q, k, v, gen = prompt_ref._inputs(dev, 81 + dim, lens, lens, heads, 2, dim, dtype, scale=6.0)
    slopes = torch.rand(heads, device=dev, generator=gen) if biased else None
    kw = dict(sm_scale=dim ** -0.5, softcap=softcap, slopes=slopes)
    alone = [prompt_ref._call(q[:50], k[:50], v[:50], [50], [50], **kw)]
    for factor in (0.0, 1.0, 2.0 ** 9, math.nan):
        q2, k2 = q.clone(), k.clone()
        q2[50:], k2[50:] = q[50:] * factor, k[50:] * factor
        # a launch whose scores are far from these ones, for the tensor memory that it leaves behind
        prompt_ref._call(torch.full_like(q, 200.0), torch.full_like(k, 200.0), v, lens, lens, sm_scale=1.0)
        got = prompt_ref._call(q2, k2, v, lens, lens, **kw)
        alone.append(type(got)(got.output[:50], got.logsumexp[:50]))
    for got in alone[1:]:
        assert torch.equal(got.logsumexp, alone[0].logsumexp) and torch.equal(got.output, alone[0].output)


# ---- caps far above a prompt's scores

@pytest.mark.parametrize("cap", [3.0e3, 1.0e5, 1.0e7, 1.0e30])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("biased", [False, True])
def test_prompt_under_a_cap_far_above_its_scores(dev, dim, cap, biased):
    lens = [200, 45]
    q, k, v, gen = prompt_ref._inputs(dev, 51 + dim, lens, lens, 4, 2, dim, torch.bfloat16, scale=1.0)
    kw = dict(sm_scale=dim ** -0.5, slopes=torch.rand(4, device=dev, generator=gen) if biased else None)
    want = prompt_ref._formula(q, k, v, lens, lens, **kw)
    prompt_ref._check(prompt_ref._call(q, k, v, lens, lens, softcap=cap, **kw), _uncapped(want, cap), 200)


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_prompt_of_a_capped_head_beside_heads_far_below_the_cap(dev, dim, dtype):
    cap, lens = 1.0e6, [300]
    q, k, v, _ = prompt_ref._inputs(dev, 61 + dim, lens, lens, 8, 1, dim, dtype, scale=1.0)
    kw = dict(sm_scale=dim ** -0.5)
    if dtype == torch.float16:                                      # its largest value holds the scores back: a smaller query
        q *= 2.0 ** -10
        kw = dict(sm_scale=dim ** -0.5 * 2.0 ** 10)
    want = prompt_ref._formula(q[:, 1:], k, v, lens, lens, **kw)
    q[:, 0] *= 2.0 ** 21
    got = prompt_ref._call(q, k, v, lens, lens, softcap=cap, **kw)
    prompt_ref._check(type(got)(got.output[:, 1:], got.logsumexp[:, 1:]), _uncapped(want, cap), 300)


# ---- the rotation's angle

@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dim,rotary", [(128, 128), (66, 34)])
def test_cos_and_sin_to_their_last_bits(dev, interleaved, dim, rotary):
    """Rows (1, 0): the rotated pair is (cos, sin) itself.  The angle is reduced in 64 bits (three roundings of 2^-53 of its
    turns); cos and sin of a turn's fraction, 1 ulp of the result each, and one rounding of their correction: 2^-22 of the
    value, nothing relative to 1."""
    from semblo_b200.rotary import apply_rotary, rotary_frequencies
    tokens = 4096
    x = torch.zeros(tokens, 1, dim, device=dev)
    first = slice(0, rotary, 2) if interleaved else slice(0, rotary // 2)
    second = slice(1, rotary, 2) if interleaved else slice(rotary // 2, rotary)
    x[..., first] = 1.0
    pos = torch.arange(tokens, device=dev) * 251 + 5
    freq = rotary_frequencies(rotary, 500000.0, device=dev)
    y, _ = apply_rotary(x, None, pos, freq, interleaved=interleaved)
    angle = pos.double()[:, None] * freq.inv_freq
    slack = angle * 2.0 ** -51 + 2.0 ** -44                         # the angle in 64 bits, here and there; second order
    for part, want in ((first, angle.cos()), (second, angle.sin())):
        err = (y[:, 0, part].double() - want).abs()
        bound = want.abs() * 2.0 ** -22 + slack
        assert bool((err <= bound).all()), float((err / bound).max())


# ---- rows that no document has

@pytest.mark.parametrize("dim", [128, 256])
@pytest.mark.parametrize("front,tail", [(7, 0), (300, 41), (63, 65)])
def test_rows_in_front_of_the_first_document(dev, dim, front, tail):
    """As behind the last one: 0 and -inf in a fresh result, untouched in a given one."""
    from semblo_b200.dense_prefill import dense_prefill_attention
    lens = [20, 75]
    q, k, v, _ = prompt_ref._inputs(dev, 71, [front] + lens + [tail], [front] + lens + [tail], 4, 2, dim, torch.bfloat16)
    cu = torch.tensor([front, front + 20, front + 95], dtype=torch.int32, device=dev)
    inside = slice(front, front + 95)
    want = prompt_ref._formula(q[inside], k[inside], v[inside], lens, lens, sm_scale=0.1)
    junk = torch.full((1 << 22,), 3.0, device=dev)                  # freed: what a fresh buffer would show
    del junk
    got = dense_prefill_attention(q, k, v, cu_seqlens_q=cu, sm_scale=0.1, return_logsumexp=True)
    prompt_ref._check(type(got)(got.output[inside], got.logsumexp[inside]), want, 75)
    outside = torch.ones(len(q), dtype=torch.bool, device=dev)
    outside[inside] = False
    assert bool((got.output[outside] == 0).all()) and bool((got.logsumexp[outside] == -math.inf).all())
    out = torch.full_like(q, 7.0)
    given = dense_prefill_attention(q, k, v, cu_seqlens_q=cu, sm_scale=0.1, out=out, return_logsumexp=True)
    assert torch.equal(out[inside], got.output[inside]) and bool((out[outside] == 7).all())
    assert bool((given.logsumexp[outside] == -math.inf).all())


# ---- outputs in the buffer of the inputs

def test_rotary_in_the_buffer_of_its_inputs(dev):
    """Queries and keys turned in place in one fused buffer, and into another one's slices: the bytes of separate calls, and
    nothing else touched."""
    from semblo_b200.rotary import apply_rotary, rotary_frequencies
    qkv = torch.randn(300, 12, 128, device=dev).to(torch.bfloat16)
    held, pos = qkv.clone(), torch.arange(300, device=dev)
    freq = rotary_frequencies(128, device=dev)
    want = apply_rotary(qkv[:, :8], qkv[:, 8:10], pos, freq)
    other = torch.full_like(qkv, 3.0)
    apply_rotary(qkv[:, :8], qkv[:, 8:10], pos, freq, q_out=other[:, :8], k_out=other[:, 8:10])
    apply_rotary(qkv[:, :8], qkv[:, 8:10], pos, freq, q_out=qkv[:, :8], k_out=qkv[:, 8:10])
    for got, rest in ((qkv, held[:, 10:]), (other, torch.full_like(held[:, 10:], 3.0))):
        assert torch.equal(got[:, :8], want[0]) and torch.equal(got[:, 8:10], want[1]) and torch.equal(got[:, 10:], rest)
